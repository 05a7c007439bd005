"""Sizes that linear_attention_fn does not serve, and scales that the attention over a paged cache does not (no GPU)."""
import pytest
import torch

from mamba_amd import _lib
from mamba_amd.ops.linear_attention import linear_attention_fn
from mamba_amd.ops.paged_attention import paged_attention_update

MOST_HEADS = 2 ** 22  # x 256 values of a head: a position's values are counted in 32 bits


@pytest.mark.parametrize("heads,kv", [(MOST_HEADS + 1, 1), (MOST_HEADS + 2, MOST_HEADS // 2 + 1)])
def test_heads(heads, kv):
    x = lambda n: torch.zeros(1, 1, 1, 1).expand(1, 1, n, 1)
    with pytest.raises(RuntimeError, match="2\\^22 heads"):
        linear_attention_fn(x(heads), x(kv), x(kv), torch.zeros(1).expand(heads))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        linear_attention_fn(x(MOST_HEADS), x(1), x(1), torch.zeros(1).expand(MOST_HEADS))


@pytest.mark.parametrize("fn", ["linear_attn_fwd_ws_bytes", "linear_attn_bwd_ws_bytes"])
def test_heads_of_the_c_entries(fn):
    p = _lib.LinearAttnParams()
    p.batch = p.seqlen = p.nkvheads = p.headdim_k = p.headdim_v = 1
    p.scale = 1.0
    p.q = p.k = p.v = p.log_decay = 256
    p.nheads = MOST_HEADS + 1
    assert getattr(_lib.load(), fn)(p) == -2
    p.nheads = MOST_HEADS
    assert getattr(_lib.load(), fn)(p) >= 0


@pytest.mark.parametrize("sign", [1, -1])
def test_scales_that_are_none_times_log2_of_e(sign):
    ints = lambda *v: torch.tensor(v, dtype=torch.int32)
    z = torch.zeros
    args = (z(1, 1, 1), None, None, z(1, 1, 1, 1), z(1, 1, 1, 1), ints([0]), ints(1))
    with pytest.raises(ValueError, match="scale"):
        paged_attention_update(*args, scale=sign * 2.5e38)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        paged_attention_update(*args, scale=sign * 2e38)
    p = _lib.PagedAttnParams()
    for n in ("batch", "nheads", "nkvheads", "headdim_k", "headdim_v", "num_pages", "page_size", "max_pages"):
        setattr(p, n, 1)
    for scale, code in ((2.5e38, -1), (2e38, 1)):
        p.scale = sign * scale
        assert _lib.load().paged_attn_parts(p) == code
