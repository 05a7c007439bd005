"""Sizes that linear_attention_fn does not serve (no GPU)."""
import pytest
import torch

from mamba_amd import _lib
from mamba_amd.ops.linear_attention import linear_attention_fn

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
