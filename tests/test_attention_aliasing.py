"""The C entry points of linear attention, its step and the attention over a paged cache refuse results in the memory of operands,
which some workgroups would write while others read."""
import ctypes

import pytest
import torch

from mamba_amd import _lib

SIZES = dict(batch=1, seqlen=4, nheads=4, nkvheads=2, headdim_k=8, headdim_v=8, scale=1.0)
ROWS = ["q", "k", "v", "out", "dout", "dq", "dk", "dv", "log_decay", "ws", "state", "k_cache", "v_cache", "block_table", "cache_seqlens"]
STATE = 4 * 8 * 8 * 4  # bytes


def _params(cls, **changes):
    """Stand-ins for pointers, a MiB apart: every call here ends before a launch."""
    p = getattr(_lib, cls)()
    names = [f[0] for f in p._fields_]
    for n, v in dict(SIZES, state_rows=1, num_pages=3, page_size=4, max_pages=2, nsplit=1).items():
        if n in names:
            setattr(p, n, v)
    for i, n in enumerate(ROWS):
        if n in names:
            setattr(p, n, (i + 1) << 20)
    for n, v in changes.items():
        setattr(p, n, v)
    return p


AT = {n: (i + 1) << 20 for i, n in enumerate(ROWS)}
FREE = 1 << 30


@pytest.mark.parametrize("fn,cls,changes", [
    *[("linear_attn_fwd", "LinearAttnParams", c) for c in (
        dict(initial_states=FREE, final_states=FREE), dict(initial_states=FREE, final_states=FREE + STATE - 4),
        dict(initial_states=FREE + STATE - 4, final_states=FREE), dict(out=AT["q"]), dict(out=AT["k"]), dict(out=AT["v"]),
        dict(nseq=3, cu_seqlens=256, initial_states=FREE, final_states=FREE + 2 * STATE))],
    *[("linear_attn_bwd", "LinearAttnParams", c) for c in (
        dict(initial_states=FREE, dinitial_states=FREE), dict(dfinal_states=FREE, dinitial_states=FREE),
        dict(dfinal_states=FREE, dinitial_states=FREE + STATE // 2), dict(dq=AT["q"]), dict(dk=AT["dout"]), dict(dv=AT["v"]),
        dict(dq=AT["dk"]), dict(dv=AT["dk"]), dict(dv=AT["dq"]))],
    *[("linear_attn_state_update", "LinearAttnStepParams", dict(out=AT[n])) for n in ("state", "q", "k", "v")],
    *[("paged_attn_update", "PagedAttnParams", dict(out=AT[n])) for n in ("k", "v", "k_cache", "v_cache")],
])
def test_results_in_the_memory_of_operands_are_refused(fn, cls, changes):
    assert getattr(_lib.load(), fn)(_params(cls, **changes), None) == -1


@pytest.mark.gpu
@pytest.mark.parametrize("L", [5, 700])
def test_states_side_by_side_are_taken(L):
    from mamba_amd.ops import linear_attention as ops
    g = torch.Generator(device="cuda").manual_seed(0)
    q, k, v = (torch.randn(1, L, 4, 8, device="cuda", generator=g) for _ in range(3))
    decay = -torch.rand(4, device="cuda", generator=g)
    for first in (0, 1):
        states = torch.randn(2, 1, 4, 8, 8, device="cuda", generator=g)
        want, want_final = ops.linear_attention_fn(q, k, v, decay, initial_states=states[first].clone(), return_final_states=True)
        lib = _lib.load()
        p = ops._params(q, k, v, decay, states[first], None, 8 ** -0.5)
        out = torch.empty_like(want)
        p.out, p.final_states = out.data_ptr(), states[1 - first].data_ptr()
        ops._strides(p, out=out)
        ws = torch.empty(max(lib.linear_attn_fwd_ws_bytes(p), 16), dtype=torch.uint8, device="cuda")
        p.ws = ws.data_ptr()
        _lib.check(lib.linear_attn_fwd(ctypes.byref(p), _lib.current_stream(q.device)), "fwd")
        assert torch.equal(out, want) and torch.equal(states[1 - first], want_final)
