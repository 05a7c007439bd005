"""What an infinity or a NaN at one position does to linear attention: the outputs of its block and of later positions, and the
states, that it has part in are no finite numbers, all others are as they were."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("which", ["q", "k", "v", "initial_states"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("L", [50, 700])
def test_where_it_shows(L, dtype, which, value):
    from mamba_amd.ops.linear_attention import linear_attention_fn
    g = torch.Generator().manual_seed(L)
    t = dict(q=torch.randn(1, L, 2, 16, generator=g).to(dtype), k=torch.randn(1, L, 2, 16, generator=g).to(dtype),
             v=torch.randn(1, L, 2, 24, generator=g).to(dtype), initial_states=torch.randn(1, 2, 16, 24, generator=g))
    call = lambda: linear_attention_fn(t["q"].cuda(), t["k"].cuda(), t["v"].cuda(), torch.tensor([-0.01, -0.001], device="cuda"),
                                       initial_states=t["initial_states"].cuda(), return_final_states=True)
    want, want_final = call()
    at, head, x = L * 3 // 4, 1, 5
    if which == "initial_states":
        t[which][0, head, 3, x] = value
        at = 0
    else:
        t[which][0, at, head, x] = value
    out, final = call()
    assert torch.equal(out[:, :, 0], want[:, :, 0]) and torch.equal(final[:, 0], want_final[:, 0])
    mine, other = out[0, :, head], want[0, :, head]
    values = torch.arange(24) == x if which in ("v", "initial_states") else torch.ones(24, dtype=torch.bool)
    # blocks are of 32 positions at most, from the start of a segment, whose lengths are multiples of that
    before = at // 32 * 32
    assert torch.equal(mine[:before], other[:before]) and torch.equal(mine[:, ~values], other[:, ~values])
    if which == "q":  # one row of outputs
        assert not bool(mine[at].isfinite().any())
        rest = torch.arange(L) != at
        assert torch.equal(mine[rest], other[rest]) and torch.equal(final, want_final)
        return
    assert not bool(mine[at:, values].isfinite().any())
    state = final[0, head]
    assert torch.equal(state[:, ~values], want_final[0, head][:, ~values])
    if which == "k":
        assert not bool(state[x].isfinite().any())
    elif which == "v":
        assert not bool(state[:, x].isfinite().any())
    else:
        assert not bool(state[3, x].isfinite())
