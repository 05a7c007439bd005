"""gated_linear_scan_fn and gated_linear_state_update where a decay or a gate is at the end of its type's range: softplus of
what lies far below zero, and products of softplus and sigmoid around fp32's smallest normal number 2^-126."""
import pytest
import torch

from oracle.gated_linear import gated_linear_oracle, within

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
GRADS = ["dx", "dgate_a", "dgate_x", "ddecay", "dinitial"]


def _check(gate_a, decay, cu=None, dtype=torch.float32, seed=0):
    """Outputs, states and every gradient within the oracle's bounds, all of them finite; gate_a (L), decay (dim)."""
    from mamba_amd.ops.gated_linear_scan import gated_linear_scan_fn
    g = torch.Generator().manual_seed(seed)
    L, dim = gate_a.numel(), decay.numel()
    seqs = 1 if cu is None else len(cu) - 1
    r = lambda *s, dt=dtype: torch.randn(*s, generator=g).to(dt)
    x, gx, dout = r(1, L, dim), r(1, L, dim), r(1, L, dim)
    ga = gate_a.to(dtype)[None, :, None].expand(1, L, dim).contiguous()
    init, dfinal = r(seqs, dim, dt=torch.float32), r(seqs, dim, dt=torch.float32)
    leaves = [t.cuda().requires_grad_() for t in (x, ga, gx, decay, init)]
    bounds = None if cu is None else torch.tensor(cu, dtype=torch.int32, device="cuda")
    out, final = gated_linear_scan_fn(*leaves[:4], initial_states=leaves[4], cu_seqlens=bounds, return_final_states=True)
    grads = torch.autograd.grad([out, final], leaves, [dout.cuda(), dfinal.cuda()])
    ref, bound = gated_linear_oracle(x, ga, gx, decay, 8.0, init, cu, dout, dfinal)
    for n, v in zip(["out", "final"] + GRADS, [out, final, *grads]):
        assert torch.isfinite(v).all(), n
        within(n, v, ref[n], bound[n])


# -2.36e38 is the least number whose product with log2(e) fp32 still holds
FAR = [-float("inf"), -3.3e38, -2.4e38, -2.3e38, -1e30, -6e4, -1000.0, -200.0, -150.0, -1.0, 0.5]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("L,cu", [(9, None), (150, None), (150, [0, 1, 70, 70, 149])])
def test_decays_far_below_zero(L, cu, dtype):
    """softplus is 0 there: the state stays what it was, and no gradient is lost to it."""
    g = torch.Generator().manual_seed(L)
    decay = torch.tensor([torch.finfo(dtype).min, *FAR]).to(dtype)
    assert torch.isinf(decay).any() and not torch.isnan(decay).any()
    _check(torch.randn(L, generator=g), decay, cu)


@pytest.mark.parametrize("dtype", DTYPES)
def test_step_with_decays_far_below_zero(dtype):
    from mamba_amd.ops.gated_linear_scan import gated_linear_state_update
    g = torch.Generator().manual_seed(0)
    decay = torch.tensor([torch.finfo(dtype).min, *FAR]).to(dtype)
    x, ga, gx, init = (torch.randn(3, decay.numel(), generator=g) for _ in range(4))
    state = init.cuda()
    out = gated_linear_state_update(state, x.cuda(), ga.cuda(), gx.cuda(), decay.cuda())
    ref, bound = gated_linear_oracle(x[:, None], ga[:, None], gx[:, None], decay, 8.0, init)
    within("out", out, ref["out"][:, 0], bound["out"][:, 0])
    within("state", state, ref["final"], bound["final"])


# k r from above 2^-126 to far below it: shut gates with ordinary decays, decays of next to nothing with open gates, and both
SHUT = [-80.0, -82.0, -83.5, -84.0, -85.0, -85.5, -86.0, -86.5, -87.0, -87.3, -50.0, -49.0, -48.0, -47.0, -46.0, -44.0, -3.5, -2.0,
        -1.0, 0.0, 3.0]
NEXT_TO_NOTHING = [-8.0, -7.0, -6.0, -5.0, -4.0, -3.0, -2.0, -1.0, 0.0, 2.0, -36.0, -37.0, -38.0, -39.0, -40.0, -41.0, -42.0, -83.0,
                   -84.0, -85.0, -86.0, -87.0, -120.0]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("times,cu", [(1, None), (8, None), (8, [0, 3, 60, 61, 100, 168])])
def test_gates_and_decays_next_to_nothing(times, cu, dtype):
    """k r below 2^-126 is no normal number: what the root takes for 0 must not come back as an infinity from its reciprocal."""
    _check(torch.tensor(SHUT * times), torch.tensor(NEXT_TO_NOTHING), cu, dtype)


def test_many_gates_around_the_smallest_normal_number():
    """Every form of the backward pass' tiles is short of 3000 positions; here one position in three has a k r around 2^-126."""
    g = torch.Generator().manual_seed(1)
    gate = torch.randn(3000, generator=g)
    gate[::3] = -80.0 - 8.0 * torch.rand(1000, generator=g)
    _check(gate, -6.0 + 6.0 * torch.rand(130, generator=g))
