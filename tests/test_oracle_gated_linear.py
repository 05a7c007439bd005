"""The oracles of the gated linear recurrence and of the norm between two blocks: against autograd, finite differences and
formulations of their own; and the plain-torch statements next to the operators against the oracles."""
import pytest
import torch

from oracle.gated_linear import block_norm_oracle, gated_linear_oracle, within


def _inputs(batch, L, dim, seed=0, dtype=torch.float64, seqs=None):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64).to(dtype)
    n = batch if seqs is None else seqs
    return dict(x=r(batch, L, dim), gate_a=r(batch, L, dim), gate_x=r(batch, L, dim), decay=r(dim), initial_states=r(n, dim),
                dout=r(batch, L, dim), dfinal=r(n, dim))


def _forward(x, gate_a, gate_x, decay, initial, rate=8.0):
    """The recurrence as one lower-triangular product per channel: h_t = sum_s exp(sum of log a over s+1..t) b_s."""
    log_a = -rate * torch.nn.functional.softplus(decay) * torch.sigmoid(gate_a)
    b = torch.sqrt(-torch.expm1(2 * log_a)) * torch.sigmoid(gate_x) * x
    cum = log_a.cumsum(1)
    L = x.shape[1]
    low = torch.tril(torch.ones(L, L, dtype=torch.float64))[None, :, :, None]
    w = torch.exp(torch.where(low > 0, cum[:, :, None] - cum[:, None], torch.zeros((), dtype=torch.float64))) * low
    h = (w * b[:, None]).sum(2) + torch.exp(cum) * initial[:, None]
    return h, h[:, -1]


def test_scan_oracle_against_the_quadratic_form_and_autograd():
    t = _inputs(2, 9, 3)
    names = ["x", "gate_a", "gate_x", "decay", "initial_states"]
    leaves = {n: t[n].clone().requires_grad_() for n in names}
    h, final = _forward(*[leaves[n] for n in names])
    grads = torch.autograd.grad([h, final], list(leaves.values()), [t["dout"], t["dfinal"]])
    res, _ = gated_linear_oracle(**t)
    torch.testing.assert_close(res["out"], h.detach(), rtol=1e-12, atol=1e-12)
    torch.testing.assert_close(res["final"], final.detach(), rtol=1e-12, atol=1e-12)
    for n, g in zip(["dx", "dgate_a", "dgate_x", "ddecay", "dinitial"], grads):
        torch.testing.assert_close(res[n], g, rtol=1e-9, atol=1e-11)


def test_scan_oracle_against_differences():
    t = _inputs(1, 6, 2, seed=3)
    res, _ = gated_linear_oracle(**t)
    value = lambda q: float((q["out"] * t["dout"]).sum() + (q["final"] * t["dfinal"]).sum())
    forward = {k: v for k, v in t.items() if k not in ("dout", "dfinal")}
    for name, grad in (("x", "dx"), ("gate_a", "dgate_a"), ("gate_x", "dgate_x"), ("decay", "ddecay"), ("initial_states", "dinitial")):
        for at in range(t[name].numel()):
            side = []
            for step in (1e-6, -1e-6):
                moved = t[name].clone()
                moved.view(-1)[at] += step
                side.append(value(gated_linear_oracle(**{**forward, name: moved})[0]))
            assert abs((side[0] - side[1]) / 2e-6 - float(res[grad].view(-1)[at])) < 1e-6, (name, at)


def test_scan_oracle_packed_equals_separate():
    cu = [2, 5, 5, 6, 13]  # positions before the first sequence, an empty one, one of one position, padding behind
    t = _inputs(1, 15, 4, seed=1, seqs=4)
    for n in ("x", "gate_a", "gate_x", "dout"):
        t[n][:, :2] = float("nan")
        t[n][:, 13:] = float("inf")
    res, bound = gated_linear_oracle(**t, cu_seqlens=cu)
    total = torch.zeros(4, dtype=torch.float64)
    for q in range(4):
        lo, hi = cu[q], cu[q + 1]
        if lo == hi:
            assert torch.equal(res["final"][q], t["initial_states"][q]) and torch.equal(res["dinitial"][q], t["dfinal"][q])
            continue
        part = {n: t[n][:, lo:hi] for n in ("x", "gate_a", "gate_x", "dout")}
        one, _ = gated_linear_oracle(**part, decay=t["decay"], initial_states=t["initial_states"][q:q + 1], dfinal=t["dfinal"][q:q + 1])
        for n in ("out", "dx", "dgate_a", "dgate_x"):
            torch.testing.assert_close(res[n][:, lo:hi], one[n], rtol=1e-13, atol=0)
        for n in ("final", "dinitial"):
            torch.testing.assert_close(res[n][q:q + 1], one[n], rtol=1e-13, atol=0)
        total += one["ddecay"]
    torch.testing.assert_close(res["ddecay"], total, rtol=1e-12, atol=0)
    for n in ("out", "dx", "dgate_a", "dgate_x"):
        assert float(res[n][:, :2].abs().max()) == 0 and float(res[n][:, 13:].abs().max()) == 0
        assert float(bound[n][:, :2].abs().max()) == 0 and float(bound[n][:, 13:].abs().max()) == 0


@pytest.mark.parametrize("rms", [True, False])
@pytest.mark.parametrize("gate", [True, False])
@pytest.mark.parametrize("scale", ["tensor", 0.5, None])
@pytest.mark.parametrize("bias", [True, False])
def test_norm_oracle_against_autograd(rms, gate, scale, bias):
    g = torch.Generator().manual_seed(2)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)
    t = dict(x=r(2, 3, 7), residual=r(2, 3, 7), norm_weight=r(7), next_weight=r(7), z=r(2, 3, 7) if gate else None,
             scale=r(7) if scale == "tensor" else scale, norm_bias=r(7) if bias else None, next_bias=r(7) if bias else None)
    dout, dsum = r(2, 3, 7), r(2, 3, 7)
    leaves = {n: v.clone().requires_grad_() for n, v in t.items() if isinstance(v, torch.Tensor)}
    a = {**t, **leaves}
    norm = lambda v, w, b: ((torch.nn.functional.rms_norm(v, (7,), w, 1e-5) + (0 if b is None else b)) if rms
                            else torch.nn.functional.layer_norm(v, (7,), w, b, 1e-5))
    y = norm(a["x"], a["norm_weight"], a["norm_bias"])
    if gate:
        y = y * torch.nn.functional.silu(a["z"])
    total = a["residual"] + (y if scale is None else y * a["scale"])
    out = norm(total, a["next_weight"], a["next_bias"])
    grads = torch.autograd.grad([out, total], list(leaves.values()), [dout, dsum])
    res, _ = block_norm_oracle(**t, is_rms_norm=rms, dout=dout, dsum=dsum)
    torch.testing.assert_close(res["out"], out.detach(), rtol=1e-10, atol=1e-10)
    torch.testing.assert_close(res["residual_out"], total.detach(), rtol=1e-10, atol=1e-10)
    for n, v in zip(leaves, grads):
        torch.testing.assert_close(res["d" + n], v, rtol=1e-8, atol=1e-9)


def test_norm_oracle_against_differences():
    g = torch.Generator().manual_seed(5)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)
    t = dict(x=r(2, 5), residual=r(2, 5), norm_weight=r(5), next_weight=r(5), z=r(2, 5), scale=r(5), norm_bias=r(5), next_bias=r(5))
    dout, dsum = r(2, 5), r(2, 5)
    res, _ = block_norm_oracle(**t, is_rms_norm=False, dout=dout, dsum=dsum)
    value = lambda q: float((q["out"] * dout).sum() + (q["residual_out"] * dsum).sum())
    for name in t:
        for at in range(t[name].numel()):
            side = []
            for step in (1e-6, -1e-6):
                moved = t[name].clone()
                moved.view(-1)[at] += step
                side.append(value(block_norm_oracle(**{**t, name: moved}, is_rms_norm=False)[0]))
            assert abs((side[0] - side[1]) / 2e-6 - float(res["d" + name].view(-1)[at])) < 2e-6, (name, at)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_plain_statements_agree_with_the_oracles(dtype):
    from mamba_amd.ops.block_norm import block_norm_ref
    from mamba_amd.ops.gated_linear_scan import gated_linear_scan_ref, gated_linear_state_update_ref
    t = _inputs(2, 11, 5, seed=4, dtype=dtype)
    t["initial_states"] = t["initial_states"].float()
    five = [t[n] for n in ("x", "gate_a", "gate_x", "decay")]
    res, bound = gated_linear_oracle(*five, initial_states=t["initial_states"])
    out, final = gated_linear_scan_ref(*five, initial_states=t["initial_states"], return_final_states=True)
    within("out", out, res["out"], bound["out"])
    within("final", final, res["final"], bound["final"])
    state = t["initial_states"].clone()
    for q in range(11):
        y = gated_linear_state_update_ref(state, *[v[:, q] for v in five[:3]], five[3])
        within("step", y, res["out"][:, q], bound["out"][:, q])
    within("state", state, res["final"], bound["final"])
    g = torch.Generator().manual_seed(6)
    r = lambda *s: torch.randn(*s, generator=g).to(dtype)
    n = dict(x=r(3, 9), residual=r(3, 9), norm_weight=r(9), next_weight=r(9), z=r(3, 9), scale=r(9), norm_bias=r(9), next_bias=r(9))
    for rms in (True, False):
        res, bound = block_norm_oracle(**n, is_rms_norm=rms)
        out, total = block_norm_ref(**n, is_rms_norm=rms)
        within("out", out, res["out"], bound["out"])
        within("residual_out", total, res["residual_out"], bound["residual_out"])
