"""block_norm_fn against the 64-bit oracle, and the operators of a gated linear recurrent block one after the other."""
import pytest
import torch

from oracle.gated_linear import block_norm_oracle, gated_linear_oracle, within

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
NAMES = ["x", "residual", "norm_weight", "next_weight", "z", "scale", "norm_bias", "next_bias"]


def _fn(*args, **kw):
    from mamba_amd.ops.block_norm import block_norm_fn
    return block_norm_fn(*args, **kw)


def _inputs(shape, dtype, stream=None, params=torch.float32, gate=True, scale=True, bias=True, seed=0, shift=0.0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)
    dim = shape[-1]
    return dict(x=(r(*shape) + shift).to(dtype), residual=(2 * r(*shape)).to(stream or dtype), norm_weight=(1 + 0.2 * r(dim)).to(params),
                next_weight=(1 + 0.2 * r(dim)).to(params), z=r(*shape).to(dtype) if gate else None,
                scale=(0.5 + 0.1 * r(dim)).to(params) if scale is True else scale, norm_bias=0.3 * r(dim).to(params) if bias else None,
                next_bias=0.3 * r(dim).to(params) if bias else None, dout=r(*shape).to(dtype), dsum=r(*shape).to(stream or dtype))


def _run(t, rms, with_dsum=True, eps=1e-5):
    d = {k: (v.cuda() if isinstance(v, torch.Tensor) else v) for k, v in t.items()}
    leaves = [n for n in NAMES if isinstance(d[n], torch.Tensor)]
    for n in leaves:
        d[n].requires_grad_()
    out, total = _fn(*[d[n] for n in NAMES], eps=eps, is_rms_norm=rms)
    outs, douts = ([out, total], [d["dout"], d["dsum"]]) if with_dsum else ([out], [d["dout"]])
    grads = torch.autograd.grad(outs, [d[n] for n in leaves], douts)
    return dict(out=out.detach(), residual_out=total.detach(), **{"d" + n: g for n, g in zip(leaves, grads)})


def _check(t, rms, with_dsum=True, eps=1e-5):
    got = _run(t, rms, with_dsum, eps)
    ref, bound = block_norm_oracle(*[t[n] for n in NAMES], eps=eps, is_rms_norm=rms, dout=t["dout"], dsum=t["dsum"] if with_dsum else None)
    assert got["out"].dtype == t["x"].dtype and got["residual_out"].dtype == t["residual"].dtype
    for n, v in got.items():
        within(n, v, ref[n], bound[n])
    return got


@pytest.mark.parametrize("rms", [True, False])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,dim", [(1, 1), (3, 2), (1, 7), (5, 8), (2, 63), (4, 64), (1, 100), (9, 256), (3, 257), (2, 511), (7, 512),
                                      (2, 520), (3, 768), (2, 1001), (5, 1024), (1, 1032), (2, 2048), (3, 2560), (1, 4096), (2, 4104),
                                      (2, 5121), (3, 6144), (2, 6152), (1, 8192), (2, 8200), (1, 10000), (1, 32768)])
def test_sizes(rows, dim, dtype, rms):
    _check(_inputs((rows, dim), dtype, seed=dim), rms)


@pytest.mark.parametrize("rows,dim", [(1100, 64), (700, 520), (5000, 8), (1500, 130), (300, 2560), (2100, 768), (600, 6144), (600, 6152), (900, 8192)])
def test_many_rows(rows, dim):
    _check(_inputs((rows, dim), torch.bfloat16, stream=torch.float32, seed=rows), True)


@pytest.mark.parametrize("rms", [True, False])
@pytest.mark.parametrize("gate", [True, False])
@pytest.mark.parametrize("scale", [True, 0.25, None, 0.0])
@pytest.mark.parametrize("bias", [True, False])
@pytest.mark.parametrize("dim", [72, 75, 1056])
def test_options(dim, bias, scale, gate, rms):
    _check(_inputs((6, dim), torch.float32, gate=gate, scale=scale, bias=bias), rms)


@pytest.mark.parametrize("dim", [160, 2562])
@pytest.mark.parametrize("params", DTYPES)
@pytest.mark.parametrize("stream", ["same", "fp32"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_types(dtype, stream, params, dim):
    got = _check(_inputs((2, 5, dim), dtype, stream=torch.float32 if stream == "fp32" else dtype, params=params), False)
    assert got["dnorm_weight"].dtype == params and got["dscale"].dtype == params and got["dresidual"].dtype == got["residual_out"].dtype


def test_parameters_of_different_types():
    t = _inputs((4, 48), torch.bfloat16)
    t["norm_weight"], t["scale"] = t["norm_weight"].bfloat16(), t["scale"].half()
    got = _check(t, True)
    assert got["dnorm_weight"].dtype == torch.bfloat16 and got["dscale"].dtype == torch.float16 and got["dnext_weight"].dtype == torch.float32


@pytest.mark.parametrize("one_bias", ["norm_bias", "next_bias"])
@pytest.mark.parametrize("with_dsum", [True, False])
def test_one_bias_and_one_gradient(one_bias, with_dsum):
    t = _inputs((5, 96), torch.float32)
    t[one_bias] = None
    _check(t, False, with_dsum)


@pytest.mark.parametrize("rms", [True, False])
def test_rows_of_one_value_and_of_none(rms):
    """Rows of zeros, of one repeated value, far from zero, and large and small ones."""
    t = _inputs((6, 200), torch.float32)
    t["x"][0], t["residual"][0] = 0.0, 0.0
    t["x"][1], t["residual"][1] = 3.0, -2.0
    t["x"][2] += 100.0
    t["x"][3] *= 1e-4
    t["x"][4] *= 1e4
    t["residual"][5] *= 1e-3
    _check(t, rms)
    t["norm_weight"][:], t["norm_bias"][:], t["scale"][:] = 0.0, 0.0, 0.0
    _check(t, rms)


def test_a_row_without_numbers_stays_alone():
    t = _inputs((40, 136), torch.bfloat16)
    clean = _run(t, True)
    t["x"][7, 3], t["residual"][21, 0], t["z"][30, 5] = float("nan"), float("inf"), float("nan")
    got = _run(t, True)
    keep = [r for r in range(40) if r not in (7, 21, 30)]
    for n in ("out", "residual_out", "dx", "dresidual", "dz"):
        assert torch.equal(got[n][keep], clean[n][keep]), n
    assert torch.isnan(got["out"][7]).all() and torch.isnan(got["out"][30]).all()


@pytest.mark.parametrize("dim,offset", [(64, 0), (64, 1), (75, 2), (1032, 8), (2560, 4)])
def test_strided_rows(dim, offset):
    t = _inputs((5, dim), torch.bfloat16, stream=torch.float32)
    plain = _run(t, True)
    wide = torch.zeros(5, 2 * dim + offset, dtype=torch.bfloat16, device="cuda")
    x, z = wide[:, offset:offset + dim], wide[:, offset + dim:]
    x.copy_(t["x"]), z.copy_(t["z"])
    d = {k: (v.cuda() if isinstance(v, torch.Tensor) else v) for k, v in t.items()}
    d["x"], d["z"] = x.detach(), z.detach()
    leaves = [d[n].requires_grad_() for n in NAMES]
    out, total = _fn(*leaves)
    grads = torch.autograd.grad([out, total], leaves, [d["dout"], d["dsum"]])
    # an unaligned row may be summed in another order: two results within the bounds of the same values
    ref, bound = block_norm_oracle(*[t[n] for n in NAMES], is_rms_norm=True, dout=t["dout"], dsum=t["dsum"])
    for n, v in zip(["out", "residual_out"] + ["d" + n for n in NAMES], [out, total, *grads]):
        within(n, v, ref[n], bound[n])
    apart = d["residual"].detach().t().contiguous().t()
    assert torch.equal(_fn(t["x"].cuda(), apart, *[d[n] for n in NAMES[2:4]], t["z"].cuda(), *[d[n] for n in NAMES[5:]])[0], plain["out"])


def test_nothing_to_norm():
    t = _inputs((0, 3, 16), torch.float32)
    got = _run(t, True)
    assert got["out"].shape == (0, 3, 16) and torch.count_nonzero(got["dnorm_weight"]) == 0


def test_results_repeat_bit_for_bit():
    t = _inputs((2000, 264), torch.bfloat16, stream=torch.float32)
    first = _run(t, True)
    for _ in range(3):
        again = _run(t, True)
        assert all(torch.equal(first[n], again[n]) for n in first)


def test_no_second_derivatives():
    t = _inputs((2, 16), torch.float32)
    x = t["x"].cuda().requires_grad_()
    out, _ = _fn(x, *[t[n].cuda() for n in NAMES[1:]])
    g, = torch.autograd.grad(out, x, t["dout"].cuda(), create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_gradients_against_differences():
    """(f(p + s v) - f(p - s v)) / 2 s along a direction v, as for the scan: 1e-3 of the product of the norms."""
    t = {k: v.cuda() for k, v in _inputs((6, 40), torch.float32).items()}
    f = lambda a: _fn(*[a[n] for n in NAMES], is_rms_norm=False)
    g = torch.Generator(device="cuda").manual_seed(1)
    for n in NAMES:
        leaf = t[n].clone().requires_grad_()
        grad, = torch.autograd.grad(f({**t, n: leaf}), leaf, [t["dout"], t["dsum"]])
        v = torch.randn(leaf.shape, device="cuda", generator=g)
        s, side = 2.0 ** -6, []
        for step in (s, -s):
            out, total = f({**t, n: t[n] + step * v})
            side.append(float((out.double() * t["dout"]).sum() + (total.double() * t["dsum"]).sum()))
        want = float((grad.double() * v).sum())
        assert abs((side[0] - side[1]) / (2 * s) - want) <= 1e-3 * float(grad.norm() * v.norm()), n


def test_captured_pass_replays():
    shape = (130, 264)
    static = {k: v.cuda() for k, v in _inputs(shape, torch.bfloat16).items()}
    leaves = [static[n].requires_grad_() for n in NAMES]

    def step():
        out, total = _fn(*leaves)
        return [out.detach(), total.detach(), *torch.autograd.grad([out, total], leaves, [static["dout"], static["dsum"]])]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed in range(4):
        new = _inputs(shape, torch.bfloat16, seed=seed + 9)
        with torch.no_grad():
            for n, v in new.items():
                static[n].copy_(v)
        graph.replay()
        want = _run(new, True)
        torch.cuda.synchronize()
        for n, v in zip(["out", "residual_out"] + ["d" + n for n in NAMES], got):
            assert torch.equal(v, want[n]), (seed, n)


# ------------------------------------------------------------------ together
def test_a_block_in_training_prefill_and_decode():
    """One gated linear recurrent block as it is used: the norm in front, projections, the scan, the output projection and
    the norm that closes the block; its gradients against the same block of plain statements in float64, and the
    block over a prompt followed by single tokens against the block over the whole sequence."""
    from mamba_amd.ops.block_norm import block_norm_ref
    from mamba_amd.ops.gated_linear_scan import gated_linear_scan_fn, gated_linear_state_update
    from mamba_amd.ops.triton.layer_norm import rms_norm_fn
    g = torch.Generator(device="cuda").manual_seed(0)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)
    batch, L, d, width = 2, 70, 48, 64
    p = dict(first=1 + 0.1 * r(d), w_in=r(3 * width, d) / 7, w_out=r(d, width) / 8, decay=r(width) - 3, post=1 + 0.1 * r(d),
             nxt=1 + 0.1 * r(d), scale=0.5 + 0.1 * r(d), w_gate=r(d, d) / 7)
    h0 = r(batch, L, d)

    def block(h, q, state=None):
        u = rms_norm_fn(h, q["first"], None, eps=1e-5)
        x, ga, gx = (u @ q["w_in"].t()).split(width, -1)
        y, last = gated_linear_scan_fn(x, ga, gx, q["decay"], initial_states=state, return_final_states=True)
        out, total = _fn(y @ q["w_out"].t(), h, q["post"], q["nxt"], z=u @ q["w_gate"].t(), scale=q["scale"])
        return out, total, last

    def plain(h, q):
        norm = lambda v, w: v / torch.sqrt((v * v).mean(-1, keepdim=True) + 1e-5) * w
        u = norm(h, q["first"])
        x, ga, gx = (u @ q["w_in"].t()).split(width, -1)
        log_a = -8 * torch.nn.functional.softplus(q["decay"]) * torch.sigmoid(ga)
        b = torch.sqrt(-torch.expm1(2 * log_a)) * torch.sigmoid(gx) * x
        s, ys = torch.zeros_like(b[:, 0]), []
        for t in range(L):
            s = torch.exp(log_a[:, t]) * s + b[:, t]
            ys.append(s)
        total = h + q["scale"] * norm(torch.stack(ys, 1) @ q["w_out"].t(), q["post"]) * torch.nn.functional.silu(u @ q["w_gate"].t())
        return norm(total, q["nxt"]), total

    leaves = {k: v.clone().requires_grad_() for k, v in p.items()}
    h = h0.clone().requires_grad_()
    out, total, _ = block(h, leaves)
    wide = {k: v.double().cpu().requires_grad_() for k, v in p.items()}
    hw = h0.double().cpu().requires_grad_()
    out_w, total_w = plain(hw, wide)
    dout, dsum = r(batch, L, d), r(batch, L, d)
    got = torch.autograd.grad([out, total], [h, *leaves.values()], [dout, dsum])
    want = torch.autograd.grad([out_w, total_w], [hw, *wide.values()], [dout.double().cpu(), dsum.double().cpu()])
    # fp32 throughout: a chain of ~10 operators, each within 1e-6 of its own result, through factors of size 1 to 10
    for name, a, b in zip(["out", "total", "h", *p], [out, total, *got], [out_w, total_w, *want]):
        err = float((a.double().cpu() - b).norm() / b.norm())
        assert err < 2e-5, (name, err)
    # prompt, then tokens
    with torch.no_grad():
        whole, sums, _ = block(h0, p)
        o, t, state = block(h0[:, :60], p)
        outs, totals = [o], [t]
        for q in range(60, L):
            hq = h0[:, q]
            u = rms_norm_fn(hq, p["first"], None, eps=1e-5)
            x, ga, gx = (u @ p["w_in"].t()).split(width, -1)
            y = gated_linear_state_update(state, x, ga, gx, p["decay"])
            o, t = _fn(y @ p["w_out"].t(), hq, p["post"], p["nxt"], z=u @ p["w_gate"].t(), scale=p["scale"])
            outs.append(o[:, None]), totals.append(t[:, None])
        for a, b in ((torch.cat(outs, 1), whole), (torch.cat(totals, 1), sums)):
            assert float((a - b).norm() / b.norm()) < 1e-5
