"""gated_linear_scan_fn and gated_linear_state_update against the 64-bit oracle: outputs, states and every gradient within
the bounds that stand beside the oracle's results plus half a step of the result's type."""
import pytest
import torch

from oracle.gated_linear import gated_linear_oracle, within

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
NAMES = ["x", "gate_a", "gate_x", "decay", "initial_states"]
GRADS = ["dx", "dgate_a", "dgate_x", "ddecay", "dinitial"]


def _fn(*args, **kw):
    from mamba_amd.ops.gated_linear_scan import gated_linear_scan_fn
    return gated_linear_scan_fn(*args, **kw)


def _inputs(batch, L, dim, dtype, seed=0, seqs=None, states=True, long_memory=False):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s, dt=dtype: torch.randn(*s, generator=g).to(dt)
    n = batch if seqs is None else seqs
    t = dict(x=r(batch, L, dim), gate_a=r(batch, L, dim), gate_x=r(batch, L, dim), decay=r(dim, dt=torch.float32),
             initial_states=r(n, dim, dt=torch.float32) if states else None, dout=r(batch, L, dim),
             dfinal=r(n, dim, dt=torch.float32) if states else None)
    if long_memory:
        keep = 0.9 + 0.099 * torch.rand(dim, generator=g)
        t["decay"] = torch.log(torch.expm1(-torch.log(keep) / 8))
    return t


def _run(t, cu=None, rate=8.0, backward=True):
    """The operator's results under the oracle's names."""
    d = {k: (v.cuda() if v is not None else None) for k, v in t.items()}
    leaves = [n for n in NAMES if d[n] is not None]
    for n in leaves:
        d[n].requires_grad_(backward)
    cu = torch.tensor(cu, dtype=torch.int32, device="cuda") if cu is not None else None
    out, final = _fn(d["x"], d["gate_a"], d["gate_x"], d["decay"], rate=rate, initial_states=d["initial_states"], cu_seqlens=cu,
                     return_final_states=True)
    res = dict(out=out.detach(), final=final.detach())
    if backward:
        outs, douts = ([out, final], [d["dout"], d["dfinal"]]) if d["dfinal"] is not None else ([out], [d["dout"]])
        res.update(zip([GRADS[NAMES.index(n)] for n in leaves], torch.autograd.grad(outs, [d[n] for n in leaves], douts)))
    return res


def _check(t, cu=None, rate=8.0):
    got = _run(t, cu, rate)
    ref, bound = gated_linear_oracle(t["x"], t["gate_a"], t["gate_x"], t["decay"], rate, t["initial_states"], cu, t["dout"], t["dfinal"])
    assert got["out"].dtype == t["x"].dtype and got["final"].dtype == torch.float32
    for n, v in got.items():
        within(n, v, ref[n], bound[n])
    return got


# one channel and one position; lengths and channel counts around the sizes of a wave, of its rows and of several tiles
SHAPES = [(1, 1, 1), (1, 1, 64), (3, 2, 5), (2, 3, 127), (1, 7, 128), (1, 8, 129), (2, 9, 256), (1, 16, 130), (1, 31, 1), (2, 33, 66),
          (1, 63, 255), (1, 64, 128), (1, 65, 257), (3, 100, 70), (1, 127, 4), (1, 128, 130), (2, 129, 128), (1, 255, 34), (1, 256, 6),
          (2, 257, 130), (1, 513, 3), (1, 1025, 8), (2, 2100, 2), (1, 4500, 1)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("batch,L,dim", SHAPES)
def test_shapes(batch, L, dim, dtype):
    _check(_inputs(batch, L, dim, dtype, seed=L + dim, states=(L + dim) % 3 != 0))


# both sides of the lines at which a pass takes other tiles, and rows enough that every tile hands its state on by itself
@pytest.mark.parametrize("batch,L,dim,dtype", [
    (2, 32, 130, torch.bfloat16), (2, 33, 130, torch.bfloat16),
    (16, 64 * 32, 2, torch.float32), (16, 64 * 32 + 1, 2, torch.float32), (9, 3700, 129, torch.bfloat16),
    (64, 64 * 32, 1, torch.float32), (64, 64 * 32 + 5, 2, torch.bfloat16), (22, 6200, 130, torch.float16),
    (130, 300, 5, torch.float32), (140, 1000, 2, torch.bfloat16)])
def test_sizes_of_other_tiles(batch, L, dim, dtype):
    _check(_inputs(batch, L, dim, dtype, seed=L, states=L % 2 == 0, long_memory=dtype == torch.float32))


@pytest.mark.parametrize("total,dim", [(17000, 257), (66100, 129)])
def test_long_packed_rows(total, dim):
    g = torch.Generator().manual_seed(total)
    cu = [0, 3] + (torch.randperm(total - 500, generator=g)[:21] + 20).sort().values.tolist()
    _check(_inputs(1, total, dim, torch.bfloat16, seqs=len(cu) - 1), cu)


@pytest.mark.parametrize("L", [300, 3000])
def test_long_memory(L):
    """Decays as such layers are initialised: a state lasts for hundreds of positions."""
    _check(_inputs(2, L, 6, torch.float32, seed=7, long_memory=True))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cu", [
    [0, 9], [0, 1, 2, 3, 4, 5, 6, 7], [0, 0, 5, 5, 5, 40, 40], [3, 10, 64, 65, 128, 129, 200], [0, 8, 16, 24, 64, 128, 256, 300],
    [17, 17, 17], [0, 300], [300, 300, 300], [0, 130, 131, 257, 258, 259, 299]], ids=str)
def test_packed(cu, dtype):
    """Sequences of every length from none on, with positions that hold no numbers before the first and behind the last."""
    t = _inputs(1, 300, 130, dtype, seed=len(cu), seqs=len(cu) - 1)
    for n in ("x", "gate_a", "gate_x", "dout"):
        t[n][:, :cu[0]] = float("nan")
        t[n][:, cu[-1]:] = float("inf")
    got = _check(t, cu)
    for n in ("out", "dx", "dgate_a", "dgate_x"):
        assert torch.count_nonzero(got[n][:, :cu[0]]) == 0 and torch.count_nonzero(got[n][:, cu[-1]:]) == 0


def test_many_short_sequences():
    g = torch.Generator().manual_seed(3)
    lengths = torch.randint(0, 5, (700,), generator=g)
    cu = [0] + lengths.cumsum(0).tolist()
    _check(_inputs(1, cu[-1] + 3, 9, torch.bfloat16, seed=5, seqs=700), cu)


def test_a_sequence_keeps_no_numbers_out_of_the_next():
    t = _inputs(1, 200, 8, torch.float32, seqs=2)
    t["x"][:, :100] = float("inf")
    t["gate_a"][:, 50] = float("nan")
    t["dout"][:, :100] = float("nan")
    got = _run(t, [0, 100, 200])
    part = {n: (t[n][:, 100:] if n in ("x", "gate_a", "gate_x", "dout") else t[n][1:] if n != "decay" else t[n]) for n in t}
    one = _run(part)
    for n in ("out", "dx", "dgate_a", "dgate_x"):
        assert torch.isfinite(got[n][:, 100:]).all()
        torch.testing.assert_close(got[n][:, 100:], one[n], rtol=1e-5, atol=1e-6)
    torch.testing.assert_close(got["final"][1:], one["final"], rtol=1e-5, atol=1e-6)
    # ... and the other way round
    u = _inputs(1, 200, 8, torch.float32, seqs=2)
    u["x"][:, 100:] = float("nan")
    u["dout"][:, 100:] = float("inf")
    got = _run(u, [0, 100, 200])
    for n in ("out", "dx", "dgate_a", "dgate_x"):
        assert torch.isfinite(got[n][:, :100]).all()
    assert torch.isfinite(got["dinitial"][0]).all() and not torch.isfinite(got["out"][:, 100:]).any()


@pytest.mark.parametrize("L", [70, 700])
def test_what_is_no_number_stays_in_its_row_and_channel(L):
    t = _inputs(2, L, 5, torch.float32)
    t["x"][1, 40, 3] = float("nan")
    out = _run(t, backward=False)["out"]
    clean = _run(_inputs(2, L, 5, torch.float32), backward=False)["out"]
    assert torch.isnan(out[1, 40:, 3]).all()
    out[1, 40:, 3] = clean[1, 40:, 3]
    assert torch.equal(out, clean)


def test_gates_and_decays_at_their_ends():
    """Shut and open gates to the last bit and beyond, decays of nothing and of everything, a rate of 0."""
    t = _inputs(1, 40, 16, torch.float32)
    ends = torch.tensor([-1e4, -100.0, -88.0, -20.0, -1e-30, 0.0, 20.0, 88.0, 100.0, 1e4])
    t["gate_a"][0, :, :10] = ends
    t["gate_x"][0, ::2, 2:12] = ends
    t["decay"][:6] = torch.tensor([-100.0, -20.0, 30.0, 100.0, -60.0, 0.0])
    got = _check(t)
    assert all(torch.isfinite(v).all() for v in got.values())
    got = _check(t, rate=0.0)
    assert torch.equal(got["out"], t["initial_states"][:, None].cuda().expand_as(got["out"]))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,offset", [(64, 0), (66, 1), (33, 3), (130, 2)])
def test_strided_rows(dim, offset, dtype):
    """x and the gates as slices of one projection's output, off any alignment; batch rows far apart; a gradient that is an
    expanded number; channels that lie apart (copied first)."""
    t = _inputs(2, 50, dim, dtype)
    wide = torch.zeros(3, 50, 3 * dim + offset, dtype=dtype, device="cuda")
    parts = [wide[::2][:, :, offset + j * dim:offset + (j + 1) * dim] for j in range(3)]
    for p, n in zip(parts, NAMES):
        p.copy_(t[n])
    plain = _run(t)
    leaves = [p.detach().requires_grad_() for p in parts]
    assert leaves[1].stride(1) == 3 * dim + offset
    decay = t["decay"].cuda().requires_grad_()
    out, final = _fn(*leaves, decay, initial_states=t["initial_states"].cuda(), return_final_states=True)
    grads = torch.autograd.grad([out, final], leaves + [decay], [t["dout"].cuda(), t["dfinal"].cuda()])
    for n, v in zip(["out", "final"] + GRADS, [out, final, *grads]):
        assert torch.equal(v, plain[n]), n
    apart = [t[n].cuda().transpose(1, 2).contiguous().transpose(1, 2) for n in NAMES[:3]]
    assert torch.equal(_fn(*apart, decay, initial_states=t["initial_states"].cuda()), plain["out"])
    t["dout"] = torch.full_like(t["dout"], 0.5)
    leaves = [t[n].cuda().requires_grad_() for n in NAMES[:3]]
    _fn(*leaves, decay, initial_states=t["initial_states"].cuda()).backward(torch.full((), 0.5, dtype=dtype, device="cuda").expand(2, 50, dim))
    want = _run({**t, "dfinal": None})
    assert all(torch.equal(v.grad, want[n]) for v, n in zip(leaves, GRADS))


@pytest.mark.parametrize("gates", [torch.float32, torch.float16])
def test_types_next_to_bf16(gates):
    """Gates, decays and states in types of their own: gradients come back in those."""
    t = _inputs(1, 40, 24, torch.bfloat16)
    x, ga, gx = (t[n].cuda().to(d).requires_grad_() for n, d in zip(NAMES, (torch.bfloat16, gates, gates)))
    decay, init = t["decay"].cuda().half().requires_grad_(), t["initial_states"].cuda().bfloat16().requires_grad_()
    out = _fn(x, ga, gx, decay, initial_states=init)
    grads = torch.autograd.grad(out, [x, ga, gx, decay, init], t["dout"].cuda())
    assert [g.dtype for g in grads] == [torch.bfloat16, gates, gates, torch.float16, torch.bfloat16]
    t.update(decay=t["decay"].half(), initial_states=t["initial_states"].bfloat16(), dfinal=None)
    ref, bound = gated_linear_oracle(t["x"], t["gate_a"], t["gate_x"], t["decay"], 8.0, t["initial_states"], None, t["dout"])
    within("out", out, ref["out"], bound["out"])
    for n, g in zip(GRADS, grads):
        # the gates' gradients are rounded to bf16 and then to the gates' own type, by half a step of it: in fp16 2^-11 of
        # the value, and 2^-25 of its smallest numbers
        own = (2.0 ** -11 * ref[n].abs() + 2.0 ** -25) if g.dtype == torch.float16 else 0.0
        within(n, g.to(torch.bfloat16) if n in ("dgate_a", "dgate_x") else g, ref[n], bound[n] + own)


@pytest.mark.parametrize("shape", [(0, 5, 4), (2, 0, 4), (2, 5, 0)])
def test_nothing_to_scan(shape):
    t = _inputs(*shape, torch.float32)
    got = _run(t)
    assert got["out"].shape == shape and got["final"].shape == (shape[0], shape[2])
    if shape[1] == 0:
        assert torch.equal(got["final"].cpu(), t["initial_states"]) and torch.equal(got["dinitial"].cpu(), t["dfinal"])
    assert torch.count_nonzero(got["ddecay"]) == 0 and got["ddecay"].shape == (shape[2],)


def test_only_what_is_asked_for():
    t = _inputs(2, 90, 40, torch.float32)
    d = {k: v.cuda() for k, v in t.items()}
    x = d["x"].requires_grad_()
    args = (x, d["gate_a"], d["gate_x"], d["decay"])
    _, final = _fn(*args, initial_states=d["initial_states"], return_final_states=True)
    dx, = torch.autograd.grad(final, x, d["dfinal"])
    ref, bound = gated_linear_oracle(*[t[n] for n in NAMES[:4]], 8.0, t["initial_states"], None, None, t["dfinal"])
    within("dx", dx, ref["dx"], bound["dx"])
    out, final = _fn(*args, initial_states=d["initial_states"], return_final_states=True)
    final.detach()
    dx, = torch.autograd.grad(out, x, d["dout"])
    ref, bound = gated_linear_oracle(*[t[n] for n in NAMES[:4]], 8.0, t["initial_states"], None, t["dout"], None)
    within("dx", dx, ref["dx"], bound["dx"])
    out = _fn(*args)
    g, = torch.autograd.grad(out, x, d["dout"], create_graph=True)
    with pytest.raises(RuntimeError):  # no second derivatives
        g.sum().backward()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("batch,L,dim", [(2, 1500, 130), (1, 5000, 33)])
def test_results_repeat_bit_for_bit(batch, L, dim, dtype):
    t = _inputs(batch, L, dim, dtype)
    first = _run(t)
    for _ in range(3):
        again = _run(t)
        for n in first:
            assert torch.equal(first[n], again[n]), n


def test_gradients_against_differences():
    """Along a direction v: (f(p + s v) - f(p - s v)) / 2 s = gradient . v, f in fp32 and summed in fp64.  With s = 2^-6 and
    terms of size 1 the third derivative adds s^2 / 6 of them, 4e-5, and the rounding of f 2^-20 / s, 6e-5: 1e-3 of the
    product of the norms covers both."""
    t = {k: v.cuda() for k, v in _inputs(1, 150, 20, torch.float32, long_memory=True).items()}

    def f(**moved):
        a = {**t, **moved}
        out, final = _fn(a["x"], a["gate_a"], a["gate_x"], a["decay"], initial_states=a["initial_states"], return_final_states=True)
        return out, final, float((out.double() * t["dout"]).sum() + (final.double() * t["dfinal"]).sum())

    g = torch.Generator(device="cuda").manual_seed(1)
    for n in NAMES:
        leaf = t[n].clone().requires_grad_()
        out, final, _ = f(**{n: leaf})
        grad, = torch.autograd.grad([out, final], leaf, [t["dout"], t["dfinal"]])
        v = torch.randn(leaf.shape, device="cuda", generator=g) * grad.abs().mean().sign()
        s = 2.0 ** -6
        with torch.no_grad():
            slope = (f(**{n: t[n] + s * v})[2] - f(**{n: t[n] - s * v})[2]) / (2 * s)
        want = float((grad.double() * v).sum())
        assert abs(slope - want) <= 1e-3 * float(grad.norm() * v.norm()), (n, slope, want)


def test_a_state_hands_a_sequence_on():
    t = _inputs(2, 700, 70, torch.float32)
    whole = _run(t, backward=False)
    d = {k: v.cuda() for k, v in t.items()}
    state, outs = d["initial_states"], []
    for lo, hi in ((0, 1), (1, 130), (130, 131), (131, 640), (640, 700)):
        out, state = _fn(*[d[n][:, lo:hi] for n in NAMES[:3]], d["decay"], initial_states=state, return_final_states=True)
        outs.append(out)
    # both are within the oracle's bounds of the same values; here they are held to twice the whole's
    ref, bound = gated_linear_oracle(t["x"], t["gate_a"], t["gate_x"], t["decay"], 8.0, t["initial_states"])
    within("out", torch.cat(outs, 1), ref["out"], 2 * bound["out"])
    within("final", state, ref["final"], 2 * bound["final"])
    within("whole", whole["out"], ref["out"], bound["out"])


def test_captured_pass_replays():
    """Forward and backward in one captured graph, replayed with eager passes between the replays."""
    t = {k: v.cuda() for k, v in _inputs(1, 900, 130, torch.bfloat16).items()}
    static = {k: v.clone() for k, v in t.items()}
    leaves = [static[n].requires_grad_() for n in NAMES]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())

    def step():
        out, final = _fn(*leaves[:4], initial_states=leaves[4], return_final_states=True)
        return [out.detach(), final.detach(), *torch.autograd.grad([out, final], leaves, [static["dout"], static["dfinal"]])]

    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed in range(4):
        new = _inputs(1, 900, 130, torch.bfloat16, seed=seed + 20)
        with torch.no_grad():
            for n, v in new.items():
                static[n].copy_(v)
        graph.replay()
        want = _run(new)
        torch.cuda.synchronize()
        for n, v in zip(["out", "final"] + GRADS, got):
            assert torch.equal(v, want[n]), (seed, n)


def test_two_streams_at_once():
    ts = [{k: v.cuda() for k, v in _inputs(1, 3000, 130, torch.bfloat16, seed=s).items()} for s in range(2)]
    want = [_fn(*[t[n] for n in NAMES[:4]], initial_states=t["initial_states"]) for t in ts]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for s, t, o in zip(streams, ts, got):
            with torch.cuda.stream(s):
                o.append(_fn(*[t[n] for n in NAMES[:4]], initial_states=t["initial_states"]))
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for os, w in zip(got, want) for o in os)


def test_under_autocast():
    t = _inputs(1, 60, 32, torch.bfloat16)
    plain = _run(t, backward=False)["out"]
    with torch.autocast("cuda", dtype=torch.bfloat16):
        got = _run(t, backward=False)["out"]
    assert torch.equal(plain, got)


# ------------------------------------------------------------------ one position
def _step(*args, **kw):
    from mamba_amd.ops.gated_linear_scan import gated_linear_state_update
    return gated_linear_state_update(*args, **kw)


@pytest.mark.parametrize("state_dtype", DTYPES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("batch,dim", [(1, 1), (1, 64), (3, 127), (2, 512), (7, 257), (1, 2560), (300, 10), (5, 2049)])
def test_step(batch, dim, dtype, state_dtype):
    t = _inputs(batch, 1, dim, dtype, seed=dim)
    state = t["initial_states"].to(state_dtype)
    dev = state.cuda()
    out = _step(dev, *[t[n][:, 0].cuda() for n in NAMES[:3]], t["decay"].cuda())
    ref, bound = gated_linear_oracle(t["x"], t["gate_a"], t["gate_x"], t["decay"], 8.0, state.float())
    assert out.dtype == dtype
    within("out", out, ref["out"][:, 0], bound["out"][:, 0])
    within("state", dev, ref["final"], bound["final"])


@pytest.mark.parametrize("index_dtype", [torch.int32, torch.int64])
def test_step_in_a_pool_of_rows(index_dtype):
    t = _inputs(9, 1, 130, torch.bfloat16)
    pool = torch.randn(20, 130)
    rows = [3, -1, 19, 0, 20, 7, -5, 11, 2 ** 31 - 1]
    dev = pool.cuda()
    out = _step(dev, *[t[n][:, 0].cuda() for n in NAMES[:3]], t["decay"].cuda(),
                state_batch_indices=torch.tensor(rows, dtype=index_dtype).cuda())
    used = [b for b, r in enumerate(rows) if 0 <= r < 20]
    ref, bound = gated_linear_oracle(*[t[n][used] for n in NAMES[:3]], t["decay"], 8.0, pool[[rows[b] for b in used]])
    within("out", out[used], ref["out"][:, 0], bound["out"][:, 0])
    within("state", dev[[rows[b] for b in used]], ref["final"], bound["final"])
    rest = [r for r in range(20) if r not in rows]
    assert torch.equal(dev[rest].cpu(), pool[rest])
    assert torch.count_nonzero(out[[b for b in range(9) if b not in used]]) == 0


def test_step_forms():
    t = _inputs(4, 1, 66, torch.bfloat16)
    args = [t[n][:, 0].cuda() for n in NAMES[:3]]
    decay, init = t["decay"].cuda(), t["initial_states"].cuda()
    a = init.clone()
    want = _step(a, *args, decay)
    # slices of one projection, off any alignment, and a state that is a slice of a longer row
    wide = torch.zeros(4, 3 * 66 + 1, dtype=torch.bfloat16, device="cuda")
    parts = [wide[:, 1 + 66 * j:67 + 66 * j] for j in range(3)]
    for p, v in zip(parts, args):
        p.copy_(v)
    row = torch.full((4, 100), 7.0, device="cuda")
    row[:, 3:69] = init
    assert torch.equal(_step(row[:, 3:69], *parts, decay), want) and torch.equal(row[:, 3:69], a)
    assert torch.equal(row[:, :3], torch.full((4, 3), 7.0, device="cuda")) and torch.equal(row[:, 69:], torch.full((4, 31), 7.0, device="cuda"))
    # channels apart in the inputs, gates in fp32, no entries, a pool without rows
    b = init.clone()
    assert torch.equal(_step(b, *[v.t().contiguous().t() for v in args], decay), want) and torch.equal(a, b)
    b = init.clone()
    assert torch.equal(_step(b, args[0], args[1].float(), args[2].float(), decay), want) and torch.equal(a, b)
    assert _step(init, *[v[:0] for v in args], decay).shape == (0, 66)
    none = _step(init[:0], *args, decay, state_batch_indices=torch.zeros(4, dtype=torch.int32, device="cuda"))
    assert torch.count_nonzero(none) == 0


def test_steps_follow_a_scan():
    """A prompt by the scan, the tokens after it by steps, in eager calls and in replays of a captured one."""
    t = _inputs(3, 90, 72, torch.float32)
    d = {k: v.cuda() for k, v in t.items()}
    whole = _fn(*[d[n] for n in NAMES[:4]], initial_states=d["initial_states"])
    _, state = _fn(*[d[n][:, :80] for n in NAMES[:3]], d["decay"], initial_states=d["initial_states"], return_final_states=True)
    eager = state.clone()
    outs = [_step(eager, *[d[n][:, q] for n in NAMES[:3]], d["decay"]) for q in range(80, 90)]
    ref, bound = gated_linear_oracle(t["x"], t["gate_a"], t["gate_x"], t["decay"], 8.0, t["initial_states"])
    within("out", torch.stack(outs, 1), ref["out"][:, 80:], 2 * bound["out"][:, 80:])
    within("whole", whole, ref["out"], bound["out"])
    within("state", eager, ref["final"], 2 * bound["final"])
    static = [d[n][:, 0].clone() for n in NAMES[:3]]
    live = state.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _step(torch.zeros_like(live), *static, d["decay"])
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _step(live, *static, d["decay"])
    for q in range(80, 90):
        for s, n in zip(static, NAMES):
            s.copy_(d[n][:, q])
        graph.replay()
        assert torch.equal(out, outs[q - 80])
    assert torch.equal(live, eager)
