"""linear_attention_fn against the 64-bit oracle: outputs, states and every gradient within the bounds that stand beside the
oracle's results plus half a step of the result's type."""
import pytest
import torch

from oracle.linear_attention import linear_attention_oracle, within

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
NAMES = ["q", "k", "v", "initial_states"]
GRADS = ["dq", "dk", "dv", "dinitial"]


def _fn(*args, **kw):
    from mamba_amd.ops.linear_attention import linear_attention_fn
    return linear_attention_fn(*args, **kw)


def _inputs(batch, L, heads, dk, dv, dtype, kv=None, seed=0, seqs=None, states=True):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s, dt=dtype: torch.randn(*s, generator=g).to(dt)
    n, kv = batch if seqs is None else seqs, kv or heads
    return dict(q=r(batch, L, heads, dk), k=r(batch, L, kv, dk), v=r(batch, L, kv, dv),
                log_decay=torch.log1p(-torch.exp2(-torch.linspace(0.5, 12, heads))),
                initial_states=r(n, heads, dk, dv, dt=torch.float32) if states else None, dout=r(batch, L, heads, dv),
                dfinal=r(n, heads, dk, dv, dt=torch.float32) if states else None)


def _run(t, cu=None, scale=None, backward=True):
    """The operator's results under the oracle's names."""
    d = {k: (v.cuda() if v is not None else None) for k, v in t.items()}
    leaves = [n for n in NAMES if d[n] is not None]
    for n in leaves:
        d[n].requires_grad_(backward)
    cu = torch.tensor(cu, dtype=torch.int32, device="cuda") if cu is not None else None
    out, final = _fn(d["q"], d["k"], d["v"], d["log_decay"], scale=scale, initial_states=d["initial_states"], cu_seqlens=cu,
                     return_final_states=True)
    res = dict(out=out.detach(), final=final.detach())
    if backward:
        outs, douts = ([out, final], [d["dout"], d["dfinal"]]) if d["dfinal"] is not None else ([out], [d["dout"]])
        res.update(zip([GRADS[NAMES.index(n)] for n in leaves], torch.autograd.grad(outs, [d[n] for n in leaves], douts)))
    return res


def _check(t, cu=None, scale=None):
    got = _run(t, cu, scale)
    ref, bound = linear_attention_oracle(t["q"], t["k"], t["v"], t["log_decay"], scale, t["initial_states"], cu, t["dout"], t["dfinal"])
    assert got["out"].dtype == t["q"].dtype and got["final"].dtype == torch.float32
    for n, v in got.items():
        within(n, v, ref[n], bound[n])
    return got


# one position; lengths around the positions of a block and of several; head sizes around those the kernels are made for, odd ones
# and ones beyond the values of a workgroup
SHAPES = [(1, 1, 1, 1, 1), (2, 1, 3, 64, 64), (1, 2, 2, 8, 16), (3, 15, 2, 33, 7), (1, 16, 2, 16, 16), (1, 31, 1, 5, 70), (2, 32, 2, 64, 32),
          (1, 33, 2, 40, 72), (1, 63, 2, 128, 128), (2, 64, 1, 80, 104), (1, 65, 2, 100, 100), (1, 100, 2, 128, 64), (1, 127, 1, 64, 128),
          (1, 128, 2, 72, 130), (1, 129, 2, 130, 72), (1, 200, 1, 256, 256), (2, 70, 1, 200, 136), (1, 77, 1, 255, 253), (1, 66, 2, 1, 256),
          (1, 90, 1, 256, 1), (2, 257, 3, 48, 48)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("batch,L,heads,dk,dv", SHAPES)
def test_shapes(batch, L, heads, dk, dv, dtype):
    _check(_inputs(batch, L, heads, dk, dv, dtype, seed=L + dk, states=(L + dk) % 3 != 0))


# lengths that are cut into segments, one position over, and ones with so many heads that they are not
@pytest.mark.parametrize("batch,L,heads,dk,dv,dtype", [
    (1, 512, 2, 64, 64, torch.bfloat16), (1, 513, 2, 64, 64, torch.float32), (2, 777, 3, 128, 128, torch.bfloat16),
    (1, 1025, 2, 40, 100, torch.float16), (1, 1500, 1, 256, 64, torch.bfloat16), (1, 2049, 1, 64, 256, torch.float32),
    (3, 4000, 1, 32, 32, torch.bfloat16), (1, 700, 300, 16, 16, torch.bfloat16), (70, 300, 8, 8, 8, torch.float16)])
def test_long_rows(batch, L, heads, dk, dv, dtype):
    _check(_inputs(batch, L, heads, dk, dv, dtype, seed=L, states=L % 2 == 1))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv,dk,dv,L", [(4, 1, 32, 48, 70), (6, 3, 64, 64, 130), (8, 2, 100, 36, 40), (16, 2, 16, 128, 600)])
def test_shared_keys_and_values(heads, kv, dk, dv, L, dtype):
    _check(_inputs(2, L, heads, dk, dv, dtype, kv=kv, seed=heads))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cu", [
    [0, 9], [0, 1, 2, 3, 4, 5, 6, 7], [0, 0, 5, 5, 5, 40, 40], [3, 10, 64, 65, 128, 129, 200], [0, 8, 16, 24, 64, 128, 256, 300],
    [17, 17, 17], [0, 300], [300, 300, 300], [0, 130, 131, 257, 258, 259, 299]], ids=str)
def test_packed(cu, dtype):
    """Sequences of every length from none on, with positions that hold no numbers before the first and behind the last."""
    t = _inputs(1, 300, 4, 40, 24, dtype, kv=2, seed=len(cu), seqs=len(cu) - 1)
    for n in ("q", "k", "v", "dout"):
        t[n][:, :cu[0]] = float("nan")
        t[n][:, cu[-1]:] = float("inf")
    got = _check(t, cu)
    for n in ("out", "dq", "dk", "dv"):
        assert torch.count_nonzero(got[n][:, :cu[0]]) == 0 and torch.count_nonzero(got[n][:, cu[-1]:]) == 0


@pytest.mark.parametrize("total,heads,dtype", [(5000, 2, torch.bfloat16), (9000, 1, torch.float32)])
def test_long_packed_rows(total, heads, dtype):
    """Sequences that are cut into segments beside ones that are not, and padding at both ends."""
    g = torch.Generator().manual_seed(total)
    cu = [7, 9, 9] + (torch.randperm(total - 600, generator=g)[:6] + 20).sort().values.tolist() + [total - 300]
    _check(_inputs(1, total, heads, 32, 32, dtype, seqs=len(cu) - 1), cu)


def test_many_short_sequences():
    g = torch.Generator().manual_seed(3)
    lengths = torch.randint(0, 5, (700,), generator=g)
    cu = [0] + lengths.cumsum(0).tolist()
    _check(_inputs(1, cu[-1] + 3, 2, 16, 8, torch.bfloat16, seed=5, seqs=700), cu)


@pytest.mark.parametrize("dtype", DTYPES)
def test_decays_at_their_ends(dtype):
    """No decay, one that forgets everything, ones far below zero, and one above, which counts as none."""
    t = _inputs(1, 150, 6, 24, 40, dtype, seed=4)
    t["log_decay"] = torch.tensor([0.0, -float("inf"), -90.0, -3e38, -1e-30, 2.0])
    _check(t)


def test_no_number_as_a_decay_stays_in_its_head():
    t = _inputs(1, 100, 3, 24, 40, torch.float32, seed=4)
    want = _run(t)
    t["log_decay"][1] = float("nan")
    got = _run(t)
    for n in want:
        axis = 1 if n in ("final", "dinitial") else 2
        a, b = got[n].movedim(axis, 0), want[n].movedim(axis, 0)
        assert bool(a[1].isnan().all()) and torch.equal(a[[0, 2]], b[[0, 2]])


@pytest.mark.parametrize("scale", [0.0, 1.0, -2.5])
def test_scales(scale):
    _check(_inputs(1, 80, 2, 32, 32, torch.bfloat16, seed=9), scale=scale)


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("which", ["q", "k", "v", "dout"])
def test_what_is_no_number_stays_in_its_sequence_and_head(which, value):
    cu = [0, 100, 230, 300]
    t = _inputs(1, 300, 4, 24, 16, torch.bfloat16, seqs=3)
    want = _run(t, cu)
    t[which][0, 150, 1, 3] = value
    got = _run(t, cu)
    for n, a in got.items():
        b = want[n]
        if n in ("final", "dinitial"):
            keep = torch.ones(3, 4, dtype=torch.bool)
            keep[1, 1] = False
        else:
            keep = torch.ones(1, 300, 4, dtype=torch.bool)
            keep[0, 100:230, 1] = False
        assert torch.equal(a[keep.cuda()], b[keep.cuda()]), n
    # and before the block that it is in, nothing sees it
    if which in ("k", "v"):
        assert torch.equal(got["out"][0, 100:100 + 32], want["out"][0, 100:100 + 32])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("offset,dk,dv", [(0, 64, 64), (1, 64, 64), (3, 40, 24), (1, 33, 7)])
def test_strided_rows(offset, dk, dv, dtype):
    """q, k, v as slices of one projection's output, off any alignment; a gradient that is no dense tensor."""
    batch, L, heads, kv = 2, 70, 4, 2
    g = torch.Generator().manual_seed(offset)
    width = heads * dk + kv * (dk + dv) + 2 * offset
    big = torch.randn(batch, L, width, generator=g).to(dtype)
    at = [offset, offset + heads * dk, offset + heads * dk + kv * dk]
    cut = lambda x: (x[..., at[0]:at[1]].unflatten(-1, (heads, dk)), x[..., at[1]:at[2]].unflatten(-1, (kv, dk)),
                     x[..., at[2]:at[2] + kv * dv].unflatten(-1, (kv, dv)))
    t = _inputs(batch, L, heads, dk, dv, dtype, kv=kv)
    t.update(zip("qkv", cut(big)))
    leaf = big.cuda().requires_grad_()
    q, k, v = cut(leaf)
    out, final = _fn(q, k, v, t["log_decay"].cuda(), initial_states=t["initial_states"].cuda(), return_final_states=True)
    dout = torch.empty(heads, batch, dv, L, dtype=dtype, device="cuda").permute(1, 3, 0, 2)
    dout.copy_(t["dout"])
    grad, = torch.autograd.grad([out, final], leaf, [dout, t["dfinal"].cuda().transpose(2, 3).contiguous().transpose(2, 3)])
    ref, bound = linear_attention_oracle(t["q"], t["k"], t["v"], t["log_decay"], None, t["initial_states"], None, t["dout"], t["dfinal"])
    within("out", out, ref["out"], bound["out"])
    within("final", final, ref["final"], bound["final"])
    for n, x in zip(("dq", "dk", "dv"), cut(grad)):
        within(n, x, ref[n], bound[n])


def test_other_orders_of_axes():
    """Heads before positions, and a head's values that are not side by side."""
    t = _inputs(2, 40, 3, 16, 24, torch.bfloat16)
    want = _run(t)
    t = {k: (v.transpose(1, 2).contiguous().transpose(1, 2) if k in ("q", "v") else v.transpose(2, 3).contiguous().transpose(2, 3) if k == "k" else v)
         for k, v in t.items()}
    got = _run(t)
    for n in want:
        assert torch.equal(got[n], want[n])


@pytest.mark.parametrize("kinds", [(torch.bfloat16, torch.float32, torch.float16), (torch.float32, torch.bfloat16, torch.float32)])
def test_other_types_are_taken_in_that_of_q(kinds):
    t = _inputs(1, 50, 2, 16, 16, torch.float32, seed=2)
    leaves = [t[n].to(d).cuda().requires_grad_() for n, d in zip("qkv", kinds)]
    out = _fn(*leaves, t["log_decay"].double().float().cuda())
    same = [x.detach().to(kinds[0]).requires_grad_() for x in leaves]
    want = _fn(*same, t["log_decay"].cuda())
    assert out.dtype == kinds[0] and torch.equal(out, want)
    dout = t["dout"].to(kinds[0]).cuda()
    for a, b, leaf in zip(torch.autograd.grad(out, leaves, dout), torch.autograd.grad(want, same, dout), leaves):
        assert a.dtype == leaf.dtype and torch.equal(a, b.to(a.dtype))
    half = _fn(*same, t["log_decay"].bfloat16().cuda())
    assert torch.equal(half, _fn(*same, t["log_decay"].bfloat16().float().cuda()))


@pytest.mark.parametrize("shape", [(0, 5, 2), (2, 0, 2), (2, 5, 0)])
def test_nothing_to_do(shape):
    batch, L, heads = shape
    q = torch.zeros(*shape, 8, device="cuda", requires_grad=True)
    v = torch.zeros(batch, L, heads, 4, device="cuda", requires_grad=True)
    init = torch.randn(batch, heads, 8, 4, device="cuda", requires_grad=True)
    out, final = _fn(q, q, v, torch.zeros(heads, device="cuda"), initial_states=init, return_final_states=True)
    assert out.shape == (batch, L, heads, 4) and torch.equal(final, init)
    g = torch.randn_like(final)
    dq, dinit = torch.autograd.grad([out, final], [q, init], [torch.zeros_like(out), g])
    assert dq.shape == q.shape and torch.equal(dinit, g)
    out = _fn(q, q, v, torch.zeros(heads, device="cuda"), return_final_states=True)[1]
    assert torch.count_nonzero(out) == 0


def test_only_what_is_asked_for():
    """Gradients of the final states alone, of some of the tensors, no states at all."""
    t = _inputs(1, 90, 2, 32, 32, torch.float32, seed=6)
    ref, bound = linear_attention_oracle(t["q"], t["k"], t["v"], t["log_decay"], None, t["initial_states"], None, None, t["dfinal"])
    d = {k: v.cuda() for k, v in t.items()}
    for n in NAMES:
        d[n].requires_grad_()
    out, final = _fn(*(d[n] for n in ("q", "k", "v", "log_decay")), initial_states=d["initial_states"], return_final_states=True)
    for n, g in zip(GRADS, torch.autograd.grad(final, [d[n] for n in NAMES], d["dfinal"])):
        within(n, g, ref[n], bound[n])
    q, k, v = (d[n].detach() for n in "qkv")
    k.requires_grad_()
    out = _fn(q, k, v, d["log_decay"])
    assert isinstance(out, torch.Tensor)
    ref, bound = linear_attention_oracle(t["q"], t["k"], t["v"], t["log_decay"], dout=t["dout"])
    within("out", out, ref["out"], bound["out"])
    within("dk", torch.autograd.grad(out, k, d["dout"])[0], ref["dk"], bound["dk"])


def test_gradients_against_differences():
    t = _inputs(1, 37, 2, 8, 8, torch.float32, seed=8)
    got = _run(t)
    g = torch.Generator().manual_seed(1)
    d = {k: v.cuda() for k, v in t.items()}

    def value(**moved):
        a = {**d, **moved}
        out, final = _fn(a["q"], a["k"], a["v"], a["log_decay"], initial_states=a["initial_states"], return_final_states=True)
        return float((out.double() * d["dout"]).sum() + (final.double() * d["dfinal"]).sum())

    # the value is linear in each tensor alone: a difference over a step of 1 is off by rounding only, about 1e-6 of the terms
    for name, grad in zip(NAMES, GRADS):
        move = torch.randn(d[name].shape, generator=g).cuda()
        there = value(**{name: d[name] + move}) - value(**{name: d[name] - move})
        here = 2 * float((got[grad].double() * move).sum())
        size = 2 * float((got[grad].double() * move).abs().sum())
        assert abs(there - here) < 1e-4 * size, name


@pytest.mark.parametrize("batch,L,heads,kv,dk,dv,dtype", [
    (2, 700, 4, 4, 64, 64, torch.bfloat16), (1, 2000, 6, 2, 80, 40, torch.float16), (3, 100, 3, 1, 33, 20, torch.float32)])
def test_results_repeat_bit_for_bit(batch, L, heads, kv, dk, dv, dtype):
    t = _inputs(batch, L, heads, dk, dv, dtype, kv=kv)
    first = _run(t)
    for _ in range(3):
        again = _run(t)
        assert all(torch.equal(first[n], again[n]) for n in first)


def test_a_state_hands_a_sequence_on():
    """A sequence in two calls, the state of the first handed to the second, with its gradient."""
    t = _inputs(1, 300, 2, 64, 64, torch.float32, seed=11)
    d = {k: v.cuda() for k, v in t.items()}
    for n in NAMES:
        d[n].requires_grad_()
    cut = 123
    one, state = _fn(d["q"][:, :cut], d["k"][:, :cut], d["v"][:, :cut], d["log_decay"], initial_states=d["initial_states"],
                     return_final_states=True)
    two, final = _fn(d["q"][:, cut:], d["k"][:, cut:], d["v"][:, cut:], d["log_decay"], initial_states=state, return_final_states=True)
    out = torch.cat([one, two], 1)
    ref, bound = linear_attention_oracle(t["q"], t["k"], t["v"], t["log_decay"], None, t["initial_states"], None, t["dout"], t["dfinal"])
    within("out", out, ref["out"], 2 * bound["out"])
    within("final", final, ref["final"], 2 * bound["final"])
    for n, g in zip(GRADS, torch.autograd.grad([out, final], [d[n] for n in NAMES], [d["dout"], d["dfinal"]])):
        within(n, g, ref[n], 2 * bound[n])


def _captured(fn):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            fn()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fn()
    return graph, out


@pytest.mark.parametrize("packed", [False, True])
def test_captured_pass_replays(packed):
    t = {k: v.cuda() for k, v in _inputs(1, 2500, 2, 32, 32, torch.bfloat16, seqs=3 if packed else 1).items()}
    cu = torch.tensor([0, 100, 1900, 2400], dtype=torch.int32, device="cuda") if packed else None
    call = lambda: _fn(t["q"], t["k"], t["v"], t["log_decay"], initial_states=t["initial_states"], cu_seqlens=cu, return_final_states=True)
    with torch.no_grad():
        graph, (out, final) = _captured(call)
        for seed in range(4):
            t["q"].copy_(torch.randn(t["q"].shape, generator=torch.Generator().manual_seed(seed)))
            if packed:
                cu.copy_(torch.tensor([seed, 100 * seed + 7, 1900 - seed, 2500 - seed]))
            graph.replay()
            want = call()
            torch.cuda.synchronize()
            assert torch.equal(out, want[0]) and torch.equal(final, want[1])


def test_two_graphs_at_once():
    """Two captured passes replayed on two streams together: each has a workspace of its own."""
    pairs = [{k: v.cuda() for k, v in _inputs(1, 3000, 1, 64, 64, torch.bfloat16, seed=s).items()} for s in (1, 2)]
    call = lambda t: _fn(t["q"], t["k"], t["v"], t["log_decay"])
    want = [call(t) for t in pairs]
    graphs = [_captured(lambda t=t: call(t)) for t in pairs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, (graph, _) in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for (_, out), w in zip(graphs, want):
        assert torch.equal(out, w)


def test_two_streams_at_once():
    calls = [{k: v.cuda() for k, v in _inputs(1, 2500, 2, 32, 32, torch.float32, seed=s).items()} for s in range(2)]
    call = lambda t: _fn(t["q"], t["k"], t["v"], t["log_decay"])
    want = [call(t) for t in calls]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for n, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[n].append(call(calls[n]))
    torch.cuda.synchronize()
    for n in range(2):
        assert all(torch.equal(g, want[n]) for g in got[n])


def test_under_autocast():
    t = {k: v.cuda() for k, v in _inputs(1, 60, 2, 16, 16, torch.bfloat16).items()}
    want = _fn(t["q"], t["k"], t["v"], t["log_decay"])
    with torch.autocast("cuda", dtype=torch.float16):
        assert torch.equal(_fn(t["q"], t["k"], t["v"], t["log_decay"]), want)
