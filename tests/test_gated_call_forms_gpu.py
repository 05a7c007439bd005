"""gated_linear_scan_fn, gated_linear_state_update and block_norm_fn beside their plain use: forward-mode gradients,
functorch's transforms, jit traces, in-place writes, the ctypes host side, rows beyond 32-bit offsets, sequence bounds that are
none, a graph of the backward pass alone, two graphs at once, and second derivatives."""
import functools

import pytest
import torch
import torch.autograd.forward_ad as fwAD

from oracle.gated_linear import gated_linear_oracle, within

pytestmark = pytest.mark.gpu


@functools.lru_cache(maxsize=None)
def _fixed(which, *shape):
    return 0.2 * torch.randn(*shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(which))


def _operands(seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return tuple(torch.randn(2, 90, 48, device="cuda", generator=g) for _ in range(2))


def _scan(x, z):
    from mamba_amd.ops.gated_linear_scan import gated_linear_scan_fn
    return gated_linear_scan_fn(x, z, _fixed(0, 2, 90, 48), _fixed(1, 48))


def _scan_states(x, z):
    from mamba_amd.ops.gated_linear_scan import gated_linear_scan_fn
    return gated_linear_scan_fn(x, z, _fixed(0, 2, 90, 48), _fixed(1, 48), initial_states=_fixed(2, 2, 48), return_final_states=True)[0]


def _norm(x, z):
    from mamba_amd.ops.block_norm import block_norm_fn
    return block_norm_fn(x, _fixed(3, 2, 90, 48), _fixed(4, 48), _fixed(5, 48), z=z, scale=_fixed(6, 48))[0]


CALLS = {f.__name__[1:]: f for f in (_scan, _scan_states, _norm)}
each_call = pytest.mark.parametrize("call", list(CALLS.values()), ids=list(CALLS))


@each_call
@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_is_refused(call, grad):
    x, z = _operands()
    with torch.set_grad_enabled(grad), fwAD.dual_level():
        with pytest.raises(NotImplementedError):
            call(fwAD.make_dual(x, torch.ones_like(x)), z)


@each_call
def test_functorch_transforms_are_refused(call):
    x, z = _operands()
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda t: call(t, z), (x,), (torch.ones_like(x),))
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda t: call(x, z) + t)(torch.zeros(2, 1, device="cuda"))


@each_call
def test_traced_call_replays(call):
    x, z = _operands()
    with torch.no_grad():
        call(x, z)
        traced = torch.jit.trace(call, (x, z), check_trace=False)
        for seed in (1, 2, 3):
            x, z = _operands(seed)
            assert torch.equal(traced(x, z), call(x, z))


@each_call
@pytest.mark.parametrize("ext", [True, False], ids=["ext", "ctypes"])
def test_output_takes_in_place_writes(call, ext, monkeypatch):
    from mamba_amd import _lib
    if not ext:
        monkeypatch.setattr(_lib, "_torch_ext", None)
    x, z = _operands()
    x.requires_grad_()
    want, = torch.autograd.grad(call(x, z), x, torch.ones_like(x))
    out = call(x, z)
    out += 1.0
    got, = torch.autograd.grad(out, x, torch.ones_like(x))
    assert torch.equal(got, want)


@each_call
def test_backward_twice(call):
    x, z = _operands()
    x.requires_grad_()
    out = call(x, z)
    first, = torch.autograd.grad(out, x, torch.ones_like(x), retain_graph=True)
    second, = torch.autograd.grad(out, x, 2 * torch.ones_like(x), retain_graph=True)
    third, = torch.autograd.grad(out, x, torch.ones_like(x))
    assert torch.equal(first, third)
    torch.testing.assert_close(second, 2 * first, rtol=1e-5, atol=1e-6)


@each_call
def test_second_derivatives_are_refused_not_dropped(call):
    x, z = _operands()
    x.requires_grad_()
    out = call(x, z)
    g, = torch.autograd.grad(out, x, torch.ones_like(x), create_graph=True)
    with pytest.raises(RuntimeError):
        (g.square().sum() + x.sum()).backward()


@each_call
def test_the_ctypes_host_side_gives_the_same(call, monkeypatch):
    from mamba_amd import _lib
    x, z = (t.requires_grad_() for t in _operands())
    want = call(x, z)
    grads = torch.autograd.grad(want, (x, z), torch.ones_like(x))
    monkeypatch.setattr(_lib, "_torch_ext", None)
    got = call(x, z)
    assert torch.equal(got, want)
    for a, b in zip(torch.autograd.grad(got, (x, z), torch.ones_like(x)), grads):
        assert torch.equal(a, b)


def test_the_ctypes_step_gives_the_same(monkeypatch):
    from mamba_amd import _lib
    from mamba_amd.ops.gated_linear_scan import gated_linear_state_update
    args = [t[:, 0] for t in _operands()] + [_fixed(0, 2, 48), _fixed(1, 48)]
    a, b = _fixed(2, 5, 48).clone(), _fixed(2, 5, 48).clone()
    rows = torch.tensor([4, -1], dtype=torch.int32, device="cuda")
    want = gated_linear_state_update(a, *args, state_batch_indices=rows)
    monkeypatch.setattr(_lib, "_torch_ext", None)
    assert torch.equal(gated_linear_state_update(b, *args, state_batch_indices=rows), want) and torch.equal(a, b)


def test_rows_beyond_32_bit_offsets():
    """Batch rows and positions that lie more than 2^31 elements apart, in the scan, the step and the norm."""
    from mamba_amd.ops.block_norm import block_norm_fn
    from mamba_amd.ops.gated_linear_scan import gated_linear_scan_fn, gated_linear_state_update
    big = torch.zeros(2 ** 31 + 5000, dtype=torch.bfloat16, device="cuda")
    g = torch.Generator().manual_seed(0)
    x, ga, gx = (torch.randn(2, 3, 70, generator=g).bfloat16() for _ in range(3))
    far = big.as_strided((2, 3, 70), (2 ** 31 + 100, 80, 1))
    far.copy_(x)
    decay = torch.zeros(70)
    ref, bound = gated_linear_oracle(x, ga, gx, decay)
    within("batch", gated_linear_scan_fn(far, ga.cuda(), gx.cuda(), decay.cuda()), ref["out"], bound["out"])
    far = big.as_strided((1, 3, 70), (0, 2 ** 30 + 200, 1))
    far.copy_(x[:1])
    ref, bound = gated_linear_oracle(x[:1], ga[:1], gx[:1], decay)
    within("position", gated_linear_scan_fn(far, ga[:1].cuda(), gx[:1].cuda(), decay.cuda()), ref["out"], bound["out"])
    state = big.as_strided((2, 70), (2 ** 31 + 300, 1))
    state.zero_()
    ref, bound = gated_linear_oracle(x[:, :1], ga[:, :1], gx[:, :1], decay)
    out = gated_linear_state_update(state, *(t[:, 0].cuda() for t in (x, ga, gx)), decay.cuda())
    within("step", out, ref["out"][:, 0], bound["out"][:, 0])
    within("state", state, ref["final"], bound["final"])
    rows = big.as_strided((3, 70), (2 ** 30 + 400, 1))
    rows.copy_(x[0])
    ones = torch.ones(70, device="cuda")
    near = block_norm_fn(x[0].cuda(), gx[0].cuda(), ones, ones, z=ga[0].cuda())
    for a, b in zip(block_norm_fn(rows, gx[0].cuda(), ones, ones, z=ga[0].cuda()), near):
        assert torch.equal(a, b)


@pytest.mark.parametrize("cu,taken", [([-7, 10, 400], [0, 10, 200]), ([0, 500, 600], [0, 200, 200]), ([-9, -5, 300], [0, 0, 200])])
def test_bounds_outside_of_the_row_are_taken_to_its_ends(cu, taken):
    from mamba_amd.ops.gated_linear_scan import gated_linear_scan_fn
    g = torch.Generator(device="cuda").manual_seed(0)
    x, ga, gx, dout = (torch.randn(1, 200, 33, device="cuda", generator=g) for _ in range(4))
    init = torch.randn(2, 33, device="cuda", generator=g)

    def run(bounds):
        leaves = [t.clone().requires_grad_() for t in (x, ga, gx, init)]
        out, final = gated_linear_scan_fn(*leaves[:3], _fixed(7, 33), initial_states=leaves[3],
                                          cu_seqlens=torch.tensor(bounds, dtype=torch.int32, device="cuda"), return_final_states=True)
        return [out, final, *torch.autograd.grad([out, final], leaves, [dout, torch.ones_like(final)])]

    assert all(torch.equal(a, b) for a, b in zip(run(cu), run(taken)))


def test_bounds_in_disorder_end():
    """No use, but no harm: the call comes back, and rows after it are as ever."""
    from mamba_amd.ops.gated_linear_scan import gated_linear_scan_fn
    x, z = (t[:1] for t in _operands())
    want = _scan(*_operands())
    for cu in ([50, 3, 90, 20], [90, 0], [7, 7, 7, 1]):
        gated_linear_scan_fn(x, z, _fixed(0, 2, 90, 48)[:1], _fixed(1, 48), cu_seqlens=torch.tensor(cu, dtype=torch.int32, device="cuda"),
                             return_final_states=True)
    torch.cuda.synchronize()
    assert torch.equal(_scan(*_operands()), want)


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


def test_a_graph_of_the_backward_pass_alone():
    """Through the C entry points: a backward pass captured by itself gives every replay's own gradients."""
    from mamba_amd import _lib
    from mamba_amd.ops import gated_linear_scan as ops
    lib = _lib.load()
    x, z = _operands()
    gx, decay = _fixed(0, 2, 90, 48), _fixed(1, 48)
    p = ops._params(x, z, gx, decay, None, None, 8.0)
    ckpt = torch.empty(lib.gated_scan_ckpt_bytes(p), dtype=torch.uint8, device="cuda")
    ws = torch.empty(lib.gated_scan_bwd_ws_bytes(p), dtype=torch.uint8, device="cuda")
    out, dout, ddecay = torch.empty_like(x), torch.ones_like(x), torch.empty_like(decay)
    grads = [torch.empty_like(x) for _ in range(3)]
    p.ckpt, p.ws, p.out, p.out_bs, p.out_ls = ckpt.data_ptr(), ws.data_ptr(), out.data_ptr(), x.stride(0), x.stride(1)
    p.dout, p.dout_bs, p.dout_ls = dout.data_ptr(), x.stride(0), x.stride(1)
    p.dx, p.dgate_a, p.dgate_x = (g.data_ptr() for g in grads)
    p.dx_bs = p.dgate_a_bs = p.dgate_x_bs = x.stride(0)
    p.dx_ls = p.dgate_a_ls = p.dgate_x_ls = x.stride(1)
    p.ddecay = ddecay.data_ptr()
    _lib.check(lib.gated_scan_fwd(p, _lib.current_stream(x.device)), "fwd")
    graph, _ = _captured(lambda: _lib.check(lib.gated_scan_bwd(p, _lib.current_stream(x.device)), "bwd"))
    for seed in range(4):
        dout.copy_(torch.randn(x.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)))
        graph.replay()
        leaf = x.clone().requires_grad_()
        want, = torch.autograd.grad(_scan(leaf, z), leaf, dout)
        assert torch.equal(grads[0], want)


def test_two_graphs_at_once():
    """Two captured scans replayed on two streams together: each has a workspace of its own."""
    pairs = [_operands(s) for s in (1, 2)]
    want = [_scan(*p) for p in pairs]
    graphs = [_captured(lambda p=p: _scan(*p)) for p in pairs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, (graph, _) in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for (_, out), w in zip(graphs, want):
        assert torch.equal(out, w)


@pytest.mark.parametrize("which", range(4))
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_in_packed_sequences_no_number_goes_as_far_as_in_rows_of_their_own(which, value):
    """A NaN or an infinity at one position: packed and alone the same results and gradients are no numbers, and the other
    sequences' are untouched."""
    from mamba_amd.ops.gated_linear_scan import gated_linear_scan_fn
    cu = [0, 40, 190, 191, 300]
    g = torch.Generator(device="cuda").manual_seed(0)
    tensors = [torch.randn(1, 300, 6, device="cuda", generator=g) for _ in range(4)]
    for at, channel in ((5, 0), (60, 1), (189, 2), (190, 3), (191, 4)):
        tensors[which][0, at, channel] = value

    def run(ts, bounds):
        leaves = [t.clone().requires_grad_() for t in ts[:3]]
        out, final = gated_linear_scan_fn(*leaves, _fixed(8, 6), return_final_states=True, cu_seqlens=bounds)
        return [out, final, *torch.autograd.grad([out, final], leaves, [ts[3], torch.ones_like(final)])]

    packed = run(tensors, torch.tensor(cu, dtype=torch.int32, device="cuda"))
    alone = [run([t[:, a:b] for t in tensors], None) for a, b in zip(cu, cu[1:])]
    for n, got in enumerate(packed):
        want = torch.cat([a[n] for a in alone], 0 if n == 1 else 1)
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isinf(), want.isinf())
        torch.testing.assert_close(got, want, rtol=2e-4, atol=2e-5, equal_nan=True)


def test_row_numbers_of_64_bits_turn_into_no_others():
    from mamba_amd.ops.gated_linear_scan import gated_linear_scan_fn, gated_linear_state_update
    args = [t[:, :3].reshape(6, 48) for t in _operands()] + [_fixed(0, 2, 90, 48)[:, :3].reshape(6, 48), _fixed(1, 48)]
    rows = [1, -1, 2 ** 32, 2 ** 32 + 2, 2 ** 31, -(2 ** 32) + 3]
    states = [_fixed(2, 5, 48).clone() for _ in range(2)]
    outs = [gated_linear_state_update(s, *args, state_batch_indices=torch.tensor(r, dtype=d, device="cuda"))
            for s, r, d in zip(states, ([1] + [-1] * 5, rows), (torch.int32, torch.int64))]
    assert torch.equal(*outs) and torch.equal(*states)
    x, z = (t[:1] for t in _operands())
    outs = [gated_linear_scan_fn(x, z, _fixed(0, 2, 90, 48)[:1], _fixed(1, 48), cu_seqlens=torch.tensor(c, dtype=d, device="cuda"))
            for c, d in (([0, 7, 90], torch.int32), ([-(2 ** 32), 7, 2 ** 32 + 5], torch.int64))]
    assert torch.equal(*outs)
    with pytest.raises(RuntimeError, match="must not overlap"):
        gated_linear_state_update(_fixed(2, 5, 48)[:1].expand(6, 48), *args)
