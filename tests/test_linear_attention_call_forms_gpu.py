"""linear_attention_fn beside its plain use: forward-mode gradients, functorch's transforms, jit traces, in-place writes, the
ctypes host side, rows beyond 32-bit offsets, sequence bounds that are none, a graph of the backward pass alone, second
derivatives."""
import functools

import pytest
import torch
import torch.autograd.forward_ad as fwAD

from oracle.linear_attention import linear_attention_oracle, within

pytestmark = pytest.mark.gpu


@functools.lru_cache(maxsize=None)
def _fixed(which, *shape):
    return 0.2 * torch.randn(*shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(which))


def _operands(seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return tuple(torch.randn(2, 90, 3, 48, device="cuda", generator=g) for _ in range(2))


def _fn(*args, **kw):
    from mamba_amd.ops.linear_attention import linear_attention_fn
    return linear_attention_fn(*args, **kw)


DECAY = lambda: -_fixed(1, 3).abs()


def _plain(x, z):
    return _fn(x, z, _fixed(0, 2, 90, 3, 48), DECAY())


def _states(x, z):
    return _fn(x, _fixed(2, 2, 90, 1, 48), z[:, :, :1], DECAY(), initial_states=_fixed(3, 2, 3, 48, 48), return_final_states=True)[0]


each_call = pytest.mark.parametrize("call", [_plain, _states], ids=["plain", "states"])


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
    assert torch.equal(first, third) and torch.equal(second, 2 * first)


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


@pytest.mark.parametrize("ext", [True, False], ids=["ext", "ctypes"])
def test_a_decay_that_wants_a_gradient_is_refused(ext, monkeypatch):
    from mamba_amd import _lib
    if not ext:
        monkeypatch.setattr(_lib, "_torch_ext", None)
    x, z = _operands()
    decay = DECAY().requires_grad_()
    with pytest.raises(RuntimeError, match="takes no gradients"):
        _fn(x, z, z, decay)
    with torch.no_grad():
        assert torch.equal(_fn(x, z, z, decay), _fn(x, z, z, decay.detach()))


def test_rows_beyond_32_bit_offsets():
    big = torch.zeros(2 ** 31 + 5000, dtype=torch.bfloat16, device="cuda")
    g = torch.Generator().manual_seed(0)
    q, k, v, do = (torch.randn(2, 3, 2, 24, generator=g).bfloat16() for _ in range(4))
    decay = torch.tensor([-0.1, 0.0])

    def check(name, far, n):
        far.copy_(q[:n])
        leaves = [far.requires_grad_(), *(t[:n].cuda().requires_grad_() for t in (k, v))]
        ref, bound = linear_attention_oracle(q[:n], k[:n], v[:n], decay, dout=do[:n])
        for which in range(3):  # the far rows as q, as k and as v
            order = [leaves[(i + which) % 3] for i in range(3)]
            inputs = [(q, k, v)[(i + which) % 3][:n] for i in range(3)]
            out = _fn(*order, decay.cuda())
            ref, bound = linear_attention_oracle(*inputs, decay, dout=do[:n])
            within(name, out, ref["out"], bound["out"])
            for key, x in zip(("dq", "dk", "dv"), torch.autograd.grad(out, order, do[:n].cuda())):
                within(f"{name} {key}", x, ref[key], bound[key])

    check("batch", big.as_strided((2, 3, 2, 24), (2 ** 31 + 100, 60, 24, 1)), 2)
    check("position", big.as_strided((1, 3, 2, 24), (0, 2 ** 30 + 200, 24, 1)), 1)
    check("head", big.as_strided((1, 3, 2, 24), (0, 24, 2 ** 31 + 200, 1)), 1)


@pytest.mark.parametrize("total,room", [(200, 1), (3000, 10)])
@pytest.mark.parametrize("cu,taken", [([-7, 10, 9999], [0, 10, "end"]), ([0, 5000, 6000], [0, "end", "end"]), ([-9, -5, 300], [0, 0, 300])])
def test_bounds_outside_of_the_row_are_taken_to_its_ends(total, room, cu, taken):
    g = torch.Generator(device="cuda").manual_seed(0)
    q, k, v, dout = (torch.randn(1, total, 1, 16, device="cuda", generator=g) for _ in range(4))
    init = torch.randn(2, 1, 16, 16, device="cuda", generator=g)
    taken = [min(total, total if t == "end" else t) for t in taken]

    def run(bounds):
        leaves = [t.clone().requires_grad_() for t in (q, k, v, init)]
        out, final = _fn(*leaves[:3], _fixed(7, 1), initial_states=leaves[3],
                         cu_seqlens=torch.tensor(bounds, dtype=torch.int32, device="cuda"), return_final_states=True)
        return [out, final, *torch.autograd.grad([out, final], leaves, [dout, torch.ones_like(final)])]

    assert all(torch.equal(a, b) for a, b in zip(run(cu), run(taken)))


@pytest.mark.parametrize("total", [90, 4000])
def test_bounds_in_disorder_end(total):
    """No use, but no harm: the call comes back, and calls after it are as ever."""
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(1, total, 2, 16, device="cuda", generator=g)
    decay = -_fixed(1, 2).abs()
    want = _fn(x, x, x, decay)
    for cu in ([50, 3, total, 20], [total, 0], [7, 7, 7, 1], [0, total, 0, total, 0, total, 0, total]):
        _fn(x, x, x, decay, cu_seqlens=torch.tensor(cu, dtype=torch.int32, device="cuda"), return_final_states=True)
    torch.cuda.synchronize()
    assert torch.equal(_fn(x, x, x, decay), want)


def test_bounds_of_64_bits_turn_into_no_others():
    x, z = (t[:1] for t in _operands())
    outs = [_fn(x, z, z, DECAY(), cu_seqlens=torch.tensor(c, dtype=d, device="cuda"))
            for c, d in (([0, 7, 90], torch.int32), ([-(2 ** 32), 7, 2 ** 32 + 5], torch.int64))]
    assert torch.equal(*outs)


def test_a_graph_of_the_backward_pass_alone():
    """Through the C entry points: a backward pass captured by itself gives every replay's own gradients, shared heads' too."""
    from mamba_amd import _lib
    from mamba_amd.ops import linear_attention as ops
    lib = _lib.load()
    q, z = _operands()
    k = v = z[:, :, :1].contiguous()
    decay, dout = DECAY(), torch.ones_like(q)
    p = ops._params(q, k, v, decay, None, None, 0.3)
    grads = [torch.empty_like(t) for t in (q, k, v)]
    ws = torch.empty(lib.linear_attn_bwd_ws_bytes(p), dtype=torch.uint8, device="cuda")
    p.ws, p.dout = ws.data_ptr(), dout.data_ptr()
    p.dq, p.dk, p.dv = (g.data_ptr() for g in grads)
    ops._strides(p, dout=dout, dq=grads[0], dk=grads[1], dv=grads[2])
    launch = lambda: _lib.check(lib.linear_attn_bwd(p, _lib.current_stream(q.device)), "bwd")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        launch()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        launch()
    for seed in range(4):
        dout.copy_(torch.randn(q.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)))
        for g in grads:
            g.fill_(float("nan"))
        graph.replay()
        leaves = [t.clone().requires_grad_() for t in (q, k, v)]
        want = torch.autograd.grad(_fn(*leaves, decay, scale=0.3), leaves, dout)
        assert all(torch.equal(a, b) for a, b in zip(grads, want))
