"""gated_linear_state_update beside its plain use: it writes the state in place and has no gradients, and torch has to see
both - the state's version, forward-mode gradients, functorch's transforms, jit traces, and backward passes that reach it."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

pytestmark = pytest.mark.gpu

NAMES = ["state", "x", "gate_a", "gate_x", "decay"]


@pytest.fixture(params=[True, False], ids=["ext", "ctypes"])
def host(request, monkeypatch):
    from mamba_amd import _lib
    if not request.param:
        monkeypatch.setattr(_lib, "_torch_ext", None)


def _step(*args, **kw):
    from mamba_amd.ops.gated_linear_scan import gated_linear_state_update
    return gated_linear_state_update(*args, **kw)


def _operands(seed=0, rows=3):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)
    return dict(state=r(rows, 72), x=r(3, 72), gate_a=r(3, 72), gate_x=r(3, 72), decay=r(72))


def _clone(t):
    return {n: v.clone() for n, v in t.items()}


def test_the_state_has_a_new_version(host):
    t = _operands(rows=6)
    state = t.pop("state")
    for index_dtype in (None, torch.int32, torch.int64):
        rows = None if index_dtype is None else torch.tensor([4, -1, 0], dtype=index_dtype, device="cuda")
        before, view = state._version, state[:3]
        _step(state, **t, state_batch_indices=rows)
        assert state._version > before and view._version == state._version
        before = state._version
        _step(state[2:5], **t)  # rows of a pool: the pool's version too
        assert state._version > before


def test_a_state_that_a_graph_has_saved(host):
    t = _operands()
    leaf = torch.ones(3, 72, device="cuda", requires_grad=True)
    loss = (leaf * t["state"]).sum()  # its gradient is the state
    _step(**t)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_a_state_of_inference_mode(host):
    t = _operands()
    want = _step(**_clone(t))
    with torch.inference_mode():
        state = t["state"].clone()
        assert torch.equal(_step(state, **{n: t[n] for n in NAMES[1:]}), want)
        state = t["state"].clone()
    with torch.no_grad():
        assert torch.equal(_step(state, **{n: t[n] for n in NAMES[1:]}), want)
    with torch.inference_mode():
        state = t["state"].clone()
        rest = {n: t[n].clone() for n in NAMES[1:4]}
    t["decay"].requires_grad_()  # a call that autograd records
    assert torch.equal(_step(state, **rest, decay=t["decay"]), want)


@pytest.mark.parametrize("which", NAMES)
@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_is_refused(host, which, grad):
    t = _operands()
    with torch.set_grad_enabled(grad), fwAD.dual_level():
        t[which] = fwAD.make_dual(t[which], torch.ones_like(t[which]))
        with pytest.raises(NotImplementedError):
            _step(**t)


def test_functorch_transforms_are_refused(host):
    t = _operands()
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda x: _step(**{**t, "x": x}), (t["x"],), (torch.ones_like(t["x"]),))
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda v: _step(**t) + v)(torch.zeros(2, 1, device="cuda"))


@pytest.mark.parametrize("index_dtype", [None, torch.int32, torch.int64])
def test_traced_call_replays(host, index_dtype):
    rows = () if index_dtype is None else (torch.tensor([4, -1, 0], dtype=index_dtype, device="cuda"),)
    call = lambda state, x, ga, gx, decay, *i: _step(state, x, ga, gx, decay, state_batch_indices=i[0] if i else None)
    with torch.no_grad():
        traced = torch.jit.trace(call, (*_operands(0, 6).values(), *rows), check_trace=False)
        for seed in (1, 2, 3):
            a, b = _operands(seed, 6), _operands(seed, 6)
            assert torch.equal(traced(*a.values(), *rows), call(*b.values(), *rows))
            assert torch.equal(a["state"], b["state"])


@pytest.mark.parametrize("which", NAMES[1:])
@pytest.mark.parametrize("pooled", [False, True])
def test_a_gradient_through_a_step_is_refused_not_dropped(host, which, pooled):
    """The call itself gives what it gives without gradients; a backward pass that reaches it raises, whatever else lies on
    the way to the leaf."""
    kw = dict(state_batch_indices=torch.tensor([4, -1, 0], dtype=torch.int32, device="cuda")) if pooled else {}
    t = _operands(rows=6)
    plain = _clone(t)
    want = _step(**plain, **kw)
    t[which].requires_grad_()
    before = t["state"]._version
    out = _step(**t, **kw)
    assert torch.equal(out, want) and torch.equal(t["state"], plain["state"])
    assert out.requires_grad and not t["state"].requires_grad and t["state"]._version > before
    loss = out.sum() + t[which].sum()
    with pytest.raises(RuntimeError, match="no gradients"):
        torch.autograd.grad(loss, t[which], retain_graph=True)
    with pytest.raises(RuntimeError, match="no gradients"):
        loss.backward()
    with torch.no_grad():
        again = _step(**{**t, "state": _operands(rows=6)["state"]}, **kw)
    assert torch.equal(again, want) and not again.requires_grad


def test_a_state_that_wants_gradients_is_refused(host):
    from mamba_amd.ops.gated_linear_scan import gated_linear_scan_fn
    t = _operands()
    for state in (t["state"].clone().requires_grad_(), t["state"] * torch.ones(1, device="cuda", requires_grad=True)):
        kept = state.detach().clone()
        with pytest.raises(RuntimeError, match="state is updated in place"):
            _step(**{**t, "state": state})
        assert torch.equal(state, kept)
    x = t["x"][:, None].clone().requires_grad_()
    _, final = gated_linear_scan_fn(x, t["gate_a"][:, None], t["gate_x"][:, None], t["decay"], return_final_states=True)
    a, b = final.detach(), final.detach().clone()
    with torch.no_grad():
        want = _step(**{**t, "state": final.clone()})
        assert torch.equal(_step(**{**t, "state": final}), want)
    assert torch.equal(a, final)  # updated in place
    assert torch.equal(_step(**{**t, "state": b}), want)


def test_steps_in_a_captured_graph_after_recorded_ones(host):
    """A step whose decay is a parameter, captured without gradients and replayed, with recorded eager steps in between."""
    t = _operands()
    t["decay"].requires_grad_()
    live, static = t["state"].clone(), [t[n].clone() for n in NAMES[1:4]]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.no_grad():
        with torch.cuda.stream(side):
            _step(torch.zeros_like(live), *static, t["decay"])
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = _step(live, *static, t["decay"])
    eager = t["state"].clone()
    for seed in range(4):
        new = _operands(seed + 5)
        for s, n in zip(static, NAMES[1:4]):
            s.copy_(new[n])
        graph.replay()
        want = _step(eager, *[new[n] for n in NAMES[1:4]], t["decay"])
        assert want.requires_grad and torch.equal(out, want) and torch.equal(live, eager)
