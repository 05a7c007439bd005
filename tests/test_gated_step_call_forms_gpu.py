"""gated_linear_state_update beside its plain use: it writes the state in place, and torch has to see that."""
import pytest
import torch

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
