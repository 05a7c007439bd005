"""Forward-mode gradients through the step of the gated recurrence are refused before it changes its state."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

from mamba_amd import _lib
from mamba_amd.ops.gated_linear_scan import gated_linear_state_update


def _refused(device, name, grad):
    g = torch.Generator().manual_seed(0)
    args = {n: torch.randn(*s, generator=g).to(device) for n, s in
            (("state", (3, 8)), ("x", (2, 8)), ("gate_a", (2, 8)), ("gate_x", (2, 8)), ("decay", (8,)))}
    before = {n: t.clone() for n, t in args.items()}
    with torch.set_grad_enabled(grad), fwAD.dual_level():
        dual = fwAD.make_dual(args[name], torch.ones_like(args[name]))
        with pytest.raises(NotImplementedError):
            gated_linear_state_update(**{**args, name: dual})
    return args, before


NAMES = ["state", "x", "gate_a", "gate_x", "decay"]


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("name", NAMES)
def test_a_tangent_is_refused_before_anything_else(name, grad):
    _refused("cpu", name, grad)


@pytest.mark.gpu
@pytest.mark.parametrize("host", ["ext", "ctypes"])
@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("name", NAMES)
def test_a_refused_call_changes_nothing(name, grad, host, monkeypatch):
    if host == "ctypes":
        monkeypatch.setattr(_lib, "_torch_ext", None)
    args, before = _refused("cuda", name, grad)
    torch.cuda.synchronize()
    for n, t in args.items():
        assert torch.equal(t, before[n]), n
