"""Forward-mode gradients through linear attention, its step and the attention over a paged cache are refused, not dropped, and a
refused call changes neither states nor caches."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

from mamba_amd import _lib
from mamba_amd.ops.linear_attention import linear_attention_fn, linear_attention_state_update
from mamba_amd.ops.paged_attention import paged_attention_update


def _arguments(device="cpu"):
    g = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g).to(device)
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device=device)
    linear = dict(q=r(1, 6, 4, 8), k=r(1, 6, 2, 8), v=r(1, 6, 2, 5), log_decay=-r(4).abs(), initial_states=r(1, 4, 8, 5))
    step = dict(state=r(3, 4, 8, 5), q=r(2, 4, 8), k=r(2, 2, 8), v=r(2, 2, 5), log_decay=-r(4).abs())
    paged = dict(q=r(2, 4, 8), k=r(2, 2, 8), v=r(2, 2, 5), k_cache=r(7, 4, 2, 8), v_cache=r(7, 4, 2, 5),
                 block_table=ints([0, 1], [2, 3]), cache_seqlens=ints(3, 5))
    return {"linear": (linear_attention_fn, linear), "step": (linear_attention_state_update, step), "paged": (paged_attention_update, paged)}


CALLS = [(op, name) for op, (_, args) in _arguments().items() for name, t in args.items() if t.is_floating_point()]


def _refused(device, op, name, grad):
    fn, args = _arguments(device)[op]
    before = {n: t.clone() for n, t in args.items()}
    with torch.set_grad_enabled(grad), fwAD.dual_level():
        dual = fwAD.make_dual(args[name], torch.ones_like(args[name]))
        with pytest.raises(NotImplementedError):
            fn(**{**args, name: dual})
    return args, before


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("op,name", CALLS)
def test_a_tangent_is_refused_before_anything_else(op, name, grad):
    _refused("cpu", op, name, grad)


@pytest.mark.parametrize("op", ["linear", "step", "paged"])
def test_a_level_without_tangents_refuses_nothing(op):
    fn, args = _arguments()[op]
    with fwAD.dual_level(), pytest.raises(RuntimeError, match="no CPU fallback"):
        fn(**args)


@pytest.mark.gpu
@pytest.mark.parametrize("host", ["ext", "ctypes"])
@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("op,name", CALLS)
def test_a_refused_call_changes_nothing(op, name, grad, host, monkeypatch):
    if host == "ctypes":
        monkeypatch.setattr(_lib, "_torch_ext", None)
    args, before = _refused("cuda", op, name, grad)
    torch.cuda.synchronize()
    for n, t in args.items():
        assert torch.equal(t, before[n]), n


@pytest.mark.gpu
@pytest.mark.parametrize("op,name", [("step", "q"), ("paged", "k")])
def test_a_transform_that_is_refused_changes_nothing(op, name):
    fn, args = _arguments("cuda")[op]
    before = {n: t.clone() for n, t in args.items()}
    call = lambda t: fn(**{**args, name: t})
    with pytest.raises(RuntimeError):
        torch.func.jvp(call, (args[name],), (torch.ones_like(args[name]),))
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda s: call(args[name]) + s)(torch.zeros(2, 1, device="cuda"))
    torch.cuda.synchronize()
    for n, t in args.items():
        assert torch.equal(t, before[n]), n
