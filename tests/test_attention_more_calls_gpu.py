"""Calls of linear attention, its step and the attention over a paged cache beside those of the other tests: a whole training step in a
captured graph, batches larger than a dimension of a launch, a gradient for the caller's part of the operands only."""
import pytest
import torch

from oracle.linear_attention import linear_step_oracle, within

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kv", [4, 2])
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("host", ["ext", "ctypes"])
def test_a_captured_training_step_replays(packed, kv, host, monkeypatch):
    from mamba_amd import _lib
    from mamba_amd.ops.linear_attention import linear_attention_fn
    if host == "ctypes":
        monkeypatch.setattr(_lib, "_torch_ext", None)
    g = torch.Generator(device="cuda").manual_seed(0)
    r = lambda *s, dtype=torch.bfloat16: torch.randn(*s, device="cuda", generator=g).to(dtype)
    L, seqs = 1500, 3 if packed else 1
    leaves = [r(1, L, 4, 32), r(1, L, kv, 32), r(1, L, kv, 48), r(seqs, 4, 32, 48, dtype=torch.float32)]
    dout, dfinal, decay = r(1, L, 4, 48), r(seqs, 4, 32, 48, dtype=torch.float32), -torch.rand(4, device="cuda", generator=g)
    cu = torch.tensor([0, 40, 1200, 1490], dtype=torch.int32, device="cuda") if packed else None
    for t in leaves:
        t.requires_grad_()

    def step():
        out, final = linear_attention_fn(*leaves[:3], decay, initial_states=leaves[3], cu_seqlens=cu, return_final_states=True)
        return [out.detach(), final.detach(), *torch.autograd.grad([out, final], leaves, [dout, dfinal])]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for n in range(4):
        with torch.no_grad():
            for t in (*leaves, dout, dfinal):
                t.copy_(torch.randn(t.shape, device="cuda", generator=g))
        if packed:
            cu.copy_(torch.tensor([n, 40 + 300 * n, 1200, 1500 - n]))
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_a_step_of_more_than_65535_users():
    from mamba_amd.ops.linear_attention import linear_attention_state_update
    g = torch.Generator().manual_seed(0)
    batch, rows = 70_000, 70_100
    t = dict(state=torch.randn(rows, 1, 2, 3, generator=g), q=torch.randn(batch, 1, 2, generator=g), k=torch.randn(batch, 1, 2, generator=g),
             v=torch.randn(batch, 1, 3, generator=g), log_decay=torch.tensor([-0.5]))
    at = torch.randperm(rows, generator=g)[:batch].to(torch.int32)
    at[::7] = -1
    d = {n: x.cuda() for n, x in t.items()}
    out = linear_attention_state_update(*d.values(), state_batch_indices=at.cuda())
    used = at >= 0
    assert torch.count_nonzero(out[~used.cuda()]) == 0
    mine = at[used].long()
    ref, bound = linear_step_oracle(t["state"][mine], t["q"][used], t["k"][used], t["v"][used], t["log_decay"])
    within("out", out[used.cuda()], ref["out"], bound["out"])
    within("state", d["state"].cpu()[mine], ref["state"], bound["state"])
    rest = torch.ones(rows, dtype=torch.bool)
    rest[mine] = False
    assert torch.equal(d["state"].cpu()[rest], t["state"][rest])


@pytest.mark.parametrize("wanted", [(0,), (1,), (2,), (3,), (0, 2), (1, 3)])
def test_gradients_of_some_operands(wanted):
    from mamba_amd.ops.linear_attention import linear_attention_fn
    g = torch.Generator(device="cuda").manual_seed(0)
    operands = [torch.randn(*s, device="cuda", generator=g) for s in ((2, 70, 4, 16), (2, 70, 2, 16), (2, 70, 2, 24), (2, 4, 16, 24))]
    decay = torch.tensor([-0.5, -0.1, -0.01, 0.0], device="cuda")
    grads = []
    for some in (range(4), wanted):
        leaves = [t.clone().requires_grad_(n in some) for n, t in enumerate(operands)]
        out = linear_attention_fn(*leaves[:3], decay, initial_states=leaves[3])
        grads.append(torch.autograd.grad(out.square().sum(), [leaves[n] for n in some]))
    for n, x in zip(wanted, grads[1]):
        assert torch.equal(x, grads[0][n])


def test_a_step_and_a_paged_call_on_another_stream_than_the_allocations():
    from mamba_amd.ops.linear_attention import linear_attention_state_update
    from mamba_amd.ops.paged_attention import paged_attention_update
    g = torch.Generator(device="cuda").manual_seed(0)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)
    state, q, k, v, decay = r(2, 4, 16, 24), r(2, 4, 16), r(2, 2, 16), r(2, 2, 24), -r(4).abs()
    caches = r(300, 16, 2, 16), r(300, 16, 2, 24)
    table = torch.arange(300, dtype=torch.int32, device="cuda").view(2, 150)
    lens = torch.tensor([2000, 7], dtype=torch.int32, device="cuda")
    other = state.clone(), *(c.clone() for c in caches)
    want = linear_attention_state_update(other[0], q, k, v, decay), paged_attention_update(q, k, v, *other[1:], table, lens)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = linear_attention_state_update(state, q, k, v, decay), paged_attention_update(q, k, v, *caches, table, lens)
    side.synchronize()
    for a, b in zip((*got, state, *caches), (*want, *other)):
        assert torch.equal(a, b)
