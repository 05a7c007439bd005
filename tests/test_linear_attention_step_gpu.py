"""linear_attention_state_update against the 64-bit oracle, and beside linear_attention_fn."""
import pytest
import torch

from oracle.linear_attention import linear_attention_oracle, linear_step_oracle, within

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _step(*args, **kw):
    from mamba_amd.ops.linear_attention import linear_attention_state_update
    return linear_attention_state_update(*args, **kw)


@pytest.fixture(params=["ext", "ctypes"])
def host(request, monkeypatch):
    from mamba_amd import _lib
    if request.param == "ctypes":
        monkeypatch.setattr(_lib, "_torch_ext", None)
    return request.param


def _inputs(batch, heads, kv, dk, dv, dtype, state_dtype=torch.float32, rows=None, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s, dt=dtype: torch.randn(*s, generator=g).to(dt)
    return dict(state=r(rows or batch, heads, dk, dv, dt=state_dtype), q=r(batch, heads, dk), k=r(batch, kv, dk), v=r(batch, kv, dv),
                log_decay=torch.log1p(-torch.exp2(-torch.linspace(0.5, 12, heads))))


def _check(t, rows=None, index_dtype=torch.int32, **kw):
    ref, bound = linear_step_oracle(t["state"], t["q"], t["k"], t["v"], t["log_decay"], rows=rows, **kw)
    d = {k: v.cuda() for k, v in t.items()}
    at = torch.tensor(rows, dtype=index_dtype, device="cuda") if rows is not None else None
    out = _step(*d.values(), state_batch_indices=at, **kw)
    assert out.dtype == t["q"].dtype and d["state"].dtype == t["state"].dtype
    within("out", out, ref["out"], bound["out"])
    within("state", d["state"], ref["state"], bound["state"])
    return out, d["state"]


@pytest.mark.parametrize("state_dtype", DTYPES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("batch,heads,kv,dk,dv", [
    (1, 1, 1, 1, 1), (2, 4, 4, 64, 64), (3, 6, 2, 33, 7), (1, 2, 1, 128, 130), (5, 3, 3, 256, 256), (2, 8, 1, 80, 104), (1, 2, 2, 9, 63), (2, 3, 1, 255, 65)])
def test_step(batch, heads, kv, dk, dv, dtype, state_dtype):
    _check(_inputs(batch, heads, kv, dk, dv, dtype, state_dtype, seed=dk))


def test_a_large_batch():
    _check(_inputs(300, 20, 20, 16, 24, torch.bfloat16))


@pytest.mark.parametrize("index_dtype", [torch.int32, torch.int64])
def test_in_a_pool_of_rows(index_dtype):
    t = _inputs(6, 4, 2, 40, 48, torch.bfloat16, rows=9)
    rows = [7, -1, 0, 9, 3, -5]
    out, state = _check(t, rows, index_dtype)
    assert torch.count_nonzero(out[[1, 3, 5]]) == 0
    assert torch.equal(state.cpu()[[1, 2, 4, 5, 6, 8]], t["state"][[1, 2, 4, 5, 6, 8]])


def test_row_numbers_of_64_bits_turn_into_no_others():
    t = _inputs(5, 2, 2, 16, 16, torch.float32, rows=4)
    rows = [1, 2 ** 32, 2 ** 32 + 2, 2 ** 31, -(2 ** 32) + 3]
    _check(t, [1, -1, -1, -1, -1])
    d = {k: v.cuda() for k, v in t.items()}
    out = _step(*d.values(), state_batch_indices=torch.tensor(rows, device="cuda"))
    assert torch.count_nonzero(out[1:]) == 0 and torch.equal(d["state"].cpu()[[0, 2, 3]], t["state"][[0, 2, 3]])


def test_pools_without_rows_and_batches_of_none():
    t = {k: v.cuda() for k, v in _inputs(2, 4, 2, 8, 8, torch.float32).items()}
    none = _step(t["state"][:0], t["q"], t["k"], t["v"], t["log_decay"], state_batch_indices=torch.tensor([0, -1], dtype=torch.int32, device="cuda"))
    assert torch.count_nonzero(none) == 0 and none.shape == (2, 4, 8)
    assert _step(t["state"], t["q"][:0], t["k"][:0], t["v"][:0], t["log_decay"]).shape == (0, 4, 8)


@pytest.mark.parametrize("scale", [0.0, -3.0])
def test_scales_and_decays_at_their_ends(scale):
    t = _inputs(2, 5, 1, 24, 40, torch.bfloat16)
    t["log_decay"] = torch.tensor([0.0, -float("inf"), -90.0, -1e-30, 2.0])
    _check(t, scale=scale)


def test_strided_operands_and_rows_of_a_larger_buffer():
    t = _inputs(3, 4, 2, 16, 24, torch.float16, seed=5)
    want_out, want_state = _check(t)
    big = torch.zeros(3, 4 * 16 * 24 + 7, device="cuda")
    state = big[:, 3:3 + 4 * 16 * 24].unflatten(1, (4, 16, 24))
    state.copy_(t["state"])
    q = torch.empty(4, 3, 16, dtype=torch.float16, device="cuda").transpose(0, 1).copy_(t["q"])
    k = torch.empty(3, 16, 2, dtype=torch.float16, device="cuda").transpose(1, 2).copy_(t["k"])
    v = torch.empty(3, 2, 30, dtype=torch.float16, device="cuda")[..., 1:25].copy_(t["v"])
    out = _step(state, q, k, v, t["log_decay"].cuda())
    assert torch.equal(out, want_out) and torch.equal(state, want_state)
    assert torch.count_nonzero(big[:, :3]) == 0 and torch.count_nonzero(big[:, -4:]) == 0


def test_rows_beyond_32_bit_offsets():
    t = _inputs(2, 2, 2, 16, 16, torch.bfloat16, torch.bfloat16)
    want_out, want_state = _check(t)
    big = torch.zeros(2 ** 31 + 5000, dtype=torch.bfloat16, device="cuda")
    state = big.as_strided((2, 2, 16, 16), (2 ** 31 + 300, 256, 16, 1)).copy_(t["state"])
    out = _step(state, *(t[n].cuda() for n in ("q", "k", "v", "log_decay")))
    assert torch.equal(out, want_out) and torch.equal(state, want_state)


@pytest.mark.parametrize("dtype", DTYPES)
def test_steps_follow_a_sequence(dtype):
    """A prompt through linear_attention_fn, then tokens one by one: what the whole sequence gives."""
    from mamba_amd.ops.linear_attention import linear_attention_fn
    g = torch.Generator().manual_seed(0)
    q, k, v = torch.randn(2, 90, 4, 32, generator=g).to(dtype), torch.randn(2, 90, 2, 32, generator=g).to(dtype), torch.randn(2, 90, 2, 48, generator=g).to(dtype)
    decay = torch.tensor([-0.5, -0.1, -0.01, 0.0])
    ref, bound = linear_attention_oracle(q, k, v, decay)
    out, state = linear_attention_fn(*(t[:, :80].cuda() for t in (q, k, v)), decay.cuda(), return_final_states=True)
    within("prompt", out, ref["out"][:, :80], bound["out"][:, :80])
    for t in range(80, 90):
        out = _step(state, *(x[:, t].cuda() for x in (q, k, v)), decay.cuda())
        within("token", out, ref["out"][:, t], bound["out"][:, t])
    within("state", state, ref["final"], bound["final"])


def test_the_host_sides_give_the_same(monkeypatch):
    from mamba_amd import _lib
    t = _inputs(3, 4, 2, 40, 48, torch.bfloat16, rows=5)
    want = _check(t, [4, 1, 0])
    monkeypatch.setattr(_lib, "_torch_ext", None)
    assert all(torch.equal(a, b) for a, b in zip(_check(t, [4, 1, 0]), want))


def test_the_state_has_a_new_version(host):
    t = {k: v.cuda() for k, v in _inputs(2, 2, 2, 8, 8, torch.float32).items()}
    version = t["state"]._version
    _step(*t.values())
    assert t["state"]._version == version + 1
    leaf = torch.ones((), device="cuda", requires_grad=True)
    used = leaf * t["state"]
    _step(*t.values())
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        used.sum().backward()


def test_a_state_of_inference_mode(host):
    with torch.inference_mode():
        t = {k: v.cuda() for k, v in _inputs(2, 2, 2, 8, 8, torch.float32).items()}
        want = t["state"].clone()
        out = _step(want, *list(t.values())[1:])
        assert torch.equal(_step(*t.values()), out) and torch.equal(t["state"], want)


@pytest.mark.parametrize("which", ["q", "k", "v"])
def test_a_gradient_through_a_step_is_refused_not_dropped(host, which):
    t = {k: v.cuda() for k, v in _inputs(2, 4, 2, 8, 8, torch.float32).items()}
    t[which].requires_grad_()
    out = _step(*t.values())
    assert out.requires_grad
    with pytest.raises(RuntimeError, match="no gradients"):
        out.sum().backward()


def test_a_state_that_wants_gradients_is_refused(host):
    t = {k: v.cuda() for k, v in _inputs(2, 4, 2, 8, 8, torch.float32).items()}
    t["state"].requires_grad_()
    with pytest.raises(RuntimeError, match="takes no gradients"):
        _step(*t.values())
    with torch.no_grad():
        _step(*t.values())


def test_transforms_are_refused_and_traces_replay(host):
    import torch.autograd.forward_ad as fwAD
    t = {k: v.cuda() for k, v in _inputs(2, 4, 2, 8, 8, torch.float32).items()}
    rest = (t["k"], t["v"], t["log_decay"])
    with fwAD.dual_level(), pytest.raises(NotImplementedError):
        _step(t["state"], fwAD.make_dual(t["q"], torch.ones_like(t["q"])), *rest)
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda s: _step(t["state"], t["q"], *rest) + s)(torch.zeros(2, 1, device="cuda"))
    with torch.no_grad():
        traced = torch.jit.trace(lambda s, q: _step(s, q, *rest), (t["state"].clone(), t["q"]), check_trace=False)
        for seed in range(3):
            state = torch.randn_like(t["state"])
            want_state = state.clone()
            want = _step(want_state, t["q"], *rest)
            assert torch.equal(traced(state, t["q"]), want) and torch.equal(state, want_state)


def test_steps_in_a_captured_graph():
    t = {k: v.cuda() for k, v in _inputs(3, 4, 2, 32, 32, torch.bfloat16, rows=5).items()}
    rows = torch.tensor([4, -1, 0], dtype=torch.int32, device="cuda")
    start = t["state"].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _step(*t.values(), state_batch_indices=rows)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _step(*t.values(), state_batch_indices=rows)
    t["state"].copy_(start)
    other = start.clone()
    for n in range(4):
        rows.copy_(torch.tensor([[4, -1, 0], [1, 2, 3], [0, 4, 9], [3, 1, -1]][n]))
        t["q"].copy_(torch.randn(t["q"].shape, generator=torch.Generator().manual_seed(n)))
        graph.replay()
        want = _step(other, *list(t.values())[1:], state_batch_indices=rows)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(t["state"], other)
