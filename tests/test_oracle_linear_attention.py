"""The oracles of linear attention and of the attention over a paged cache: against autograd, finite differences and
formulations of their own; and the plain-torch statements next to the operators against the oracles."""
import pytest
import torch

from oracle.linear_attention import linear_attention_oracle, linear_step_oracle, paged_attention_oracle, within


def _inputs(batch=2, L=9, heads=4, kv=2, dk=3, dv=5, seed=0, dtype=torch.float64, seqs=None):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64).to(dtype)
    n = batch if seqs is None else seqs
    return dict(q=r(batch, L, heads, dk), k=r(batch, L, kv, dk), v=r(batch, L, kv, dv), log_decay=-r(heads).abs(),
                initial_states=r(n, heads, dk, dv), dout=r(batch, L, heads, dv), dfinal=r(n, heads, dk, dv))


def _quadratic(q, k, v, log_decay, start, scale):
    """out as one lower-triangular product per head, the final state as one product."""
    L, group = q.shape[1], q.shape[2] // k.shape[2]
    k, v = k.repeat_interleave(group, 2), v.repeat_interleave(group, 2)
    t = torch.arange(L)
    apart = t[:, None] - t
    decay = torch.where(apart >= 0, torch.exp(log_decay[:, None, None] * apart.clamp(min=0)), 0)
    out = torch.einsum("bthk,bshk,hts,bshv->bthv", q, k, decay, v)
    out = out + torch.einsum("bthk,ht,bhkv->bthv", q, torch.exp(log_decay[:, None] * (t + 1)), start)
    final = torch.einsum("bshk,hs,bshv->bhkv", k, torch.exp(log_decay[:, None] * (L - 1 - t)), v)
    return scale * out, final + torch.exp(log_decay * L)[:, None, None] * start


@pytest.mark.parametrize("scale", [None, -0.7])
def test_oracle_against_the_quadratic_form_and_autograd(scale):
    t = _inputs()
    names = ["q", "k", "v", "initial_states"]
    leaves = {n: t[n].clone().requires_grad_() for n in names}
    out, final = _quadratic(leaves["q"], leaves["k"], leaves["v"], t["log_decay"], leaves["initial_states"], scale or 3 ** -0.5)
    grads = torch.autograd.grad([out, final], list(leaves.values()), [t["dout"], t["dfinal"]])
    res, _ = linear_attention_oracle(scale=scale, **t)
    torch.testing.assert_close(res["out"], out.detach(), rtol=1e-12, atol=1e-12)
    torch.testing.assert_close(res["final"], final.detach(), rtol=1e-12, atol=1e-12)
    for n, g in zip(["dq", "dk", "dv", "dinitial"], grads):
        torch.testing.assert_close(res[n], g, rtol=1e-11, atol=1e-12)


def test_oracle_against_differences():
    t = _inputs(1, 4, 2, 1, 2, 2, seed=3)
    res, _ = linear_attention_oracle(**t)
    value = lambda r: float((r["out"] * t["dout"]).sum() + (r["final"] * t["dfinal"]).sum())
    forward = {k: v for k, v in t.items() if k not in ("dout", "dfinal")}
    for name, grad in (("q", "dq"), ("k", "dk"), ("v", "dv"), ("initial_states", "dinitial")):
        for at in range(t[name].numel()):
            side = []
            for step in (1e-6, -1e-6):
                moved = t[name].clone()
                moved.view(-1)[at] += step
                side.append(value(linear_attention_oracle(**{**forward, name: moved})[0]))
            assert abs((side[0] - side[1]) / 2e-6 - float(res[grad].view(-1)[at])) < 1e-6, (name, at)


def test_oracle_packed_equals_separate():
    cu = [2, 5, 5, 6, 13]  # positions before the first sequence, an empty one, one of one position, padding behind
    t = _inputs(1, 15, seed=1, seqs=4)
    for n in ("q", "k", "v", "dout"):
        t[n][:, :2], t[n][:, 13:] = float("nan"), float("nan")
    res, _ = linear_attention_oracle(cu_seqlens=cu, **t)
    for n in range(4):
        part = {k: (v[:, cu[n]:cu[n + 1]] if v.dim() == 4 and v.shape[0] == 1 else v[n:n + 1] if v.dim() == 4 else v) for k, v in t.items()}
        one, _ = linear_attention_oracle(**part)
        for name in ("out", "dq", "dk", "dv"):
            torch.testing.assert_close(res[name][:, cu[n]:cu[n + 1]], one[name], rtol=1e-12, atol=1e-12)
        for name in ("final", "dinitial"):
            torch.testing.assert_close(res[name][n:n + 1], one[name], rtol=1e-12, atol=1e-12)
    for name in ("out", "dq", "dk", "dv"):
        assert torch.count_nonzero(res[name][:, :2]) == 0 and torch.count_nonzero(res[name][:, 13:]) == 0


def test_no_decay_is_a_running_sum_and_full_decay_is_one_position():
    t = _inputs(1, 6, 2, 2, 3, 4)
    t["log_decay"] = torch.tensor([0.0, -float("inf")], dtype=torch.float64)
    res, _ = linear_attention_oracle(t["q"], t["k"], t["v"], t["log_decay"], scale=1.0)
    sums = (t["k"][..., :, None] * t["v"][..., None, :]).cumsum(1)
    torch.testing.assert_close(res["out"][:, :, 0], (t["q"][..., None] * sums).sum(-2)[:, :, 0])
    torch.testing.assert_close(res["out"][:, :, 1], ((t["q"] * t["k"]).sum(-1, keepdim=True) * t["v"])[:, :, 1])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_statements_beside_the_operators(dtype):
    from mamba_amd.ops.linear_attention import linear_attention_ref, linear_attention_state_update_ref
    t = _inputs(2, 7, dtype=dtype)
    t["initial_states"], t["log_decay"] = t["initial_states"].float(), t["log_decay"].float()
    res, bound = linear_attention_oracle(t["q"], t["k"], t["v"], t["log_decay"], initial_states=t["initial_states"])
    out, final = linear_attention_ref(t["q"], t["k"], t["v"], t["log_decay"], initial_states=t["initial_states"], return_final_states=True)
    within("out", out, res["out"], bound["out"])
    within("final", final, res["final"], bound["final"])
    state = t["initial_states"].clone()
    ref, bound = linear_step_oracle(state, t["q"][:, 0], t["k"][:, 0], t["v"][:, 0], t["log_decay"])
    torch.testing.assert_close(ref["out"], res["out"][:, 0])
    out = linear_attention_state_update_ref(state, t["q"][:, 0], t["k"][:, 0], t["v"][:, 0], t["log_decay"])
    within("step", out, ref["out"], bound["out"])
    within("state", state, ref["state"], bound["state"])


def _cache(seed=0, dtype=torch.float64):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64).to(dtype)
    return dict(q=r(4, 6, 8), k=r(4, 3, 8), v=r(4, 3, 5), k_cache=r(9, 4, 3, 8), v_cache=r(9, 4, 3, 5)), [
        [7, 2, 0], [1, 3, 4], [5, -1, -1], [6, 8, -1]], [9, 11, 0, -1]


@pytest.mark.parametrize("window", [None, 1, 5])
@pytest.mark.parametrize("new", [True, False])
def test_attention_oracle_against_dense_attention(window, new):
    t, table, lens = _cache()
    if not new:
        t["k"] = t["v"] = None
    res, _ = paged_attention_oracle(block_table=table, cache_seqlens=lens, window=window, **t)
    for b, n in enumerate(lens):
        if n + new <= 0:
            assert torch.count_nonzero(res["out"][b]) == 0
            continue
        rows = [page for page in table[b] if page >= 0]
        keys, values = res["k_cache"][rows].flatten(0, 1)[:n + new], res["v_cache"][rows].flatten(0, 1)[:n + new]
        if new:
            assert torch.equal(keys[-1], t["k"][b]) and torch.equal(values[-1], t["v"][b])
        if window:
            keys, values = keys[-window:], values[-window:]
        want = torch.nn.functional.scaled_dot_product_attention(
            t["q"][b][:, None], keys.transpose(0, 1).repeat_interleave(2, 0), values.transpose(0, 1).repeat_interleave(2, 0))
        torch.testing.assert_close(res["out"][b], want[:, 0], rtol=1e-12, atol=1e-12)


def test_attention_oracle_leaves_out_pages_that_are_none():
    t, table, _ = _cache()
    short = {k: v[:1] if v.shape[0] == 4 else v for k, v in t.items()}
    whole, _ = paged_attention_oracle(block_table=[[7, 2]], cache_seqlens=[5], **short)
    holes, _ = paged_attention_oracle(block_table=[[7, 99, 2]], cache_seqlens=[9], **short)
    assert torch.equal(holes["out"], whole["out"])
    # a new token behind the table's end takes part, and is written nowhere
    full, _ = paged_attention_oracle(block_table=[[7, 2]], cache_seqlens=[50], **short)
    again, _ = paged_attention_oracle(block_table=[[7, 2, -1]], cache_seqlens=[8], **short)
    assert torch.equal(full["out"], again["out"]) and torch.equal(full["k_cache"], t["k_cache"])


@pytest.mark.parametrize("window", [None, 3])
def test_attention_statement_beside_the_operator(window):
    from mamba_amd.ops.paged_attention import paged_attention_update_ref
    t, table, lens = _cache(dtype=torch.float32)
    res, bound = paged_attention_oracle(block_table=table, cache_seqlens=lens, window=window, **t)
    out = paged_attention_update_ref(block_table=torch.tensor(table), cache_seqlens=torch.tensor(lens), window=window, **t)
    within("out", out, res["out"], bound["out"])
    assert torch.equal(t["k_cache"], res["k_cache"]) and torch.equal(t["v_cache"], res["v_cache"])
