"""Oracles of linear attention with a decay per head and of the attention of one token over a paged cache (test
infrastructure, CPU, plain PyTorch).

Everything is formed in 64 bits, position by position, with the gradients written out;
tests/test_oracle_linear_attention.py pins both against torch.autograd, finite differences and formulations of their own.

Next to each result stands a bound of what the operators' arithmetic may be off by.  u = 2^-24 is half a step of fp32.

Linear attention.  Every result is a sum of products of three of the inputs' numbers and a decay; beside each result stands A,
the same sum of absolute values, and the result is off by a number of steps times A.
 * fp32 arithmetic, K u: the sums over a head size and over a block (at most 256 + 64 terms, in any order), twice, 2 (256 + 64);
   a decay f^n = 2^(n l log2 e): its argument x is off by 3 u |x|, so it by 3 u min(|x|, 126) below which it is 0, in the block and
   from the blocks before, 2 * 378; its exponential, products and scale, 16; and once per block (of 32 positions or more) that a
   state has gone through, its factor and the product with it, 6 u + 3 u |x|, where the x of all blocks together count once more
   as above, 378.  K = 1800 + 6 (n / 32 + 1) for a sequence of n positions.
 * What is rounded on its way from one product to the next.  bf16: the decayed scores (at a sequence's end in two parts) and the
   state, as operands of out, dq, dk and dv, to 8 bits, 2^-8 of each; the decayed values that a state takes up, in two parts, 2^-16.
   fp16: everything computed, in two parts, with the products of two second parts left out, 2^-15.  Where a state is a result, the
   values it takes up are in three parts, and in fp16 the products of second and third parts are left out, 2^-23.  fp32: nothing.
   Gradients of shared heads are sums in fp32.
   (K covers sums of any numbers; tests/test_linear_attention_precision_gpu.py has results of one product each, to a fortieth of it.)

Attention.  A score is off by d = (headdim_k + 8) u scale |q| . |k|, its weight 2^(..) relative to the others by 2 d and 16 u; the
weights' sums and products in fp32 by n u for n positions; weights that go into the product with V are rounded to the type, 2^-8
(bf16) or 2^-11 and 2^-40 in all (fp16) of the largest weight of their run, which is not above the sum of all.
"""
import torch

from oracle.gated_linear import U, within  # noqa: F401  (the bounds and their check are the same)

ROUND = {torch.float32: (0.0, 0.0), torch.bfloat16: (2.0 ** -8 + 2.0 ** -16, 2.0 ** -23), torch.float16: (2.0 ** -14, 2.0 ** -23)}


def _d(t):
    return None if t is None else t.detach().double().cpu()


def linear_attention_oracle(q, k, v, log_decay, scale=None, initial_states=None, cu_seqlens=None, dout=None, dfinal=None):
    """Returns two dicts, results and bounds, with out, final and, where dout or dfinal is given, dq, dk, dv, dinitial.
    cu_seqlens: a list."""
    of_outs, of_states = ROUND.get(q.dtype, (0.0, 0.0))
    batch, total, heads, size_k = q.shape
    group = heads // k.shape[2]
    scale = size_k ** -0.5 if scale is None else scale
    q, k, v = _d(q), _d(k).repeat_interleave(group, 2), _d(v).repeat_interleave(group, 2)
    size_v = v.shape[-1]
    f = torch.exp(_d(log_decay).clamp(max=0.0))[:, None, None]
    spans = [(slice(None), slice(None), 0, total)] if cu_seqlens is None else [
        (slice(n, n + 1), slice(0, 1), cu_seqlens[n], cu_seqlens[n + 1]) for n in range(len(cu_seqlens) - 1)]
    seqs = batch if cu_seqlens is None else len(spans)
    start = torch.zeros(seqs, heads, size_k, size_v, dtype=torch.float64) if initial_states is None else _d(initial_states)
    steps = lambda n: (1800 + 6 * (n / 32 + 1)) * U
    zeros = lambda *s: torch.zeros(*s, dtype=torch.float64)
    out, dq = zeros(batch, total, heads, size_v), zeros(batch, total, heads, size_k)
    final, out_b, dq_b, final_b = zeros(*start.shape), zeros(*out.shape), zeros(*dq.shape), zeros(*start.shape)
    back = dout is not None or dfinal is not None
    do = _d(dout) if dout is not None else zeros(*out.shape)
    df = _d(dfinal) if dfinal is not None else zeros(*start.shape)
    outer = lambda a, b: a[..., :, None] * b[..., None, :]
    left = lambda a, s: (a[..., :, None] * s).sum(-2)   # a S
    right = lambda s, b: (s * b[..., None, :]).sum(-1)  # S b
    for seq, row, lo, hi in spans:
        S, A, e = start[seq], start[seq].abs(), steps(hi - lo)
        for t in range(lo, hi):
            S = f * S + outer(k[row, t], v[row, t])
            A = f * A + outer(k[row, t].abs(), v[row, t].abs())
            out[row, t], out_b[row, t] = scale * left(q[row, t], S), abs(scale) * left(q[row, t].abs(), A) * (of_outs + e)
            if back:
                dq[row, t], dq_b[row, t] = scale * right(S, do[row, t]), abs(scale) * right(A, do[row, t].abs()) * (of_outs + e)
        final[seq], final_b[seq] = S, A * (of_states + e)
    res, bound = dict(out=out, final=final), dict(out=out_b, final=final_b)
    if not back:
        return res, bound
    dk, dv = zeros(*k.shape), zeros(*v.shape)
    dk_b, dv_b, dstart, dstart_b = zeros(*k.shape), zeros(*v.shape), zeros(*start.shape), zeros(*start.shape)
    for seq, row, lo, hi in spans:
        R, A, e = df[seq], df[seq].abs(), steps(hi - lo)
        for t in range(hi - 1, lo - 1, -1):
            R = R + scale * outer(q[row, t], do[row, t])
            A = A + abs(scale) * outer(q[row, t].abs(), do[row, t].abs())
            dk[row, t], dk_b[row, t] = right(R, v[row, t]), right(A, v[row, t].abs()) * (of_outs + e)
            dv[row, t], dv_b[row, t] = left(k[row, t], R), left(k[row, t].abs(), A) * (of_outs + e)
            R, A = f * R, f * A
        dstart[seq], dstart_b[seq] = R, A * (of_states + e)
    shared = lambda t: t.view(batch, total, heads // group, group, t.shape[-1]).sum(3)
    res.update(dq=dq, dk=shared(dk), dv=shared(dv), dinitial=dstart)
    bound.update(dq=dq_b, dk=shared(dk_b) * (1 + group * U), dv=shared(dv_b) * (1 + group * U), dinitial=dstart_b)
    return res, bound


def linear_step_oracle(state, q, k, v, log_decay, scale=None, rows=None):
    """The new states and outputs of one token, and their bounds: a state's element is one product and one sum (4 u of the
    absolute terms with its decay), an output a sum over a head size."""
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    group = q.shape[1] // k.shape[1]
    q, k, v, state = _d(q), _d(k).repeat_interleave(group, 1), _d(v).repeat_interleave(group, 1), _d(state).clone()
    f = torch.exp(_d(log_decay).clamp(max=0.0))[:, None, None]
    out, state_b = torch.zeros(*q.shape[:2], v.shape[-1], dtype=torch.float64), torch.zeros_like(state)
    out_b = torch.zeros_like(out)
    for place, row in enumerate(range(len(q)) if rows is None else rows):
        if not 0 <= row < len(state):
            continue
        term = k[place][..., :, None] * v[place][..., None, :]
        size = f * state[row].abs() + term.abs()
        state[row] = f * state[row] + term
        state_b[row] = 400 * U * size
        out[place] = scale * (q[place][..., None] * state[row]).sum(-2)
        out_b[place] = abs(scale) * (q[place].abs()[..., None] * size).sum(-2) * (400 + 264) * U
    return dict(out=out, state=state), dict(out=out_b, state=state_b)


def paged_attention_oracle(q, k, v, k_cache, v_cache, block_table, cache_seqlens, scale=None, window=None):
    """The outputs, the caches behind the call and the outputs' bounds.  block_table, cache_seqlens: nested lists."""
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    dtype, (pages, page, kv, size_k) = q.dtype, k_cache.shape
    group = q.shape[1] // kv
    k_cache, v_cache = k_cache.clone().cpu(), v_cache.clone().cpu()
    out = torch.zeros(*q.shape[:2], v_cache.shape[-1], dtype=torch.float64)
    bound = torch.zeros_like(out)
    for b, n in enumerate(cache_seqlens):
        if n < 0:
            continue
        n = min(n, len(block_table[b]) * page)
        places = [(block_table[b][p // page], p % page) for p in range(n)]
        keys = [(_d(k_cache[at]), _d(v_cache[at])) if 0 <= at[0] < pages else None for at in places]
        if k is not None:
            keys.append((_d(k[b]), _d(v[b])))
            if n < len(block_table[b]) * page and 0 <= block_table[b][n // page] < pages:
                k_cache[block_table[b][n // page], n % page] = k[b].cpu()
                v_cache[block_table[b][n // page], n % page] = v[b].cpu()
        keys = [pair for pair in (keys[-window:] if window is not None else keys) if pair is not None]
        if not keys:
            continue
        K, V = (torch.stack([pair[i] for pair in keys]).repeat_interleave(group, 1) for i in (0, 1))  # positions, heads, size
        s = scale * (K * _d(q[b])).sum(-1)
        p = torch.softmax(s, 0)[..., None]
        out[b] = (p * V).sum(0)
        d = ((size_k + 8) * U * abs(scale) * (K.abs() * _d(q[b]).abs()).sum(-1)).amax(0)[:, None]
        rounding = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}.get(dtype, 0.0)
        small = 2.0 ** -40 * V.abs().sum(0) if dtype == torch.float16 else 0.0
        bound[b] = (p * V.abs()).sum(0) * (4 * d + (32 + 2 * len(keys)) * U + rounding) + small
    return dict(out=out, k_cache=k_cache, v_cache=v_cache), dict(out=bound)
