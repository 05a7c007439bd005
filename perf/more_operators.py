"""The operators of linear attention layers and of the attention layers between them, timed as a program that trains or serves
such layers calls them.

  linear     linear_attention_fn             S_t = exp(log_decay) S_{t-1} + k_t v_t^T,  out_t = scale q_t S_t  per head; forward
                                             (prefill) or forward + backward (training), rows of a batch or packed sequences
  step       linear_attention_state_update   one token of the same recurrence, the states updated in place
  attention  paged_attention_update          one token's attention over a paged key-value cache, its key and value appended

`own` says which side `run` takes: the plain form in torch's elementary operations, or the package's operators.
`listed()` has the cases, `draw()` gives more of the same ranges.
"""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
CHUNK = 64


def listed():
    return [
        # the few tokens that a draft proposed, checked for four users in one call from their states: launch time counts
        dict(name="linear_draft_b4_l9", op="linear", batch=4, seqlen=9, heads=12, kv_heads=12, dk=64, dv=64, dtype="bf16", grad=False,
             sequences=0, states=True),
        # prefill of one prompt, whatever its length is, and the states that decoding starts from
        dict(name="linear_prefill_b1_l777", op="linear", batch=1, seqlen=777, heads=20, kv_heads=20, dk=128, dv=128, dtype="bf16",
             grad=False, sequences=0, states=True),
        # prefill of the prompts of several users in one packed row; head sizes off the powers of two, keys of pairs of heads shared
        dict(name="linear_prefill_packed", op="linear", batch=1, seqlen=8191, heads=16, kv_heads=8, dk=80, dv=104, dtype="fp16",
             grad=False, sequences=23, states=True),
        # training in fp32, a small model
        dict(name="linear_train_fp32", op="linear", batch=2, seqlen=2048, heads=12, kv_heads=12, dk=64, dv=64, dtype="fp32", grad=True,
             sequences=0, states=False),
        # training at full size, d_model 2560
        dict(name="linear_train", op="linear", batch=8, seqlen=4096, heads=20, kv_heads=20, dk=128, dv=128, dtype="bf16", grad=True,
             sequences=0, states=False),
        # training on one long row of packed sequences, keys and values shared by four heads each
        dict(name="linear_train_packed", op="linear", batch=1, seqlen=32768, heads=32, kv_heads=8, dk=64, dv=64, dtype="bf16", grad=True,
             sequences=16, states=False),
        # one token for one user
        dict(name="step_b1", op="step", batch=1, heads=20, kv_heads=20, dk=128, dv=128, dtype="bf16", state="fp32", pooled=False),
        # one token for a full serving batch, states in a pool of rows, some of the batch's places empty
        dict(name="step_b256_pooled", op="step", batch=256, heads=20, kv_heads=20, dk=128, dv=128, dtype="bf16", state="fp32", pooled=True),
        # the first tokens of a chat: a short cache, launch time counts
        dict(name="attention_b1_l100", op="attention", batch=1, context=100, heads=32, kv_heads=8, dk=128, dv=128, page=16, dtype="bf16",
             window=0),
        # a serving batch of ragged lengths, four query heads for each key head
        dict(name="attention_b32_l8192", op="attention", batch=32, context=8192, heads=32, kv_heads=8, dk=128, dv=128, page=64, dtype="bf16",
             window=0),
        # a head for every key, an odd head size, and a window over the last positions
        dict(name="attention_fp16_window", op="attention", batch=48, context=2047, heads=12, kv_heads=12, dk=80, dv=80, page=16, dtype="fp16",
             window=777),
        # one user with a very long context: all parallelism lies along the cache
        dict(name="attention_b1_l131072", op="attention", batch=1, context=131072, heads=32, kv_heads=8, dk=128, dv=128, page=256,
             dtype="bf16", window=0),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _heads(rng):
    kv = rng.choice([1, 2, 4, 5, 8, 12, 16, 20])
    return kv * rng.choice([1, 1, 1, 2, 4, 8] if kv <= 8 else [1]), kv


def _head_size(rng):
    return rng.choice([32, 64, 64, 128, 128, 128, 256, 48, 80, 96, 112, 72, 33, 100, 1])


def draw(rng):
    op = rng.choice(["linear"] * 6 + ["step"] * 2 + ["attention"] * 4)
    dtype = rng.choice(["bf16"] * 4 + ["fp16", "fp32"])
    heads, kv_heads = _heads(rng)
    dk = _head_size(rng)
    dv = dk if rng.random() < 0.7 else _head_size(rng)
    case = dict(op=op, heads=heads, kv_heads=kv_heads, dk=dk, dv=dv, dtype=dtype)
    if op == "linear":
        most = min(32768 * 20 * 256 // (heads * (dk + dv)), 32768 * 20 * 128 * 128 // (heads * dk * dv)) // (4 if dtype == "fp32" else 1)
        grad = rng.random() < 0.6
        if rng.random() < 0.35:
            total = min(_log(rng, 33, 32768), most)
            return dict(case, batch=1, seqlen=total, grad=grad, sequences=min(_log(rng, 2, 64), total), states=rng.random() < 0.5)
        batch = _log(rng, 1, 16)
        seqlen = max(1, min(_log(rng, 1, 8192) if rng.random() < 0.7 else _log(rng, 1, 64) * 128, most // batch))
        return dict(case, batch=batch, seqlen=seqlen, grad=grad, sequences=0, states=rng.random() < 0.5)
    if op == "step":
        batch = min(_log(rng, 1, 1024), 256 * 20 * 128 * 128 // (heads * dk * dv))
        return dict(case, batch=batch, state=rng.choice(["fp32", "fp32", dtype]), pooled=rng.random() < 0.5)
    context = _log(rng, 1, 131072)
    batch = max(1, min(_log(rng, 1, 128), 131072 * 8 * 256 // (context * kv_heads * (dk + dv)) // (2 if dtype == "fp32" else 1)))
    context = min(context, 131072 * 8 * 256 // (kv_heads * (dk + dv)) // (2 if dtype == "fp32" else 1))
    return dict(case, batch=batch, context=context, page=rng.choice([1, 16, 16, 32, 64, 128, 256, 24]),
                window=_log(rng, 1, context) if rng.random() < 0.3 else 0)


# ------------------------------------------------------------------ inputs
def _bounds(case, seed):
    """First positions of a row's packed sequences, and its end: ragged, every sequence of one position at least."""
    n, total = case["sequences"], case["seqlen"]
    g = torch.Generator().manual_seed(seed + 17)
    cuts = (torch.randperm(total - 1, generator=g)[:n - 1] + 1).sort().values
    return torch.cat([torch.zeros(1, dtype=torch.int64), cuts, torch.tensor([total])])


def _log_decay(heads, g):
    """Heads that forget within a few positions to heads that remember thousands, as such layers have them."""
    power = torch.linspace(1.0, 12.0, heads, device="cuda") + 0.2 * torch.rand(heads, device="cuda", generator=g)
    return torch.log1p(-torch.exp2(-power))


def _same(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    randn = lambda *shape, dtype=dtype: torch.randn(*shape, device="cuda", generator=g).to(dtype)
    heads, kv, dk, dv, batch = case["heads"], case["kv_heads"], case["dk"], case["dv"], case["batch"]
    s = dict(case=case, scale=dk ** -0.5)
    if case["op"] == "linear":
        rows = (batch, case["seqlen"])
        s.update(q=randn(*rows, heads, dk), k=randn(*rows, kv, dk), v=randn(*rows, kv, dv), log_decay=_log_decay(heads, g), cu_seqlens=None,
                 initial=None)
        if case["sequences"]:
            s["cu_seqlens"] = _bounds(case, seed).to("cuda", torch.int32)
        if case["states"]:
            s["initial"] = randn(case["sequences"] or batch, heads, dk, dv, dtype=torch.float32)
        if case["grad"]:
            s["dout"] = randn(*rows, heads, dv)
            s["dfinal"] = randn(*s["initial"].shape, dtype=torch.float32) if case["states"] else None
    elif case["op"] == "step":
        rows = batch + batch // 8 + 1 if case["pooled"] else batch
        s.update(q=randn(batch, heads, dk), k=randn(batch, kv, dk), v=randn(batch, kv, dv), log_decay=_log_decay(heads, g),
                 state=randn(rows, heads, dk, dv, dtype=DTYPES[case["state"]]), indices=None)
        if case["pooled"]:
            indices = torch.randperm(rows, device="cuda", generator=g)[:batch].to(torch.int32)
            if batch > 8:
                indices[5::8] = -1
            s["indices"] = indices
    else:
        page, context = case["page"], case["context"]
        # positions that are in the cache before the call; a batch of ragged lengths has an empty place too
        lens = torch.full((batch,), context - 1, device="cuda", dtype=torch.int64)
        if batch > 1:
            lens = torch.randint(0, context, (batch,), device="cuda", generator=g)
        if batch > 8:
            lens[5] = -1
        wide = -(-context // page)
        used = (lens + page) // page  # pages that hold positions 0 .. lens
        first = torch.cumsum(used, 0) - used
        pages = batch * wide
        order = torch.randperm(pages, device="cuda", generator=g)
        column = torch.arange(wide, device="cuda")
        table = torch.where(column < used[:, None], order[(first[:, None] + column).clamp(max=pages - 1)], -1)
        # the pool has the pages of this batch and some of others; -1 behind a sequence's last page
        s.update(q=2 * randn(batch, heads, dk), k=randn(batch, kv, dk), v=randn(batch, kv, dv), k_cache=randn(pages, page, kv, dk),
                 v_cache=randn(pages, page, kv, dv), block_table=table.to(torch.int32), cache_seqlens=lens.to(torch.int32))
    return s


LEAVES = ("q", "k", "v", "initial")


def prepare(case, seed):
    s = _same(case, seed)
    if case.get("grad"):
        for name in LEAVES:
            if s[name] is not None:
                s[name].requires_grad_()
    return s


# ------------------------------------------------------------------ the plain forms
def _blocks(cu, total, reverse):
    """Positions of every sequence in blocks of CHUNK, in the order of the walk: (blocks, CHUNK) positions (`total` where there is
    none), whose sequence each block belongs to, and how many positions it has."""
    count = total // CHUNK + cu.shape[0]
    n = cu[1:] - cu[:-1]
    ends = torch.cumsum((n + CHUNK - 1) // CHUNK, 0)
    b = torch.arange(count, device=cu.device)
    seq = torch.searchsorted(ends, b, right=True)
    here = seq < n.shape[0]
    seq = seq.clamp(max=n.shape[0] - 1)
    at = (b - (ends - (n + CHUNK - 1) // CHUNK)[seq])[:, None] * CHUNK + torch.arange(CHUNK, device=cu.device)
    inside = here[:, None] & (at < n[seq][:, None])
    pos = torch.where(inside, cu[1:][seq][:, None] - 1 - at if reverse else cu[:-1][seq][:, None] + at, total)
    return pos, torch.where(here, seq, -1), inside.sum(1)


def _pass(a, b, c, log_decay, cu, start, mix, read, write, reverse):
    """y_t = mix sum_{s <= t} f^(t - s) (a_t . b_s) c_s + read f^(t + e) a_t start, and start f^n + write sum f^(n - e' - s) b_s c_s^T at the
    end of n positions, f = exp(log_decay), along the sequences or against them: there a state has been scaled when it comes in.
    a, b, c: (positions, heads, size).  Within a block as a product with the decays, from block to block by the blocks' states."""
    total, heads = a.shape[:2]
    late = 0 if reverse else 1
    pos, seq, n = _blocks(cu, total, reverse)
    rows = lambda t: torch.cat([t, torch.zeros_like(t[:1])])[pos].permute(2, 0, 1, 3)  # heads, blocks, CHUNK, size
    a, b, c = rows(a), rows(b), rows(c)
    i = torch.arange(CHUNK, device=pos.device)
    power = lambda e: torch.exp(log_decay.view(-1, *[1] * e.dim()) * e)
    apart = i[:, None] - i
    p = torch.matmul(a, b.transpose(-1, -2)) * torch.where(apart >= 0, power(apart.clamp(min=0)), 0)[:, None]
    y = mix * torch.matmul(p, c)
    left = (n[:, None] - late - i).clamp(min=0)
    own_states = write * torch.matmul((b * power(left)[..., None]).transpose(-1, -2), c)
    # f^(positions between two blocks) from each block of a sequence to its later ones
    ends = torch.cumsum(n, 0)
    between = (ends - n)[:, None] - ends
    same = (seq[:, None] == seq) & (seq[:, None] >= 0)
    later = same & (torch.arange(len(seq), device=pos.device)[:, None] > torch.arange(len(seq), device=pos.device))
    carry = torch.where(later, power(between.clamp(min=0)), 0)
    shape = own_states.shape
    states = torch.matmul(carry, own_states.flatten(2)).view(shape)
    # what a sequence starts from, at each of its blocks
    first = torch.cumsum(n, 0) - n - cu[:-1][seq.clamp(min=0)] + cu[0]
    start = start.permute(1, 0, 2, 3)
    states = states + power(first)[..., None, None] * start[:, seq.clamp(min=0)]
    y = y + read * torch.matmul(a * power(i + late)[:, None, :, None], states)
    out = torch.zeros(total + 1, heads, c.shape[-1], device=a.device)
    out[pos] = y.permute(1, 2, 0, 3)
    # the state behind each sequence: all of its blocks' contributions, and what it started from
    length = cu[1:] - cu[:-1]
    behind = cu[1:, None] - cu[0] - ends
    mine = torch.arange(length.shape[0], device=pos.device)[:, None] == seq
    last = torch.matmul(torch.where(mine, power(behind.clamp(min=0)), 0), own_states.flatten(2)).view(heads, -1, *shape[2:])
    last = last + power(length)[..., None, None] * start
    return out[:total], last.permute(1, 0, 2, 3)


def _linear_run_plain(s):
    case, dtype, scale = s["case"], s["q"].dtype, s["scale"]
    with torch.no_grad():
        batch, seqlen, heads, dk = s["q"].shape
        group = heads // case["kv_heads"]
        rows = lambda t: t.float().flatten(0, 1)
        q, k, v = rows(s["q"]), rows(s["k"]).repeat_interleave(group, 1), rows(s["v"]).repeat_interleave(group, 1)
        cu = s["cu_seqlens"].long() if s["cu_seqlens"] is not None else torch.arange(batch + 1, device=q.device) * seqlen
        start = s["initial"] if s["initial"] is not None else torch.zeros(len(cu) - 1, heads, dk, v.shape[-1], device=q.device)
        out, final = _pass(q, k, v, s["log_decay"], cu, start, scale, scale, 1.0, False)
        back = lambda t, like: t.view(like.shape[:2] + (-1,) + t.shape[-1:]).to(dtype)
        res = {"out": back(out, s["q"])}
        if case["states"]:
            res["final"] = final
        if not case["grad"]:
            return res
        do = rows(s["dout"])
        dfinal = s["dfinal"] if case["states"] else torch.zeros_like(start)
        dq, _ = _pass(do, v, k, s["log_decay"], cu, start.transpose(-1, -2), scale, scale, 1.0, False)
        dk_, _ = _pass(v, do, q, s["log_decay"], cu, dfinal.transpose(-1, -2), scale, 1.0, scale, True)
        dv_, dstart = _pass(k, q, do, s["log_decay"], cu, dfinal, scale, 1.0, scale, True)
        shared = lambda t: t.view(t.shape[0], -1, group, t.shape[-1]).sum(2)
        res.update(dq=back(dq, s["q"]), dk=back(shared(dk_), s["k"]), dv=back(shared(dv_), s["v"]))
        if case["states"]:
            res["dinitial"] = dstart
        return res


def _places(used):
    """The batch's places with the first used one's number in place of the empty ones: their work is done twice, with the same result."""
    return torch.where(used, torch.arange(len(used), device=used.device), used.int().argmax())


def _step_run_plain(s):
    state = s["state"]
    rows = s["indices"].long() if s["indices"] is not None else torch.arange(len(s["q"]), device=state.device)
    at = _places(rows >= 0)
    group = s["case"]["heads"] // s["case"]["kv_heads"]
    q, k, v = s["q"][at].float(), s["k"][at].float().repeat_interleave(group, 1), s["v"][at].float().repeat_interleave(group, 1)
    h = torch.exp(s["log_decay"])[:, None, None] * state[rows[at]].float() + k[..., None] * v[..., None, :]
    state[rows[at]] = h.to(state.dtype)
    out = s["scale"] * (q[..., None] * h).sum(-2)
    return {"out": torch.where((rows >= 0)[:, None, None], out, 0).to(s["q"].dtype), "state": state}


def _attention_run_plain(s):
    case, page = s["case"], s["case"]["page"]
    batch, kv, group = case["batch"], case["kv_heads"], case["heads"] // case["kv_heads"]
    lens, table = s["cache_seqlens"].long(), s["block_table"].long()
    used = lens >= 0
    here = _places(used)
    last = lens[here]
    row = torch.gather(table[here], 1, (last // page)[:, None])[:, 0] * page + last % page
    s["k_cache"].flatten(0, 1)[row] = s["k"][here]
    s["v_cache"].flatten(0, 1)[row] = s["v"][here]
    k = s["k_cache"][table.clamp(min=0)].flatten(1, 2).float().transpose(1, 2)  # batch, kv heads, positions, size
    v = s["v_cache"][table.clamp(min=0)].flatten(1, 2).float().transpose(1, 2)
    pos = torch.arange(k.shape[2], device=k.device)
    seen = pos <= lens[:, None]
    if case["window"]:
        seen &= pos > lens[:, None] - case["window"]
    q = s["q"].float().view(batch, kv, group, -1)
    logits = torch.where(seen[:, None, None], s["scale"] * torch.matmul(q, k.transpose(-1, -2)), -math.inf)
    top = logits.amax(-1, keepdim=True)
    p = torch.where(seen[:, None, None], torch.exp(logits - top), 0)
    out = torch.matmul(p, v) / p.sum(-1, keepdim=True)
    out = torch.where(used[:, None, None, None], out, 0).flatten(1, 2)
    return {"out": out.to(s["q"].dtype), "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


# ------------------------------------------------------------------ the package's operators
def _linear_run_own(s):
    from mamba_amd.ops.linear_attention import linear_attention_fn
    case = s["case"]
    res = linear_attention_fn(s["q"], s["k"], s["v"], s["log_decay"], scale=s["scale"], initial_states=s["initial"],
                              cu_seqlens=s["cu_seqlens"], return_final_states=case["states"])
    out = {"out": res[0], "final": res[1]} if case["states"] else {"out": res}
    if not case["grad"]:
        return out
    outs, douts = [out["out"]], [s["dout"]]
    if case["states"]:
        outs.append(out["final"])
        douts.append(s["dfinal"])
    names = [n for n in LEAVES if s[n] is not None]
    for name, g in zip(names, torch.autograd.grad(outs, [s[n] for n in names], douts)):
        out["d" + name] = g
    return {k: v.detach() for k, v in out.items()}


def _step_run_own(s):
    from mamba_amd.ops.linear_attention import linear_attention_state_update
    out = linear_attention_state_update(s["state"], s["q"], s["k"], s["v"], s["log_decay"], scale=s["scale"],
                                        state_batch_indices=s["indices"])
    return {"out": out, "state": s["state"]}


def _attention_run_own(s):
    from mamba_amd.ops.paged_attention import paged_attention_update
    out = paged_attention_update(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["block_table"], s["cache_seqlens"], scale=s["scale"],
                                 window=s["case"]["window"] or None)
    return {"out": out, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def run(state):
    op = state["case"]["op"]
    if own:
        return {"linear": _linear_run_own, "step": _step_run_own, "attention": _attention_run_own}[op](state)
    return {"linear": _linear_run_plain, "step": _step_run_plain, "attention": _attention_run_plain}[op](state)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    size = lambda dtype: 4 if dtype == "fp32" else 2
    e, heads, kv, dk, dv, batch = size(case["dtype"]), case["heads"], case["kv_heads"], case["dk"], case["dv"], case["batch"]
    if case["op"] == "linear":
        rows = batch * case["seqlen"]
        states = (case["sequences"] or batch) * heads * dk * dv * 4 if case["states"] else 0
        # q, k, v read and out written; with gradients also q, k, v, dout read and dq, dk, dv written
        forward, leaves = heads * (dk + dv) + kv * (dk + dv), heads * dk + kv * (dk + dv)
        if not case["grad"]:
            return {"bytes": rows * forward * e + 2 * states, "flops": 4 * rows * heads * dk * dv}
        return {"bytes": rows * (forward + 2 * leaves + heads * dv) * e + 4 * states, "flops": 14 * rows * heads * dk * dv}
    if case["op"] == "step":
        used = batch - len(range(5, batch, 8)) if case["pooled"] and batch > 8 else batch
        return {"bytes": used * heads * dk * dv * 2 * size(case["state"]) + batch * (heads + kv) * (dk + dv) * e,
                "flops": 5 * used * heads * dk * dv}
    # ragged lengths: uniform, so half of the longest in the mean
    length = case["context"] if batch == 1 else (case["context"] + 1) / 2
    if case["window"]:
        w, c = case["window"], case["context"]
        length = min(w, c) if batch == 1 else (w * (c - w) + w * (w + 1) / 2) / c
    rows = length * (batch - (1 if batch > 8 else 0))
    return {"bytes": rows * kv * (dk + dv) * e + batch * (heads + kv) * (dk + dv) * e, "flops": 2 * rows * heads * (dk + dv)}


# ------------------------------------------------------------------ the definitions in 64 bits
def _linear_exact(s):
    case = s["case"]
    batch, total, heads, dk = s["q"].shape
    dv, group = case["dv"], heads // case["kv_heads"]
    seqs = case["sequences"] or batch
    q, k, v = s["q"].double(), s["k"].double().repeat_interleave(group, 2), s["v"].double().repeat_interleave(group, 2)
    cu = s["cu_seqlens"].tolist() if case["sequences"] else [0, total]
    f = torch.exp(s["log_decay"].double())[:, None, None]
    rows = lambda n: slice(n, n + 1) if case["sequences"] else slice(0, batch)
    zeros = lambda: torch.zeros(seqs, heads, dk, dv, dtype=torch.float64, device=q.device)
    start = s["initial"].double() if case["states"] else zeros()
    do = s["dout"].double() if case["grad"] else None
    out = torch.zeros(batch, total, heads, dv, dtype=torch.float64, device=q.device)
    dq, final = torch.zeros_like(q), zeros()
    for n in range(len(cu) - 1):
        state = start[rows(n)]
        for t in range(cu[n], cu[n + 1]):
            state = torch.addcmul(f * state, k[:, t, :, :, None], v[:, t, :, None, :])
            out[:, t] = s["scale"] * torch.matmul(q[:, t, :, None], state)[..., 0, :]
            if case["grad"]:
                dq[:, t] = s["scale"] * torch.matmul(state, do[:, t, :, :, None])[..., 0]
        final[rows(n)] = state
    res = {"out": out}
    if case["states"]:
        res["final"] = final
    if not case["grad"]:
        return res
    dk_, dv_, dstart = torch.zeros_like(k), torch.zeros_like(v), zeros()
    for n in range(len(cu) - 1):
        grad = s["dfinal"].double()[rows(n)] if case["states"] else zeros()[rows(n)]
        for t in range(cu[n + 1] - 1, cu[n] - 1, -1):
            grad = torch.addcmul(grad, s["scale"] * q[:, t, :, :, None], do[:, t, :, None, :])
            dk_[:, t] = torch.matmul(grad, v[:, t, :, :, None])[..., 0]
            dv_[:, t] = torch.matmul(k[:, t, :, None], grad)[..., 0, :]
            grad = f * grad
        dstart[rows(n)] = grad
    shared = lambda t: t.view(batch, total, -1, group, t.shape[-1]).sum(3)
    res.update(dq=dq, dk=shared(dk_), dv=shared(dv_))
    if case["states"]:
        res["dinitial"] = dstart
    return res


def _step_exact(s):
    group = s["case"]["heads"] // s["case"]["kv_heads"]
    q, k, v, state = s["q"].double(), s["k"].double(), s["v"].double(), s["state"].double()
    f = torch.exp(s["log_decay"].double())
    out = torch.zeros(*q.shape[:2], v.shape[-1], dtype=torch.float64, device=q.device)
    for place, row in enumerate(s["indices"].tolist() if s["indices"] is not None else range(q.shape[0])):
        if row < 0:
            continue
        outer = torch.einsum("hi,hj->hij", k[place], v[place]).repeat_interleave(group, 0)
        state[row] = f[:, None, None] * state[row] + outer
        out[place] = s["scale"] * torch.einsum("hi,hij->hj", q[place], state[row])
    return {"out": out, "state": state}


def _attention_exact(s):
    case, page = s["case"], s["case"]["page"]
    group = case["heads"] // case["kv_heads"]
    kc, vc = s["k_cache"].double(), s["v_cache"].double()
    out = torch.zeros(case["batch"], case["heads"], case["dv"], dtype=torch.float64, device=kc.device)
    for b, n in enumerate(s["cache_seqlens"].tolist()):
        if n < 0:
            continue
        pages = s["block_table"][b].tolist()
        kc[pages[n // page], n % page] = s["k"][b].double()
        vc[pages[n // page], n % page] = s["v"][b].double()
        here = torch.tensor(pages[:n // page + 1], device=kc.device)
        first = max(0, n + 1 - case["window"]) if case["window"] else 0
        k, v = kc[here].flatten(0, 1)[first:n + 1], vc[here].flatten(0, 1)[first:n + 1]
        for h in range(case["heads"]):
            weights = torch.softmax(s["scale"] * (k[:, h // group] @ s["q"][b, h].double()), 0)
            out[b, h] = weights @ v[:, h // group]
    return {"out": out, "k_cache": kc, "v_cache": vc}


def exact(case, seed):
    s = _same(case, seed)
    return {"linear": _linear_exact, "step": _step_exact, "attention": _attention_exact}[case["op"]](s)
