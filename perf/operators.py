"""The operators of gated linear recurrent blocks, timed as a program that trains or serves such blocks calls them.

  scan   gated_linear_scan_fn       h_t = a_t h_{t-1} + sqrt(1 - a_t^2) sigmoid(gate_x_t) x_t with
                                    log a_t = -rate softplus(decay) sigmoid(gate_a_t), per channel; forward (prefill) or
                                    forward + backward (training), rows of a batch or packed sequences
  step   gated_linear_state_update  one token of the same recurrence, the states updated in place
  norm   block_norm_fn              residual + scale * norm(x) * silu(z) and the next block's norm of that sum, forward
                                    (serving) or forward + backward (training)

`own` says which side `run` takes: the plain form in torch's elementary operations, or the package's operators.
`listed()` has the cases, `draw()` gives more of the same ranges.
"""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
RATE = 8.0
EPS = 1e-5


def listed():
    return [
        # the few tokens that a draft proposed, checked for four users in one call from their states: launch time counts
        dict(name="scan_draft_b4_l9", op="scan", batch=4, dim=1536, seqlen=9, dtype="bf16", grad=False, sequences=0, states=True),
        # prefill of one prompt, whatever its length is, and the state that decoding starts from
        dict(name="scan_prefill_b1_l777", op="scan", batch=1, dim=1536, seqlen=777, dtype="bf16", grad=False, sequences=0,
             states=True),
        # prefill of the prompts of several users in one packed row, odd number of channels
        dict(name="scan_prefill_packed", op="scan", batch=1, dim=2561, seqlen=8191, dtype="fp16", grad=False, sequences=23,
             states=True),
        # training in fp32, a small model
        dict(name="scan_train_fp32", op="scan", batch=2, dim=1536, seqlen=2048, dtype="fp32", grad=True, sequences=0, states=False),
        # training at full size, the shape of the Mamba-1 benchmark
        dict(name="scan_train_large", op="scan", batch=8, dim=5120, seqlen=4096, dtype="bf16", grad=True, sequences=0, states=False),
        # training on one long row of packed sequences, as the packed SSD benchmark has it
        dict(name="scan_train_packed", op="scan", batch=1, dim=4096, seqlen=32768, dtype="bf16", grad=True, sequences=16, states=False),
        # one token for one user: host time and one launch
        dict(name="step_b1", op="step", batch=1, dim=2560, dtype="bf16", state="fp32", pooled=False),
        # one token for a full serving batch, states in a pool of rows, some of the batch's places empty
        dict(name="step_b256_pooled", op="step", batch=256, dim=5120, dtype="bf16", state="fp32", pooled=True),
        # between two blocks of one decoded token
        dict(name="norm_token", op="norm", rows=1, dim=2560, dtype="bf16", stream="bf16", params="bf16", rms=True, gate=True, scale=True,
             bias=False, grad=False),
        # LayerNorm with biases over a prompt, an odd number of channels
        dict(name="norm_prefill_odd", op="norm", rows=1531, dim=1001, dtype="fp16", stream="fp16", params="fp16", rms=False, gate=True,
             scale=False, bias=True, grad=False),
        # training in fp32, a small model with LayerNorm
        dict(name="norm_train_fp32", op="norm", rows=4096, dim=768, dtype="fp32", stream="fp32", params="fp32", rms=False, gate=False,
             scale=True, bias=True, grad=True),
        # a training step at full size: 16384 positions of d_model 2560, fp32 residual stream and parameters
        dict(name="norm_train", op="norm", rows=16384, dim=2560, dtype="bf16", stream="fp32", params="fp32", rms=True, gate=True,
             scale=True, bias=False, grad=True),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["scan"] * 6 + ["step"] * 2 + ["norm"] * 4)
    dtype = rng.choice(["bf16"] * 4 + ["fp16", "fp32"])
    if op == "scan":
        dim = _log(rng, 64, 640) * 8 + rng.choice([0, 0, 0, 1, 6])
        grad = rng.random() < 0.6
        most = 8 * 5120 * 4096 // (4 if dtype == "fp32" else 2)
        if rng.random() < 0.3:
            total = min(_log(rng, 33, 32768), most // dim)
            return dict(op=op, batch=1, dim=dim, seqlen=total, dtype=dtype, grad=grad,
                        sequences=min(_log(rng, 2, 64), total), states=rng.random() < 0.5)
        batch = _log(rng, 1, 16)
        seqlen = min(_log(rng, 1, 8192) if rng.random() < 0.7 else _log(rng, 2, 64) * 128, most // (dim * batch))
        return dict(op=op, batch=batch, dim=dim, seqlen=seqlen, dtype=dtype, grad=grad, sequences=0, states=rng.random() < 0.5)
    if op == "step":
        return dict(op=op, batch=_log(rng, 1, 1024), dim=_log(rng, 64, 640) * 8 + rng.choice([0, 0, 0, 1, 6]), dtype=dtype,
                    state=rng.choice(["fp32", dtype]), pooled=rng.random() < 0.5)
    grad = rng.random() < 0.6
    dim = _log(rng, 64, 1024) * 8 + rng.choice([0, 0, 0, 1, 6])
    rows = min(_log(rng, 1, 16384), 16384 * 2560 // dim)
    rms = rng.random() < 0.6
    return dict(op=op, rows=rows, dim=dim, dtype=dtype, stream=rng.choice([dtype, "fp32"]), params=rng.choice([dtype, "fp32"]), rms=rms,
                gate=rng.random() < 0.7, scale=rng.random() < 0.7, bias=not rms, grad=grad)


# ------------------------------------------------------------------ inputs
def _bounds(case, seed):
    """First positions of a row's packed sequences, and its end: ragged, every sequence of one position at least."""
    n, total = case["sequences"], case["seqlen"]
    g = torch.Generator().manual_seed(seed + 17)
    cuts = (torch.randperm(total - 1, generator=g)[:n - 1] + 1).sort().values
    return torch.cat([torch.zeros(1, dtype=torch.int64), cuts, torch.tensor([total])])


def _decay(dim, g):
    """Parameters for which a fully open gate keeps 0.9 to 0.999 of the state, as such layers are initialised."""
    keep = 0.9 + 0.099 * torch.rand(dim, device="cuda", generator=g)
    return torch.log(torch.expm1(-torch.log(keep) / RATE))


def _same(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    randn = lambda *shape, dtype=dtype: torch.randn(*shape, device="cuda", generator=g).to(dtype)
    s = dict(case=case)
    if case["op"] == "scan":
        shape = (case["batch"], case["seqlen"], case["dim"])
        s.update(x=randn(*shape), gate_a=randn(*shape), gate_x=randn(*shape), decay=_decay(case["dim"], g), cu_seqlens=None,
                 initial=None)
        if case["sequences"]:
            s["cu_seqlens"] = _bounds(case, seed).to("cuda", torch.int32)
        if case["states"]:
            s["initial"] = randn(case["sequences"] or case["batch"], case["dim"], dtype=torch.float32)
        if case["grad"]:
            s["dout"] = randn(*shape)
            s["dfinal"] = randn(*s["initial"].shape, dtype=torch.float32) if case["states"] else None
    elif case["op"] == "step":
        batch, dim = case["batch"], case["dim"]
        rows = batch + batch // 2 + 1 if case["pooled"] else batch
        s.update(x=randn(batch, dim), gate_a=randn(batch, dim), gate_x=randn(batch, dim), decay=_decay(dim, g),
                 state=randn(rows, dim, dtype=DTYPES[case["state"]]), indices=None)
        if case["pooled"]:
            indices = torch.randperm(rows, device="cuda", generator=g)[:batch].to(torch.int32)
            if batch > 8:
                indices[5::8] = -1
            s["indices"] = indices
    else:
        rows, dim = case["rows"], case["dim"]
        stream, params = DTYPES[case["stream"]], DTYPES[case["params"]]
        s.update(x=randn(rows, dim), residual=(2 * randn(rows, dim, dtype=torch.float32)).to(stream),
                 z=randn(rows, dim) if case["gate"] else None,
                 norm_weight=(1 + 0.1 * randn(dim, dtype=torch.float32)).to(params),
                 next_weight=(1 + 0.1 * randn(dim, dtype=torch.float32)).to(params), norm_bias=None, next_bias=None, scale=None)
        if case["bias"]:
            s.update(norm_bias=(0.1 * randn(dim, dtype=torch.float32)).to(params),
                     next_bias=(0.1 * randn(dim, dtype=torch.float32)).to(params))
        if case["scale"]:
            s["scale"] = (0.5 + 0.1 * randn(dim, dtype=torch.float32)).to(params)
        if case["grad"]:
            s.update(dout=randn(rows, dim), dsum=randn(rows, dim, dtype=stream))
    return s


LEAVES = {"scan": ("x", "gate_a", "gate_x", "decay", "initial"),
          "norm": ("x", "residual", "norm_weight", "next_weight", "z", "scale", "norm_bias", "next_bias")}


def prepare(case, seed):
    s = _same(case, seed)
    if case.get("grad"):
        for name in LEAVES[case["op"]]:
            if s[name] is not None:
                s[name].requires_grad_()
    return s


# ------------------------------------------------------------------ the plain forms
def _scan_plain(a, b):
    """h_t = a_t h_{t-1} + b_t along dim 1 from h = 0, by doubling: after the step n, position t holds its last 2 n terms."""
    n = 1
    while n < a.shape[1]:
        b = torch.cat([b[:, :n], b[:, n:] + a[:, n:] * b[:, :-n]], 1)
        a = torch.cat([a[:, :n], a[:, n:] * a[:, :-n]], 1)
        n *= 2
    return b


def _edges(s):
    """Indices (row, position) of the first and the last position of every sequence."""
    case, device = s["case"], s["x"].device
    if s["cu_seqlens"] is not None:
        cu = s["cu_seqlens"].long()
        row = torch.zeros_like(cu[1:])
        return (row, cu[:-1]), (row, cu[1:] - 1)
    row = torch.arange(case["batch"], device=device)
    return (row, torch.zeros_like(row)), (row, torch.full_like(row, case["seqlen"] - 1))


def _scan_run_plain(s):
    case, dtype = s["case"], s["x"].dtype
    with torch.no_grad():
        first, last = _edges(s)
        x, decay = s["x"].float(), s["decay"].float()
        r, i = torch.sigmoid(s["gate_a"].float()), torch.sigmoid(s["gate_x"].float())
        k = RATE * torch.log1p(torch.exp(decay))
        log_a = -k * r
        a, m = torch.exp(log_a), torch.sqrt(-torch.expm1(2 * log_a))
        b = m * i * x
        # what enters a sequence is added to its first position, whose own factor then keeps the one before out
        if s["initial"] is not None:
            b[first] += a[first] * s["initial"]
        a0 = a.clone()
        a0[first] = 0
        h = _scan_plain(a0, b)
        out = {"out": h.to(dtype)}
        if case["states"]:
            out["final"] = h[last]
        if not case["grad"]:
            return out
        # gradient of h, from the last position on: g_t = dout_t + a_{t+1} g_{t+1}
        g = s["dout"].float()
        if case["states"]:
            g[last] += s["dfinal"]
        back = torch.cat([a0[:, 1:], torch.zeros_like(a0[:, :1])], 1)
        g = _scan_plain(back.flip(1), g.flip(1)).flip(1)
        before = torch.cat([torch.zeros_like(h[:, :1]), h[:, :-1]], 1)
        before[first] = s["initial"] if s["initial"] is not None else 0
        dlog_a = g * (a * before - a * a / m * i * x)
        gi = g * m
        out["dx"] = (gi * i).to(dtype)
        out["dgate_a"] = (dlog_a * -k * r * (1 - r)).to(dtype)
        out["dgate_x"] = (gi * x * i * (1 - i)).to(dtype)
        out["ddecay"] = (dlog_a * r).sum((0, 1)) * -RATE * torch.sigmoid(decay)
        if s["initial"] is not None:
            out["dinitial"] = (a * g)[first]
        return out


def _step_run_plain(s):
    state, x = s["state"], s["x"].float()
    r, i = torch.sigmoid(s["gate_a"].float()), torch.sigmoid(s["gate_x"].float())
    log_a = -RATE * torch.log1p(torch.exp(s["decay"].float())) * r
    b = torch.sqrt(-torch.expm1(2 * log_a)) * i * x
    if s["indices"] is None:
        h = torch.exp(log_a) * state.float() + b
        state.copy_(h)
        return {"out": h.to(s["x"].dtype), "state": state}
    rows = s["indices"].long()
    used = rows >= 0
    # an empty place of the batch is sent to a row of its own behind the pool
    more = torch.cat([state, torch.zeros_like(state[:1])])
    at = torch.where(used, rows, state.shape[0])
    h = torch.exp(log_a) * more[at].float() + b
    more[at] = h.to(state.dtype)
    state.copy_(more[:-1])
    return {"out": torch.where(used[:, None], h, 0).to(s["x"].dtype), "state": state}


def _norm_plain(x, weight, bias, rms):
    """Normalised rows, the factor of each, and the norm's result."""
    d = x if rms else x - x.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt(d.square().mean(-1, keepdim=True) + EPS)
    n = d * rstd
    return n, rstd, n * weight + bias if bias is not None else n * weight


def _norm_back(dy, n, rstd, weight, rms):
    dn = dy * weight
    d = dn - n * (dn * n).mean(-1, keepdim=True)
    return rstd * (d if rms else d - dn.mean(-1, keepdim=True))


def _norm_run_plain(s):
    case, rms = s["case"], s["case"]["rms"]
    with torch.no_grad():
        f = lambda name: s[name].float() if s[name] is not None else None
        x, residual, z, scale = f("x"), f("residual"), f("z"), f("scale")
        n1, rstd1, y = _norm_plain(x, f("norm_weight"), f("norm_bias"), rms)
        gate = z * torch.sigmoid(z) if z is not None else torch.ones_like(x[:1])
        factor = scale if scale is not None else torch.ones_like(x[0])
        total = residual + factor * y * gate
        n2, rstd2, o = _norm_plain(total, f("next_weight"), f("next_bias"), rms)
        out = {"out": o.to(s["x"].dtype), "residual_out": total.to(s["residual"].dtype)}
        if not case["grad"]:
            return out
        dout = s["dout"].float()
        d = s["dsum"].float() + _norm_back(dout, n2, rstd2, f("next_weight"), rms)
        dy = d * factor * gate
        params = s["norm_weight"].dtype
        out["dx"] = _norm_back(dy, n1, rstd1, f("norm_weight"), rms).to(s["x"].dtype)
        out["dresidual"] = d.to(s["residual"].dtype)
        out["dnorm_weight"] = (dy * n1).sum(0).to(params)
        out["dnext_weight"] = (dout * n2).sum(0).to(params)
        if z is not None:
            t = torch.sigmoid(z)
            out["dz"] = (d * factor * y * t * (1 + z * (1 - t))).to(s["z"].dtype)
        if scale is not None:
            out["dscale"] = (d * y * gate).sum(0).to(params)
        if case["bias"]:
            out["dnorm_bias"] = dy.sum(0).to(params)
            out["dnext_bias"] = dout.sum(0).to(params)
        return out


# ------------------------------------------------------------------ the package's operators
def _grads(s, outs, douts, out):
    names = [n for n in LEAVES[s["case"]["op"]] if s[n] is not None]
    for name, g in zip(names, torch.autograd.grad(outs, [s[n] for n in names], douts)):
        out["d" + name] = g
    return {k: v.detach() for k, v in out.items()}


def _scan_run_own(s):
    from mamba_amd.ops.gated_linear_scan import gated_linear_scan_fn
    case = s["case"]
    res = gated_linear_scan_fn(s["x"], s["gate_a"], s["gate_x"], s["decay"], rate=RATE, initial_states=s["initial"],
                               cu_seqlens=s["cu_seqlens"], return_final_states=case["states"])
    out = {"out": res[0], "final": res[1]} if case["states"] else {"out": res}
    if not case["grad"]:
        return out
    if case["states"]:
        return _grads(s, [out["out"], out["final"]], [s["dout"], s["dfinal"]], out)
    return _grads(s, [out["out"]], [s["dout"]], out)


def _step_run_own(s):
    from mamba_amd.ops.gated_linear_scan import gated_linear_state_update
    out = gated_linear_state_update(s["state"], s["x"], s["gate_a"], s["gate_x"], s["decay"], rate=RATE, state_batch_indices=s["indices"])
    return {"out": out, "state": s["state"]}


def _norm_run_own(s):
    from mamba_amd.ops.block_norm import block_norm_fn
    case = s["case"]
    o, total = block_norm_fn(s["x"], s["residual"], s["norm_weight"], s["next_weight"], z=s["z"], scale=s["scale"],
                             norm_bias=s["norm_bias"], next_bias=s["next_bias"], eps=EPS, is_rms_norm=case["rms"])
    out = {"out": o, "residual_out": total}
    return _grads(s, [o, total], [s["dout"], s["dsum"]], out) if case["grad"] else out


def run(state):
    op = state["case"]["op"]
    if own:
        return {"scan": _scan_run_own, "step": _step_run_own, "norm": _norm_run_own}[op](state)
    return {"scan": _scan_run_plain, "step": _step_run_plain, "norm": _norm_run_plain}[op](state)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    size = lambda dtype: 4 if dtype == "fp32" else 2
    e = size(case["dtype"])
    if case["op"] == "scan":
        n, states = case["batch"] * case["seqlen"] * case["dim"], (case["sequences"] or case["batch"]) * case["dim"] * 4
        tensors, rows = (8, 4) if case["grad"] else (4, 2)
        return {"bytes": tensors * n * e + (rows * states if case["states"] else 0), "flops": (50 if case["grad"] else 18) * n}
    if case["op"] == "step":
        n = case["batch"] * case["dim"]
        return {"bytes": n * (4 * e + 2 * size(case["state"])), "flops": 18 * n}
    n = case["rows"] * case["dim"]
    gate = 1 if case["gate"] else 0
    # in: x, z, residual; out: out, residual_out; with gradients also in: dout, dsum; out: dx, dz, dresidual
    acts, streams = (4 + 2 * gate, 4) if case["grad"] else (2 + gate, 2)
    return {"bytes": n * (acts * e + streams * size(case["stream"])), "flops": (60 if case["grad"] else 20) * n}


# ------------------------------------------------------------------ the definitions in 64 bits
def _scan_exact(s):
    case = s["case"]
    x, ga, gx, lam = (s[n].double() for n in ("x", "gate_a", "gate_x", "decay"))
    batch, total, dim = x.shape
    cu = s["cu_seqlens"].tolist() if case["sequences"] else [0, total]
    seqs = len(cu) - 1
    r, i = 1 / (1 + torch.exp(-ga)), 1 / (1 + torch.exp(-gx))
    k = RATE * torch.log1p(torch.exp(lam))
    a = torch.exp(-k * r)
    m = torch.sqrt(-torch.expm1(-2 * k * r))
    b = m * i * x
    start = s["initial"].double() if case["states"] else torch.zeros(seqs * batch, dim, dtype=torch.float64, device=x.device)
    h, before, final = torch.empty_like(x), torch.empty_like(x), torch.empty_like(start)
    rows = lambda q: slice(q, q + 1) if case["sequences"] else slice(0, batch)
    for q in range(seqs):
        now = start[rows(q)]
        for t in range(cu[q], cu[q + 1]):
            before[:, t] = now
            now = torch.addcmul(b[:, t], a[:, t], now)
            h[:, t] = now
        final[rows(q)] = now
    out = {"out": h}
    if case["states"]:
        out["final"] = final
    if not case["grad"]:
        return out
    g, dstart = s["dout"].double(), torch.zeros_like(start)
    for q in range(seqs):
        carry = s["dfinal"].double()[rows(q)] if case["states"] else torch.zeros_like(start[rows(q)])
        for t in range(cu[q + 1] - 1, cu[q] - 1, -1):
            g[:, t] += carry
            carry = a[:, t] * g[:, t]
        dstart[rows(q)] = carry
    da = g * (before - a / m * i * x)
    drate = da * a * -r
    out.update(dx=g * m * i, dgate_a=da * a * -k * r * (1 - r), dgate_x=g * m * x * i * (1 - i),
               ddecay=drate.sum((0, 1)) * RATE / (1 + torch.exp(-lam)))
    if case["states"]:
        out["dinitial"] = dstart
    return out


def _step_exact(s):
    x, ga, gx, lam, state = (s[n].double() for n in ("x", "gate_a", "gate_x", "decay", "state"))
    log_a = -RATE * torch.log1p(torch.exp(lam)) / (1 + torch.exp(-ga))
    out, state = torch.zeros_like(x), state.clone()
    rows = s["indices"].tolist() if s["indices"] is not None else range(x.shape[0])
    for place, row in enumerate(rows):
        if row >= 0:
            h = torch.exp(log_a[place]) * state[row] + torch.sqrt(-torch.expm1(2 * log_a[place])) * x[place] / (1 + torch.exp(-gx[place]))
            out[place] = h
            state[row] = h
    return {"out": out, "state": state}


def _norm_exact(s):
    names = [n for n in LEAVES["norm"] if s[n] is not None]
    t = {n: s[n].detach().double().requires_grad_() for n in names}

    def norm(v, weight, bias):
        if not s["case"]["rms"]:
            v = v - v.mean(-1, keepdim=True)
        v = v / torch.sqrt((v * v).mean(-1, keepdim=True) + EPS) * weight
        return v + bias if bias is not None else v

    y = norm(t["x"], t["norm_weight"], t.get("norm_bias"))
    if "z" in t:
        y = y * t["z"] / (1 + torch.exp(-t["z"]))
    if "scale" in t:
        y = y * t["scale"]
    total = t["residual"] + y
    o = norm(total, t["next_weight"], t.get("next_bias"))
    out = {"out": o, "residual_out": total}
    if s["case"]["grad"]:
        grads = torch.autograd.grad([o, total], [t[n] for n in names], [s["dout"].double(), s["dsum"].double()])
        out.update({"d" + n: g for n, g in zip(names, grads)})
    return {k: v.detach() for k, v in out.items()}


def exact(case, seed):
    s = _same(case, seed)
    return {"scan": _scan_exact, "step": _step_exact, "norm": _norm_exact}[case["op"]](s)
