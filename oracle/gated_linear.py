"""Oracles of the gated linear recurrence and of the norm between two blocks (test infrastructure, CPU, plain PyTorch).

Everything is formed in 64 bits, position by position, with the gradients written out; tests/test_oracle_gated_linear.py
pins both against torch.autograd, finite differences and independent formulations.

Next to each result stands a bound of what 32-bit arithmetic may be off by.  u = 2^-24 is half a step of fp32; a rounded
operation is off by u, the GPU's exponential, reciprocal and square root by 2 u, an exponential besides by the error of
its argument.  sigmoid(v) = 1 / (1 + exp(-v)): the argument v log2(e) is off by 2 u |v|, the whole by (5 + 2 |v|) u at
most.  a = exp(-k r): the argument k r log2(e) is off by (5 + 2 |v| + 3) u k r, so a by Ca = 2 + k r (8 + 2 |v|) steps of
u, v = gate_a (beyond |v| = 100 the sigmoid is 0 or 1 to the last bit).  sqrt(1 - a^2) has half the relative error of
2 k r where that is small, and less than Ca where it is not; with the other factors of a position, at |v| up to 8, C = 32
steps cover it.  Through the recurrence an error moves like the state: |error_t| <= a_t |error_{t-1}| + u (Ca a_t H_{t-1} +
(C + Ca) |b_t|), H the recurrence of |b|: a product of n decays is off by at most n times what one is, which is what the
sum over the positions says too, in whatever order the decays are multiplied.  A sigmoid r, or a
product k r, below fp32's smallest normal number 2^-126 may come out as 0: m = sqrt(2 k r (1 - k r ...)) is then off by
sqrt(2 max(k, 1) 2^-126) at most, and so, by the formulas below, is what m multiplies; k r / m = m / 2 there, so dgate_a
and, as the decay's slope is k itself where k is small, ddecay are off by as much.  tiny = 2^-62 sqrt(max(k, 1)) times the
other factors is added for it.
"""
import torch

U = 2.0 ** -24
C = 32


def _d(t):
    return None if t is None else t.detach().double().cpu()


def gated_linear_oracle(x, gate_a, gate_x, decay, rate=8.0, initial_states=None, cu_seqlens=None, dout=None, dfinal=None):
    """Returns two dicts, results and bounds, with out, final and, where dout or dfinal is given, dx, dgate_a, dgate_x,
    ddecay, dinitial.  cu_seqlens: a list."""
    x, ga, gx, lam = _d(x), _d(gate_a), _d(gate_x), _d(decay)
    batch, L, dim = x.shape
    # sequences as (their states, their row, first position, end); the rows of a batch are walked together
    if cu_seqlens is None:
        spans = [(slice(None), slice(None), 0, L)]
    else:
        spans = [(q, 0, cu_seqlens[q], cu_seqlens[q + 1]) for q in range(len(cu_seqlens) - 1)]
    seqs = batch if cu_seqlens is None else len(spans)
    inside = torch.zeros(batch, L, 1, dtype=torch.float64)
    for _, row, lo, hi in spans:
        inside[row, lo:hi] = 1
    x, ga, gx = (torch.where(inside > 0, t, torch.zeros_like(t)) for t in (x, ga, gx))
    init = _d(initial_states) if initial_states is not None else torch.zeros(seqs, dim, dtype=torch.float64)
    r, i = torch.sigmoid(ga), torch.sigmoid(gx)
    k = rate * torch.nn.functional.softplus(lam, threshold=1e9)
    a = torch.exp(-k * r)
    m = torch.sqrt(-torch.expm1(-2 * k * r))
    b = m * i * x
    Ca = C + k * r * (8 + 2 * ga.abs().clamp(max=100.0))
    tiny = 2.0 ** -62 * k.clamp(min=1.0).sqrt()
    small, size_b = tiny * (i * x).abs(), b.abs()
    h, before = torch.zeros_like(x), torch.zeros_like(x)
    Eh, Ebefore, final, Efinal = torch.zeros_like(x), torch.zeros_like(x), init.clone(), torch.zeros_like(init)
    for q, row, lo, hi in spans:
        now, H, E = init[q].clone(), init[q].abs(), torch.zeros_like(init[q])
        for t in range(lo, hi):
            before[row, t], Ebefore[row, t] = now, E
            E = a[row, t] * E + U * Ca[row, t] * (a[row, t] * H + 2 * size_b[row, t]) + small[row, t]
            H = a[row, t] * H + size_b[row, t]
            now = a[row, t] * now + b[row, t]
            h[row, t], Eh[row, t] = now, E
        final[q], Efinal[q] = now, E
    res, bound = dict(out=h, final=final), dict(out=Eh, final=Efinal)
    if dout is None and dfinal is None:
        return res, bound
    dout = _d(dout) if dout is not None else torch.zeros_like(x)
    dfinal = _d(dfinal) if dfinal is not None else torch.zeros_like(init)
    dout = torch.where(inside > 0, dout, torch.zeros_like(dout))
    g, Eg = torch.zeros_like(x), torch.zeros_like(x)
    dinit, Edinit = torch.zeros_like(init), torch.zeros_like(init)
    for q, row, lo, hi in spans:
        carry, H, E = dfinal[q].clone(), dfinal[q].abs(), torch.zeros_like(init[q])
        for t in range(hi - 1, lo - 1, -1):
            g[row, t], Eg[row, t] = dout[row, t] + carry, E + U * (dout[row, t].abs() + H)
            H = a[row, t] * (dout[row, t].abs() + H)
            E = a[row, t] * Eg[row, t] + Ca[row, t] * U * H
            carry = a[row, t] * g[row, t]
        dinit[q], Edinit[q] = carry, E
    ix, im = i * x, torch.where(m > 0, 1 / m, torch.zeros_like(m))
    e = g * a * (a * ix * r * im - before * r)
    size = a * (a * ix.abs() * r * im + before.abs() * r)
    Ee = Eg * size + g.abs() * a * r * (Ebefore + 4 * Ca * U * (a * ix.abs() * im + before.abs()))
    slope = rate * torch.sigmoid(lam)
    res.update(dx=g * m * i, dgate_x=g * m * ix * (1 - i), dgate_a=k * (1 - r) * e, ddecay=slope * e.sum((0, 1)), dinitial=dinit)
    lost = tiny * g.abs() * ix.abs()
    bound.update(dx=m * i * (Eg + 3 * Ca * U * g.abs()) + tiny * g.abs() * i,
                 dgate_x=m * ix.abs() * ((1 - i) * (Eg + 4 * Ca * U * g.abs()) + C * U * g.abs()) + lost,  # 1 - i: off by C u i at most
                 dgate_a=k * ((1 - r) * Ee + 3 * C * U * e.abs()) + lost,  # 1 - r: off by C u r at most
                 ddecay=slope * (Ee + (C + x.shape[0] * L) * U * (g * size).abs()).sum((0, 1)) + lost.sum((0, 1)), dinitial=Edinit)
    return res, bound


def block_norm_oracle(x, residual, norm_weight, next_weight, z=None, scale=None, norm_bias=None, next_bias=None, eps=1e-5,
                      is_rms_norm=True, dout=None, dsum=None):
    """Results and bounds, as above: out, residual_out and the gradients of the tensors given.

    The bounds: a row's statistics are sums of dim terms of one sign, or of terms whose size the bound holds; every
    result of a row is a sum of a few products of at most eight rounded factors.  K = 256 steps of u of the largest sum of
    absolute terms in the row cover them: 8 factors, 16 steps each for exponentials and divisions, twice for the sums."""
    K = 256
    f = lambda t: _d(t)
    x, residual, w1, w2, z, b1, b2 = map(f, (x, residual, norm_weight, next_weight, z, norm_bias, next_bias))
    sc = _d(scale) if isinstance(scale, torch.Tensor) else torch.tensor(1.0 if scale is None else scale, dtype=torch.float64)
    zero = torch.zeros(x.shape[-1], dtype=torch.float64)
    mean = lambda v: v.mean(-1, keepdim=True)
    top = lambda v: v.abs().amax(-1, keepdim=True).expand_as(v)

    def norm(v, size):
        """n, rstd and the size of n's terms: of v and its mean, and of what a statistic off by u moves n by"""
        mu = torch.zeros_like(mean(v)) if is_rms_norm else mean(v)
        d = v - mu
        rstd = 1 / torch.sqrt(mean(d * d) + eps)
        n = d * rstd
        spread = (size + mean(size) * (0 if is_rms_norm else 1)) * rstd
        return n, rstd, spread + n.abs() * mean(n.abs() * spread)

    n1, rstd1, N1 = norm(x, x.abs())
    y, Y = n1 * w1 + (zero if b1 is None else b1), N1 * w1.abs() + (zero if b1 is None else b1.abs())
    s1 = torch.sigmoid(z) if z is not None else None
    gate = z * s1 if z is not None else torch.ones_like(x)
    total, S = residual + sc * y * gate, residual.abs() + sc.abs() * Y * gate.abs()
    n2, rstd2, N2 = norm(total, S)
    out = n2 * w2 + (zero if b2 is None else b2)
    res = dict(out=out, residual_out=total)
    bound = dict(out=K * U * top(N2 * w2.abs() + (zero if b2 is None else b2.abs())), residual_out=K * U * S)
    if dout is None:
        return res, bound
    dout = _d(dout)
    ds = _d(dsum) if dsum is not None else torch.zeros_like(x)

    def back(dy, w, n, rstd, DY, N):
        dn, DN = dy * w, DY * w.abs()
        d = dn - n * mean(dn * n) - (0 if is_rms_norm else mean(dn))
        return rstd * d, rstd * (DN + N * mean(DN * N) + mean(DN)) * (1 + mean(N * N))  # (the last factor: rstd's own error)

    dn2, D2 = back(dout, w2, n2, rstd2, dout.abs(), N2)
    d, D = ds + dn2, ds.abs() + D2
    dy, DY = d * sc * gate, D * sc.abs() * gate.abs()
    dx, DX = back(dy, w1, n1, rstd1, DY, N1)
    rows = tuple(range(x.dim() - 1))
    col = lambda v: v.sum(rows)
    res.update(dx=dx, dresidual=d, dnorm_weight=col(dy * n1), dnext_weight=col(dout * n2))
    bound.update(dx=K * U * top(DX), dresidual=K * U * top(D), dnorm_weight=K * U * col(top(DY) * N1),
                 dnext_weight=K * U * col(dout.abs() * N2))
    if z is not None:
        slope = s1 * (1 + z * (1 - s1))
        res["dz"], bound["dz"] = d * sc * y * slope, K * U * top(D * sc.abs() * Y * (s1 * (1 + z.abs() * (1 - s1))))
    if isinstance(scale, torch.Tensor):
        res["dscale"], bound["dscale"] = col(d * y * gate), K * U * col(top(D) * Y * gate.abs())
    if b1 is not None:
        res["dnorm_bias"], bound["dnorm_bias"] = col(dy), K * U * col(top(DY))
    if b2 is not None:
        res["dnext_bias"], bound["dnext_bias"] = col(dout), K * U * col(dout.abs())
    return res, bound


def within(name, got, ref, bound):
    """Asserts |got - ref| <= bound + half a step of got's type (relative, or of its smallest numbers)."""
    info = torch.finfo(got.dtype)
    tol = bound + ref.abs() * (info.eps / 2) * (1 + 2.0 ** -10) + info.smallest_normal * info.eps / 2 + 1e-30
    got = got.detach().double().cpu()
    assert got.shape == ref.shape, f"{name}: shape {tuple(got.shape)}, not {tuple(ref.shape)}"
    bad = ~((got - ref).abs() <= tol)
    if bool(bad.any()):
        at = tuple(int(v) for v in bad.nonzero()[0])
        raise AssertionError(f"{name}: {int(bad.sum())} of {bad.numel()} off, first at {at}: {float(got[at])} for {float(ref[at])}, "
                             f"allowed {float(tol[at]):.3e}; largest excess {float(((got - ref).abs() / tol).nan_to_num(9e9).max()):.2f}")
