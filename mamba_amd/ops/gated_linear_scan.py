"""Gated linear recurrence with one state per channel, on the HIP kernels: the scan of a sequence with its gradients
(`gated_linear_scan_fn`) and the step of one generated token (`gated_linear_state_update`), the counterparts of
`selective_scan_fn` and `selective_state_update` for blocks whose recurrence is

    r_t = sigmoid(gate_a_t),  i_t = sigmoid(gate_x_t),  log a_t = -rate * softplus(decay) * r_t
    h_t = a_t * h_{t-1} + sqrt(1 - a_t^2) * i_t * x_t

per channel.  The first position of a sequence is like any other: what enters there is scaled by sqrt(1 - a_t^2) too (there is no
form with the factor 1 in its place).  The states, the decays and every sum are held in fp32.  There is no CPU or PyTorch fallback: CPU tensors
raise.  `gated_linear_scan_ref` and `gated_linear_state_update_ref` state the arithmetic in plain torch; no operator
calls them.
"""
import torch
import torch.nn.functional as F

from mamba_amd import _lib


def _unit(t):
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _check_decay(what, decay, dim, device):
    if tuple(decay.shape) != (dim,):
        raise RuntimeError(f"{what}: decay must be ({dim},), got {tuple(decay.shape)}")
    if decay.dtype not in _lib.DTYPE_CODE:
        raise RuntimeError(f"{what}: decay must be fp32, fp16 or bf16")


def _check_rate(what, rate):
    rate = float(rate)
    if not 0.0 <= rate < float("inf"):
        raise ValueError(f"{what}: rate must be finite and not negative, got {rate}")
    return rate


def _one_device(what, first, *others):
    for t in others:
        if t is not None and t.device != first.device:
            raise RuntimeError(f"{what}: all tensors must be on {first.device}, got one on {t.device}")


def _check_sizes(what, *sizes):
    if max(sizes) > 2 ** 31 - 1:
        raise RuntimeError(f"{what}: sizes are counted in 32 bits, got {max(sizes)}")


def _int32(t, low, high):
    """Bounds or row numbers in 32 bits; 64-bit ones are first taken to [low, high], so that none turns into another."""
    return (t if t.dtype == torch.int32 else t.clamp(low, high).to(torch.int32)).contiguous()


def _params(x, gate_a, gate_x, decay, initial_states, cu_seqlens, rate):
    p = _lib.GatedScanParams()
    p.batch, p.seqlen, p.dim = x.shape
    p.nseq = cu_seqlens.shape[0] - 1 if cu_seqlens is not None else 0
    p.dtype, p.decay_dtype, p.rate = _lib.DTYPE_CODE[x.dtype], _lib.DTYPE_CODE[decay.dtype], rate
    p.x, p.gate_a, p.gate_x, p.decay = x.data_ptr(), gate_a.data_ptr(), gate_x.data_ptr(), decay.data_ptr()
    p.initial_states, p.cu_seqlens = _lib.ptr(initial_states), _lib.ptr(cu_seqlens)
    p.x_bs, p.x_ls = x.stride(0), x.stride(1)
    p.gate_a_bs, p.gate_a_ls = gate_a.stride(0), gate_a.stride(1)
    p.gate_x_bs, p.gate_x_ls = gate_x.stride(0), gate_x.stride(1)
    return p


def _bytes(n, what, device):
    if n < 0:
        _lib.check(int(n), what)
    return torch.empty(n, dtype=torch.uint8, device=device)


class GatedLinearScanFn(torch.autograd.Function):
    """Arguments as `gated_linear_scan_fn` has checked and converted them; returns (out, final_states or None)."""

    @staticmethod
    def forward(ctx, x, gate_a, gate_x, decay, initial_states, cu_seqlens, rate, return_final_states):
        x, gate_a, gate_x = _unit(x), _unit(gate_a), _unit(gate_x)
        batch, seqlen, dim = x.shape
        seqs = cu_seqlens.shape[0] - 1 if cu_seqlens is not None else batch
        out = torch.empty(batch, seqlen, dim, dtype=x.dtype, device=x.device)
        final = torch.empty(seqs, dim, dtype=torch.float32, device=x.device) if return_final_states else None
        ckpt = None
        if out.numel() > 0:
            with torch.cuda.device(x.device):
                lib = _lib.load()
                p = _params(x, gate_a, gate_x, decay, initial_states, cu_seqlens, rate)
                ckpt = _bytes(lib.gated_scan_ckpt_bytes(p), "gated_scan_ckpt_bytes", x.device)
                p.ckpt, p.out, p.final_states = ckpt.data_ptr(), out.data_ptr(), _lib.ptr(final)
                p.out_bs, p.out_ls = out.stride(0), out.stride(1)
                _lib.check(lib.gated_scan_fwd(p, _lib.current_stream(x.device)), "gated_scan_fwd")
        elif final is not None:  # no position: the states are what they were
            final.copy_(initial_states) if initial_states is not None else final.zero_()
        ctx.save_for_backward(x, gate_a, gate_x, decay, initial_states, cu_seqlens, ckpt)
        ctx.rate = rate
        ctx.set_materialize_grads(False)
        return out, final

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout, dfinal):
        x, gate_a, gate_x, decay, initial_states, cu_seqlens, ckpt = ctx.saved_tensors
        if dout is None and dfinal is None:
            return (None,) * 8
        new = lambda: torch.empty(x.shape, dtype=x.dtype, device=x.device)
        if dout is None:
            dout = torch.zeros(x.shape, dtype=x.dtype, device=x.device)
        dout = _unit(dout)
        dfinal = dfinal.contiguous() if dfinal is not None else None
        dx, dgate_a, dgate_x = new(), new(), new()
        dinitial = torch.empty_like(initial_states) if initial_states is not None else None
        if x.numel() == 0:
            if dinitial is not None:
                dinitial.copy_(dfinal) if dfinal is not None else dinitial.zero_()
            return dx, dgate_a, dgate_x, torch.zeros_like(decay), dinitial, None, None, None
        ddecay = torch.empty_like(decay)
        with torch.cuda.device(x.device):
            lib = _lib.load()
            p = _params(x, gate_a, gate_x, decay, initial_states, cu_seqlens, ctx.rate)
            ws = _bytes(lib.gated_scan_bwd_ws_bytes(p), "gated_scan_bwd_ws_bytes", x.device)
            p.ckpt, p.ws = ckpt.data_ptr(), ws.data_ptr()
            p.dout, p.dfinal_states = dout.data_ptr(), _lib.ptr(dfinal)
            p.dx, p.dgate_a, p.dgate_x = dx.data_ptr(), dgate_a.data_ptr(), dgate_x.data_ptr()
            p.ddecay, p.dinitial_states = ddecay.data_ptr(), _lib.ptr(dinitial)
            p.dout_bs, p.dout_ls = dout.stride(0), dout.stride(1)
            p.dx_bs, p.dx_ls = p.dgate_a_bs, p.dgate_a_ls = p.dgate_x_bs, p.dgate_x_ls = dx.stride(0), dx.stride(1)
            _lib.check(lib.gated_scan_bwd(p, _lib.current_stream(x.device)), "gated_scan_bwd")
        return dx, dgate_a, dgate_x, ddecay, dinitial, None, None, None


def gated_linear_scan_fn(x, gate_a, gate_x, decay, rate=8.0, initial_states=None, cu_seqlens=None,
                         return_final_states=False):
    """The recurrence over whole sequences, differentiable in every tensor but cu_seqlens.

    Argument:
        x, gate_a, gate_x: (batch, seqlen, dim) in fp32, fp16 or bf16 (the gates are taken in x's dtype), any strides;
            rows with unit channel stride, such as slices of one projection's output, are read as they lie
        decay: (dim,) in any of the three dtypes
        rate: the recurrence's constant, a number >= 0
        initial_states: (batch, dim), or (number of sequences, dim) with cu_seqlens; None: zeros
        cu_seqlens: (number of sequences + 1,) int32, not decreasing: x is one row (batch 1) of packed sequences,
            sequence q at positions cu_seqlens[q] .. cu_seqlens[q + 1] - 1.  A sequence may be empty (its final state is
            its initial one).  Positions outside of all of them, padding behind the last for instance, do not count,
            whatever they hold: their outputs and gradients are 0.
    Return:
        out: (batch, seqlen, dim) in x's dtype, and with return_final_states also the states after the last positions,
        fp32, of initial_states' shape
    """
    ext = _lib.torch_ext()
    if ext is not None:
        # the same checks, node and launches in C++ (csrc/torch_gated.cpp); None = a case for the code below
        r = ext.gated_linear_scan(x, gate_a, gate_x, decay, rate, initial_states, cu_seqlens, bool(return_final_states))
        if r is not None:
            return r
    what = "gated_linear_scan"
    if x.dim() != 3 or x.dtype not in _lib.DTYPE_CODE:
        raise RuntimeError(f"{what}: x must be (batch, seqlen, dim) in fp32, fp16 or bf16")
    batch, seqlen, dim = x.shape
    _check_sizes(what, batch, seqlen, dim)
    for name, t in (("gate_a", gate_a), ("gate_x", gate_x)):
        if t.shape != x.shape:
            raise RuntimeError(f"{what}: {name} must have x's shape {tuple(x.shape)}, got {tuple(t.shape)}")
    _check_decay(what, decay, dim, x.device)
    rate = _check_rate(what, rate)
    seqs = batch
    if cu_seqlens is not None:
        if cu_seqlens.dim() != 1 or cu_seqlens.shape[0] < 2 or cu_seqlens.dtype not in (torch.int32, torch.int64):
            raise RuntimeError(f"{what}: cu_seqlens must be (number of sequences + 1,) int32")
        if batch != 1:
            raise RuntimeError(f"{what}: with cu_seqlens x must be one row of packed sequences (batch 1)")
        seqs = cu_seqlens.shape[0] - 1
    if initial_states is not None and tuple(initial_states.shape) != (seqs, dim):
        raise RuntimeError(f"{what}: initial_states must be ({seqs}, {dim}), got {tuple(initial_states.shape)}")
    _lib.require_gpu(x, gate_a, gate_x, decay, initial_states, cu_seqlens)
    _one_device(what, x, gate_a, gate_x, decay, initial_states, cu_seqlens)
    if cu_seqlens is not None:
        cu_seqlens = _int32(cu_seqlens, 0, seqlen)
    if initial_states is not None:
        initial_states = initial_states.float().contiguous()
    out, final = GatedLinearScanFn.apply(x, gate_a.to(x.dtype), gate_x.to(x.dtype), decay.contiguous(), initial_states,
                                         cu_seqlens, rate, bool(return_final_states))
    return (out, final) if return_final_states else out


class GatedLinearStateUpdateFn(torch.autograd.Function):
    """Arguments as `gated_linear_state_update` has checked and converted them.  The step has no gradients: as a node it lets
    the transforms and traces of torch see the call, and raises where a backward pass comes to it."""

    @staticmethod
    def forward(ctx, state, x, gate_a, gate_x, decay, state_batch_indices, rate):
        batch, dim = x.shape
        out = torch.empty(batch, dim, dtype=x.dtype, device=x.device)
        if out.numel() == 0:
            return out
        if state.shape[0] == 0:  # a pool without rows: every entry is a padding entry
            return out.zero_()
        x, gate_a, gate_x = _unit(x), _unit(gate_a), _unit(gate_x)
        p = _lib.GatedStepParams()
        p.batch, p.dim, p.state_rows = batch, dim, state.shape[0]
        p.dtype, p.state_dtype, p.decay_dtype = (_lib.DTYPE_CODE[t.dtype] for t in (x, state, decay))
        p.rate = rate
        p.state, p.x, p.gate_a, p.gate_x, p.decay, p.out = (t.data_ptr() for t in (state, x, gate_a, gate_x, decay, out))
        p.state_batch_indices = _lib.ptr(state_batch_indices)
        p.state_rs, p.x_rs, p.gate_a_rs, p.gate_x_rs, p.out_rs = (t.stride(0) for t in (state, x, gate_a, gate_x, out))
        with torch.cuda.device(x.device):
            _lib.check(_lib.load().gated_state_update(p, _lib.current_stream(x.device)), "gated_state_update")
        if not state.is_inference():
            torch.autograd.graph.increment_version(state)  # a graph that has saved it has to notice
        return out

    @staticmethod
    def backward(ctx, dout):
        raise RuntimeError("gated_linear_state_update has no gradients; gated_linear_scan_fn over one position has")


def gated_linear_state_update(state, x, gate_a, gate_x, decay, rate=8.0, state_batch_indices=None):
    """One token of the same recurrence: `state` is updated in place.  It is made for generating and has no gradients: a
    backward pass through `out` raises, and so does a call with a state that wants a gradient.

    Argument:
        state: (rows, dim) in fp32, fp16 or bf16, unit channel stride
        x, gate_a, gate_x: (batch, dim) in fp32, fp16 or bf16 (the gates are taken in x's dtype)
        decay: (dim,) in any of the three dtypes; rate: a number >= 0
        state_batch_indices: (batch,) int32, row of `state` per batch entry, each row at most once; an index outside
            [0, rows) is a padding entry (state untouched, out = 0).  Without it row b belongs to entry b.
    Return:
        out: (batch, dim) in x's dtype, the new states
    """
    ext = _lib.torch_ext()
    if ext is not None:
        out = ext.gated_linear_state_update(state, x, gate_a, gate_x, decay, rate, state_batch_indices)
        if out is not None:
            return out
    what = "gated_linear_state_update"
    if x.dim() != 2 or state.dim() != 2 or state.shape[1] != x.shape[1]:
        raise RuntimeError(f"{what}: state must be (rows, dim) and x (batch, dim)")
    batch, dim = x.shape
    _check_sizes(what, batch, dim, state.shape[0])
    if dim > 2 ** 30:
        raise RuntimeError(f"{what}: rows of at most 2^30 channels are served, got {dim}")
    if state_batch_indices is None and state.shape[0] < batch:
        raise RuntimeError(f"{what}: state has {state.shape[0]} rows for a batch of {batch} and no state_batch_indices")
    for name, t in (("gate_a", gate_a), ("gate_x", gate_x)):
        if t.shape != x.shape:
            raise RuntimeError(f"{what}: {name} must have x's shape {tuple(x.shape)}, got {tuple(t.shape)}")
    if x.dtype not in _lib.DTYPE_CODE or state.dtype not in _lib.DTYPE_CODE:
        raise RuntimeError(f"{what}: x and state must be fp32, fp16 or bf16")
    if state.stride(1) != 1 and dim > 1:
        raise RuntimeError(f"{what}: state must have unit channel stride (it is updated in place)")
    if state.stride(0) < dim and state.shape[0] > 1:
        raise RuntimeError(f"{what}: state's rows must not overlap (they are updated in place)")
    _check_decay(what, decay, dim, x.device)
    rate = _check_rate(what, rate)
    if state_batch_indices is not None:
        if tuple(state_batch_indices.shape) != (batch,) or state_batch_indices.dtype not in (torch.int32, torch.int64):
            raise RuntimeError(f"{what}: state_batch_indices must be ({batch},) int32")
    if torch.is_grad_enabled() and state.requires_grad:
        raise RuntimeError(f"{what}: state is updated in place and takes no gradients: detach it, or call under torch.no_grad()")
    _lib.refuse_tangents(what, state, x, gate_a, gate_x, decay)
    _lib.require_gpu(state, x, gate_a, gate_x, decay, state_batch_indices)
    _one_device(what, x, state, gate_a, gate_x, decay, state_batch_indices)
    if state_batch_indices is not None:
        state_batch_indices = _int32(state_batch_indices, -1, 2 ** 31 - 1)
    return GatedLinearStateUpdateFn.apply(state, x, gate_a.to(x.dtype), gate_x.to(x.dtype), decay.contiguous(), state_batch_indices,
                                          rate)


def gated_linear_state_update_ref(state, x, gate_a, gate_x, decay, rate=8.0):
    """One step from plain torch operators, in place on `state`; row b of the state belongs to entry b."""
    log_a = -rate * F.softplus(decay.float()) * torch.sigmoid(gate_a.float())
    m = torch.sqrt(-torch.expm1(2 * log_a))
    h = torch.exp(log_a) * state.float() + m * torch.sigmoid(gate_x.float()) * x.float()
    state.copy_(h)
    return h.to(x.dtype)


def gated_linear_scan_ref(x, gate_a, gate_x, decay, rate=8.0, initial_states=None, return_final_states=False):
    """The recurrence position by position from plain torch operators, on whatever device the inputs live on."""
    log_a = -rate * F.softplus(decay.float()) * torch.sigmoid(gate_a.float())
    a, b = torch.exp(log_a), torch.sqrt(-torch.expm1(2 * log_a)) * torch.sigmoid(gate_x.float()) * x.float()
    h = torch.zeros_like(b[:, 0]) if initial_states is None else initial_states.float()
    out = []
    for t in range(x.shape[1]):
        h = a[:, t] * h + b[:, t]
        out.append(h)
    out = torch.stack(out, 1).to(x.dtype)
    return (out, h) if return_final_states else out
