"""Linear attention with a decay per head, on the HIP kernels: whole sequences with their gradients (`linear_attention_fn`)
and the step of one generated token (`linear_attention_state_update`), the counterparts of `mamba_chunk_scan_combined` and
`selective_state_update` for layers whose heads have keys and values of their own and forget at a fixed rate:

    S_t = exp(log_decay) * S_{t-1} + k_t v_t^T,    out_t = scale * q_t S_t

per head, with a state of headdim_k x headdim_v.  Keys and values may be shared by neighbouring heads.  The states and every sum
are held in fp32; operands of the matrix products are not, with q in 16 bits.  bf16: a block's scores and the state (initial states
too) are rounded to bf16, 8 bits, where outputs and gradients are formed from them (the scores of a sequence's last blocks, or of a
sequence of fewer than 96 positions, keep 16).  fp16: they keep 16 bits.  Rows that a state takes up keep
16 bits, and 24 where states are returned (the step: all of them).  fp32: nothing is rounded.

There is no CPU or PyTorch fallback: CPU tensors raise.  `linear_attention_ref` and `linear_attention_state_update_ref` state the
arithmetic in plain torch; no operator calls them.
"""
import torch

from mamba_amd import _lib

MAX_HEADDIM = 256


def _unit(t):
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _one_device(what, first, *others):
    for t in others:
        if t is not None and t.device != first.device:
            raise RuntimeError(f"{what}: all tensors must be on {first.device}, got one on {t.device}")


def _int32(t, low, high):
    """Bounds or row numbers in 32 bits; 64-bit ones are first taken to [low, high], so that none turns into another."""
    return (t if t.dtype == torch.int32 else t.clamp(low, high).to(torch.int32)).contiguous()


def _check_heads(what, q, k, v, lead):
    """Sizes (nheads, nkvheads, headdim_k, headdim_v) of q (*lead, nheads, headdim_k), k and v (*lead, nkvheads, ..)."""
    names = "(" + ", ".join(lead)
    if q.dim() != len(lead) + 2 or q.dtype not in _lib.DTYPE_CODE:
        raise RuntimeError(f"{what}: q must be {names}, nheads, headdim_k) in fp32, fp16 or bf16")
    for name, t in (("k", k), ("v", v)):
        if t.dim() != q.dim() or t.shape[:-2] != q.shape[:-2]:
            raise RuntimeError(f"{what}: {name} must be {names}, nkvheads, head size) beside q {tuple(q.shape)}, got {tuple(t.shape)}")
        if t.dtype not in _lib.DTYPE_CODE:
            raise RuntimeError(f"{what}: {name} must be fp32, fp16 or bf16")
    nheads, headdim_k = q.shape[-2:]
    nkv, headdim_v = v.shape[-2:]
    if k.shape[-1] != headdim_k:
        raise RuntimeError(f"{what}: q and k must have the same head size, got {headdim_k} and {k.shape[-1]}")
    if k.shape[-2] != nkv:
        raise RuntimeError(f"{what}: k and v must have the same number of heads, got {k.shape[-2]} and {nkv}")
    if nkv == 0 and nheads > 0 or nkv > 0 and nheads % nkv != 0:
        raise RuntimeError(f"{what}: the heads of k and v ({nkv}) must divide those of q ({nheads})")
    if not (1 <= headdim_k <= MAX_HEADDIM and 1 <= headdim_v <= MAX_HEADDIM):
        raise RuntimeError(f"{what}: head sizes of 1 to {MAX_HEADDIM} are served, got {headdim_k} and {headdim_v}")
    return nheads, nkv, headdim_k, headdim_v


def _check_decay(what, log_decay, nheads):
    if tuple(log_decay.shape) != (nheads,):
        raise RuntimeError(f"{what}: log_decay must be ({nheads},), got {tuple(log_decay.shape)}")
    if log_decay.dtype not in _lib.DTYPE_CODE:
        raise RuntimeError(f"{what}: log_decay must be fp32, fp16 or bf16")
    if torch.is_grad_enabled() and log_decay.requires_grad:
        raise RuntimeError(f"{what}: log_decay is a constant of the layer and takes no gradients: detach it "
                           "(mamba_chunk_scan_combined has gradients of its decays)")


def _check_scale(what, scale, headdim, most=3.4e38):
    scale = headdim ** -0.5 if scale is None else float(scale)
    if not abs(scale) <= most:
        raise ValueError(f"{what}: scale must be finite, of at most {most:g}, got {scale}")
    return scale


def _strides(p, **tensors):
    for name, t in tensors.items():
        for suffix, n in zip(("bs", "ls", "hs") if t.dim() == 4 else ("bs", "hs"), t.stride()):
            setattr(p, f"{name}_{suffix}", n)


def _params(q, k, v, log_decay, initial_states, cu_seqlens, scale):
    p = _lib.LinearAttnParams()
    p.batch, p.seqlen, p.nheads, p.headdim_k = q.shape
    p.nkvheads, p.headdim_v = v.shape[2:]
    p.nseq = cu_seqlens.shape[0] - 1 if cu_seqlens is not None else 0
    p.dtype, p.scale = _lib.DTYPE_CODE[q.dtype], scale
    p.q, p.k, p.v, p.log_decay = q.data_ptr(), k.data_ptr(), v.data_ptr(), log_decay.data_ptr()
    p.initial_states, p.cu_seqlens = _lib.ptr(initial_states), _lib.ptr(cu_seqlens)
    _strides(p, q=q, k=k, v=v)
    return p


def _workspace(n, what, device):
    if n < 0:
        _lib.check(int(n), what)
    return torch.empty(n, dtype=torch.uint8, device=device) if n > 0 else None


class LinearAttentionFn(torch.autograd.Function):
    """Arguments as `linear_attention_fn` has checked and converted them; returns (out, final_states or None)."""

    @staticmethod
    def forward(ctx, q, k, v, log_decay, initial_states, cu_seqlens, scale, return_final_states):
        q, k, v = _unit(q), _unit(k), _unit(v)
        batch, seqlen, nheads, headdim_k = q.shape
        headdim_v = v.shape[-1]
        seqs = cu_seqlens.shape[0] - 1 if cu_seqlens is not None else batch
        out = torch.empty(batch, seqlen, nheads, headdim_v, dtype=q.dtype, device=q.device)
        final = None
        if return_final_states:
            final = torch.empty(seqs, nheads, headdim_k, headdim_v, dtype=torch.float32, device=q.device)
        if out.numel() > 0:
            with torch.cuda.device(q.device):
                lib = _lib.load()
                p = _params(q, k, v, log_decay, initial_states, cu_seqlens, scale)
                p.out, p.final_states = out.data_ptr(), _lib.ptr(final)
                _strides(p, out=out)
                ws = _workspace(lib.linear_attn_fwd_ws_bytes(p), "linear_attn_fwd_ws_bytes", q.device)
                p.ws = _lib.ptr(ws)
                _lib.check(lib.linear_attn_fwd(p, _lib.current_stream(q.device)), "linear_attn_fwd")
        elif final is not None:  # no position: the states are what they were
            final.copy_(initial_states) if initial_states is not None else final.zero_()
        ctx.save_for_backward(q, k, v, log_decay, initial_states, cu_seqlens)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        return out, final

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout, dfinal):
        q, k, v, log_decay, initial_states, cu_seqlens = ctx.saved_tensors
        if dout is None and dfinal is None:
            return (None,) * 8
        if dout is None:
            dout = torch.zeros(*q.shape[:3], v.shape[-1], dtype=q.dtype, device=q.device)
        dout = _unit(dout)
        dfinal = dfinal.contiguous() if dfinal is not None else None
        dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v))
        dinitial = torch.empty_like(initial_states) if initial_states is not None else None
        if q.numel() == 0:
            if dinitial is not None:
                dinitial.copy_(dfinal) if dfinal is not None else dinitial.zero_()
            return dq, dk.zero_(), dv.zero_(), None, dinitial, None, None, None
        with torch.cuda.device(q.device):
            lib = _lib.load()
            p = _params(q, k, v, log_decay, initial_states, cu_seqlens, ctx.scale)
            p.dout, p.dfinal_states, p.dinitial_states = dout.data_ptr(), _lib.ptr(dfinal), _lib.ptr(dinitial)
            p.dq, p.dk, p.dv = dq.data_ptr(), dk.data_ptr(), dv.data_ptr()
            _strides(p, dout=dout, dq=dq, dk=dk, dv=dv)
            ws = _workspace(lib.linear_attn_bwd_ws_bytes(p), "linear_attn_bwd_ws_bytes", q.device)
            p.ws = _lib.ptr(ws)
            _lib.check(lib.linear_attn_bwd(p, _lib.current_stream(q.device)), "linear_attn_bwd")
        return dq, dk, dv, None, dinitial, None, None, None


def linear_attention_fn(q, k, v, log_decay, scale=None, initial_states=None, cu_seqlens=None, return_final_states=False):
    """Linear attention over whole sequences, differentiable in q, k, v and initial_states.

    Argument:
        q: (batch, seqlen, nheads, headdim_k) in fp32, fp16 or bf16, any strides; rows with unit stride along the head, such as
            slices of one projection's output, are read as they lie
        k: (batch, seqlen, nkvheads, headdim_k), v: (batch, seqlen, nkvheads, headdim_v), taken in q's dtype; head h of q has head
            h // (nheads // nkvheads) of k and v.  Head sizes of 1 to 256
        log_decay: (nheads,), at most 0, a constant of the layer (no gradient): a state keeps exp(log_decay) of itself from
            position to position.  Minus infinity forgets everything; values above 0 count as 0
        scale: a number, headdim_k ** -0.5 unless given
        initial_states: (batch, nheads, headdim_k, headdim_v), or (number of sequences, ..) with cu_seqlens; None: zeros
        cu_seqlens: (number of sequences + 1,) int32, not decreasing: q is one row (batch 1) of packed sequences, sequence n at
            positions cu_seqlens[n] .. cu_seqlens[n + 1] - 1.  A sequence may be empty (its final state is its initial one).
            Positions outside of all of them, padding behind the last for instance, do not count, whatever they hold: their
            outputs and gradients are 0.
    Return:
        out: (batch, seqlen, nheads, headdim_v) in q's dtype, and with return_final_states also the states after the last
        positions, fp32, of initial_states' shape

    Products are formed in blocks of 32 positions (fp32: 16) of a sequence.  An infinity or a NaN in k or v at one position leaves no finite
    numbers in what it has part in, infinities or NaN: the states and the outputs from there on, and those of the positions in its block that
    lie before it.  Other sequences and heads never see it.
    """
    ext = _lib.torch_ext()
    if ext is not None:
        # the same checks, node and launches in C++ (csrc/torch_attention.cpp); None = a case for the code below
        r = ext.linear_attention(q, k, v, log_decay, scale, initial_states, cu_seqlens, bool(return_final_states))
        if r is not None:
            return r
    what = "linear_attention"
    nheads, nkv, headdim_k, headdim_v = _check_heads(what, q, k, v, ("batch", "seqlen"))
    batch, seqlen = q.shape[:2]
    if batch > 2 ** 31 - 1 or seqlen > 2 ** 30 or nheads > 2 ** 22:
        raise RuntimeError(f"{what}: rows of up to 2^30 positions with up to 2^22 heads are served, got {batch} of {seqlen} with {nheads}")
    _check_decay(what, log_decay, nheads)
    scale = _check_scale(what, scale, headdim_k)
    seqs = batch
    if cu_seqlens is not None:
        if cu_seqlens.dim() != 1 or cu_seqlens.shape[0] < 2 or cu_seqlens.dtype not in (torch.int32, torch.int64):
            raise RuntimeError(f"{what}: cu_seqlens must be (number of sequences + 1,) int32")
        if batch != 1:
            raise RuntimeError(f"{what}: with cu_seqlens q must be one row of packed sequences (batch 1)")
        seqs = cu_seqlens.shape[0] - 1
    if initial_states is not None and tuple(initial_states.shape) != (seqs, nheads, headdim_k, headdim_v):
        raise RuntimeError(f"{what}: initial_states must be ({seqs}, {nheads}, {headdim_k}, {headdim_v}), got {tuple(initial_states.shape)}")
    _lib.refuse_tangents(what, q, k, v, log_decay, initial_states)
    _lib.require_gpu(q, k, v, log_decay, initial_states, cu_seqlens)
    _one_device(what, q, k, v, log_decay, initial_states, cu_seqlens)
    if cu_seqlens is not None:
        cu_seqlens = _int32(cu_seqlens, 0, seqlen)
    if initial_states is not None:
        initial_states = initial_states.float().contiguous()
    out, final = LinearAttentionFn.apply(q, k.to(q.dtype), v.to(q.dtype), log_decay.detach().float().contiguous(), initial_states,
                                         cu_seqlens, scale, bool(return_final_states))
    return (out, final) if return_final_states else out


class LinearAttentionStateUpdateFn(torch.autograd.Function):
    """Arguments as `linear_attention_state_update` has checked and converted them.  The step has no gradients: as a node it
    lets the transforms and traces of torch see the call, and raises where a backward pass comes to it."""

    @staticmethod
    def forward(ctx, state, q, k, v, log_decay, state_batch_indices, scale):
        batch, nheads, headdim_k = q.shape
        nkv, headdim_v = v.shape[1:]
        out = torch.empty(batch, nheads, headdim_v, dtype=q.dtype, device=q.device)
        if out.numel() == 0:
            return out
        if state.shape[0] == 0:  # a pool without rows: every entry is a padding entry
            return out.zero_()
        q, k, v = _unit(q), _unit(k), _unit(v)
        p = _lib.LinearAttnStepParams()
        p.batch, p.nheads, p.nkvheads, p.headdim_k, p.headdim_v, p.state_rows = batch, nheads, nkv, headdim_k, headdim_v, state.shape[0]
        p.dtype, p.state_dtype, p.scale = _lib.DTYPE_CODE[q.dtype], _lib.DTYPE_CODE[state.dtype], scale
        p.state, p.q, p.k, p.v, p.log_decay, p.out = (t.data_ptr() for t in (state, q, k, v, log_decay, out))
        p.state_batch_indices = _lib.ptr(state_batch_indices)
        p.state_rs = state.stride(0)
        _strides(p, q=q, k=k, v=v, out=out)
        with torch.cuda.device(q.device):
            _lib.check(_lib.load().linear_attn_state_update(p, _lib.current_stream(q.device)), "linear_attn_state_update")
        if not state.is_inference():
            torch.autograd.graph.increment_version(state)  # a graph that has saved it has to notice
        return out

    @staticmethod
    def backward(ctx, dout):
        raise RuntimeError("linear_attention_state_update has no gradients; linear_attention_fn over one position has")


def linear_attention_state_update(state, q, k, v, log_decay, scale=None, state_batch_indices=None):
    """One token of the same recurrence: `state` is updated in place.  It is made for generating and has no gradients: a
    backward pass through `out` raises, and so does a call with a state that wants a gradient.

    Argument:
        state: (rows, nheads, headdim_k, headdim_v) in fp32, fp16 or bf16, each row contiguous
        q: (batch, nheads, headdim_k) in fp32, fp16 or bf16; k: (batch, nkvheads, headdim_k), v: (batch, nkvheads, headdim_v), taken
            in q's dtype
        log_decay: (nheads,), scale: as in linear_attention_fn
        state_batch_indices: (batch,) int32, row of `state` per batch entry, each row at most once; an index outside
            [0, rows) is a padding entry (state untouched, out = 0).  Without it row b belongs to entry b.
    Return:
        out: (batch, nheads, headdim_v) in q's dtype, scale * q S of the new states
    """
    ext = _lib.torch_ext()
    if ext is not None:
        out = ext.linear_attention_state_update(state, q, k, v, log_decay, scale, state_batch_indices)
        if out is not None:
            return out
    what = "linear_attention_state_update"
    nheads, nkv, headdim_k, headdim_v = _check_heads(what, q, k, v, ("batch",))
    batch = q.shape[0]
    if state.dim() != 4 or tuple(state.shape[1:]) != (nheads, headdim_k, headdim_v):
        raise RuntimeError(f"{what}: state must be (rows, {nheads}, {headdim_k}, {headdim_v}), got {tuple(state.shape)}")
    if state.dtype not in _lib.DTYPE_CODE:
        raise RuntimeError(f"{what}: state must be fp32, fp16 or bf16")
    if max(batch, state.shape[0]) > 2 ** 31 - 1 or nheads > 65535:
        raise RuntimeError(f"{what}: up to 65535 heads and 2^31 - 1 rows are served")
    if state_batch_indices is None and state.shape[0] < batch:
        raise RuntimeError(f"{what}: state has {state.shape[0]} rows for a batch of {batch} and no state_batch_indices")
    if state.shape[0] > 0 and not state[0].is_contiguous():
        raise RuntimeError(f"{what}: every row of state must be contiguous (it is updated in place)")
    if state.shape[0] > 1 and state.stride(0) < nheads * headdim_k * headdim_v:
        raise RuntimeError(f"{what}: state's rows must not overlap (they are updated in place)")
    _check_decay(what, log_decay, nheads)
    scale = _check_scale(what, scale, headdim_k)
    if state_batch_indices is not None:
        if tuple(state_batch_indices.shape) != (batch,) or state_batch_indices.dtype not in (torch.int32, torch.int64):
            raise RuntimeError(f"{what}: state_batch_indices must be ({batch},) int32")
    if torch.is_grad_enabled() and state.requires_grad:
        raise RuntimeError(f"{what}: state is updated in place and takes no gradients: detach it, or call under torch.no_grad()")
    _lib.refuse_tangents(what, state, q, k, v, log_decay)
    _lib.require_gpu(state, q, k, v, log_decay, state_batch_indices)
    _one_device(what, q, state, k, v, log_decay, state_batch_indices)
    if state_batch_indices is not None:
        state_batch_indices = _int32(state_batch_indices, -1, 2 ** 31 - 1)
    return LinearAttentionStateUpdateFn.apply(state, q, k.to(q.dtype), v.to(q.dtype), log_decay.detach().float().contiguous(),
                                              state_batch_indices, scale)


def linear_attention_state_update_ref(state, q, k, v, log_decay, scale=None):
    """One step from plain torch operators, in place on `state`; row b of the state belongs to entry b."""
    group = q.shape[1] // k.shape[1]
    k, v = k.float().repeat_interleave(group, 1), v.float().repeat_interleave(group, 1)
    h = torch.exp(log_decay.float())[:, None, None] * state.float() + k[..., None] * v[..., None, :]
    state.copy_(h)
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    return (scale * (q.float()[..., None] * h).sum(-2)).to(q.dtype)


def linear_attention_ref(q, k, v, log_decay, scale=None, initial_states=None, return_final_states=False):
    """The recurrence position by position from plain torch operators, on whatever device the inputs live on."""
    batch, seqlen, nheads, headdim_k = q.shape
    group = nheads // k.shape[2]
    k, v = k.float().repeat_interleave(group, 2), v.float().repeat_interleave(group, 2)
    f = torch.exp(log_decay.float())[:, None, None]
    scale = headdim_k ** -0.5 if scale is None else scale
    if initial_states is None:
        state = torch.zeros(batch, nheads, headdim_k, v.shape[-1], device=q.device)
    else:
        state = initial_states.float()
    out = []
    for t in range(seqlen):
        state = f * state + k[:, t, :, :, None] * v[:, t, :, None, :]
        out.append(scale * (q[:, t].float()[..., None] * state).sum(-2))
    out = torch.stack(out, 1).to(q.dtype)
    return (out, state) if return_final_states else out
