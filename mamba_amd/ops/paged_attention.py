"""Attention of one generated token over a paged cache of keys and values, on the HIP kernels (`paged_attention_update`): what
`selective_state_update` and `causal_conv1d_update` are for the recurrent layers of a hybrid model, for its attention layers.
Scores and sums are formed in fp32; the weights are rounded to q's type for the product with the values (their sum is not).
There is no CPU or PyTorch fallback: CPU tensors raise.  `paged_attention_update_ref` states the arithmetic in plain torch; no
operator calls it.
"""
import torch

from mamba_amd import _lib
from mamba_amd.ops.linear_attention import _check_heads, _check_scale, _int32, _one_device, _strides, _unit


def _rows_apart(t):
    """Whether no two elements of a tensor lie in one place."""
    if t.numel() == 0:
        return True
    end = 1
    for stride, size in sorted((st, n) for st, n in zip(t.stride(), t.shape) if n > 1):
        if stride < end:
            return False
        end = stride * (size - 1) + end
    return True


class PagedAttentionUpdateFn(torch.autograd.Function):
    """Arguments as `paged_attention_update` has checked and converted them.  It has no gradients: as a node it lets the
    transforms and traces of torch see the call, and raises where a backward pass comes to it."""

    @staticmethod
    def forward(ctx, q, k, v, k_cache, v_cache, block_table, cache_seqlens, scale, window):
        batch, nheads, headdim_k = q.shape
        num_pages, page_size, nkv, headdim_v = v_cache.shape
        out = torch.empty(batch, nheads, headdim_v, dtype=q.dtype, device=q.device)
        if out.numel() == 0:
            return out
        q = _unit(q)
        p = _lib.PagedAttnParams()
        p.batch, p.nheads, p.nkvheads, p.headdim_k, p.headdim_v = batch, nheads, nkv, headdim_k, headdim_v
        p.num_pages, p.page_size, p.max_pages, p.window = num_pages, page_size, block_table.shape[1], window
        p.dtype, p.scale = _lib.DTYPE_CODE[q.dtype], scale
        if k is not None:
            k, v = _unit(k), _unit(v)
            p.k, p.v = k.data_ptr(), v.data_ptr()
            _strides(p, k=k, v=v)
        p.q, p.k_cache, p.v_cache, p.block_table, p.cache_seqlens, p.out = (
            t.data_ptr() for t in (q, k_cache, v_cache, block_table, cache_seqlens, out))
        _strides(p, q=q, out=out)
        p.kc_ps, p.kc_ls, p.kc_hs = k_cache.stride()[:3]
        p.vc_ps, p.vc_ls, p.vc_hs = v_cache.stride()[:3]
        p.table_bs = block_table.stride(0)
        with torch.cuda.device(q.device):
            lib = _lib.load()
            p.nsplit = lib.paged_attn_parts(p)
            if p.nsplit < 0:
                _lib.check(p.nsplit, "paged_attn_parts")
            n = lib.paged_attn_ws_bytes(p)
            ws = torch.empty(n, dtype=torch.uint8, device=q.device) if n > 0 else None
            p.ws = _lib.ptr(ws)
            _lib.check(lib.paged_attn_update(p, _lib.current_stream(q.device)), "paged_attn_update")
        if k is not None:
            for t in (k_cache, v_cache):
                if not t.is_inference():
                    torch.autograd.graph.increment_version(t)  # a graph that has saved it has to notice
        return out

    @staticmethod
    def backward(ctx, dout):
        raise RuntimeError("paged_attention_update has no gradients: it is made for generating")


def paged_attention_update(q, k, v, k_cache, v_cache, block_table, cache_seqlens, scale=None, window=None):
    """Softmax attention of one new token per sequence over its cache, the token's key and value appended to the cache in place.
    It is made for generating and has no gradients: a backward pass through `out` raises.

    Argument:
        q: (batch, nheads, headdim_k) in fp32, fp16 or bf16
        k: (batch, nkvheads, headdim_k), v: (batch, nkvheads, headdim_v), the new token's, taken in q's dtype; head h of q has head
            h // (nheads // nkvheads) of them.  Both None: the cache is read as it is, the sequence ends with it.  Head sizes of 1 to 256
        k_cache: (number of pages, page size, nkvheads, headdim_k), v_cache: (number of pages, page size, nkvheads, headdim_v), in
            q's dtype, unit stride along the head, any other strides (other orders of the first three axes, say)
        block_table: (batch, most pages of a sequence) int32: position p of sequence b lies in page block_table[b, p // page size] at
            p % page size.  Sequences may share pages that none of them writes.  Entries behind a sequence's last page are not used; a
            page outside of [0, number of pages) has no positions, and a new token whose page is one is not written (it still counts)
        cache_seqlens: (batch,) int32, positions in the cache before the call: the new token is position cache_seqlens[b].  A negative
            number is a padding entry (nothing written, out = 0); so is an entry without positions.  A number beyond the table's
            positions counts as theirs
        scale: a number of at most 2e38 in size, headdim_k ** -0.5 unless given.  Scores beyond 2.3e38 are infinities
        window: only the last `window` positions, the new one among them, count; None: all
    Return:
        out: (batch, nheads, headdim_v) in q's dtype
    """
    ext = _lib.torch_ext()
    if ext is not None:
        out = ext.paged_attention_update(q, k, v, k_cache, v_cache, block_table, cache_seqlens, scale, window)
        if out is not None:
            return out
    what = "paged_attention_update"
    if (k is None) != (v is None):
        raise RuntimeError(f"{what}: k and v come together or not at all")
    for name, t in (("k_cache", k_cache), ("v_cache", v_cache)):
        if t.dim() != 4 or t.dtype != q.dtype:
            raise RuntimeError(f"{what}: {name} must be (pages, page size, nkvheads, head size) in q's dtype")
    if k_cache.shape[:3] != v_cache.shape[:3]:
        raise RuntimeError(f"{what}: k_cache and v_cache must have the same pages and heads, got {tuple(k_cache.shape)} and {tuple(v_cache.shape)}")
    if k is None:
        token = lambda t: torch.empty(*q.shape[:1], *t.shape[2:], dtype=t.dtype, device="meta")
        nheads, nkv, headdim_k, headdim_v = _check_heads(what, q, token(k_cache), token(v_cache), ("batch",))
    else:
        nheads, nkv, headdim_k, headdim_v = _check_heads(what, q, k, v, ("batch",))
        if tuple(k_cache.shape[2:]) != (nkv, headdim_k) or tuple(v_cache.shape[2:]) != (nkv, headdim_v):
            raise RuntimeError(f"{what}: the caches must have the heads of k and v, got {tuple(k_cache.shape)} and {tuple(v_cache.shape)}")
    batch = q.shape[0]
    num_pages, page_size = k_cache.shape[:2]
    if num_pages == 0 or page_size == 0:
        raise RuntimeError(f"{what}: the caches need a page at least, of a position at least")
    for name, t in (("k_cache", k_cache), ("v_cache", v_cache)):
        if t.stride(3) != 1 and t.shape[3] > 1:
            raise RuntimeError(f"{what}: {name} must have unit stride along the head")
        if k is not None and not _rows_apart(t):
            raise RuntimeError(f"{what}: {name}'s rows must not overlap (they are written in place)")
        if k is not None and torch.is_grad_enabled() and t.requires_grad:
            raise RuntimeError(f"{what}: {name} is updated in place and takes no gradients: detach it, or call under torch.no_grad()")
    if block_table.dim() != 2 or block_table.shape[0] != batch or block_table.shape[1] < 1 or block_table.dtype not in (torch.int32, torch.int64):
        raise RuntimeError(f"{what}: block_table must be ({batch}, pages of a sequence) int32")
    if tuple(cache_seqlens.shape) != (batch,) or cache_seqlens.dtype not in (torch.int32, torch.int64):
        raise RuntimeError(f"{what}: cache_seqlens must be ({batch},) int32")
    if batch > 65535 or num_pages > 2 ** 31 - 1 or block_table.shape[1] * page_size > 2 ** 30:
        raise RuntimeError(f"{what}: up to 65535 sequences and tables of up to 2^30 positions are served")
    scale = _check_scale(what, scale, headdim_k, 2e38)
    if window is not None and not 1 <= int(window) <= 2 ** 31 - 1:
        raise ValueError(f"{what}: window must be at least 1, got {window}")
    _lib.refuse_tangents(what, q, k, v, k_cache, v_cache)
    _lib.require_gpu(q, k, v, k_cache, v_cache, block_table, cache_seqlens)
    _one_device(what, q, k, v, k_cache, v_cache, block_table, cache_seqlens)
    block_table = _int32(block_table, -1, 2 ** 31 - 1)
    cache_seqlens = _int32(cache_seqlens, -1, 2 ** 31 - 1)
    return PagedAttentionUpdateFn.apply(q, k.to(q.dtype) if k is not None else None, v.to(q.dtype) if v is not None else None, k_cache,
                                        v_cache, block_table, cache_seqlens, scale, int(window) if window is not None else 0)


def paged_attention_update_ref(q, k, v, k_cache, v_cache, block_table, cache_seqlens, scale=None, window=None):
    """One call from plain torch operators, sequence by sequence, in place on the caches; every page named has to exist."""
    group, page = q.shape[1] // k_cache.shape[2], k_cache.shape[1]
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    out = torch.zeros(*q.shape[:2], v_cache.shape[-1], dtype=q.dtype, device=q.device)
    for b, n in enumerate(cache_seqlens.tolist()):
        if n < 0:
            continue
        pages = block_table[b].long()
        if k is not None:
            k_cache[pages[n // page], n % page] = k[b].to(k_cache.dtype)
            v_cache[pages[n // page], n % page] = v[b].to(v_cache.dtype)
            n += 1
        first = max(0, n - window) if window is not None else 0
        if n == 0:
            continue
        pos = torch.arange(first, n, device=q.device)
        keys = k_cache[pages[pos // page], pos % page].float().repeat_interleave(group, 1)
        values = v_cache[pages[pos // page], pos % page].float().repeat_interleave(group, 1)
        p = torch.softmax(scale * (keys * q[b].float()).sum(-1), 0)
        out[b] = (p[..., None] * values).sum(0).to(q.dtype)
    return out
