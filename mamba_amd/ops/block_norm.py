"""The norm behind a block, its gate and residual scale, the residual add and the norm in front of the next block in
one pass over the rows, on the HIP kernels:

    residual_out = residual + scale * norm(x; norm_weight, norm_bias) * silu(z)
    out = norm(residual_out; next_weight, next_bias)

`layer_norm_fn` / `rms_norm_fn` (mamba_amd.ops.triton.layer_norm) are the add + norm of blocks without a norm of their
own behind them.  There is no CPU or PyTorch fallback: CPU tensors raise.  `block_norm_ref` states the arithmetic in
plain torch; no operator calls it.
"""
import torch
import torch.nn.functional as F

from mamba_amd import _lib


def _rows(t):
    t = t.reshape(-1, t.shape[-1])
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _params(x, residual, norm_weight, next_weight, z, scale, norm_bias, next_bias, eps, is_rms_norm):
    p = _lib.NormBlockParams()
    p.rows, p.dim = x.shape
    p.dtype, p.res_dtype, p.weight_dtype = (_lib.DTYPE_CODE[t.dtype] for t in (x, residual, norm_weight))
    p.is_rms, p.eps = int(is_rms_norm), eps
    p.scale_value = 1.0 if isinstance(scale, torch.Tensor) else scale
    p.x, p.z, p.residual = x.data_ptr(), _lib.ptr(z), residual.data_ptr()
    p.norm_weight, p.next_weight = norm_weight.data_ptr(), next_weight.data_ptr()
    p.norm_bias, p.next_bias = _lib.ptr(norm_bias), _lib.ptr(next_bias)
    p.scale = scale.data_ptr() if isinstance(scale, torch.Tensor) else None
    p.x_rs, p.residual_rs, p.z_rs = x.stride(0), residual.stride(0), z.stride(0) if z is not None else 0
    return p


class BlockNormFn(torch.autograd.Function):
    """Arguments as `block_norm_fn` has checked and converted them (scale: a tensor or a number); returns
    (out, residual_out)."""

    @staticmethod
    def forward(ctx, x, residual, norm_weight, next_weight, z, scale, norm_bias, next_bias, eps, is_rms_norm):
        shape = x.shape
        x, residual, z = _rows(x), _rows(residual), _rows(z) if z is not None else None
        rows, dim = x.shape
        # in x's shape, no views of rows: an output of several that is a view takes no in-place writes
        out = torch.empty(shape, dtype=x.dtype, device=x.device)
        total = torch.empty(shape, dtype=residual.dtype, device=x.device)
        stats = torch.empty(rows, 4, dtype=torch.float32, device=x.device)
        if rows > 0:
            p = _params(x, residual, norm_weight, next_weight, z, scale, norm_bias, next_bias, eps, is_rms_norm)
            p.out, p.residual_out, p.stats = out.data_ptr(), total.data_ptr(), stats.data_ptr()
            p.out_rs = p.residual_out_rs = dim
            with torch.cuda.device(x.device):
                _lib.check(_lib.load().norm_block_fwd(p, _lib.current_stream(x.device)), "norm_block_fwd")
        ctx.save_for_backward(x, residual, norm_weight, next_weight, z, scale if isinstance(scale, torch.Tensor) else None,
                              norm_bias, next_bias, stats)
        ctx.scale = None if isinstance(scale, torch.Tensor) else scale
        ctx.eps, ctx.is_rms_norm, ctx.shape = eps, is_rms_norm, shape
        ctx.set_materialize_grads(False)
        return out, total

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout, dsum):
        x, residual, norm_weight, next_weight, z, scale, norm_bias, next_bias, stats = ctx.saved_tensors
        if dout is None and dsum is None:
            return (None,) * 10
        rows, dim = x.shape
        dout = _rows(dout) if dout is not None else torch.zeros(rows, dim, dtype=x.dtype, device=x.device)
        dsum = _rows(dsum) if dsum is not None else None
        dx, dresidual = (torch.empty(ctx.shape, dtype=t.dtype, device=x.device) for t in (x, residual))
        dz = torch.empty(ctx.shape, dtype=x.dtype, device=x.device) if z is not None else None
        given = [(n, t) for n, t in (("dnorm_weight", norm_weight), ("dnext_weight", next_weight), ("dscale", scale),
                                     ("dnorm_bias", norm_bias), ("dnext_bias", next_bias)) if t is not None]
        sums = (torch.empty if rows > 0 else torch.zeros)(len(given), dim, dtype=norm_weight.dtype, device=x.device)
        grads = {n: sums[i] for i, (n, _) in enumerate(given)}
        if rows > 0:
            p = _params(x, residual, norm_weight, next_weight, z, scale if scale is not None else ctx.scale, norm_bias,
                        next_bias, ctx.eps, ctx.is_rms_norm)
            p.stats = stats.data_ptr()
            p.dout, p.dsum, p.dx, p.dresidual, p.dz = dout.data_ptr(), _lib.ptr(dsum), dx.data_ptr(), dresidual.data_ptr(), _lib.ptr(dz)
            p.dout_rs, p.dsum_rs = dout.stride(0), dsum.stride(0) if dsum is not None else 0
            p.dx_rs = p.dresidual_rs = p.dz_rs = dim
            for n, g in grads.items():
                setattr(p, n, g.data_ptr())
            with torch.cuda.device(x.device):
                lib = _lib.load()
                p.nparts = lib.norm_block_bwd_nparts(p)
                nsums = 2 + (norm_bias is not None) + (next_bias is not None)
                parts = torch.empty(nsums, p.nparts, dim, dtype=torch.float32, device=x.device)
                p.parts = parts.data_ptr()
                _lib.check(lib.norm_block_bwd(p, _lib.current_stream(x.device)), "norm_block_bwd")
        return (dx, dresidual, grads["dnorm_weight"], grads["dnext_weight"], dz, grads.get("dscale"), grads.get("dnorm_bias"),
                grads.get("dnext_bias"), None, None)


def block_norm_fn(x, residual, norm_weight, next_weight, z=None, scale=None, norm_bias=None, next_bias=None, eps=1e-5,
                  is_rms_norm=True):
    """Closes one block and opens the next; differentiable in every tensor.

    Argument:
        x: (..., dim), the block's output, in fp32, fp16 or bf16
        residual: x's shape, the residual stream, in x's dtype or fp32
        norm_weight, norm_bias: (dim,), the norm behind the block; next_weight, next_bias: (dim,), the norm in front of
            the next one; the biases may be None
        z: x's shape, the block's gate (silu(z) multiplies the normed rows), or None
        scale: the factor on what is added to the stream: (dim,), a number, or None (1)
        is_rms_norm: RMSNorm (True) or LayerNorm
    The parameters may be in any of the three dtypes; where they differ among themselves they are taken in fp32.
    Return:
        out in x's dtype, residual_out in residual's (the sum is normed before it is rounded to that)
    """
    tensor_scale = scale if isinstance(scale, torch.Tensor) else None
    number = 1.0 if scale is None or tensor_scale is not None else float(scale)
    ext = _lib.torch_ext()
    if ext is not None:
        # the same node in C++ (csrc/torch_gated.cpp); None = a case for the code below
        r = ext.block_norm(x, residual, norm_weight, next_weight, z, tensor_scale, number, norm_bias, next_bias, eps, bool(is_rms_norm))
        if r is not None:
            return r
    what = "block_norm"
    if x.dim() < 1 or x.dtype not in _lib.DTYPE_CODE:
        raise RuntimeError(f"{what}: x must be (..., dim) in fp32, fp16 or bf16")
    for name, t in (("residual", residual), ("z", z)):
        if t is not None and t.shape != x.shape:
            raise RuntimeError(f"{what}: {name} must have x's shape {tuple(x.shape)}, got {tuple(t.shape)}")
    if residual.dtype not in (x.dtype, torch.float32):
        raise RuntimeError(f"{what}: the residual stream must be in x's dtype or fp32")
    dim = x.shape[-1]
    if dim < 1 or dim > 32768:
        raise RuntimeError(f"{what}: rows of 1 to 32768 channels are served, got {dim}")
    if x.numel() // dim > 2 ** 31 - 1:
        raise RuntimeError(f"{what}: rows are counted in 32 bits, got {x.numel() // dim}")
    params = dict(norm_weight=norm_weight, next_weight=next_weight, scale=tensor_scale, norm_bias=norm_bias, next_bias=next_bias)
    for name, t in params.items():
        if t is not None and (tuple(t.shape) != (dim,) or t.dtype not in _lib.DTYPE_CODE):
            raise RuntimeError(f"{what}: {name} must be ({dim},) in fp32, fp16 or bf16")
    _lib.require_gpu(x, residual, z, *params.values())
    for t in (residual, z, *params.values()):
        if t is not None and t.device != x.device:
            raise RuntimeError(f"{what}: all tensors must be on {x.device}, got one on {t.device}")
    one = len({t.dtype for t in params.values() if t is not None}) == 1
    conv = lambda t: None if t is None else (t if one else t.float()).contiguous()
    return BlockNormFn.apply(x, residual, conv(norm_weight), conv(next_weight), z.to(x.dtype) if z is not None else None,
                             conv(scale) if tensor_scale is not None else number, conv(norm_bias), conv(next_bias), float(eps),
                             bool(is_rms_norm))


def block_norm_ref(x, residual, norm_weight, next_weight, z=None, scale=None, norm_bias=None, next_bias=None, eps=1e-5,
                   is_rms_norm=True):
    """The arithmetic in plain torch, in fp32, on whatever device the inputs live on."""
    def norm(v, weight, bias):
        v = v if is_rms_norm else v - v.mean(-1, keepdim=True)
        v = v * torch.rsqrt(v.square().mean(-1, keepdim=True) + eps) * weight.float()
        return v if bias is None else v + bias.float()

    y = norm(x.float(), norm_weight, norm_bias)
    if z is not None:
        y = y * F.silu(z.float())
    if scale is not None:
        y = y * (scale.float() if isinstance(scale, torch.Tensor) else scale)
    total = residual.float() + y
    return norm(total, next_weight, next_bias).to(x.dtype), total.to(residual.dtype)
