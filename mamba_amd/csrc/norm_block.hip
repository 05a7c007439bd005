// The norm behind a block with its gate and residual scale, the residual add and the norm in front of the next block
// (gfx950):
//   s = residual + scale * norm(x) * silu(z);  out = norm'(s)
// norm: n = (v - mean) rstd, y = n weight + bias, mean 0 for RMSNorm.  Backward, with d = dsum + norm''s gradient:
//   dn'  = dout next_weight;    d  = dsum + rstd' (dn' - n' mean(n' dn') - mean(dn'))
//   dy   = d scale silu(z);     dx = rstd (dy w - n mean(n dy w) - mean(dy w)),   dz = d scale y silu'(z)
//   sums over the rows: dout n', dout (next_weight, next_bias), dy n, dy (norm_weight, norm_bias), d y silu(z) (scale)
// s is formed again in the backward pass from the same inputs: its rounding to the stream's type then enters neither
// the norm nor the sums.
#include "norm_common.hpp"

namespace {

constexpr int kThreads = 256;

DEVI float block_sum(float v, float *red) {
  v = wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return red[0] + red[1] + red[2] + red[3];
}

// One row, read again from memory for every pass over it.
template <typename T, typename R> struct Row {
  const NormBlockParams &p;
  int64_t row;
  float mean1 = 0.f, rstd1 = 0.f, mean2 = 0.f, rstd2 = 0.f;
  DEVI Row(const NormBlockParams &q, int64_t r) : p(q), row(r) {}
  DEVI float par(const void *w, int c) const { return ld_param(w, p.weight_dtype, c); }
  DEVI float x(int c) const { return ld1<T>(static_cast<const T *>(p.x) + row * p.x_rs + c); }
  DEVI float z(int c) const { return ld1<T>(static_cast<const T *>(p.z) + row * p.z_rs + c); }
  DEVI float n1(int c) const { return (x(c) - mean1) * rstd1; }
  DEVI float y(int c) const { return n1(c) * par(p.norm_weight, c) + (p.norm_bias ? par(p.norm_bias, c) : 0.f); }
  DEVI float scale(int c) const { return p.scale ? par(p.scale, c) : p.scale_value; }
  DEVI float gate(int c) const {
    if (!p.z) return 1.f;
    const float v = z(c);
    return v * sigmoid_f(v);
  }
  DEVI float s(int c) const {
    return ld1<R>(static_cast<const R *>(p.residual) + row * p.residual_rs + c) + scale(c) * y(c) * gate(c);
  }
  DEVI float n2(int c) const { return (s(c) - mean2) * rstd2; }
  template <typename F> DEVI float sum(float *red, F f) const {
    float v = 0.f;
    for (int c = threadIdx.x; c < p.dim; c += kThreads) v += f(c);
    return block_sum(v, red);
  }
};

template <typename T, typename R> __global__ __launch_bounds__(kThreads) void norm_block_fwd_kernel(const NormBlockParams p) {
  __shared__ float red[4];
  const float inv = 1.f / (float)p.dim;
  for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
    Row<T, R> w(p, r);
    if (!p.is_rms) w.mean1 = w.sum(red, [&](int c) { return w.x(c); }) * inv;
    w.rstd1 = 1.f / sqrtf(w.sum(red, [&](int c) { const float d = w.x(c) - w.mean1; return d * d; }) * inv + p.eps);
    if (!p.is_rms) w.mean2 = w.sum(red, [&](int c) { return w.s(c); }) * inv;
    w.rstd2 = 1.f / sqrtf(w.sum(red, [&](int c) { const float d = w.s(c) - w.mean2; return d * d; }) * inv + p.eps);
    for (int c = threadIdx.x; c < p.dim; c += kThreads) {
      st1<R>(static_cast<R *>(p.residual_out) + r * p.residual_out_rs + c, w.s(c));
      st1<T>(static_cast<T *>(p.out) + r * p.out_rs + c,
             w.n2(c) * w.par(p.next_weight, c) + (p.next_bias ? w.par(p.next_bias, c) : 0.f));
    }
    if (p.stats && threadIdx.x == 0)
      *reinterpret_cast<f32x4 *>(p.stats + r * 4) = f32x4{w.mean1, w.rstd1, w.mean2, w.rstd2};
  }
}

// The sums' places in `parts`: next_weight, norm_weight, scale, next_bias, norm_bias, those that are wanted, each
// (nparts, dim).
struct Sums {
  float *next_w, *norm_w, *scale, *next_b, *norm_b;
};

template <typename T, typename R> __global__ __launch_bounds__(kThreads) void norm_block_bwd_kernel(const NormBlockParams p, const Sums sums) {
  __shared__ float red[4];
  const float inv = 1.f / (float)p.dim;
  const int64_t mine = (int64_t)blockIdx.x * p.dim;
  for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
    Row<T, R> w(p, r);
    const f32x4 st = *reinterpret_cast<const f32x4 *>(p.stats + r * 4);
    w.mean1 = st.x, w.rstd1 = st.y, w.mean2 = st.z, w.rstd2 = st.w;
    auto dout = [&](int c) { return ld1<T>(static_cast<const T *>(p.dout) + r * p.dout_rs + c); };
    auto dn2 = [&](int c) { return dout(c) * w.par(p.next_weight, c); };
    const float c1 = w.sum(red, [&](int c) { return dn2(c) * w.n2(c); }) * inv;
    const float c2 = p.is_rms ? 0.f : w.sum(red, dn2) * inv;
    auto d = [&](int c) {
      const float ds = p.dsum ? ld1<R>(static_cast<const R *>(p.dsum) + r * p.dsum_rs + c) : 0.f;
      return ds + w.rstd2 * (dn2(c) - w.n2(c) * c1 - c2);
    };
    auto dn1 = [&](int c) { return d(c) * w.scale(c) * w.gate(c) * w.par(p.norm_weight, c); };
    const float c3 = w.sum(red, [&](int c) { return dn1(c) * w.n1(c); }) * inv;
    const float c4 = p.is_rms ? 0.f : w.sum(red, dn1) * inv;
    const bool first = r == blockIdx.x;
    for (int c = threadIdx.x; c < p.dim; c += kThreads) {
      const float dv = d(c), g = w.gate(c), y = w.y(c), n1 = w.n1(c), dy = dv * w.scale(c) * g;
      st1<R>(static_cast<R *>(p.dresidual) + r * p.dresidual_rs + c, dv);
      st1<T>(static_cast<T *>(p.dx) + r * p.dx_rs + c, w.rstd1 * (dn1(c) - n1 * c3 - c4));
      if (p.dz) {
        const float z = w.z(c), sg = sigmoid_f(z);
        st1<T>(static_cast<T *>(p.dz) + r * p.dz_rs + c, dv * w.scale(c) * y * sg * (1.f + z * (1.f - sg)));
      }
      auto add = [&](float *part, float v) {
        if (part) part[mine + c] = first ? v : part[mine + c] + v;
      };
      add(sums.next_w, dout(c) * w.n2(c));
      add(sums.next_b, dout(c));
      add(sums.norm_w, dy * n1);
      add(sums.norm_b, dy);
      add(sums.scale, dv * y * g);
    }
  }
}

int check(const NormBlockParams *p, bool bwd) {
  if (!p || !p->x || !p->residual || !p->norm_weight || !p->next_weight) return MAMBA_E_BADARG;
  if (p->rows <= 0 || p->dim <= 0) return MAMBA_E_BADARG;
  if (p->dim > 32768) return MAMBA_E_UNSUPPORTED;
  if (p->dtype < MAMBA_F32 || p->dtype > MAMBA_F16 || p->weight_dtype < MAMBA_F32 || p->weight_dtype > MAMBA_F16)
    return MAMBA_E_BADARG;
  if (p->res_dtype != p->dtype && p->res_dtype != MAMBA_F32) return MAMBA_E_UNSUPPORTED;
  if (p->stats && !aligned16(p->stats)) return MAMBA_E_BADARG;
  if (!bwd) return p->out && p->residual_out ? MAMBA_OK : MAMBA_E_BADARG;
  if (!p->stats || !p->dout || !p->dx || !p->dresidual || !p->dnorm_weight || !p->dnext_weight || !p->parts) return MAMBA_E_BADARG;
  if (!p->z != !p->dz || !p->scale != !p->dscale || !p->norm_bias != !p->dnorm_bias || !p->next_bias != !p->dnext_bias)
    return MAMBA_E_BADARG;
  return p->nparts >= 1 && p->nparts <= 65536 ? MAMBA_OK : MAMBA_E_BADARG;
}

template <typename T, typename R> int run(const NormBlockParams &p, bool bwd, hipStream_t st) {
  if (!bwd) {
    norm_block_fwd_kernel<T, R><<<dim3(min(p.rows, 65536)), dim3(kThreads), 0, st>>>(p);
    return hipGetLastError() == hipSuccess ? MAMBA_OK : MAMBA_E_LAUNCH;
  }
  ReduceJobs jobs{};
  int n = 0;
  const int nparts = min(p.nparts, p.rows);
  auto part = [&](void *out) -> float * {
    if (!out) return nullptr;
    float *q = p.parts + (int64_t)n * nparts * p.dim;
    jobs.part[n] = q, jobs.out[n++] = out;
    return q;
  };
  Sums sums;
  sums.next_w = part(p.dnext_weight), sums.norm_w = part(p.dnorm_weight), sums.scale = part(p.dscale);
  sums.next_b = part(p.dnext_bias), sums.norm_b = part(p.dnorm_bias);
  norm_block_bwd_kernel<T, R><<<dim3(nparts), dim3(kThreads), 0, st>>>(p, sums);
  if (hipGetLastError() != hipSuccess) return MAMBA_E_LAUNCH;
  return launch_reduce(jobs, n, p.weight_dtype, nparts, p.dim, st);
}

template <typename T> int pick(const NormBlockParams &p, bool bwd, hipStream_t st) {
  return p.res_dtype == MAMBA_F32 ? run<T, float>(p, bwd, st) : run<T, T>(p, bwd, st);
}

int dispatch(const NormBlockParams *p, bool bwd, hipStream_t st) {
  if (const int rc = check(p, bwd)) return rc;
  switch (p->dtype) {
    case MAMBA_F32: return pick<float>(*p, bwd, st);
    case MAMBA_BF16: return pick<bf16_t>(*p, bwd, st);
    default: return pick<f16_t>(*p, bwd, st);
  }
}

}  // namespace

extern "C" int norm_block_fwd(const NormBlockParams *p, mamba_stream_t stream) {
  return dispatch(p, false, static_cast<hipStream_t>(stream));
}
extern "C" int norm_block_bwd(const NormBlockParams *p, mamba_stream_t stream) {
  return dispatch(p, true, static_cast<hipStream_t>(stream));
}
extern "C" int norm_block_bwd_nparts(const NormBlockParams *p) {
  if (!p || p->rows <= 0 || p->dim <= 0) return MAMBA_E_BADARG;
  return min(p->rows, 1024);
}
