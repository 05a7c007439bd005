// The norm behind a block with its gate and residual scale, the residual add and the norm in front of the next block
// (gfx950):
//   s = residual + scale * norm(x) * silu(z);  out = norm'(s)
// norm: n = (v - mean) rstd, y = n weight + bias, mean 0 for RMSNorm.  Backward, with d = dsum + norm''s gradient:
//   dn' = dout next_weight;   d  = dsum + rstd' (dn' - n' mean(n' dn') - mean(dn'))
//   dn  = d scale silu(z) norm_weight;   dx = rstd (dn - n mean(n dn) - mean(dn)),   dz = d scale y silu'(z)
// Sums over the rows: with Q = sum d silu(z) n and P = sum d silu(z), norm_weight's is scale Q, norm_bias's scale P,
// scale's norm_weight Q + norm_bias P; next_weight's is sum dout n', next_bias's sum dout: two sums per channel are
// carried through the rows, four with biases.
// s is formed again in the backward pass from the same inputs: its rounding to the stream's type then enters neither
// the norm nor the sums.
//
// Both directions are bound by memory: 14 and 22 bytes per element for a bf16 block with gate on an fp32 stream.  A
// workgroup holds one row in registers, 8 channels per thread, and asks for its next row before it works on this one;
// the parameters and sums of a thread's channels stay in registers over the rows.  16384 x 2560 (bf16, fp32 stream): forward 107 us,
// 5.5 TB/s, backward 173 us, 5.3 TB/s, of 6.2 that a copy reaches.
#include "norm_common.hpp"

namespace {

// ------------------------------------------------------------------ rows of 8 to 8192 channels
// 8 channels of a thread.  WHOLE: the number of channels is a multiple of 8.  Otherwise the last thread that has channels
// reads the row's last 8 and moves its own to the front.  Rows lie at any alignment.
template <bool WHOLE> struct Seg {
  int c, n, dim;  // first channel, how many are there
  DEVI Seg(int dim_) : c(threadIdx.x * 8), n(min(max(dim_ - (int)threadIdx.x * 8, 0), 8)), dim(dim_) {}
  template <typename T> DEVI void fetch(const T *row, Pack8<T> &k) const { k.load_any(row + min(c, dim - 8)); }
  template <typename T> DEVI void get(const Pack8<T> &k, float (&v)[8]) const {
    k.unpack(v);
    if constexpr (!WHOLE) {
      row8_place(c, dim, v);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = n ? v[e] : 0.f;
    }
  }
  template <typename T> DEVI void put(T *row, const float (&v)[8]) const {
    if (n == 8) {
      st8_any<T>(row + c, v);
    } else if (!WHOLE) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < n) st1<T>(row + c + e, v[e]);
    }
  }
  DEVI void param(const void *base, int dtype, float missing, float (&v)[1][8]) const {
    if (base) {
      load_params<1, 1>(base, dtype, 0, min(c, dim), dim, v);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[0][e] = missing;
    }
  }
  DEVI bool has(int e) const { return WHOLE ? n != 0 : e < n; }
};

// FULL: LayerNorm or biases (is_rms decides about the mean); otherwise RMSNorm without biases.
template <typename T, typename R, bool FULL, bool GATE, bool WHOLE, int MAXT>
__global__ __launch_bounds__(MAXT) void norm_block_fwd_kernel(const NormBlockParams p) {
  __shared__ float lds[64];
  WideSum ws(lds);
  const Seg<WHOLE> seg(p.dim);
  const T *xp = static_cast<const T *>(p.x), *zp = static_cast<const T *>(p.z);
  const R *rp = static_cast<const R *>(p.residual);
  const float inv = 1.f / (float)p.dim;
  const bool centre = FULL && !p.is_rms;
  Pack8<T> bx, bz;
  Pack8<R> br;
  auto fetch = [&](int64_t r) {
    seg.fetch(xp + r * p.x_rs, bx);
    if constexpr (GATE) seg.fetch(zp + r * p.z_rs, bz);
    seg.fetch(rp + r * p.residual_rs, br);
  };
  fetch(blockIdx.x);
  float w1[1][8], w2[1][8], sc[1][8], b1[1][8], b2[1][8];
  seg.param(p.norm_weight, p.weight_dtype, 0.f, w1);
  seg.param(p.scale, p.weight_dtype, p.scale_value, sc);
  seg.param(p.next_weight, p.weight_dtype, 0.f, w2);
  if constexpr (FULL) seg.param(p.norm_bias, p.weight_dtype, 0.f, b1), seg.param(p.next_bias, p.weight_dtype, 0.f, b2);
  // rows of 8 channels in v: the mean is taken off (LayerNorm), the result is the factor of the norm
  float mean = 0.f;
  auto norm = [&](float (&v)[8]) {
    float dummy = 0.f, var = 0.f;
    mean = 0.f;
    if (centre) {
#pragma unroll
      for (int e = 0; e < 8; ++e) mean += v[e];
      ws.sum2(mean, dummy);
      mean *= inv;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = seg.has(e) ? v[e] - mean : 0.f;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) var = __builtin_fmaf(v[e], v[e], var);
    dummy = 0.f;
    ws.sum2(var, dummy);
    return 1.f / sqrtf(var * inv + p.eps);
  };
  for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
    float v[8], z[8], s[8];
    seg.get(bx, v);
    seg.get(br, s);
    if constexpr (GATE) seg.get(bz, z);
    fetch(min(r + gridDim.x, (int64_t)p.rows - 1));
    const float rstd1 = norm(v), mean1 = mean;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float y = v[e] * rstd1 * w1[0][e];
      if constexpr (FULL) y += b1[0][e];
      if constexpr (GATE) y *= z[e] * sigmoid_f(z[e]);
      s[e] = __builtin_fmaf(sc[0][e], y, s[e]);
    }
    seg.put(static_cast<R *>(p.residual_out) + r * p.residual_out_rs, s);
    const float rstd2 = norm(s), mean2 = mean;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      s[e] *= rstd2 * w2[0][e];
      if constexpr (FULL) s[e] += b2[0][e];
    }
    seg.put(static_cast<T *>(p.out) + r * p.out_rs, s);
    if (p.stats && threadIdx.x == 0) *reinterpret_cast<f32x4 *>(p.stats + r * 4) = f32x4{mean1, rstd1, mean2, rstd2};
  }
}

// The sums over a workgroup's rows: rows of `parts`, each (nparts, dim); the biases' null where there is none.
struct Sums {
  float *next_w, *q, *next_b, *p;
};

// Rows of more than 12 waves leave a thread 128 registers: the parameters are then read again for every row (from the
// caches) and the next row is not asked for ahead.  With a gate, LayerNorm or biases, rows of more than 8 waves (4104 channels and
// on) spill all the same, 12 to 232 bytes a thread: 231 us at 4096 x 8192 (bf16 with gate, fp32 stream) for 118 of bytes.
template <typename T, typename R, bool FULL, bool GATE, bool WHOLE, int MAXT>
__global__ __launch_bounds__(MAXT) void norm_block_bwd_kernel(const NormBlockParams p, const Sums sums) {
  __shared__ float lds[64];
  WideSum ws(lds);
  const Seg<WHOLE> seg(p.dim);
  const T *xp = static_cast<const T *>(p.x), *zp = static_cast<const T *>(p.z), *gp = static_cast<const T *>(p.dout);
  const R *rp = static_cast<const R *>(p.residual);
  // without dsum the residual stands in for it (read, not used)
  const bool has_dsum = p.dsum != nullptr;
  const R *dp = has_dsum ? static_cast<const R *>(p.dsum) : rp;
  const int64_t dp_rs = has_dsum ? p.dsum_rs : p.residual_rs;
  const float inv = 1.f / (float)p.dim;
  const bool centre = FULL && !p.is_rms;
  Pack8<T> bx, bz, bg;
  Pack8<R> br, bd;
  f32x4 bs;
  auto fetch = [&](int64_t r) {
    bs = *reinterpret_cast<const f32x4 *>(p.stats + r * 4);
    seg.fetch(xp + r * p.x_rs, bx);
    if constexpr (GATE) seg.fetch(zp + r * p.z_rs, bz);
    seg.fetch(rp + r * p.residual_rs, br);
    seg.fetch(gp + r * p.dout_rs, bg);
    seg.fetch(dp + r * dp_rs, bd);
  };
  constexpr bool LEAN = MAXT > 768;
  float w1[1][8], w2[1][8], sc[1][8], b1[1][8];
  auto params = [&]() {
    seg.param(p.norm_weight, p.weight_dtype, 0.f, w1);
    seg.param(p.scale, p.weight_dtype, p.scale_value, sc);
    seg.param(p.next_weight, p.weight_dtype, 0.f, w2);
    if constexpr (FULL) seg.param(p.norm_bias, p.weight_dtype, 0.f, b1);
  };
  if (!LEAN) {
    fetch(blockIdx.x);
    params();
  }
  float a_next[8], a_q[8], a_nb[FULL ? 8 : 1], a_p[FULL ? 8 : 1];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    a_next[e] = a_q[e] = 0.f;
    if constexpr (FULL) a_nb[e] = a_p[e] = 0.f;
  }
  for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
    float n1[8], z[8], n2[8], g[8], d[8];
    if (LEAN) {
      fetch(r);
      params();
    }
    seg.get(bx, n1);
    seg.get(br, n2);
    seg.get(bg, g);
    seg.get(bd, d);
    if constexpr (GATE) seg.get(bz, z);
    const f32x4 st = bs;
    if (!LEAN) fetch(min(r + gridDim.x, (int64_t)p.rows - 1));
    float c1 = 0.f, c2 = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      n1[e] = FULL ? (seg.has(e) ? (n1[e] - st.x) * st.y : 0.f) : n1[e] * st.y;
      float y = n1[e] * w1[0][e];
      if constexpr (FULL) y += b1[0][e];
      if constexpr (GATE) y *= z[e] * sigmoid_f(z[e]);
      const float s = __builtin_fmaf(sc[0][e], y, n2[e]);
      n2[e] = FULL ? (seg.has(e) ? (s - st.z) * st.w : 0.f) : s * st.w;
      a_next[e] = __builtin_fmaf(g[e], n2[e], a_next[e]);
      if constexpr (FULL) a_nb[e] += g[e];
      g[e] *= w2[0][e];
      c1 = __builtin_fmaf(g[e], n2[e], c1);
      c2 += g[e];
    }
    ws.sum2(c1, c2);
    c1 *= inv;
    c2 = centre ? c2 * inv : 0.f;
    float c3 = 0.f, c4 = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      d[e] = __builtin_fmaf(st.w, g[e] - n2[e] * c1 - c2, has_dsum ? d[e] : 0.f);
      const float sg = GATE ? sigmoid_f(z[e]) : 1.f;
      const float dg = GATE ? d[e] * (z[e] * sg) : d[e];
      a_q[e] = __builtin_fmaf(dg, n1[e], a_q[e]);
      if constexpr (FULL) a_p[e] += seg.has(e) ? dg : 0.f;
      g[e] = dg * sc[0][e] * w1[0][e];
      c3 = __builtin_fmaf(g[e], n1[e], c3);
      c4 += g[e];
      if constexpr (GATE) {
        float y = n1[e] * w1[0][e];
        if constexpr (FULL) y += b1[0][e];
        z[e] = d[e] * sc[0][e] * y * (sg * __builtin_fmaf(z[e], 1.f - sg, 1.f));
      }
    }
    seg.put(static_cast<R *>(p.dresidual) + r * p.dresidual_rs, d);
    if constexpr (GATE) seg.put(static_cast<T *>(p.dz) + r * p.dz_rs, z);
    ws.sum2(c3, c4);
    c3 *= inv;
    c4 = centre ? c4 * inv : 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) g[e] = st.y * (g[e] - n1[e] * c3 - c4);
    seg.put(static_cast<T *>(p.dx) + r * p.dx_rs, g);
  }
  const int64_t mine = (int64_t)blockIdx.x * p.dim;
  seg.put(sums.next_w + mine, a_next);
  seg.put(sums.q + mine, a_q);
  if constexpr (FULL) {
    if (sums.next_b) seg.put(sums.next_b + mine, a_nb);
    if (sums.p) seg.put(sums.p + mine, a_p);
  }
}

// ------------------------------------------------------------------ any row
// One row of any length, read again from memory for every pass over it: rows of less than 8 or more than 8192 channels.  The long
// ones are served, not made fast: 283 us forward and 941 backward at 4096 x 8198 (bf16 with gate, fp32 stream), where 8192 channels in
// registers take 88 and 231.
constexpr int kThreads = 256;

DEVI float block_sum(float v, float *red) {
  v = wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return red[0] + red[1] + red[2] + red[3];
}

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

template <typename T, typename R> __global__ __launch_bounds__(kThreads) void norm_block_any_fwd_kernel(const NormBlockParams p) {
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

template <typename T, typename R>
__global__ __launch_bounds__(kThreads) void norm_block_any_bwd_kernel(const NormBlockParams p, const Sums sums) {
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
      const float dv = d(c), g = w.gate(c), y = w.y(c), n1 = w.n1(c);
      st1<R>(static_cast<R *>(p.dresidual) + r * p.dresidual_rs + c, dv);
      st1<T>(static_cast<T *>(p.dx) + r * p.dx_rs + c, w.rstd1 * (dn1(c) - n1 * c3 - c4));
      if (p.dz) {
        const float z = w.z(c), sg = sigmoid_f(z);
        st1<T>(static_cast<T *>(p.dz) + r * p.dz_rs + c, dv * w.scale(c) * y * (sg * (1.f + z * (1.f - sg))));
      }
      auto add = [&](float *part, float v) {
        if (part) part[mine + c] = first ? v : part[mine + c] + v;
      };
      add(sums.next_w, dout(c) * w.n2(c));
      add(sums.next_b, dout(c));
      add(sums.q, dv * g * n1);
      add(sums.p, dv * g);
    }
  }
}

// ------------------------------------------------------------------ the parameters' gradients
// The sums of the parts in their order, and the gradients from them: blockIdx.y 0 is the next norm, 1 this one.  16
// channels per workgroup, 256 slices of the parts.
__global__ __launch_bounds__(1024) void norm_block_sums_kernel(const NormBlockParams p, const Sums sums, int nparts) {
  constexpr int SLICES = 256;
  __shared__ f32x4 lds[SLICES][4];
  const int q = threadIdx.x & 3, sl = threadIdx.x >> 2, c = blockIdx.x * 16 + q * 4, dim = p.dim;
  auto total = [&](const float *src) {  // in the threads of slice 0
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    auto row4 = [&](int part) {
      const float *r = src + (int64_t)part * dim + c;
      f32x4 v = {0.f, 0.f, 0.f, 0.f};
      if (c + 4 <= dim) {
        v = *(const GLOBAL_AS f32x4_a4 *)r;
      } else {
        if (c < dim) v.x = r[0];
        if (c + 1 < dim) v.y = r[1];
        if (c + 2 < dim) v.z = r[2];
      }
      return v;
    };
    int part = sl;
    for (; part + 3 * SLICES < nparts; part += 4 * SLICES) {
      const f32x4 v0 = row4(part), v1 = row4(part + SLICES), v2 = row4(part + 2 * SLICES), v3 = row4(part + 3 * SLICES);
      acc += (v0 + v1) + (v2 + v3);
    }
    for (; part < nparts; part += SLICES) acc += row4(part);
    __syncthreads();
    lds[sl][q] = acc;
    __syncthreads();
#pragma unroll
    for (int half = SLICES / 2; half >= 1; half >>= 1) {
      if (sl < half) lds[sl][q] += lds[sl + half][q];
      __syncthreads();
    }
    return lds[0][q];
  };
  auto write = [&](void *dst, f32x4 v) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (sl == 0 && c + e < dim) st_param(dst, p.weight_dtype, c + e, v[e]);
  };
  auto param = [&](const void *src, float missing) {
    f32x4 v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = src && c + e < dim ? ld_param(src, p.weight_dtype, c + e) : missing;
    return v;
  };
  if (blockIdx.y == 0) {
    write(p.dnext_weight, total(sums.next_w));
    if (sums.next_b) write(p.dnext_bias, total(sums.next_b));
    return;
  }
  const f32x4 qv = total(sums.q), scale = param(p.scale, p.scale_value);
  f32x4 pv = {0.f, 0.f, 0.f, 0.f};
  if (sums.p) pv = total(sums.p);
  write(p.dnorm_weight, scale * qv);
  if (p.dscale) write(p.dscale, param(p.norm_weight, 0.f) * qv + param(p.norm_bias, 0.f) * pv);
  if (sums.p) write(p.dnorm_bias, scale * pv);
}

// ------------------------------------------------------------------ host side
bool in_registers(int dim) { return dim >= 8 && dim <= 8192; }
// threads that hold a row, 8 channels each, in whole waves
int row_threads(int dim) { return wide_threads((dim + 7) / 8 * 8); }
// Workgroups that a launch deals its rows to.
// Forward, three waves a SIMD: 112 us at 16384 x 2560 (five 123, one 109), 12.5 at 4096 x 768 in fp32 (14.5, 18.8).
int fwd_wgs(int dim) { return cu_count() * wide_resident(row_threads(dim), 3); }
// Backward, every one more is a row of partial sums to write and read: four waves a CU, one workgroup at least.  (Four times
// as many: 173 -> 193 us at 16384 x 2560, 27 -> 36 us at 4096 x 768 in fp32.)
int bwd_wgs(int dim) { return cu_count() * max(1, 4 * 64 / row_threads(dim)); }

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

template <typename T, typename R, bool FULL, bool GATE, bool WHOLE>
void launch_rows(const NormBlockParams &p, const Sums *sums, int wgs, hipStream_t st) {
  const int t = row_threads(p.dim);
  auto go = [&](auto most) {
    if (sums) norm_block_bwd_kernel<T, R, FULL, GATE, WHOLE, most.value><<<dim3(wgs), dim3(t), 0, st>>>(p, *sums);
    else norm_block_fwd_kernel<T, R, FULL, GATE, WHOLE, most.value><<<dim3(wgs), dim3(t), 0, st>>>(p);
  };
  if (t <= 512) go(std::integral_constant<int, 512>{});
  else if (t <= 768) go(std::integral_constant<int, 768>{});
  else go(std::integral_constant<int, 1024>{});
}

template <typename T, typename R> int run(const NormBlockParams &p, bool bwd, hipStream_t st) {
  Sums sums{};
  const int nparts = min(p.nparts, p.rows);
  if (bwd) {
    int n = 0;
    auto part = [&]() { return p.parts + (int64_t)n++ * nparts * p.dim; };
    sums.next_w = part(), sums.q = part();
    if (p.next_bias) sums.next_b = part();
    if (p.norm_bias) sums.p = part();
  }
  if (in_registers(p.dim)) {
    const int wgs = bwd ? nparts : min(p.rows, fwd_wgs(p.dim));
    const Sums *s = bwd ? &sums : nullptr;
    const bool full = !p.is_rms || p.norm_bias || p.next_bias, gate = p.z, whole = p.dim % 8 == 0;
    auto pick = [&](auto f, auto g) {
      if (whole) launch_rows<T, R, f.value, g.value, true>(p, s, wgs, st);
      else launch_rows<T, R, f.value, g.value, false>(p, s, wgs, st);
    };
    if (full) gate ? pick(std::true_type{}, std::true_type{}) : pick(std::true_type{}, std::false_type{});
    else gate ? pick(std::false_type{}, std::true_type{}) : pick(std::false_type{}, std::false_type{});
  } else if (bwd) {
    norm_block_any_bwd_kernel<T, R><<<dim3(nparts), dim3(kThreads), 0, st>>>(p, sums);
  } else {
    norm_block_any_fwd_kernel<T, R><<<dim3(min(p.rows, 65536)), dim3(kThreads), 0, st>>>(p);
  }
  if (hipGetLastError() != hipSuccess) return MAMBA_E_LAUNCH;
  if (!bwd) return MAMBA_OK;
  norm_block_sums_kernel<<<dim3((p.dim + 15) / 16, 2), dim3(1024), 0, st>>>(p, sums, nparts);
  return hipGetLastError() == hipSuccess ? MAMBA_OK : MAMBA_E_LAUNCH;
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
  return min(p->rows, in_registers(p->dim) ? bwd_wgs(p->dim) : 1024);
}
