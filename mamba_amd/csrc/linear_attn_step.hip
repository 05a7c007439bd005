// One token of linear attention with a decay per head (linear_attn.hpp has the formulas), the states updated in place (gfx950):
//   S = f S + k v^T,   out = scale q S
// Every state is read and written once, which is what the operator costs (256 x 20 heads of 128 x 128 in a pool, 593 MB: 121 us, 4.9
// TB/s).  A workgroup has the columns (values) of one head that
// LANES lanes hold, 16 bytes of a row each, and walks the rows (keys), ROWS at a time; the rows' shares of out are added up over
// the lanes of a column in a fixed order.
#include "common.hpp"

#include <algorithm>
#include <type_traits>

namespace {

constexpr int kThreads = 256, LANES = 16;

DEVI float log2_decay(float l) {  // minus infinity is a decay to nothing, above 0 counts as 0, NaN stays
  l = l > 0.f ? 0.f : l;
  return (l < -1e6f ? -1e6f : l) * kLog2e;
}

template <typename S, int V> struct Piece {
  float v[V];
  DEVI void load(const S *p, int valid) {
    if constexpr (V == 4) {
      if (valid >= 4) {
        const f32x4 w = *(const GLOBAL_AS f32x4_a4 *)p;
        v[0] = w.x, v[1] = w.y, v[2] = w.z, v[3] = w.w;
        return;
      }
    } else {
      if (valid >= 8) {
        ld8_any<S>(p, v);
        return;
      }
    }
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = e < valid ? ld1<S>(p + e) : 0.f;
  }
  DEVI void store(S *p, int valid) const {
    if constexpr (V == 4) {
      if (valid >= 4) {
        *(GLOBAL_AS f32x4_a4 *)p = f32x4{v[0], v[1], v[2], v[3]};
        return;
      }
    } else {
      if (valid >= 8) {
        st8_any<S>(p, v);
        return;
      }
    }
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (e < valid) st1<S>(p + e, v[e]);
  }
};

template <typename T, typename S> __global__ __launch_bounds__(kThreads) void lin_step_kernel(const LinearAttnStepParams p) {
  constexpr int V = std::is_same_v<S, float> ? 4 : 8, ROWS = kThreads / LANES, U = 8;
  __shared__ float sums[4][LANES * V];
  const int tid = threadIdx.x, lane = tid % LANES, row0 = tid / LANES;
  const int h = blockIdx.y, col = (blockIdx.x * LANES + lane) * V, valid = p.headdim_v - col;
  const int hk = h / (p.nheads / p.nkvheads);
  const float f = fast_exp2(log2_decay(p.log_decay[h]));
  for (int b = blockIdx.z; b < p.batch; b += gridDim.z) {
    const int row = p.state_batch_indices ? p.state_batch_indices[b] : b;
    T *out = static_cast<T *>(p.out) + b * p.out_bs + h * p.out_hs + col;
    if (row < 0 || row >= p.state_rows) {
      if (row0 == 0)
        for (int e = 0; e < V; ++e)
          if (e < valid) st1<T>(out + e, 0.f);
      continue;
    }
    const T *q = static_cast<const T *>(p.q) + b * p.q_bs + h * p.q_hs, *k = static_cast<const T *>(p.k) + b * p.k_bs + hk * p.k_hs;
    const T *v = static_cast<const T *>(p.v) + b * p.v_bs + hk * p.v_hs + col;
    S *state = static_cast<S *>(p.state) + row * p.state_rs + (int64_t)h * p.headdim_k * p.headdim_v + col;
    float vv[V], acc[V];
#pragma unroll
    for (int e = 0; e < V; ++e) vv[e] = e < valid ? ld1<T>(v + e) : 0.f, acc[e] = 0.f;
    for (int r0 = row0; r0 < p.headdim_k; r0 += ROWS * U) {
      Piece<S, V> s[U];
      float kk[U], qq[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int r = r0 + u * ROWS, at = min(r, p.headdim_k - 1);
        s[u].load(state + (int64_t)at * p.headdim_v, valid);
        kk[u] = ld1<T>(k + at), qq[u] = ld1<T>(q + at);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int r = r0 + u * ROWS;
        if (r < p.headdim_k) {
#pragma unroll
          for (int e = 0; e < V; ++e) {
            s[u].v[e] = __builtin_fmaf(kk[u], vv[e], f * s[u].v[e]);
            acc[e] = __builtin_fmaf(qq[u], s[u].v[e], acc[e]);
          }
          s[u].store(state + (int64_t)r * p.headdim_v, valid);
        }
      }
    }
    // over the rows of a wave, then over the waves
#pragma unroll
    for (int e = 0; e < V; ++e)
#pragma unroll
      for (int step = LANES; step < 64; step *= 2) acc[e] += __shfl_xor(acc[e], step, 64);
    if ((tid & 63) < LANES) {
#pragma unroll
      for (int e = 0; e < V; ++e) sums[tid >> 6][lane * V + e] = acc[e];
    }
    __syncthreads();
    if (tid < LANES * V) {
      const int at = blockIdx.x * LANES * V + tid;
      if (at < p.headdim_v)
        st1<T>(out - col + at, p.scale * (sums[0][tid] + sums[1][tid] + sums[2][tid] + sums[3][tid]));
    }
    __syncthreads();
  }
}

template <typename T, typename S> int run(const LinearAttnStepParams &p, hipStream_t st) {
  constexpr int V = std::is_same_v<S, float> ? 4 : 8;
  const dim3 grid((p.headdim_v + LANES * V - 1) / (LANES * V), p.nheads, std::min(p.batch, 65535));
  lin_step_kernel<T, S><<<grid, kThreads, 0, st>>>(p);
  return hipGetLastError() == hipSuccess ? MAMBA_OK : MAMBA_E_LAUNCH;
}
template <typename T> int run_state(const LinearAttnStepParams &p, hipStream_t st) {
  switch (p.state_dtype) {
    case MAMBA_F32: return run<T, float>(p, st);
    case MAMBA_BF16: return run<T, bf16_t>(p, st);
    default: return run<T, f16_t>(p, st);
  }
}

}  // namespace

extern "C" int linear_attn_state_update(const LinearAttnStepParams *p, mamba_stream_t stream) {
  if (!p || !p->state || !p->q || !p->k || !p->v || !p->log_decay || !p->out) return MAMBA_E_BADARG;
  if (p->batch <= 0 || p->nheads <= 0 || p->nkvheads <= 0 || p->nheads % p->nkvheads != 0 || p->headdim_k <= 0 || p->headdim_v <= 0 ||
      p->state_rows <= 0)
    return MAMBA_E_BADARG;
  if (p->dtype < MAMBA_F32 || p->dtype > MAMBA_F16 || p->state_dtype < MAMBA_F32 || p->state_dtype > MAMBA_F16) return MAMBA_E_BADARG;
  if (!p->state_batch_indices && p->state_rows < p->batch) return MAMBA_E_BADARG;
  if (!(p->scale >= -3.4e38f && p->scale <= 3.4e38f)) return MAMBA_E_BADARG;
  if (p->headdim_k > 256 || p->headdim_v > 256 || p->nheads > 65535) return MAMBA_E_UNSUPPORTED;
  // written by one workgroup while another still reads
  if (p->out == p->q || p->out == p->k || p->out == p->v || p->out == p->state) return MAMBA_E_BADARG;
  hipStream_t st = static_cast<hipStream_t>(stream);
  switch (p->dtype) {
    case MAMBA_F32: return run_state<float>(*p, st);
    case MAMBA_BF16: return run_state<bf16_t>(*p, st);
    default: return run_state<f16_t>(*p, st);
  }
}
