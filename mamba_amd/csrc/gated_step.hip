// One position of the gated linear recurrence (gated_scan.hip has the formulas), the states updated in place (gfx950).
#include "gated_gates.hpp"

namespace {

// V channels per thread; blockIdx.y is the batch entry.
template <typename T, typename S, int V, bool VEC>
__global__ __launch_bounds__(256) void gated_step_kernel(const GatedStepParams p) {
  const int c = (blockIdx.x * 256 + threadIdx.x) * V, b = blockIdx.y;
  if (c >= p.dim) return;
  const int row = p.state_batch_indices ? p.state_batch_indices[b] : b;
  T *op = static_cast<T *>(p.out) + b * p.out_rs + c;
  const int n = min(V, p.dim - c);
  if (row < 0 || row >= p.state_rows) {
    for (int e = 0; e < n; ++e) st1<T>(op + e, 0.f);
    return;
  }
  const T *xp = static_cast<const T *>(p.x) + b * p.x_rs + c;
  const T *ap = static_cast<const T *>(p.gate_a) + b * p.gate_a_rs + c;
  const T *gp = static_cast<const T *>(p.gate_x) + b * p.gate_x_rs + c;
  S *sp = static_cast<S *>(p.state) + row * p.state_rs + c;
  for (int e = 0; e < n; ++e) {
    const float k = p.rate * softplus_exact(ld_param(p.decay, p.decay_dtype, c + e));
    const Gates q(ld1<T>(ap + e), ld1<T>(gp + e), k, -k * kLog2e);
    const float h = __builtin_fmaf(q.a, ld1<S>(sp + e), q.m() * q.i * ld1<T>(xp + e));
    st1<S>(sp + e, h);
    st1<T>(op + e, h);
  }
}

template <typename T, typename S> int run_step(const GatedStepParams &p, hipStream_t st) {
  gated_step_kernel<T, S, 1, false><<<dim3((p.dim + 255) / 256, p.batch), 256, 0, st>>>(p);
  return hipGetLastError() == hipSuccess ? MAMBA_OK : MAMBA_E_LAUNCH;
}
template <typename T> int step_state(const GatedStepParams &p, hipStream_t st) {
  switch (p.state_dtype) {
    case MAMBA_F32: return run_step<T, float>(p, st);
    case MAMBA_BF16: return run_step<T, bf16_t>(p, st);
    default: return run_step<T, f16_t>(p, st);
  }
}

}  // namespace

extern "C" int gated_state_update(const GatedStepParams *p, mamba_stream_t stream) {
  if (!p || !p->state || !p->x || !p->gate_a || !p->gate_x || !p->decay || !p->out) return MAMBA_E_BADARG;
  if (p->batch <= 0 || p->dim <= 0 || p->state_rows <= 0) return MAMBA_E_BADARG;
  if (!(p->rate >= 0.f && p->rate <= 3.4e38f)) return MAMBA_E_BADARG;
  if (p->dtype < MAMBA_F32 || p->dtype > MAMBA_F16) return MAMBA_E_BADARG;
  if (!p->state_batch_indices && p->state_rows < p->batch) return MAMBA_E_BADARG;
  if (p->state_dtype < MAMBA_F32 || p->state_dtype > MAMBA_F16 || p->decay_dtype < MAMBA_F32 || p->decay_dtype > MAMBA_F16)
    return MAMBA_E_BADARG;
  if (p->batch > 65535) return MAMBA_E_UNSUPPORTED;
  hipStream_t st = static_cast<hipStream_t>(stream);
  switch (p->dtype) {
    case MAMBA_F32: return step_state<float>(*p, st);
    case MAMBA_BF16: return step_state<bf16_t>(*p, st);
    default: return step_state<f16_t>(*p, st);
  }
}
