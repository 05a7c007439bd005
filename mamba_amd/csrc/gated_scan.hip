// Gated linear recurrence, one state per channel (gfx950):
//   r = sigmoid(gate_a), i = sigmoid(gate_x), k = rate softplus(decay), log a = -k r, m = sqrt(1 - a^2)
//   h_t = a_t h_{t-1} + m_t i_t x_t
// and its gradients, with g_t = dout_t + a_{t+1} g_{t+1}:
//   dx = g m i,  dgate_x = g m x i (1 - i),  dgate_a = k (1 - r) e,  ddecay = rate sigmoid(decay) sum e,
//   e = g a (a i x / m - h_{t-1}) r,  dinitial = a g at the first position
// (gated_gates.hpp has the terms of one position.)
#include "gated_gates.hpp"
#include "norm_common.hpp"

namespace {

// Where the sequences of a row lie: position t belongs to sequence `s`, which ends at `next`; outside of all of them
// `in` is false.
struct SeqWalk {
  const int32_t *cu;
  int nseq, s, next;
  DEVI SeqWalk(const int32_t *c, int n) : cu(c), nseq(n), s(-1), next(c[0]) {}
  DEVI bool first_at(int t) {  // for t = 0, 1, 2, ...: whether a sequence starts at t
    bool f = false;
    while (t >= next && s < nseq) {
      f = true;
      ++s;
      next = s < nseq ? cu[s + 1] : INT32_MAX;
    }
    return f && s < nseq;
  }
  DEVI bool in() const { return s >= 0 && s < nseq; }
};

template <typename T> __global__ __launch_bounds__(64) void gated_fwd_kernel(const GatedScanParams p) {
  const int c = blockIdx.x * 64 + threadIdx.x, b = blockIdx.y;
  if (c >= p.dim) return;
  const T *xp = static_cast<const T *>(p.x) + b * p.x_bs + c;
  const T *ap = static_cast<const T *>(p.gate_a) + b * p.gate_a_bs + c;
  const T *gp = static_cast<const T *>(p.gate_x) + b * p.gate_x_bs + c;
  T *op = static_cast<T *>(p.out) + b * p.out_bs + c;
  const float k = decay_rate(p, c);
  auto init = [&](int s) { return p.initial_states ? p.initial_states[(int64_t)s * p.dim + c] : 0.f; };
  auto final = [&](int s, float h) {
    if (p.final_states) p.final_states[(int64_t)s * p.dim + c] = h;
  };
  float h = 0.f;
  if (p.nseq == 0) {
    h = init(b);
    for (int t = 0; t < p.seqlen; ++t) {
      const Gates q(ld1<T>(ap + t * p.gate_a_ls), ld1<T>(gp + t * p.gate_x_ls), k);
      h = __builtin_fmaf(q.a, h, q.m * q.i * ld1<T>(xp + t * p.x_ls));
      st1<T>(op + t * p.out_ls, h);
    }
    final(b, h);
    return;
  }
  for (int s = 0; s < p.nseq; ++s)
    if (p.cu_seqlens[s + 1] <= p.cu_seqlens[s]) final(s, init(s));
  SeqWalk w(p.cu_seqlens, p.nseq);
  for (int t = 0; t < p.seqlen; ++t) {
    if (w.first_at(t)) h = init(w.s);
    if (w.in()) {
      const Gates q(ld1<T>(ap + t * p.gate_a_ls), ld1<T>(gp + t * p.gate_x_ls), k);
      h = __builtin_fmaf(q.a, h, q.m * q.i * ld1<T>(xp + t * p.x_ls));
      if (t + 1 == w.next) final(w.s, h);
    } else {
      h = 0.f;
    }
    st1<T>(op + t * p.out_ls, h);
  }
}

// ws: h before every position, fp32 (batch, seqlen, dim); then the sequence of every position (int32, packed rows
// only: -1 outside), then one row of ddecay terms per batch row.
template <typename T> __global__ __launch_bounds__(64) void gated_bwd_kernel(const GatedScanParams p, float *hbuf, float *parts) {
  const int c = blockIdx.x * 64 + threadIdx.x, b = blockIdx.y;
  if (c >= p.dim) return;
  const T *xp = static_cast<const T *>(p.x) + b * p.x_bs + c;
  const T *ap = static_cast<const T *>(p.gate_a) + b * p.gate_a_bs + c;
  const T *gp = static_cast<const T *>(p.gate_x) + b * p.gate_x_bs + c;
  const T *dop = static_cast<const T *>(p.dout) + b * p.dout_bs + c;
  T *dxp = static_cast<T *>(p.dx) + b * p.dx_bs + c;
  T *dap = static_cast<T *>(p.dgate_a) + b * p.dgate_a_bs + c;
  T *dgp = static_cast<T *>(p.dgate_x) + b * p.dgate_x_bs + c;
  float *hp = hbuf + (int64_t)b * p.seqlen * p.dim + c;
  const float k = decay_rate(p, c);
  auto init = [&](int s) { return p.initial_states ? p.initial_states[(int64_t)s * p.dim + c] : 0.f; };
  auto dfinal = [&](int s) { return p.dfinal_states ? p.dfinal_states[(int64_t)s * p.dim + c] : 0.f; };
  auto dinit = [&](int s, float v) {
    if (p.dinitial_states) p.dinitial_states[(int64_t)s * p.dim + c] = v;
  };
  const int nseq = p.nseq;
  float h = nseq ? 0.f : init(b), sum = 0.f;
  if (nseq) {
    for (int s = 0; s < nseq; ++s)
      if (p.cu_seqlens[s + 1] <= p.cu_seqlens[s]) dinit(s, dfinal(s));
  }
  auto seq_of = [&](int t) {  // the last sequence that starts at or before t, -1 outside
    int lo = -1, hi = nseq + 1;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (p.cu_seqlens[mid] <= t) lo = mid;
      else hi = mid;
    }
    return lo >= 0 && lo < nseq ? lo : -1;
  };
  for (int t = 0; t < p.seqlen; ++t) {
    const int s = nseq ? seq_of(t) : b;
    if (nseq && (s < 0 || p.cu_seqlens[s] == t)) h = s < 0 ? 0.f : init(s);
    hp[(int64_t)t * p.dim] = h;
    if (s >= 0) {
      const Gates q(ld1<T>(ap + t * p.gate_a_ls), ld1<T>(gp + t * p.gate_x_ls), k);
      h = __builtin_fmaf(q.a, h, q.m * q.i * ld1<T>(xp + t * p.x_ls));
    }
  }
  float carry = nseq ? 0.f : dfinal(b);
  for (int t = p.seqlen - 1; t >= 0; --t) {
    const int s = nseq ? seq_of(t) : b;
    if (s < 0) {
      st1<T>(dxp + t * p.dx_ls, 0.f);
      st1<T>(dap + t * p.dgate_a_ls, 0.f);
      st1<T>(dgp + t * p.dgate_x_ls, 0.f);
      continue;
    }
    if (nseq && p.cu_seqlens[s + 1] == t + 1) carry = dfinal(s);
    const float x = ld1<T>(xp + t * p.x_ls);
    const Gates q(ld1<T>(ap + t * p.gate_a_ls), ld1<T>(gp + t * p.gate_x_ls), k);
    const float g = ld1<T>(dop + t * p.dout_ls) + carry;
    float dx, dga, dgx, e;
    q.grads(g, hp[(int64_t)t * p.dim], x, k, dx, dga, dgx, e);
    st1<T>(dxp + t * p.dx_ls, dx);
    st1<T>(dap + t * p.dgate_a_ls, dga);
    st1<T>(dgp + t * p.dgate_x_ls, dgx);
    sum += e;
    carry = q.a * g;
    if (nseq ? p.cu_seqlens[s] == t : t == 0) dinit(s, carry);
  }
  parts[(int64_t)b * p.dim + c] = sum * decay_slope(p, c);
}

int64_t words(const GatedScanParams &p) { return (int64_t)p.batch * p.seqlen * p.dim; }

bool shapes_ok(const GatedScanParams *p) {
  if (!p || p->batch <= 0 || p->seqlen <= 0 || p->dim <= 0 || p->nseq < 0) return false;
  if (p->nseq > 0 && p->batch != 1) return false;
  if (!(p->rate >= 0.f && p->rate <= 3.4e38f)) return false;
  return p->dtype >= MAMBA_F32 && p->dtype <= MAMBA_F16 && p->decay_dtype >= MAMBA_F32 && p->decay_dtype <= MAMBA_F16;
}
int check(const GatedScanParams *p, bool bwd) {
  if (!shapes_ok(p)) return MAMBA_E_BADARG;
  if (!p->x || !p->gate_a || !p->gate_x || !p->decay || !p->ckpt || (p->nseq > 0) != (p->cu_seqlens != nullptr))
    return MAMBA_E_BADARG;
  if (!aligned16(p->ckpt)) return MAMBA_E_BADARG;
  if (!bwd && !p->out) return MAMBA_E_BADARG;
  if (bwd && (!p->dout || !p->dx || !p->dgate_a || !p->dgate_x || !p->ddecay || !p->ws || !aligned16(p->ws)))
    return MAMBA_E_BADARG;
  if (p->batch > 65535) return MAMBA_E_UNSUPPORTED;
  return MAMBA_OK;
}

template <typename T> int run_fwd(const GatedScanParams &p, hipStream_t st) {
  gated_fwd_kernel<T><<<dim3((p.dim + 63) / 64, p.batch), 64, 0, st>>>(p);
  return hipGetLastError() == hipSuccess ? MAMBA_OK : MAMBA_E_LAUNCH;
}
template <typename T> int run_bwd(const GatedScanParams &p, hipStream_t st) {
  float *h = static_cast<float *>(p.ws), *parts = h + words(p);
  gated_bwd_kernel<T><<<dim3((p.dim + 63) / 64, p.batch), 64, 0, st>>>(p, h, parts);
  if (hipGetLastError() != hipSuccess) return MAMBA_E_LAUNCH;
  ReduceJobs jobs{};
  jobs.part[0] = parts, jobs.out[0] = p.ddecay;
  return launch_reduce(jobs, 1, p.decay_dtype, p.batch, p.dim, st);
}

// ------------------------------------------------------------------ one position
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
    const Gates q(ld1<T>(ap + e), ld1<T>(gp + e), k);
    const float h = __builtin_fmaf(q.a, ld1<S>(sp + e), q.m * q.i * ld1<T>(xp + e));
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

extern "C" int64_t gated_scan_ckpt_bytes(const GatedScanParams *p) { return shapes_ok(p) ? 16 : MAMBA_E_BADARG; }
extern "C" int64_t gated_scan_bwd_ws_bytes(const GatedScanParams *p) {
  return shapes_ok(p) ? (words(*p) + (int64_t)p->batch * p->dim) * 4 : MAMBA_E_BADARG;
}
extern "C" int gated_scan_fwd(const GatedScanParams *p, mamba_stream_t stream) {
  if (const int rc = check(p, false)) return rc;
  hipStream_t st = static_cast<hipStream_t>(stream);
  switch (p->dtype) {
    case MAMBA_F32: return run_fwd<float>(*p, st);
    case MAMBA_BF16: return run_fwd<bf16_t>(*p, st);
    default: return run_fwd<f16_t>(*p, st);
  }
}
extern "C" int gated_scan_bwd(const GatedScanParams *p, mamba_stream_t stream) {
  if (const int rc = check(p, true)) return rc;
  hipStream_t st = static_cast<hipStream_t>(stream);
  switch (p->dtype) {
    case MAMBA_F32: return run_bwd<float>(*p, st);
    case MAMBA_BF16: return run_bwd<bf16_t>(*p, st);
    default: return run_bwd<f16_t>(*p, st);
  }
}
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
