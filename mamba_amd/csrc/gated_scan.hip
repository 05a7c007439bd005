// Gated linear recurrence, one state per channel (gfx950):
//   r = sigmoid(gate_a), i = sigmoid(gate_x), k = rate softplus(decay), log a = -k r, m = sqrt(1 - a^2)
//   h_t = a_t h_{t-1} + m_t i_t x_t
// and its gradients, with g_t = dout_t + a_{t+1} g_{t+1}:
//   dx = g m i,  dgate_x = dx x (1 - i),  dgate_a = k (1 - r) e,  ddecay = rate sigmoid(decay) sum e,
//   e = g a (a i x r / m - r h_{t-1}),  dinitial = a g at the first position
// The forward pass moves 4 tensors and the backward pass 7: both are bound by memory (about 80 vector slots per element
// backward, half of them the six quarter-rate instructions of a position, are below half of the time the bytes take).
// gated_tile.hpp says how a row is cut.  The forward pass leaves the state that enters every tile of the backward
// pass, which then forms its own states again: one float per tile and channel instead of the states in 32 bits.
#include "gated_tile.hpp"
#include "norm_common.hpp"

namespace {

// The decay's constants of a lane's channels.
template <int V> struct Rates {
  Vec<V> d, k, k2;
  DEVI Rates(const GatedScanParams &p, int c) {
#pragma unroll
    for (int e = 0; e < V; ++e) d[e] = ld_param(p.decay, p.decay_dtype, min(c + e, p.dim - 1));
  }
  DEVI void form(float rate) {  // once the rows have been asked for
#pragma unroll
    for (int e = 0; e < V; ++e) k[e] = rate * softplus_exact(d[e]), k2[e] = -k[e] * kLog2e;
  }
};

template <typename T, int V, bool WHOLE, bool PACKED, int R, int NW>
__global__ __launch_bounds__(NW * 64) void gated_fwd_kernel(const GatedScanParams p, const Chain q, float *ckpt, int ck_rows, int ck_tiles) {
  __shared__ WaveSteps<V, NW> steps;
  __shared__ Vec<V> enter[64];
  __shared__ int ticket;
  const int cgroups = (p.dim + 64 * V - 1) / (64 * V), nchains = cgroups * p.batch;
  const int chain = blockIdx.x % nchains, b = chain / cgroups;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), L = p.seqlen;
  const Lane<T, V, WHOLE> at((chain % cgroups) * (64 * V) + lane * V, p.dim);
  const int n = take_tile(q, chain, &ticket);
  const int t0 = (n * NW + wave) * R, rows = min(max(L - t0, 0), R);
  Rates<V> rate(p, at.c);
  const T *xp = static_cast<const T *>(p.x) + b * p.x_bs;
  const T *ap = static_cast<const T *>(p.gate_a) + b * p.gate_a_bs;
  const T *gp = static_cast<const T *>(p.gate_x) + b * p.gate_x_bs;
  Raw<T, V> x[R], ga[R], gx[R];
#pragma unroll
  for (int j = 0; j < R; ++j) {
    const int64_t t = min(t0 + j, L - 1);
    ga[j] = at.load(ap + t * p.gate_a_ls);
    gx[j] = at.load(gp + t * p.gate_x_ls);
    x[j] = at.load(xp + t * p.x_ls);
  }
  SeqRows<PACKED ? R : 1> rowsof(PACKED ? p.cu_seqlens : nullptr, PACKED ? p.nseq : -1, t0, L);
  rate.form(p.rate);
  Step<V> pos[R], own = no_step<V>();
#pragma unroll
  for (int j = 0; j < R; ++j) {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const Gates g(ga[j].get(e), gx[j].get(e), rate.k[e], rate.k2[e]);
      pos[j].a[e] = PACKED ? fmaxf(g.a, kTiny) : g.a;
      pos[j].b[e] = g.m() * g.i * x[j].get(e);
    }
    if constexpr (PACKED) {
      if (!(rowsof.in >> j & 1)) {
        pos[j].a = pos[j].b = vec_of<V>(0.f);
      } else if (rowsof.start >> j & 1) {
        if (p.initial_states) pos[j].b = apply<false>(pos[j], at.load_state(p.initial_states + (int64_t)rowsof.seq[j] * p.dim));
        pos[j].a = vec_of<V>(0.f);
      }
    } else {
      if (j >= rows) pos[j] = no_step<V>();
    }
    own = then<PACKED>(own, pos[j]);
  }
  steps.put(wave, lane, own);
  lds_barrier();
  Step<V> before = no_step<V>();
  for (int w = 0; w < wave; ++w) before = then<PACKED>(before, steps.get(w, lane));
  if (wave == NW - 1) leave_step(q, chain, n, lane, then<PACKED>(before, own));
  if (wave == 0) {
    Vec<V> first = vec_of<V>(0.f);
    if (!PACKED && p.initial_states) first = at.load_state(p.initial_states + (int64_t)b * p.dim);
    enter[lane] = entering<PACKED>(q, chain, n, lane, first);
  }
  lds_barrier();
  Vec<V> h = apply<PACKED>(before, enter[lane]);
  if (wave == NW - 1) leave_state(q, chain, n, lane, apply<PACKED>(own, h));
  if (t0 % ck_rows == 0 && rows > 0) {
    float *ck = ckpt + (((int64_t)chain * ck_tiles + t0 / ck_rows) * 64 + lane) * V;
#pragma unroll
    for (int e = 0; e < V; ++e) ck[e] = h[e];
  }
  T *op = static_cast<T *>(p.out) + b * p.out_bs;
#pragma unroll
  for (int j = 0; j < R; ++j) {
    h = apply<PACKED>(pos[j], h);
    if (j < rows) at.store(op + (int64_t)(t0 + j) * p.out_ls, h);
    if constexpr (PACKED) {
      if (p.final_states && (rowsof.last >> j & 1)) at.store_state(p.final_states + (int64_t)rowsof.seq[j] * p.dim, h);
    }
  }
  if (!PACKED && p.final_states && t0 < L && t0 + R >= L) at.store_state(p.final_states + (int64_t)b * p.dim, h);
  if constexpr (PACKED) {
    if (p.final_states && n == 0)
      empty_sequences(p.cu_seqlens, p.nseq, L, [&](int s) {
        const int64_t o = (int64_t)s * p.dim;
        at.store_state(p.final_states + o, p.initial_states ? at.load_state(p.initial_states + o) : vec_of<V>(0.f));
      });
  }
}

// Tiles from the last one on: what enters a tile is a_t g_t of the position behind it.
template <typename T, int V, bool WHOLE, bool PACKED, int R, int NW>
__global__ __launch_bounds__(NW * 64) void gated_bwd_kernel(const GatedScanParams p, const Chain q, const float *ckpt, float *parts) {
  __shared__ WaveSteps<V, NW> steps, back;
  __shared__ Vec<V> enter[64];
  __shared__ int ticket;
  const int cgroups = (p.dim + 64 * V - 1) / (64 * V), nchains = cgroups * p.batch;
  const int chain = blockIdx.x % nchains, b = chain / cgroups;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), L = p.seqlen;
  const Lane<T, V, WHOLE> at((chain % cgroups) * (64 * V) + lane * V, p.dim);
  const int n = take_tile(q, chain, &ticket), tile = q.ntiles - 1 - n;
  const int t0 = (tile * NW + wave) * R, rows = min(max(L - t0, 0), R);
  Rates<V> rate(p, at.c);
  Vec<V> h;
  const float *ck = ckpt + (((int64_t)chain * q.ntiles + tile) * 64 + lane) * V;
#pragma unroll
  for (int e = 0; e < V; ++e) h[e] = ck[e];
  const T *xp = static_cast<const T *>(p.x) + b * p.x_bs;
  const T *ap = static_cast<const T *>(p.gate_a) + b * p.gate_a_bs;
  const T *gp = static_cast<const T *>(p.gate_x) + b * p.gate_x_bs;
  const T *dp = static_cast<const T *>(p.dout) + b * p.dout_bs;
  Raw<T, V> x[R], ga[R], gx[R], dout[R];
#pragma unroll
  for (int j = 0; j < R; ++j) {
    const int64_t t = min(t0 + j, L - 1);
    ga[j] = at.load(ap + t * p.gate_a_ls);
    gx[j] = at.load(gp + t * p.gate_x_ls);
    x[j] = at.load(xp + t * p.x_ls);
    dout[j] = at.load(dp + t * p.dout_ls);
  }
  SeqRows<PACKED ? R : 1> rowsof(PACKED ? p.cu_seqlens : nullptr, PACKED ? p.nseq : -1, t0, L);
  auto starts = [&](int j) { return PACKED && (rowsof.start >> j & 1); };
  auto ends = [&](int j) { return PACKED && (rowsof.last >> j & 1); };
  auto counts = [&](int j) { return PACKED ? (rowsof.in >> j & 1) != 0 : j < rows; };
  auto state_of = [&](int j) { return (int64_t)rowsof.seq[PACKED ? j : 0] * p.dim; };
  auto initial = [&](int j) { return p.initial_states ? at.load_state(p.initial_states + state_of(j)) : vec_of<V>(0.f); };
  rate.form(p.rate);
  // of every position: a, r, i, m, x, the gradient that arrives there, and f: first r / m, then e / g
  Vec<V> a[R], r[R], i[R], m[R], f[R], xs[R], d[R];
  Step<V> own = no_step<V>();
#pragma unroll
  for (int j = 0; j < R; ++j) {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const Gates g(ga[j].get(e), gx[j].get(e), rate.k[e], rate.k2[e]);
      const float im = g.im();
      a[j][e] = PACKED ? fmaxf(g.a, kTiny) : g.a;
      r[j][e] = g.r, i[j][e] = g.i, m[j][e] = g.m2 * im, f[j][e] = g.r * im;
      xs[j][e] = x[j].get(e), d[j][e] = dout[j].get(e);
    }
    if (!counts(j)) {
      // a position past the row hands everything on, one outside of the sequences nothing
      a[j] = vec_of<V>(PACKED ? 0.f : 1.f);
      r[j] = m[j] = i[j] = f[j] = xs[j] = d[j] = vec_of<V>(0.f);
    }
    if (ends(j) && p.dfinal_states) {
      const Vec<V> v = at.load_state(p.dfinal_states + state_of(j));
#pragma unroll
      for (int e = 0; e < V; ++e) d[j][e] += v[e];
    }
    Step<V> s;
    s.a = a[j];
#pragma unroll
    for (int e = 0; e < V; ++e) s.b[e] = m[j][e] * i[j][e] * xs[j][e];
    if (starts(j)) {
      s.b = apply<false>(s, initial(j));
      s.a = vec_of<V>(0.f);
    }
    own = then<PACKED>(own, s);
  }
  Step<V> rev = no_step<V>();
#pragma unroll
  for (int j = R - 1; j >= 0; --j) {
    const bool cut = ends(j), out = PACKED && !counts(j);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float g = cut ? d[j][e] : rev.b[e] + d[j][e];
      rev.a[e] = cut || out ? 0.f : factor1<PACKED>(rev.a[e], a[j][e]);
      rev.b[e] = out ? 0.f : a[j][e] * g;
    }
  }
  steps.put(wave, lane, own);
  back.put(wave, lane, rev);
  lds_barrier();
  Step<V> behind = no_step<V>();
  for (int w = NW - 1; w > wave; --w) behind = then<PACKED>(behind, back.get(w, lane));
  if (wave == 0) leave_step(q, chain, n, lane, then<PACKED>(behind, rev));
  for (int w = 0; w < wave; ++w) h = apply<PACKED>(steps.get(w, lane), h);
#pragma unroll
  for (int j = 0; j < R; ++j) {
    if (starts(j)) h = initial(j);
    if (PACKED && !counts(j)) h = vec_of<V>(0.f);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float ix = i[j][e] * xs[j][e];
      f[j][e] = a[j][e] * __builtin_fmaf(a[j][e] * ix, f[j][e], -r[j][e] * h[e]);
      h[e] = __builtin_fmaf(a[j][e], h[e], m[j][e] * ix);
    }
  }
  if (wave == NW - 1) {
    Vec<V> first = vec_of<V>(0.f);
    if (!PACKED && p.dfinal_states) first = at.load_state(p.dfinal_states + (int64_t)b * p.dim);
    enter[lane] = entering<PACKED>(q, chain, n, lane, first);
  }
  lds_barrier();
  Vec<V> carry = apply<PACKED>(behind, enter[lane]), sum = vec_of<V>(0.f);
  if (wave == 0) leave_state(q, chain, n, lane, apply<PACKED>(rev, carry));
  T *dxp = static_cast<T *>(p.dx) + b * p.dx_bs;
  T *dap = static_cast<T *>(p.dgate_a) + b * p.dgate_a_bs;
  T *dgp = static_cast<T *>(p.dgate_x) + b * p.dgate_x_bs;
#pragma unroll
  for (int j = R - 1; j >= 0; --j) {
    Vec<V> dx, da, dg;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      float g = ends(j) ? d[j][e] : d[j][e] + carry[e];
      if (PACKED && !counts(j)) g = 0.f;
      const float ee = g * f[j][e];
      dx[e] = g * m[j][e] * i[j][e];
      da[e] = rate.k[e] * (1.f - r[j][e]) * ee;
      dg[e] = dx[e] * xs[j][e] * (1.f - i[j][e]);
      if (counts(j)) sum[e] += ee;
      carry[e] = a[j][e] * g;
    }
    if (j < rows) {
      const int64_t t = t0 + j;
      at.store(dxp + t * p.dx_ls, dx);
      at.store(dap + t * p.dgate_a_ls, da);
      at.store(dgp + t * p.dgate_x_ls, dg);
    }
    if (starts(j) && p.dinitial_states) at.store_state(p.dinitial_states + state_of(j), carry);
  }
  if (!PACKED && t0 == 0 && p.dinitial_states) at.store_state(p.dinitial_states + (int64_t)b * p.dim, carry);
  if constexpr (PACKED) {
    if (p.dinitial_states && tile == 0)
      empty_sequences(p.cu_seqlens, p.nseq, L, [&](int s) {
        const int64_t o = (int64_t)s * p.dim;
        at.store_state(p.dinitial_states + o, p.dfinal_states ? at.load_state(p.dfinal_states + o) : vec_of<V>(0.f));
      });
  }
  // the terms of ddecay over the tile (the steps were read before the last barrier)
  steps.put(wave, lane, Step<V>{sum, sum});
  lds_barrier();
  if (wave == 0) {
    for (int w = 1; w < NW; ++w) {
      const Vec<V> s = steps.get(w, lane).a;
#pragma unroll
      for (int e = 0; e < V; ++e) sum[e] += s[e];
    }
#pragma unroll
    for (int e = 0; e < V; ++e) sum[e] *= p.rate / (1.f + expf(-rate.d[e]));
    at.store_state(parts + ((int64_t)b * q.ntiles + tile) * p.dim, sum);
  }
}

// ------------------------------------------------------------------ host side
constexpr int kV = 2, kFwdRows = 16, kFwdWaves = 4, kBwdRows = 4, kBwdWaves = 8, kGroup = 8;
constexpr int kTileChannels = 64 * kV;

// Tiles of one pass and what its chains need in memory: the tickets and words, cleared before the launch, lie at the
// start of the buffer, `tail` behind them.
struct Plan {
  int cgroups, ntiles, group, ngroups;
  int64_t chains, words, head;  // head: bytes before the tail
  Plan(const GatedScanParams &p, int tile_rows) {
    cgroups = (p.dim + kTileChannels - 1) / kTileChannels;
    chains = (int64_t)p.batch * cgroups;
    ntiles = (int)(((int64_t)p.seqlen + tile_rows - 1) / tile_rows);
    group = group_of(chains, ntiles);
    ngroups = (ntiles + group - 1) / group;
    words = ntiles > 1 ? chains * (ntiles + ngroups) * kTileChannels : 0;
    head = ntiles > 1 ? (chains * 4 + 15) / 16 * 16 + words * 8 : 0;
  }
  static int group_of(int64_t chains, int ntiles) {
    (void)chains;
    return min(ntiles, kGroup);
  }
  Chain chain(void *buf) const {
    Chain q;
    q.tickets = static_cast<uint32_t *>(buf);
    q.steps = reinterpret_cast<uint64_t *>(static_cast<char *>(buf) + (chains * 4 + 15) / 16 * 16);
    q.states = q.steps + chains * ntiles * kTileChannels;
    q.ntiles = ntiles, q.group = group, q.ngroups = ngroups;
    return q;
  }
  bool fits() const { return chains * ntiles <= 0x7fffffff; }
};
Plan fwd_plan(const GatedScanParams &p) { return Plan(p, kFwdRows * kFwdWaves); }
Plan bwd_plan(const GatedScanParams &p) { return Plan(p, kBwdRows * kBwdWaves); }

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
  // positions and tiles are counted in 32 bits
  if (p->seqlen > 0x7fffffff - 4096 || p->nseq > 0x7fffffff - 64 || !fwd_plan(*p).fits() || !bwd_plan(*p).fits()) return MAMBA_E_UNSUPPORTED;
  return MAMBA_OK;
}

// f(T{}, even, packed) with the call's types as compile-time values
template <typename F> int with_forms(const GatedScanParams &p, F f) {
  auto forms = [&](auto t) {
    const bool even = p.dim % kV == 0;
    if (p.nseq > 0) return even ? f(t, std::true_type{}, std::true_type{}) : f(t, std::false_type{}, std::true_type{});
    return even ? f(t, std::true_type{}, std::false_type{}) : f(t, std::false_type{}, std::false_type{});
  };
  switch (p.dtype) {
    case MAMBA_F32: return forms(float{});
    case MAMBA_BF16: return forms(bf16_t{});
    default: return forms(f16_t{});
  }
}

}  // namespace

extern "C" int64_t gated_scan_ckpt_bytes(const GatedScanParams *p) {
  if (!shapes_ok(p)) return MAMBA_E_BADARG;
  const Plan f = fwd_plan(*p), w = bwd_plan(*p);
  return f.head + w.chains * w.ntiles * kTileChannels * 4;
}
extern "C" int64_t gated_scan_bwd_ws_bytes(const GatedScanParams *p) {
  if (!shapes_ok(p)) return MAMBA_E_BADARG;
  const Plan w = bwd_plan(*p);
  return w.head + (int64_t)p->batch * w.ntiles * p->dim * 4;
}

extern "C" int gated_scan_fwd(const GatedScanParams *p, mamba_stream_t stream) {
  if (const int rc = check(p, false)) return rc;
  const Plan plan = fwd_plan(*p);
  if (plan.head > 0)
    if (const int rc = mamba_hip_zero(p->ckpt, plan.head, stream)) return rc;
  float *ck = reinterpret_cast<float *>(static_cast<char *>(p->ckpt) + plan.head);
  return with_forms(*p, [&](auto t, auto even, auto packed) {
    gated_fwd_kernel<decltype(t), kV, even.value, packed.value, kFwdRows, kFwdWaves>
        <<<dim3((unsigned)(plan.chains * plan.ntiles)), dim3(kFwdWaves * 64), 0, static_cast<hipStream_t>(stream)>>>(
            *p, plan.chain(p->ckpt), ck, kBwdRows * kBwdWaves, bwd_plan(*p).ntiles);
    return hipGetLastError() == hipSuccess ? MAMBA_OK : MAMBA_E_LAUNCH;
  });
}
extern "C" int gated_scan_bwd(const GatedScanParams *p, mamba_stream_t stream) {
  if (const int rc = check(p, true)) return rc;
  const Plan plan = bwd_plan(*p);
  if (plan.head > 0)
    if (const int rc = mamba_hip_zero(p->ws, plan.head, stream)) return rc;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const float *ck = reinterpret_cast<const float *>(static_cast<const char *>(p->ckpt) + fwd_plan(*p).head);
  float *parts = reinterpret_cast<float *>(static_cast<char *>(p->ws) + plan.head);
  const int rc = with_forms(*p, [&](auto t, auto even, auto packed) {
    gated_bwd_kernel<decltype(t), kV, even.value, packed.value, kBwdRows, kBwdWaves>
        <<<dim3((unsigned)(plan.chains * plan.ntiles)), dim3(kBwdWaves * 64), 0, st>>>(*p, plan.chain(p->ws), ck, parts);
    return hipGetLastError() == hipSuccess ? MAMBA_OK : MAMBA_E_LAUNCH;
  });
  if (rc != MAMBA_OK) return rc;
  ReduceJobs jobs{};
  jobs.part[0] = parts, jobs.out[0] = p->ddecay;
  return launch_reduce(jobs, 1, p->decay_dtype, p->batch * plan.ntiles, p->dim, st);
}
