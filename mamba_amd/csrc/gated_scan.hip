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

template <typename T, bool EVEN, bool PACKED, int R, int NW>
__global__ __launch_bounds__(NW * 64) void gated_fwd_kernel(const GatedScanParams p, const Chain q, float *ckpt, int ck_rows, int ck_tiles) {
  __shared__ f32x4 steps[NW][64];
  __shared__ f32x2 enter[64];
  __shared__ int ticket;
  const int cgroups = (p.dim + kTileChannels - 1) / kTileChannels, nchains = cgroups * p.batch;
  const int chain = blockIdx.x % nchains, b = chain / cgroups;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), cl = lane * 2;
  const int c = (chain % cgroups) * kTileChannels + cl, L = p.seqlen;
  const Lane<T, EVEN> at(c, p.dim);
  const int n = take_tile(q, chain, &ticket);
  const int t0 = (n * NW + wave) * R, rows = min(max(L - t0, 0), R);
  const float d0 = ld_param(p.decay, p.decay_dtype, min(c, p.dim - 1)), d1 = ld_param(p.decay, p.decay_dtype, min(c + 1, p.dim - 1));
  const T *xp = static_cast<const T *>(p.x) + b * p.x_bs;
  const T *ap = static_cast<const T *>(p.gate_a) + b * p.gate_a_bs;
  const T *gp = static_cast<const T *>(p.gate_x) + b * p.gate_x_bs;
  Pair<T> x[R], ga[R], gx[R];
#pragma unroll
  for (int j = 0; j < R; ++j) {
    const int64_t t = min(t0 + j, L - 1);
    ga[j] = at.load(ap + t * p.gate_a_ls);
    gx[j] = at.load(gp + t * p.gate_x_ls);
    x[j] = at.load(xp + t * p.x_ls);
  }
  SeqRows<PACKED ? R : 1> rowsof(PACKED ? p.cu_seqlens : nullptr, PACKED ? p.nseq : -1, t0, L);
  const float k0 = p.rate * softplus_exact(d0), k1 = p.rate * softplus_exact(d1);
  f32x2 a[R], bt[R];
  Step own = no_step();
#pragma unroll
  for (int j = 0; j < R; ++j) {
    const Gates q0(ga[j].lo(), gx[j].lo(), k0), q1(ga[j].hi(), gx[j].hi(), k1);
    a[j] = PACKED ? f32x2{fmaxf(q0.a, kTiny), fmaxf(q1.a, kTiny)} : f32x2{q0.a, q1.a};
    bt[j] = f32x2{q0.m * q0.i * x[j].lo(), q1.m * q1.i * x[j].hi()};
    if constexpr (PACKED) {
      if (!(rowsof.in >> j & 1)) {
        a[j] = bt[j] = f32x2{0.f, 0.f};
      } else if (rowsof.start >> j & 1) {
        if (p.initial_states) {
          const f32x2 h = at.load_state(p.initial_states + (int64_t)rowsof.seq[j] * p.dim, c);
          bt[j] = f32x2{__builtin_fmaf(a[j].x, h.x, bt[j].x), __builtin_fmaf(a[j].y, h.y, bt[j].y)};
        }
        a[j] = f32x2{0.f, 0.f};
      }
    } else {
      if (j >= rows) a[j] = f32x2{1.f, 1.f}, bt[j] = f32x2{0.f, 0.f};
    }
    own = then<PACKED>(own, Step{a[j], bt[j]});
  }
  steps[wave][lane] = f32x4{own.a.x, own.a.y, own.b.x, own.b.y};
  lds_barrier();
  Step before = no_step();
  for (int w = 0; w < wave; ++w) {
    const f32x4 s = steps[w][lane];
    before = then<PACKED>(before, Step{f32x2{s.x, s.y}, f32x2{s.z, s.w}});
  }
  if (wave == NW - 1) leave_step(q, chain, n, cl, then<PACKED>(before, own));
  if (wave == 0) {
    f32x2 first = {0.f, 0.f};
    if (!PACKED && p.initial_states) first = at.load_state(p.initial_states + (int64_t)b * p.dim, c);
    enter[lane] = entering<PACKED>(q, chain, n, cl, first);
  }
  lds_barrier();
  f32x2 h = apply<PACKED>(before, enter[lane]);
  if (wave == NW - 1) leave_state(q, chain, n, cl, apply<PACKED>(own, h));
  if (t0 % ck_rows == 0 && rows > 0) *reinterpret_cast<f32x2 *>(ckpt + ((int64_t)chain * ck_tiles + t0 / ck_rows) * kTileChannels + cl) = h;
  T *op = static_cast<T *>(p.out) + b * p.out_bs;
#pragma unroll
  for (int j = 0; j < R; ++j) {
    h = apply<PACKED>(Step{a[j], bt[j]}, h);
    if (j < rows) at.store(op + (int64_t)(t0 + j) * p.out_ls, c, h.x, h.y);
    if constexpr (PACKED) {
      if (p.final_states && (rowsof.last >> j & 1)) at.store_state(p.final_states + (int64_t)rowsof.seq[j] * p.dim, c, h);
    }
  }
  if (!PACKED && p.final_states && t0 < L && t0 + R >= L) at.store_state(p.final_states + (int64_t)b * p.dim, c, h);
  if constexpr (PACKED) {
    if (p.final_states && n == 0)
      empty_sequences(p.cu_seqlens, p.nseq, L, [&](int s) {
        const int64_t o = (int64_t)s * p.dim;
        at.store_state(p.final_states + o, c, p.initial_states ? at.load_state(p.initial_states + o, c) : f32x2{0.f, 0.f});
      });
  }
}

// Tiles from the last one on: what enters a tile is a_t g_t of the position behind it.
template <typename T, bool EVEN, bool PACKED, int R, int NW>
__global__ __launch_bounds__(NW * 64) void gated_bwd_kernel(const GatedScanParams p, const Chain q, const float *ckpt, float *parts) {
  __shared__ f32x4 steps[NW][64], back[NW][64];
  __shared__ f32x2 enter[64];
  __shared__ int ticket;
  const int cgroups = (p.dim + kTileChannels - 1) / kTileChannels, nchains = cgroups * p.batch;
  const int chain = blockIdx.x % nchains, b = chain / cgroups;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), cl = lane * 2;
  const int c = (chain % cgroups) * kTileChannels + cl, L = p.seqlen;
  const Lane<T, EVEN> at(c, p.dim);
  const int n = take_tile(q, chain, &ticket), tile = q.ntiles - 1 - n;
  const int t0 = (tile * NW + wave) * R, rows = min(max(L - t0, 0), R);
  const float d0 = ld_param(p.decay, p.decay_dtype, min(c, p.dim - 1)), d1 = ld_param(p.decay, p.decay_dtype, min(c + 1, p.dim - 1));
  const f32x2 saved = *reinterpret_cast<const f32x2 *>(ckpt + ((int64_t)chain * q.ntiles + tile) * kTileChannels + cl);
  const T *xp = static_cast<const T *>(p.x) + b * p.x_bs;
  const T *ap = static_cast<const T *>(p.gate_a) + b * p.gate_a_bs;
  const T *gp = static_cast<const T *>(p.gate_x) + b * p.gate_x_bs;
  const T *dp = static_cast<const T *>(p.dout) + b * p.dout_bs;
  Pair<T> x[R], ga[R], gx[R], dout[R];
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
  auto initial = [&](int j) {
    return p.initial_states ? at.load_state(p.initial_states + (int64_t)rowsof.seq[PACKED ? j : 0] * p.dim, c) : f32x2{0.f, 0.f};
  };
  const float k0 = p.rate * softplus_exact(d0), k1 = p.rate * softplus_exact(d1);
  // per position: a, r, m i, x, i and, first r / m, then e / g
  f32x2 a[R], r[R], i[R], m[R], f[R], xs[R], d[R];
  Step own = no_step();
#pragma unroll
  for (int j = 0; j < R; ++j) {
    const Gates q0(ga[j].lo(), gx[j].lo(), k0), q1(ga[j].hi(), gx[j].hi(), k1);
    a[j] = PACKED ? f32x2{fmaxf(q0.a, kTiny), fmaxf(q1.a, kTiny)} : f32x2{q0.a, q1.a}, r[j] = f32x2{q0.r, q1.r}, i[j] = f32x2{q0.i, q1.i}, m[j] = f32x2{q0.m, q1.m};
    f[j] = f32x2{q0.r * q0.im, q1.r * q1.im};
    xs[j] = f32x2{x[j].lo(), x[j].hi()}, d[j] = f32x2{dout[j].lo(), dout[j].hi()};
    if (!counts(j)) {
      // a position past the row hands everything on, one outside of the sequences nothing
      a[j] = PACKED ? f32x2{0.f, 0.f} : f32x2{1.f, 1.f};
      r[j] = m[j] = i[j] = f[j] = xs[j] = d[j] = f32x2{0.f, 0.f};
    }
    if (ends(j) && p.dfinal_states) {
      const f32x2 v = at.load_state(p.dfinal_states + (int64_t)rowsof.seq[PACKED ? j : 0] * p.dim, c);
      d[j] = f32x2{d[j].x + v.x, d[j].y + v.y};
    }
    Step s = {a[j], f32x2{m[j].x * i[j].x * xs[j].x, m[j].y * i[j].y * xs[j].y}};
    if (starts(j)) {
      const f32x2 h = initial(j);
      s.b = f32x2{__builtin_fmaf(a[j].x, h.x, s.b.x), __builtin_fmaf(a[j].y, h.y, s.b.y)};
      s.a = f32x2{0.f, 0.f};
    }
    own = then<PACKED>(own, s);
  }
  Step rev = no_step();
#pragma unroll
  for (int j = R - 1; j >= 0; --j) {
    const bool cut = ends(j);
    const f32x2 g = cut ? d[j] : f32x2{rev.b.x + d[j].x, rev.b.y + d[j].y};
    if (PACKED && !counts(j)) {
      rev = Step{f32x2{0.f, 0.f}, f32x2{0.f, 0.f}};
    } else {
      rev.a = cut ? f32x2{0.f, 0.f} : factor<PACKED>(rev.a, a[j]);
      rev.b = f32x2{a[j].x * g.x, a[j].y * g.y};
    }
  }
  steps[wave][lane] = f32x4{own.a.x, own.a.y, own.b.x, own.b.y};
  back[wave][lane] = f32x4{rev.a.x, rev.a.y, rev.b.x, rev.b.y};
  lds_barrier();
  Step behind = no_step();
  for (int w = NW - 1; w > wave; --w) {
    const f32x4 s = back[w][lane];
    behind = then<PACKED>(behind, Step{f32x2{s.x, s.y}, f32x2{s.z, s.w}});
  }
  if (wave == 0) leave_step(q, chain, n, cl, then<PACKED>(behind, rev));
  f32x2 h = saved;
  for (int w = 0; w < wave; ++w) {
    const f32x4 s = steps[w][lane];
    h = apply<PACKED>(Step{f32x2{s.x, s.y}, f32x2{s.z, s.w}}, h);
  }
#pragma unroll
  for (int j = 0; j < R; ++j) {
    if (starts(j)) h = initial(j);
    if (PACKED && !counts(j)) h = f32x2{0.f, 0.f};
    const f32x2 ix = {i[j].x * xs[j].x, i[j].y * xs[j].y};
    f[j] = f32x2{a[j].x * __builtin_fmaf(a[j].x * ix.x, f[j].x, -r[j].x * h.x), a[j].y * __builtin_fmaf(a[j].y * ix.y, f[j].y, -r[j].y * h.y)};
    h = f32x2{__builtin_fmaf(a[j].x, h.x, m[j].x * ix.x), __builtin_fmaf(a[j].y, h.y, m[j].y * ix.y)};
  }
  if (wave == NW - 1) {
    f32x2 first = {0.f, 0.f};
    if (!PACKED && p.dfinal_states) first = at.load_state(p.dfinal_states + (int64_t)b * p.dim, c);
    enter[lane] = entering<PACKED>(q, chain, n, cl, first);
  }
  lds_barrier();
  f32x2 carry = apply<PACKED>(behind, enter[lane]), sum = {0.f, 0.f};
  if (wave == 0) leave_state(q, chain, n, cl, apply<PACKED>(rev, carry));
  T *dxp = static_cast<T *>(p.dx) + b * p.dx_bs;
  T *dap = static_cast<T *>(p.dgate_a) + b * p.dgate_a_bs;
  T *dgp = static_cast<T *>(p.dgate_x) + b * p.dgate_x_bs;
#pragma unroll
  for (int j = R - 1; j >= 0; --j) {
    f32x2 g = ends(j) ? d[j] : f32x2{d[j].x + carry.x, d[j].y + carry.y};
    if (PACKED && !counts(j)) g = f32x2{0.f, 0.f};
    const int64_t t = t0 + j;
    const f32x2 e = {g.x * f[j].x, g.y * f[j].y}, dx = {g.x * m[j].x * i[j].x, g.y * m[j].y * i[j].y};
    if (j < rows) {
      at.store(dxp + t * p.dx_ls, c, dx.x, dx.y);
      at.store(dap + t * p.dgate_a_ls, c, k0 * (1.f - r[j].x) * e.x, k1 * (1.f - r[j].y) * e.y);
      at.store(dgp + t * p.dgate_x_ls, c, dx.x * xs[j].x * (1.f - i[j].x), dx.y * xs[j].y * (1.f - i[j].y));
    }
    if (counts(j)) sum = f32x2{sum.x + e.x, sum.y + e.y};
    carry = f32x2{a[j].x * g.x, a[j].y * g.y};
    if (starts(j) && p.dinitial_states) at.store_state(p.dinitial_states + (int64_t)rowsof.seq[PACKED ? j : 0] * p.dim, c, carry);
  }
  if (!PACKED && t0 == 0 && p.dinitial_states) at.store_state(p.dinitial_states + (int64_t)b * p.dim, c, carry);
  if constexpr (PACKED) {
    if (p.dinitial_states && tile == 0)
      empty_sequences(p.cu_seqlens, p.nseq, L, [&](int s) {
        const int64_t o = (int64_t)s * p.dim;
        at.store_state(p.dinitial_states + o, c, p.dfinal_states ? at.load_state(p.dfinal_states + o, c) : f32x2{0.f, 0.f});
      });
  }
  // the terms of ddecay over the tile (the steps were read before the last barrier)
  f32x2 *sums = reinterpret_cast<f32x2 *>(&steps[0][0]);
  sums[wave * 64 + lane] = sum;
  lds_barrier();
  if (wave == 0) {
#pragma unroll
    for (int w = 1; w < NW; ++w) sum = f32x2{sum.x + sums[w * 64 + lane].x, sum.y + sums[w * 64 + lane].y};
    const f32x2 slope = {p.rate / (1.f + expf(-d0)), p.rate / (1.f + expf(-d1))};
    at.store_state(parts + ((int64_t)b * q.ntiles + tile) * p.dim, c, f32x2{sum.x * slope.x, sum.y * slope.y});
  }
}

// ------------------------------------------------------------------ host side
constexpr int kFwdRows = 8, kFwdWaves = 8, kBwdRows = 4, kBwdWaves = 8;

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
    return min(ntiles, 8);
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
    const bool even = p.dim % 2 == 0;
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
    gated_fwd_kernel<decltype(t), even.value, packed.value, kFwdRows, kFwdWaves>
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
    gated_bwd_kernel<decltype(t), even.value, packed.value, kBwdRows, kBwdWaves>
        <<<dim3((unsigned)(plan.chains * plan.ntiles)), dim3(kBwdWaves * 64), 0, st>>>(*p, plan.chain(p->ws), ck, parts);
    return hipGetLastError() == hipSuccess ? MAMBA_OK : MAMBA_E_LAUNCH;
  });
  if (rc != MAMBA_OK) return rc;
  ReduceJobs jobs{};
  jobs.part[0] = parts, jobs.out[0] = p->ddecay;
  return launch_reduce(jobs, 1, p->decay_dtype, p->batch * plan.ntiles, p->dim, st);
}
