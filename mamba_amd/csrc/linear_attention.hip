// Linear attention with a decay per head (linear_attn.hpp has the formulas), gfx950.
#include "linear_attn.hpp"

#include <algorithm>

namespace {
using namespace lin;

// The state of one segment alone, from zero, for the segments behind it.
template <typename T, int KD, int DVT, bool RAG> __global__ __launch_bounds__(kThreads, KD == 256 ? 1 : 2) void lin_segment_kernel(const LinLaunch p) {
  using F = Frags<T>;
  using Sh = Shape<T, KD, DVT>;
  constexpr int C = Sh::C;
  __shared__ __align__(16) typename F::E lb[C * Sh::PK], lc[C * Sh::PV];
  const Place at = place_of(p);
  if (at.none) return;
  const LinWalk &w = p.w[at.walk];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), i = lane & 15, g = lane >> 4;
  const int v0 = at.slice * Sh::VAL;
  const Item it = item_of(p, at.item);
  if (v0 >= w.val || it.zero || (it.before + 1) * p.seg_len >= it.len) return;  // the last segment's is not asked for
  const float l2 = log2_decay(p.log_decay[at.head]);
  int64_t b_ls, c_ls;
  const T *b = static_cast<const T *>(w.b.p) + rows_at(w.b, it, at.head, w.reverse, p.seg_len, b_ls);
  const T *c = static_cast<const T *>(w.c.p) + rows_at(w.c, it, at.head, w.reverse, p.seg_len, c_ls) + v0;
  Stage<T, C, KD, RAG> sb;
  Stage<T, C, Sh::VAL, RAG> sc;
  WaveState<T, KD, DVT> state;
  state.zero();
  const int vals = min(w.val - v0, Sh::VAL);
  sb.fetch(b, b_ls, min(it.n, C), w.key, tid), sc.fetch(c, c_ls, min(it.n, C), vals, tid);
  for (int t = 0; t < it.n; t += C) {
    const int n = min(it.n - t, C);
    sb.commit(lb, n, w.key, tid), sc.commit(lc, n, vals, tid);
    lds_barrier();
    if (t + C < it.n) {
      const int next = min(it.n - t - C, C);
      sb.fetch(b + (t + C) * b_ls, b_ls, next, w.key, tid), sc.fetch(c + (t + C) * c_ls, c_ls, next, vals, tid);
    }
    typename F::Raw cf[Sh::JB][DVT];
    value_frags<T, KD, DVT>(lc, cf, wave, i, g);
    state.scale(fast_exp2(l2 * (float)n));
    state.update(lb, cf, l2, w.write, n - w.late, i, g);
    lds_barrier();
  }
  f32x4 *dst = p.segs + ((((int64_t)at.walk * p.items + at.item) * p.nheads + at.head) * p.slices + at.slice) * (kWaves * Sh::TILES * 64) +
               wave * Sh::TILES * 64 + lane;
  state.each([&](f32x4 &v, int tile) { dst[tile * 64] = v; });
}

template <typename T, int KD, int DVT, bool RAG> __global__ __launch_bounds__(kThreads, KD == 256 ? 1 : 2) void lin_walk_kernel(const LinLaunch p) {
  using F = Frags<T>;
  using Sh = Shape<T, KD, DVT>;
  using E = typename F::E;
  constexpr int C = Sh::C, KB = Sh::KB, JB = Sh::JB, IT = Sh::IT, NT = F::NT, KS = F::KS, V = F::V;
  constexpr int BLOCKS = JB * IT;
  __shared__ __align__(16) E la[C * Sh::PK], lb[C * Sh::PK], lc[C * Sh::PV];
  __shared__ __align__(16) typename F::Comp lp[BLOCKS][64];
  const Place at = place_of(p);
  if (at.none) return;
  const LinWalk &w = p.w[at.walk];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), i = lane & 15, g = lane >> 4;
  const int v0 = at.slice * Sh::VAL;
  const Item it = item_of(p, at.item);
  if (v0 >= w.val || it.seq < 0) return;
  const int vals = min(w.val - v0, Sh::VAL);
  // a lane's values of y: NV side by side from value y0 on, per tile or (PAIR) for both
  constexpr int NV = Sh::PAIR ? 8 : 4, NY = Sh::PAIR ? 1 : DVT;
  int64_t y_ls;
  const int64_t y_at = rows_at(w.y, it, at.head, w.reverse, p.seg_len, y_ls) + v0;
  auto put = [&](int64_t row, int d, const float (&v)[NV]) {
    const int col = wave * Sh::WV + (Sh::PAIR ? 8 * g : 16 * d + 4 * g);
    if (w.y_f32) {
      float *dst = static_cast<float *>(w.y.p) + y_at + row * y_ls + col;
#pragma unroll
      for (int e = 0; e < NV; ++e)
        if (col + e < vals) dst[e] = v[e];
    } else {
      T *dst = static_cast<T *>(w.y.p) + y_at + row * y_ls + col;
      if (!RAG && col + NV <= vals) {
        if constexpr (std::is_same_v<T, float>) {
          *(GLOBAL_AS f32x4_a4 *)dst = f32x4{v[0], v[1], v[2], v[3]};
        } else if constexpr (NV == 8) {
          st8_any<T>(dst, v);
        } else {
          typedef u32x2 u32x2_a2 __attribute__((aligned(2)));
          if constexpr (DT<T>::id == MAMBA_BF16) *(GLOBAL_AS u32x2_a2 *)dst = u32x2{pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3])};
          else *(GLOBAL_AS u32x2_a2 *)dst = u32x2{pack_f16(v[0], v[1]), pack_f16(v[2], v[3])};
        }
      } else {
#pragma unroll
        for (int e = 0; e < NV; ++e)
          if (col + e < vals) st1<T>(dst + e, v[e]);
      }
    }
  };
  if (it.zero) {
    const float zero[NV] = {};
    for (int row = i; row < it.n; row += 16)
#pragma unroll
      for (int d = 0; d < NY; ++d) put(row, d, zero);
    return;
  }

  const float l2 = log2_decay(p.log_decay[at.head]);
  int64_t a_ls, b_ls, c_ls;
  const T *a = static_cast<const T *>(w.a.p) + rows_at(w.a, it, at.head, w.reverse, p.seg_len, a_ls);
  const T *b = static_cast<const T *>(w.b.p) + rows_at(w.b, it, at.head, w.reverse, p.seg_len, b_ls);
  const T *c = static_cast<const T *>(w.c.p) + rows_at(w.c, it, at.head, w.reverse, p.seg_len, c_ls) + v0;
  Stage<T, C, KD, RAG> sa, sb;
  Stage<T, C, Sh::VAL, RAG> sc;
  auto fetch = [&](int t) {
    const int n = min(it.n - t, C);
    sa.fetch(a + t * a_ls, a_ls, n, w.key, tid), sb.fetch(b + t * b_ls, b_ls, n, w.key, tid), sc.fetch(c + t * c_ls, c_ls, n, vals, tid);
  };
  if (it.n > 0) fetch(0);

  // the state that comes in
  WaveState<T, KD, DVT> state;
  const int64_t seq_head = ((int64_t)it.seq * p.nheads + at.head) * w.key * w.val;
  if (w.start.p) {
    const float *src = w.start.p + seq_head;
    state.each_element(i, g, w.key, w.val, v0 + wave * Sh::WV, [&](float, int k, int v, bool ok) {
      const float x = src[(int64_t)min(k, w.key - 1) * w.start.ks + (int64_t)min(v, w.val - 1) * w.start.vs];
      return ok ? x : 0.f;
    });
  } else {
    state.zero();
  }
  if (it.before > 0) {
    const float f = fast_exp2(l2 * (float)p.seg_len);
    const int64_t step = (int64_t)p.nheads * p.slices * (kWaves * Sh::TILES * 64);
    const f32x4 *src = p.segs + (((int64_t)at.walk * p.items + at.item - it.before) * p.nheads * p.slices + at.head * p.slices + at.slice) *
                                    (kWaves * Sh::TILES * 64) + wave * Sh::TILES * 64 + lane;
    for (int s = 0; s < it.before; ++s, src += step) state.each([&](f32x4 &v, int tile) { v = v * f + src[tile * 64]; });
  }

  for (int t = 0; t < it.n; t += C) {
    const int n = min(it.n - t, C);
    sa.commit(la, n, w.key, tid), sb.commit(lb, n, w.key, tid), sc.commit(lc, n, vals, tid);
    lds_barrier();
    if (t + C < it.n) fetch(t + C);
    // (a_t . b_s) f^(t - s), the blocks of KS s on and below the diagonal in turn by the waves
    int f = 0;
#pragma unroll
    for (int ib = 0; ib < IT; ++ib)
#pragma unroll
      for (int jb = 0; jb < JB; ++jb) {
        if (jb * KS > ib * 16 + 15) continue;
        if ((f++ & 3) != wave) continue;
        f32x4 acc[NT];
#pragma unroll
        for (int h = 0; h < NT; ++h) acc[h] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
          const auto ar = F::along(la + (16 * ib + i) * Sh::PK + KS * kb + V * g);
#pragma unroll
          for (int h = 0; h < NT; ++h)
            acc[h] = F::mma_raw(F::along(lb + (KS * jb + F::krow(i, h)) * Sh::PK + KS * kb + V * g), ar, acc[h]);
        }
        float v[V];
        F::gather(acc, v);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const int apart = 16 * ib + i - (KS * jb + V * g + e);
          v[e] = apart >= 0 ? v[e] * (w.mix * fast_exp2(l2 * (float)apart)) : 0.f;
        }
        lp[ib * JB + jb][lane] = F::comp(v);
      }
    // y from the state that came in
    f32x4 y[IT][DVT];
#pragma unroll
    for (int ib = 0; ib < IT; ++ib)
#pragma unroll
      for (int d = 0; d < DVT; ++d) y[ib][d] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      typename F::Comp s[DVT];
#pragma unroll
      for (int d = 0; d < DVT; ++d) {
        f32x4 tiles[NT];
#pragma unroll
        for (int h = 0; h < NT; ++h) tiles[h] = state.t[kb][h][d];
        float v[V];
        F::gather(tiles, v);
        s[d] = F::comp(v);
      }
#pragma unroll
      for (int ib = 0; ib < IT; ++ib) {
        const auto ar = F::data(F::along(la + (16 * ib + i) * Sh::PK + KS * kb + V * g));
#pragma unroll
        for (int d = 0; d < DVT; ++d) y[ib][d] = mma16(s[d], ar, y[ib][d]);
      }
    }
#pragma unroll
    for (int ib = 0; ib < IT; ++ib) {
      const float f = w.read * fast_exp2(l2 * (float)(16 * ib + i + w.late));
#pragma unroll
      for (int d = 0; d < DVT; ++d) y[ib][d] *= f;
    }
    typename F::Raw cf[JB][DVT];
    value_frags<T, KD, DVT>(lc, cf, wave, i, g);
    state.scale(fast_exp2(l2 * (float)n));
    state.update(lb, cf, l2, w.write, n - w.late, i, g);
    lds_barrier();  // nothing of the block's rows is read behind this
#pragma unroll
    for (int jb = 0; jb < JB; ++jb) {
      typename F::Data cd[DVT];
#pragma unroll
      for (int d = 0; d < DVT; ++d) cd[d] = F::data(cf[jb][d]);
#pragma unroll
      for (int ib = 0; ib < IT; ++ib) {
        if (jb * KS > ib * 16 + 15) continue;
        const typename F::Comp pf = lp[ib * JB + jb][lane];
#pragma unroll
        for (int d = 0; d < DVT; ++d) y[ib][d] = mma16(cd[d], pf, y[ib][d]);
      }
    }
#pragma unroll
    for (int ib = 0; ib < IT; ++ib) {
      const int row = 16 * ib + i;
      if (row < n) {
#pragma unroll
        for (int d = 0; d < NY; ++d) {
          float v[NV];
#pragma unroll
          for (int e = 0; e < NV; ++e) v[e] = Sh::PAIR ? y[ib][e >> 2][e & 3] : y[ib][d][e & 3];
          put(t + row, d, v);
        }
      }
    }
  }
  if (w.end.p && (it.before + 1) * (int64_t)p.seg_len >= it.len) {
    float *dst = w.end.p + seq_head;
    state.each_element(i, g, w.key, w.val, v0 + wave * Sh::WV, [&](float x, int k, int v, bool ok) {
      if (ok) dst[(int64_t)k * w.end.ks + (int64_t)v * w.end.vs] = x;
      return x;
    });
  }
}

// Items of packed sequences cut into segments: sequences in order, then what lies before the first and behind the last.  Bounds
// are taken into the row and made not to decrease, so that there are never more items than the host has counted on.
__global__ __launch_bounds__(kThreads) void lin_plan_kernel(int4 *plan, const int32_t *cu, int nseq, int seqlen, int seg_len, int items) {
  __shared__ int top[kThreads], sum[kThreads];
  const int tid = threadIdx.x;
  int end_before = 0, items_before = 0, first_start = 0;
  auto bound_at = [&](int q) { return min(max(cu[q], 0), seqlen); };
  for (int q0 = 0; q0 < nseq; q0 += kThreads) {
    const int q = q0 + tid;
    // the largest bound up to this sequence's start and end
    top[tid] = q < nseq ? max(bound_at(q), bound_at(q + 1)) : 0;
    __syncthreads();
    for (int step = 1; step < kThreads; step *= 2) {
      const int other = tid >= step ? top[tid - step] : 0;
      __syncthreads();
      top[tid] = max(top[tid], other);
      __syncthreads();
    }
    const int before = max(tid > 0 ? top[tid - 1] : 0, end_before);
    const int start = q < nseq ? max(before, bound_at(q)) : 0, end = max(max(top[tid], end_before), start);
    const int len = q < nseq ? end - start : 0, n = q < nseq ? max((len + seg_len - 1) / seg_len, 1) : 0;
    sum[tid] = n;
    __syncthreads();
    for (int step = 1; step < kThreads; step *= 2) {
      const int other = tid >= step ? sum[tid - step] : 0;
      __syncthreads();
      sum[tid] += other;
      __syncthreads();
    }
    for (int s = 0; s < n; ++s) {
      const int at = items_before + sum[tid] - n + s;
      if (at < items - 2) plan[at] = int4{q, start, len, s};
    }
    end_before = max(end_before, top[kThreads - 1]);
    items_before += sum[kThreads - 1];
    __syncthreads();
  }
  first_start = bound_at(0);
  if (tid == 0) {
    items_before = min(items_before, items - 2);
    plan[items_before] = int4{nseq, 0, first_start, 0};
    plan[items_before + 1] = int4{nseq, end_before, seqlen - end_before, 0};
    plan[items] = int4{items_before + 2, 0, 0, 0};
  }
}

// Gradients of heads that share keys and values, added up in order: parts (rows, nheads, dim) in fp32.
template <typename T> __global__ __launch_bounds__(kThreads) void lin_shared_kernel(const float *parts, T *out, int64_t n, int dim, int kv_heads, int group, int seqlen,
                                                                                   int64_t bs, int64_t ls, int64_t hs) {
  for (int64_t at = (int64_t)blockIdx.x * kThreads + threadIdx.x; at < n; at += (int64_t)gridDim.x * kThreads) {
    const int x = at % dim;
    const int64_t rh = at / dim;
    const int h = rh % kv_heads;
    const int64_t row = rh / kv_heads;
    const float *src = parts + ((row * kv_heads + h) * group) * dim + x;
    float v = 0.f;
    for (int m = 0; m < group; ++m) v += src[(int64_t)m * dim];
    st1<T>(out + row / seqlen * bs + row % seqlen * ls + h * hs + x, v);
  }
}

// ------------------------------------------------------------------ host side
// How a pass is cut: the sizes that the kernels are made for, the values of a workgroup, and segments of a sequence where
// there are too few (sequence, head, slice) walks for the chip.
struct Cut {
  int kd, dvt, slices, nseg, seg_len, items;
  bool ragged, packed;
  int64_t state_bytes, plan_bytes;
};
Cut cut_of(const LinearAttnParams &p, int nwalks) {
  Cut c;
  const int most = p.headdim_k > p.headdim_v ? p.headdim_k : p.headdim_v, v = p.dtype == MAMBA_F32 ? 4 : 8;
  const int val = nwalks == 1 ? p.headdim_v : most, key = nwalks == 1 ? p.headdim_k : most;
  c.kd = key <= 64 ? 64 : key <= 128 ? 128 : 256;
  c.dvt = val > 64 && c.kd <= 128 && p.dtype != MAMBA_F16 ? 2 : 1;  // (two tiles of values more would not fit the registers)
  c.slices = (val + 64 * c.dvt - 1) / (64 * c.dvt);
  c.ragged = p.headdim_k % v != 0 || p.headdim_v % v != 0;
  c.packed = p.nseq > 0;
  const int64_t seqs = c.packed ? p.nseq : p.batch, walks = (int64_t)p.nheads * c.slices * nwalks;
  const int64_t total = (int64_t)p.batch * p.seqlen, room = 2 * cu_count();
  // positions of a segment: as many as make every workgroup's share of the chip, four blocks at least
  const int64_t share = (total * walks + room - 1) / room, least = 256;
  int64_t len = (std::max(share, least) + 63) / 64 * 64;
  const int64_t longest = c.packed ? total : p.seqlen;
  if (seqs * walks >= room / 2 * (c.packed ? 2 : 1) || len >= longest) len = longest;
  c.nseg = (int)((longest + len - 1) / len);
  if (c.nseg < 1) c.nseg = 1;
  c.seg_len = c.nseg == 1 ? INT32_MAX : (int)len;
  c.items = c.packed ? (int)(seqs + 2 + (c.nseg > 1 ? total / len : 0)) : (int)(seqs * c.nseg);
  c.plan_bytes = c.packed && c.nseg > 1 ? ((int64_t)c.items + 1) * 16 : 0;
  c.state_bytes = c.nseg > 1 ? (int64_t)nwalks * c.items * p.nheads * c.slices * c.kd * 64 * c.dvt * 4 : 0;
  return c;
}

template <typename T, int KD, int DVT, bool RAG> int run(const LinLaunch &l, hipStream_t st) {
  const int64_t outer = ((int64_t)l.items * l.kv_heads + 7) / 8 * 8, blocks = outer * (l.nheads / l.kv_heads) * l.nwalks * l.slices;
  if (blocks > INT32_MAX) return MAMBA_E_UNSUPPORTED;
  if (l.nseg > 1) {
    lin_segment_kernel<T, KD, DVT, RAG><<<(int)blocks, kThreads, 0, st>>>(l);
    if (hipGetLastError() != hipSuccess) return MAMBA_E_LAUNCH;
  }
  lin_walk_kernel<T, KD, DVT, RAG><<<(int)blocks, kThreads, 0, st>>>(l);
  return hipGetLastError() == hipSuccess ? MAMBA_OK : MAMBA_E_LAUNCH;
}
template <typename T, int KD> int run_dvt(const LinLaunch &l, const Cut &c, hipStream_t st) {
  if constexpr (KD <= 128 && !std::is_same_v<T, f16_t>) {
    if (c.dvt == 2) return c.ragged ? run<T, KD, 2, true>(l, st) : run<T, KD, 2, false>(l, st);
  }
  return c.ragged ? run<T, KD, 1, true>(l, st) : run<T, KD, 1, false>(l, st);
}
template <typename T> int run_kd(const LinLaunch &l, const Cut &c, hipStream_t st) {
  switch (c.kd) {
    case 64: return run_dvt<T, 64>(l, c, st);
    case 128: return run_dvt<T, 128>(l, c, st);
    default: return run_dvt<T, 256>(l, c, st);
  }
}
int run_type(const LinLaunch &l, const Cut &c, int dtype, hipStream_t st) {
  switch (dtype) {
    case MAMBA_F32: return run_kd<float>(l, c, st);
    case MAMBA_BF16: return run_kd<bf16_t>(l, c, st);
    default: return run_kd<f16_t>(l, c, st);
  }
}

int check(const LinearAttnParams *p) {
  if (!p || !p->q || !p->k || !p->v || !p->log_decay) return MAMBA_E_BADARG;
  if (p->batch <= 0 || p->seqlen <= 0 || p->nheads <= 0 || p->nkvheads <= 0 || p->headdim_k <= 0 || p->headdim_v <= 0) return MAMBA_E_BADARG;
  if (p->nheads % p->nkvheads != 0 || p->dtype < MAMBA_F32 || p->dtype > MAMBA_F16) return MAMBA_E_BADARG;
  if (p->nseq < 0 || (p->nseq > 0) != (p->cu_seqlens != nullptr) || (p->nseq > 0 && p->batch != 1)) return MAMBA_E_BADARG;
  if (!(p->scale >= -3.4e38f && p->scale <= 3.4e38f)) return MAMBA_E_BADARG;
  if (p->headdim_k > 256 || p->headdim_v > 256 || p->seqlen > 1 << 30 || p->nseq > 1 << 30) return MAMBA_E_UNSUPPORTED;
  return MAMBA_OK;
}
LinRows rows(const void *t, int64_t bs, int64_t ls, int64_t hs, int group) { return LinRows{const_cast<void *>(t), bs, ls, hs, group}; }
// a buffer of a call: the plan, the segments' states, fp32 gradients of shared heads
int64_t parts_bytes(const LinearAttnParams &p) {
  return p.nheads == p.nkvheads ? 0 : (int64_t)p.batch * p.seqlen * p.nheads * (p.headdim_k + p.headdim_v) * 4;
}
LinLaunch launch_of(const LinearAttnParams &p, const Cut &c, int nwalks) {
  LinLaunch l{};
  l.log_decay = p.log_decay, l.cu = p.cu_seqlens, l.nwalks = nwalks, l.nheads = p.nheads, l.kv_heads = p.nkvheads;
  l.slices = c.slices, l.items = c.items, l.nseg = c.nseg, l.seg_len = c.seg_len, l.nseq = c.packed ? p.nseq : p.batch, l.seqlen = p.seqlen;
  l.plan = c.plan_bytes ? static_cast<const int32_t *>(p.ws) : nullptr;
  l.segs = reinterpret_cast<f32x4 *>(static_cast<char *>(p.ws) + c.plan_bytes);
  return l;
}
int plan(const LinearAttnParams &p, const Cut &c, hipStream_t st) {
  if (!c.plan_bytes) return MAMBA_OK;
  lin_plan_kernel<<<1, kThreads, 0, st>>>(static_cast<int4 *>(p.ws), p.cu_seqlens, p.nseq, p.seqlen, c.seg_len, c.items);
  return hipGetLastError() == hipSuccess ? MAMBA_OK : MAMBA_E_LAUNCH;
}
template <typename T> int shared(const LinearAttnParams &p, const float *parts, void *out, int dim, int64_t bs, int64_t ls, int64_t hs, hipStream_t st) {
  const int64_t n = (int64_t)p.batch * p.seqlen * p.nkvheads * dim;
  const int blocks = (int)std::min<int64_t>((n + kThreads - 1) / kThreads, 16 * (int64_t)cu_count());
  lin_shared_kernel<T><<<blocks, kThreads, 0, st>>>(parts, static_cast<T *>(out), n, dim, p.nkvheads, p.nheads / p.nkvheads, p.seqlen, bs, ls, hs);
  return hipGetLastError() == hipSuccess ? MAMBA_OK : MAMBA_E_LAUNCH;
}
int shared_type(const LinearAttnParams &p, const float *parts, void *out, int dim, int64_t bs, int64_t ls, int64_t hs, hipStream_t st) {
  switch (p.dtype) {
    case MAMBA_F32: return shared<float>(p, parts, out, dim, bs, ls, hs, st);
    case MAMBA_BF16: return shared<bf16_t>(p, parts, out, dim, bs, ls, hs, st);
    default: return shared<f16_t>(p, parts, out, dim, bs, ls, hs, st);
  }
}

}  // namespace

extern "C" int64_t linear_attn_fwd_ws_bytes(const LinearAttnParams *p) {
  if (const int rc = check(p)) return rc;
  const Cut c = cut_of(*p, 1);
  return c.plan_bytes + c.state_bytes;
}
extern "C" int64_t linear_attn_bwd_ws_bytes(const LinearAttnParams *p) {
  if (const int rc = check(p)) return rc;
  const Cut c = cut_of(*p, 3);
  return c.plan_bytes + c.state_bytes + parts_bytes(*p);
}

extern "C" int linear_attn_fwd(const LinearAttnParams *p, mamba_stream_t stream) {
  if (const int rc = check(p)) return rc;
  if (!p->out) return MAMBA_E_BADARG;
  const Cut c = cut_of(*p, 1);
  if (c.plan_bytes + c.state_bytes > 0 && (!p->ws || reinterpret_cast<uintptr_t>(p->ws) % 16 != 0)) return MAMBA_E_BADARG;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int group = p->nheads / p->nkvheads;
  LinLaunch l = launch_of(*p, c, 1);
  LinWalk &w = l.w[0];
  w.a = rows(p->q, p->q_bs, p->q_ls, p->q_hs, 1), w.b = rows(p->k, p->k_bs, p->k_ls, p->k_hs, group);
  w.c = rows(p->v, p->v_bs, p->v_ls, p->v_hs, group), w.y = rows(p->out, p->out_bs, p->out_ls, p->out_hs, 1);
  w.start = LinState{const_cast<float *>(p->initial_states), p->headdim_v, 1}, w.end = LinState{p->final_states, p->headdim_v, 1};
  w.mix = w.read = p->scale, w.write = 1.f, w.key = p->headdim_k, w.val = p->headdim_v, w.late = 1;
  if (const int rc = plan(*p, c, st)) return rc;
  return run_type(l, c, p->dtype, st);
}

extern "C" int linear_attn_bwd(const LinearAttnParams *p, mamba_stream_t stream) {
  if (const int rc = check(p)) return rc;
  if (!p->dout || !p->dq || !p->dk || !p->dv) return MAMBA_E_BADARG;
  const Cut c = cut_of(*p, 3);
  if (linear_attn_bwd_ws_bytes(p) > 0 && (!p->ws || reinterpret_cast<uintptr_t>(p->ws) % 16 != 0)) return MAMBA_E_BADARG;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int group = p->nheads / p->nkvheads, dk = p->headdim_k, dv = p->headdim_v;
  LinLaunch l = launch_of(*p, c, 3);
  const LinRows q = rows(p->q, p->q_bs, p->q_ls, p->q_hs, 1), k = rows(p->k, p->k_bs, p->k_ls, p->k_hs, group);
  const LinRows v = rows(p->v, p->v_bs, p->v_ls, p->v_hs, group), go = rows(p->dout, p->dout_bs, p->dout_ls, p->dout_hs, 1);
  float *initial = const_cast<float *>(p->initial_states), *dfinal = const_cast<float *>(p->dfinal_states);
  LinWalk &wq = l.w[0], &wk = l.w[1], &wv = l.w[2];
  wq.a = go, wq.b = v, wq.c = k, wq.y = rows(p->dq, p->dq_bs, p->dq_ls, p->dq_hs, 1);
  wq.start = LinState{initial, 1, dv}, wq.mix = wq.read = p->scale, wq.write = 1.f, wq.key = dv, wq.val = dk, wq.late = 1;
  wk.a = v, wk.b = go, wk.c = q, wk.start = LinState{dfinal, 1, dv}, wk.key = dv, wk.val = dk;
  wv.a = k, wv.b = q, wv.c = go, wv.start = LinState{dfinal, dv, 1}, wv.end = LinState{p->dinitial_states, dv, 1}, wv.key = dk, wv.val = dv;
  for (LinWalk *w : {&wk, &wv}) w->mix = w->write = p->scale, w->read = 1.f, w->reverse = 1;
  float *parts_k = reinterpret_cast<float *>(static_cast<char *>(p->ws) + c.plan_bytes + c.state_bytes);
  float *parts_v = parts_k + (int64_t)p->batch * p->seqlen * p->nheads * dk;
  if (group == 1) {
    wk.y = rows(p->dk, p->dk_bs, p->dk_ls, p->dk_hs, 1), wv.y = rows(p->dv, p->dv_bs, p->dv_ls, p->dv_hs, 1);
  } else {
    const int64_t hk = dk, hv = dv, H = p->nheads;
    wk.y = rows(parts_k, p->seqlen * H * hk, H * hk, hk, 1), wv.y = rows(parts_v, p->seqlen * H * hv, H * hv, hv, 1);
    wk.y_f32 = wv.y_f32 = 1;
  }
  if (const int rc = plan(*p, c, st)) return rc;
  if (const int rc = run_type(l, c, p->dtype, st)) return rc;
  if (group == 1) return MAMBA_OK;
  if (const int rc = shared_type(*p, parts_k, p->dk, dk, p->dk_bs, p->dk_ls, p->dk_hs, st)) return rc;
  return shared_type(*p, parts_v, p->dv, dv, p->dv_bs, p->dv_ls, p->dv_hs, st);
}
