// Attention of one new token over a paged cache of keys and values, split over the cache's length and joined (gfx950):
//   out = sum_p softmax_p(scale q . k_p) v_p   over the positions of the sequence's cache (the last `window` of them)
// Every key and value is read once, for all query heads that share it: that is what the operator costs (16 operations a byte for
// 16 heads).  A workgroup has one key head (up to 16 of its query heads) and a run of positions; each of its waves takes a tile of
// 32 positions (fp32: 16) at a time and keeps the running maximum m and the sums
//   l = sum 2^(s_p - m),  o = sum 2^(s_p - m) v_p,   s_p = scale log2(e) q . k_p
// As the rows of K sit in memory they are operands; the products leave the tile with 8 positions of one head in a lane, which is
// the operand that the product with V wants (mma_frag.hpp), and a head's m, l are one lane's; V goes through LDS to be read by
// columns.  Waves meet at the end, workgroups in a second launch.  Memory bounds it: 131072 positions of 8 x 128 in bf16, 537 MB,
// 98-105 us (5.1-5.5 TB/s) and 6 for the join; one tile on its way and one at work a wave, two workgroups a CU.
#include "mma_frag.hpp"

#include <algorithm>
#include <type_traits>

namespace {

constexpr int kThreads = 256, kWaves = 4, kHeads = 16;
constexpr int kRowBits = 23;  // workgroups beyond 2^23 lie along y: a launch takes fewer than 2^32 threads along x
// workgroups of a CU that the registers leave room for, with rows of whole pieces.  (With others, read element by element, there is room for
// 2, 1 and 1 at sizes of up to 64, 96 and 128: their ranges take one and a half or two rounds.  32 sequences of up to 8192 positions, 32
// heads on 8, bf16: 469 us at 100 values a head, 118 at 128.)
constexpr int workgroups(int D) { return D == 64 ? 3 : D == 256 ? 1 : 2; }
constexpr float kLow = -3.40282347e38f;  // the least number: stands for a maximum of minus infinity, so that differences are numbers

struct Span {  // positions of a sequence, in tiles
  int n;            // positions of the cache before the call; negative: an empty place of the batch
  int first, last;  // [first, last): those that count
  int tile0, tiles; // tiles that hold them
  DEVI int count() const { return max(tiles, 1); }  // (a sequence without positions is to be answered too)
};
template <int KS> DEVI Span span_of(const PagedAttnParams &p, int b) {
  Span r;
  r.n = min(p.cache_seqlens[b], p.max_pages * p.page_size);
  r.last = max(r.n, -1) + (p.k ? 1 : 0);
  r.first = p.window > 0 ? max(r.last - p.window, 0) : 0;
  r.tile0 = r.first / KS;
  r.tiles = r.last > r.first ? (r.last - 1) / KS + 1 - r.tile0 : 0;
  return r;
}
// The tiles of all sequences one behind the other, cut into nsplit even ranges, whatever the lengths: range w goes from tile w share
// on.  A range has the end of one sequence and the start of the next; the part of sequence b in range w lies in ws at w + b, and no
// other does.  (Every sequence cut into nsplit parts: 126 us instead of 109 for 32 sequences of 8192 positions at most.)
DEVI int64_t sum_of_wave(int64_t v) {
#pragma unroll
  for (int step = 1; step < 64; step *= 2) v += __shfl_xor(v, step, 64);
  return v;
}
template <int KS> DEVI int64_t tiles_before(const PagedAttnParams &p, int end) {
  int64_t sum = 0;
  for (int b = threadIdx.x % 64; b < end; b += 64) sum += span_of<KS>(p, b).count();
  return sum_of_wave(sum);
}
DEVI int64_t share_of(const PagedAttnParams &p, int64_t total) { return max((total + p.nsplit - 1) / p.nsplit, (int64_t)(2 * kWaves)); }

template <typename T, int D, bool RAG> __global__ __launch_bounds__(kThreads, RAG ? 1 : workgroups(D)) void paged_part_kernel(const PagedAttnParams p) {
  using F = Frags<T>;
  using E = typename F::E;
  using Raw = typename F::Raw;
  constexpr int LD = D == 96 ? 128 : D;  // columns of a tile in LDS, whose rows are permuted by powers of two
  using Columns = typename F::template ColumnLane<LD>;
  constexpr int KS = F::KS, NT = F::NT, V = F::V, KB = D / KS, OT = D / 16, PER = D / V, NV = KS * PER / 64;
  // l and o are kLift times the sums: weights of 2^-29 of the largest are still whole fp16 numbers, and the last ones left out are below
  // 2^-40 (without it below 2^-25, which many positions beside one that draws the weight add up to a result).
  constexpr float kLift = std::is_same_v<T, f16_t> ? 32768.f : 1.f;
  constexpr int TILE = F::size(KS, LD), SUMS = kHeads * (D + 4) * 4, AREA = TILE > SUMS ? TILE : SUMS;
  __shared__ __align__(16) char area[kWaves][AREA];
  __shared__ float wave_m[kWaves][kHeads], wave_l[kWaves][kHeads];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), i = lane & 15, g = lane >> 4;
  const int group = p.nheads / p.nkvheads, htiles = (group + kHeads - 1) / kHeads;
  // Workgroups go to the XCDs in turn; all heads of a range (or sequence) are to be on one, as a position's heads lie side by side in
  // memory and share its L2's lines where a head is not whole lines (48 x 12 heads of 80 in fp16: 39 us in order, 37 this way).
  const int rows = p.nkvheads * htiles, n = p.nsplit == 1 ? p.batch : p.nsplit;
  const uint32_t block = blockIdx.y << kRowBits | blockIdx.x;
  const int row = n >= 8 ? block / 8 % rows : block % rows, range = n >= 8 ? block / 8 / rows * 8 + block % 8 : block / rows;
  if (range >= n) return;
  const int hk = row / htiles, ht = row % htiles, h0 = hk * group + ht * kHeads, heads = min(group - ht * kHeads, kHeads);
  // tiles [lo, hi) of the batch, of which sequence b begins at `at`
  int b = 0;
  int64_t lo = 0, hi = 0, at = 0;
  if (p.nsplit == 1) {
    b = range;
  } else {
    const int64_t total = tiles_before<KS>(p, p.batch), share = share_of(p, total);
    lo = range * share, hi = min(lo + share, total);
    if (lo >= total) return;
    for (;; b += 64) {
      const int64_t own = b + lane < p.batch ? span_of<KS>(p, b + lane).count() : 0;
      int64_t to = own;
#pragma unroll
      for (int step = 1; step < 64; step *= 2) {
        const int64_t other = __shfl_up(to, step, 64);
        to += lane >= step ? other : 0;
      }
      const uint64_t beyond = __ballot(at + to > lo);
      if (beyond) {
        const int l = __builtin_ctzll(beyond);
        b += l, at += __shfl(to - own, l, 64);
        break;
      }
      at += __shfl(to, 63, 64);
    }
  }
  for (;;) {
  b = __builtin_amdgcn_readfirstlane(b);
  const Span sp = span_of<KS>(p, b);
  if (p.nsplit == 1) hi = sp.count();
  const int begin = sp.tile0 + (int)max(lo - at, (int64_t)0), end = sp.tile0 + (int)min(hi - at, (int64_t)sp.tiles);
  const bool ends_here = hi >= at + sp.count(), whole = ends_here && lo <= at;
  const int dk = p.headdim_k, dv = p.headdim_v;
  const int32_t *table = p.block_table + b * p.table_bs;
  const T *k_new = p.k ? static_cast<const T *>(p.k) + b * p.k_bs + hk * p.k_hs : nullptr;
  const T *v_new = p.k ? static_cast<const T *>(p.v) + b * p.v_bs + hk * p.v_hs : nullptr;

  // the new token's row of the cache: written here, read by nobody (its tile takes the row from the call's arguments)
  if (k_new && ht == 0 && ends_here && sp.n >= 0 && sp.n < p.max_pages * p.page_size) {
    const int id = table[sp.n / p.page_size], off = sp.n % p.page_size;
    if (id >= 0 && id < p.num_pages) {
      T *kd = static_cast<T *>(p.k_cache) + id * p.kc_ps + off * p.kc_ls + hk * p.kc_hs;
      T *vd = static_cast<T *>(p.v_cache) + id * p.vc_ps + off * p.vc_ls + hk * p.vc_hs;
      for (int x = tid; x < dk; x += kThreads) kd[x] = k_new[x];
      for (int x = tid; x < dv; x += kThreads) vd[x] = v_new[x];
    }
  }

  // q of the heads, by lanes: head i (beyond the last: the last again, not stored)
  Raw qf[KB];
  const T *q = static_cast<const T *>(p.q) + b * p.q_bs + (h0 + min(i, heads - 1)) * p.q_hs;
  // a piece of a row of `cols` columns, and what of it is in them.  (K's is looked at where it is used: in the load it waits for it, 37 us and
  // not 31 for those 48 x 12 heads.
  // V's columns beyond the last meet no others and are not stored.)
  auto piece = [&](const T *row, int col, int cols) -> Raw {
    if constexpr (RAG) {
      E v[V];
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] = *(const GLOBAL_AS E *)(row + min(col + e, cols - 1));
      return __builtin_bit_cast(Raw, v);
    } else {
      const T *at = row + min(col, cols - V);
      if constexpr (std::is_same_v<T, float>) return *(const GLOBAL_AS f32x4_a4 *)at;
      else return *(const GLOBAL_AS u32x4_a2 *)at;
    }
  };
  auto within = [&](Raw v, int col, int cols) -> Raw {
    if constexpr (RAG) {
      E e[V];
      __builtin_memcpy(e, &v, 16);
#pragma unroll
      for (int n = 0; n < V; ++n) e[n] = col + n < cols ? e[n] : E(0);
      return __builtin_bit_cast(Raw, e);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = col < cols ? v[e] : 0;
      return v;
    }
  };
#pragma unroll
  for (int kb = 0; kb < KB; ++kb) qf[kb] = within(piece(q, KS * kb + V * g, dk), KS * kb + V * g, dk);

  // rows of a tile: lane r (of KS) has the place of position r; those that do not count take the first one's that does
  struct Entry {
    int id, off;  // -1: no page
  };
  auto page_of = [&](int tile) {
    const int pos = KS * tile + (lane & (KS - 1)), index = pos / p.page_size;
    const int id = table[min(index, p.max_pages - 1)];
    return Entry{id < p.num_pages && index < p.max_pages ? id : -1, pos - index * p.page_size};
  };
  struct Rows {
    uint64_t k, v;
    uint32_t mask;
  };
  auto rows_of = [&](int tile, Entry at) {
    const int pos = KS * tile + (lane & (KS - 1));
    const bool is_new = k_new && pos == sp.n;
    const bool ok = pos >= sp.first && pos < sp.last && (is_new || at.id >= 0);
    const int64_t page = max(at.id, 0);
    const T *kr = static_cast<const T *>(p.k_cache) + page * p.kc_ps + at.off * p.kc_ls + hk * p.kc_hs;
    const T *vr = static_cast<const T *>(p.v_cache) + page * p.vc_ps + at.off * p.vc_ls + hk * p.vc_hs;
    Rows r;
    r.k = reinterpret_cast<uint64_t>(is_new ? k_new : kr), r.v = reinterpret_cast<uint64_t>(is_new ? v_new : vr);
    r.mask = (uint32_t)__ballot(ok) & (uint32_t)((1ull << KS) - 1);
    const int src = ok || !r.mask ? (lane & (KS - 1)) : __builtin_ctz(r.mask);
    r.k = __shfl(r.k, src, 64), r.v = __shfl(r.v, src, 64);
    return r;
  };
  Raw kr[KB][NT], vr[NV];
  auto load_k = [&](const Rows &r) {
#pragma unroll
    for (int h = 0; h < NT; ++h) {
      const T *row = reinterpret_cast<const T *>(__shfl(r.k, F::krow(i, h), 64));
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) kr[kb][h] = piece(row, KS * kb + V * g, dk);
    }
  };
  auto load_v = [&](const Rows &r) {
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int id = n * 64 + lane;
      vr[n] = piece(reinterpret_cast<const T *>(__shfl(r.v, id / PER, 64)), id % PER * V, dv);
    }
  };

  E *tile_v = reinterpret_cast<E *>(area[wave]);
  const float scale = p.scale * kLog2e;
  float m = -__builtin_inff(), l = 0.f;
  f32x4 o[OT];
#pragma unroll
  for (int d = 0; d < OT; ++d) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};

  int t = begin + wave;
  Rows now{}, next{};
  Entry id_next{};
  if (t < end) {
    now = rows_of(t, page_of(t));
    load_k(now), load_v(now);
    if (t + kWaves < end) id_next = page_of(t + kWaves);
  }
  for (; t < end; t += kWaves) {
    const bool more = t + kWaves < end;
    f32x4 s[NT];
    if (dk < D) {
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int h = 0; h < NT; ++h) kr[kb][h] = within(kr[kb][h], KS * kb + V * g, dk);
    }
#pragma unroll
    for (int h = 0; h < NT; ++h) {
      s[h] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) s[h] = F::mma_raw(kr[kb][h], qf[kb], s[h]);
    }
    if (more) {
      next = rows_of(t + kWaves, id_next);
      load_k(next);
      if (t + 2 * kWaves < end) id_next = page_of(t + 2 * kWaves);
    }
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int id = n * 64 + lane;
      *reinterpret_cast<Raw *>(tile_v + F::template place<LD>(id / PER, id % PER)) = vr[n];
    }
    if (more) load_v(next);
    if (now.mask) {
      float v[V];
      F::gather(s, v);
      const uint32_t mine = now.mask >> (V * g);
      float top = -__builtin_inff();
#pragma unroll
      for (int e = 0; e < V; ++e) {
        v[e] = (mine >> e & 1) ? v[e] * scale : -__builtin_inff();
        top = fmaxf(top, v[e]);
      }
      top = fmaxf(top, __shfl_xor(top, 16, 64));
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      const float m_new = fmaxf(fmaxf(m, top), kLow), shrink = fast_exp2(m - m_new);
      m = m_new;
      l *= shrink;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        v[e] = fast_exp2(v[e] - m) * kLift;
        l += v[e];
      }
      const Raw pf = F::pack(v);  // 0 .. kLift: the type's own format holds them; l has them unrounded
#pragma unroll
      for (int d = 0; d < OT; ++d) {
        o[d] *= shrink;
        o[d] = F::mma_raw(Columns(d, i, g).columns(area[wave]), pf, o[d]);
      }
    }
    now = next;
  }

  // the waves' shares together: lane (i, g) has head i, values 16 d + 4 g ..; l is the sum over a head's four lanes
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
  asm volatile("" ::: "memory");  // the same LDS as numbers of another type
  float *mine = reinterpret_cast<float *>(area[wave]) + i * (D + 4);
#pragma unroll
  for (int d = 0; d < OT; ++d) *reinterpret_cast<f32x4 *>(mine + 16 * d + 4 * g) = o[d];
  if (g == 0) wave_m[wave][i] = m, wave_l[wave][i] = l;
  __syncthreads();
  for (int x = tid; x < heads * D; x += kThreads) {
    const int h = x / D, col = x % D;
    float top = -__builtin_inff(), sum = 0.f, acc = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) top = fmaxf(top, wave_m[w][h]);
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      if (wave_m[w][h] == -__builtin_inff()) continue;  // a wave that has seen no position
      const float f = fast_exp2(wave_m[w][h] - top);
      sum = __builtin_fmaf(f, wave_l[w][h], sum);
      acc = __builtin_fmaf(f, reinterpret_cast<const float *>(area[w])[h * (D + 4) + col], acc);
    }
    const bool none = top == -__builtin_inff();
    if (whole) {
      if (col < dv) st1<T>(static_cast<T *>(p.out) + b * p.out_bs + (h0 + h) * p.out_hs + col, none ? 0.f : acc / sum);
    } else {
      const int64_t place = ((int64_t)range + b) * p.nheads + h0 + h;
      p.ws[place * D + col] = acc;
      if (col == 0) {
        float *ml = p.ws + (int64_t)(p.nsplit + p.batch) * p.nheads * D + place * 2;
        ml[0] = top, ml[1] = sum;
      }
    }
  }
  at += sp.count();
  if (at >= hi) break;
  ++b;
  __syncthreads();
  }
}

// The parts of a sequence together: one workgroup per (batch, head).  What each part's sums are multiplied by is found first, for all
// of them at once (one after another that took as long as the cache itself, 108 us for 256 parts); then the threads add up rows of
// parts, four columns each, and the rows' shares meet in LDS, in a fixed order.
constexpr int kMostParts = 512;
template <typename T, int D, int KS> __global__ __launch_bounds__(kThreads) void paged_join_kernel(const PagedAttnParams p) {
  constexpr int TURN = kThreads / (D / 4);
  __shared__ __align__(16) float acc_of[TURN][D];
  __shared__ float factor[kMostParts], wave_top[kWaves], wave_sum[kWaves];
  const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
  const int64_t share = share_of(p, tiles_before<KS>(p, p.batch)), at = tiles_before<KS>(p, b);
  const int first = (int)(at / share), parts = (int)((at + span_of<KS>(p, b).count() - 1) / share) - first + 1;
  if (parts <= 1) return;
  const int64_t place = ((int64_t)first + b) * p.nheads + h;  // of the first part; the others p.nheads further each
  const float *ml = p.ws + (int64_t)(p.nsplit + p.batch) * p.nheads * D + place * 2;
  float m[kMostParts / kThreads], l[kMostParts / kThreads], top = -__builtin_inff(), sum = 0.f;
#pragma unroll
  for (int n = 0; n < kMostParts / kThreads; ++n) {
    const int64_t from = min(n * kThreads + tid, parts - 1) * (int64_t)p.nheads * 2;
    m[n] = ml[from], l[n] = ml[from + 1];
    top = fmaxf(top, m[n]);
  }
#pragma unroll
  for (int step = 1; step < 64; step *= 2) top = fmaxf(top, __shfl_xor(top, step, 64));
  if (tid % 64 == 0) wave_top[tid / 64] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) top = fmaxf(top, wave_top[w]);
#pragma unroll
  for (int n = 0; n < kMostParts / kThreads; ++n) {
    const int s = n * kThreads + tid;
    const float f = m[n] == -__builtin_inff() ? 0.f : fast_exp2(m[n] - top);  // (a part that has seen no position)
    if (s < parts) sum = __builtin_fmaf(f, l[n], sum);
    factor[s] = f;
  }
#pragma unroll
  for (int step = 1; step < 64; step *= 2) sum += __shfl_xor(sum, step, 64);
  if (tid % 64 == 0) wave_sum[tid / 64] = sum;
  __syncthreads();
  const int col = tid % (D / 4) * 4, turn = tid / (D / 4);
  const float *src = p.ws + place * D + col;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = turn; s < parts; s += TURN) acc += factor[s] * *reinterpret_cast<const f32x4 *>(src + (int64_t)s * p.nheads * D);
  if (turn < TURN) *reinterpret_cast<f32x4 *>(&acc_of[turn][col]) = acc;  // (96 columns leave 16 threads over)
  __syncthreads();
  if (tid < p.headdim_v) {
    float v = 0.f;
    sum = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) sum += wave_sum[w];
#pragma unroll
    for (int t = 0; t < TURN; ++t) v += acc_of[t][tid];
    st1<T>(static_cast<T *>(p.out) + b * p.out_bs + h * p.out_hs + tid, top == -__builtin_inff() ? 0.f : v / sum);
  }
}

// ------------------------------------------------------------------ host side
int size_class(const PagedAttnParams &p) {
  const int most = std::max(p.headdim_k, p.headdim_v);
  return most <= 64 ? 64 : most <= 96 ? 96 : most <= 128 ? 128 : 256;
}
int rows_of_batch(const PagedAttnParams &p) { return p.nkvheads * ((p.nheads / p.nkvheads + kHeads - 1) / kHeads); }
template <typename T, int D> int run(const PagedAttnParams &p, hipStream_t st) {
  constexpr int V = Frags<T>::V;
  const int64_t n = p.nsplit == 1 ? p.batch : p.nsplit, workgroups = rows_of_batch(p) * (n >= 8 ? (n + 7) / 8 * 8 : n);
  if (workgroups > 1 << 30 || (p.nsplit > 1 && p.nheads > 1 << kRowBits)) return MAMBA_E_UNSUPPORTED;
  const dim3 grid((int)std::min<int64_t>(workgroups, 1 << kRowBits), (int)((workgroups - 1) >> kRowBits) + 1);
  if (p.headdim_k % V == 0 && p.headdim_v % V == 0) paged_part_kernel<T, D, false><<<grid, kThreads, 0, st>>>(p);
  else paged_part_kernel<T, D, true><<<grid, kThreads, 0, st>>>(p);
  if (hipGetLastError() != hipSuccess) return MAMBA_E_LAUNCH;
  if (p.nsplit > 1) {
    paged_join_kernel<T, D, Frags<T>::KS><<<dim3(p.nheads, p.batch), kThreads, 0, st>>>(p);
    if (hipGetLastError() != hipSuccess) return MAMBA_E_LAUNCH;
  }
  return MAMBA_OK;
}
template <typename T> int run_size(const PagedAttnParams &p, hipStream_t st) {
  switch (size_class(p)) {
    case 64: return run<T, 64>(p, st);
    case 96: return run<T, 96>(p, st);
    case 128: return run<T, 128>(p, st);
    default: return run<T, 256>(p, st);
  }
}
int check(const PagedAttnParams *p) {
  if (!p) return MAMBA_E_BADARG;
  if (p->batch <= 0 || p->nheads <= 0 || p->nkvheads <= 0 || p->nheads % p->nkvheads != 0 || p->headdim_k <= 0 || p->headdim_v <= 0)
    return MAMBA_E_BADARG;
  if (p->page_size <= 0 || p->num_pages <= 0 || p->max_pages <= 0 || p->window < 0 || p->dtype < MAMBA_F32 || p->dtype > MAMBA_F16)
    return MAMBA_E_BADARG;
  if (!(p->scale >= -2e38f && p->scale <= 2e38f)) return MAMBA_E_BADARG;  // (times log2(e) it is a number too)
  if (p->headdim_k > 256 || p->headdim_v > 256 || (int64_t)p->max_pages * p->page_size > 1 << 30) return MAMBA_E_UNSUPPORTED;
  return MAMBA_OK;
}

}  // namespace

extern "C" int paged_attn_parts(const PagedAttnParams *p) {
  if (const int rc = check(p)) return rc;
  const int64_t rows = rows_of_batch(*p), longest = (int64_t)p->max_pages * p->page_size, most = p->window > 0 ? std::min<int64_t>(p->window, longest) : longest;
  const int64_t tile = p->dtype == MAMBA_F32 ? 16 : 32, parts = (most + 2 * kWaves * tile - 1) / (2 * kWaves * tile);  // of a sequence
  const int64_t places = (int64_t)cu_count() * workgroups(size_class(*p));  // that the chip holds at a time
  if (parts <= 1 || p->batch * rows >= 4 * places) return 1;
  const int64_t n = std::min<int64_t>({places / rows, parts * p->batch, (int64_t)kMostParts});
  return (int)std::max<int64_t>(1, n >= 8 ? n / 8 * 8 : n);  // (as many for every XCD)
}
extern "C" int64_t paged_attn_ws_bytes(const PagedAttnParams *p) {
  if (const int rc = check(p)) return rc;
  if (p->nsplit <= 0 || p->nsplit > kMostParts) return MAMBA_E_BADARG;
  return p->nsplit == 1 ? 0 : ((int64_t)p->nsplit + p->batch) * p->nheads * (size_class(*p) + 2) * 4;
}
extern "C" int paged_attn_update(const PagedAttnParams *p, mamba_stream_t stream) {
  if (const int rc = check(p)) return rc;
  if (!p->q || !p->k_cache || !p->v_cache || !p->block_table || !p->cache_seqlens || !p->out || (p->k == nullptr) != (p->v == nullptr))
    return MAMBA_E_BADARG;
  if (p->nsplit <= 0 || p->nsplit > kMostParts || (p->nsplit > 1 && (!p->ws || reinterpret_cast<uintptr_t>(p->ws) % 16 != 0))) return MAMBA_E_BADARG;
  if (p->batch > 65535) return MAMBA_E_UNSUPPORTED;
  if (p->out == p->k || p->out == p->v || p->out == p->k_cache || p->out == p->v_cache) return MAMBA_E_BADARG;  // (others still read them)
  hipStream_t st = static_cast<hipStream_t>(stream);
  switch (p->dtype) {
    case MAMBA_F32: return run_size<float>(*p, st);
    case MAMBA_BF16: return run_size<bf16_t>(*p, st);
    default: return run_size<f16_t>(*p, st);
  }
}
