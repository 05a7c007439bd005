// Linear attention with a decay per head, forward and backward (gfx950): the walk that all of them are.
//
//   S_t = f S_{t-1} + k_t v_t^T,   o_t = scale q_t S_t,   f = exp(log_decay[head])
// With rows a, b of `key` values and rows c of `val` values, the walk
//   y_t = mix sum_{s <= t} f^(t - s) (a_t . b_s) c_s + read f^(t + late) a_t Z,     t, s = 0, 1, .. from its first position
//   Z' = f^n Z + write sum_{s < n} f^(n - late - s) b_s c_s^T                       after n positions
// is (a, b, c) = (q, k, v) for the outputs; (do, v, k) on Z^T for dq; and from the last position to the first, with late = 0
// (what comes in has been scaled already), (v, do, q) for dk and (k, q, do) for dv, whose Z ends as the gradient of the
// initial state.  All four are one kernel.
#pragma once
#include "mma_frag.hpp"

#include <type_traits>

// Rows by position and head: element (b, t, h, x) at p[b * bs + t * ls + h * hs + x].
struct LinRows {
  void *p;
  int64_t bs, ls, hs;
  int32_t group; // q heads that share a head of this tensor
};
struct LinState { // element (sequence, head, k, v) at p[(sequence * nheads + head) * key * val + k * ks + v * vs]
  float *p;
  int32_t ks, vs;
};
struct LinWalk {
  LinRows a, b, c, y; // y is written
  LinState start, end; // p null: zeros, not wanted
  float mix, read, write;
  int32_t key, val, reverse, late;
  int32_t y_f32; // y in fp32, whatever the operands' type
};
struct LinLaunch {
  LinWalk w[3];
  const float *log_decay;
  const int32_t *cu;   // null: the rows of the batch are the sequences
  const int32_t *plan; // null, or per item: sequence, first position, positions, number of items of its sequence before it
  f32x4 *segs;         // states of the segments, as the lanes hold them
  int32_t nwalks, nheads, kv_heads, slices, items, nseg, seg_len, nseq, seqlen;
};

namespace lin {

constexpr int kThreads = 256, kWaves = 4;
// A launch takes fewer than 2^32 threads along x: workgroups beyond 2^23 lie along y.
constexpr int kRowBits = 23;

// The positions that a workgroup walks: [first, first + n) of row `b`, counted in the order of the walk.
struct Item {
  int b, seq, first, n, before, len; // before: segments of the sequence before this one; len: the sequence's positions
  bool zero;                         // positions outside of all sequences
};

DEVI Item item_of(const LinLaunch &p, int index) {
  Item it;
  it.zero = false;
  if (p.plan) {
    const int4 v = reinterpret_cast<const int4 *>(p.plan)[index];
    const int n_all = reinterpret_cast<const int4 *>(p.plan)[p.items].x;
    it.b = 0, it.seq = v.x, it.first = v.y, it.len = v.z, it.before = v.w;
    if (index >= n_all) it.seq = -1, it.len = 0, it.before = 0;
    if (it.seq >= p.nseq) it.zero = true;
  } else if (p.cu) {
    it.b = 0, it.before = 0, it.seq = index;
    if (index < p.nseq) {
      it.first = min(max(p.cu[index], 0), p.seqlen);
      it.len = min(max(p.cu[index + 1], it.first), p.seqlen) - it.first;
    } else {  // what lies before the first sequence, and behind the last
      it.zero = true;
      const int at = min(max(p.cu[index == p.nseq ? 0 : p.nseq], 0), p.seqlen);
      it.first = index == p.nseq ? 0 : at;
      it.len = index == p.nseq ? at : p.seqlen - at;
    }
  } else {
    it.b = it.seq = index / p.nseg, it.before = index % p.nseg;
    it.first = 0, it.len = p.seqlen;
  }
  it.n = min(it.len - it.before * p.seg_len, p.seg_len);
  if (it.zero || p.nseg == 1) it.n = it.len;
  return it;
}

// What a workgroup is: a walk, an item, a head, a slice of the values.  The walks, the slices and the heads that share keys read
// the same rows at the same time: they are neighbours on one XCD (workgroups go to the 8 XCDs in turn).
struct Place {
  int walk, item, head, slice;
  bool none;
};
DEVI Place place_of(const LinLaunch &p) {
  Place at;
  const int group = p.nheads / p.kv_heads, inner = p.nwalks * p.slices * group;
  const int block = blockIdx.y << kRowBits | blockIdx.x, xcd = block & 7, r = block >> 3;
  int in = r % inner;
  const int outer = (r / inner) * 8 + xcd;
  at.none = outer >= p.items * p.kv_heads;
  at.walk = in % p.nwalks, in /= p.nwalks;
  at.slice = in % p.slices, in /= p.slices;
  at.item = outer / p.kv_heads;
  at.head = (outer % p.kv_heads) * group + in;
  return at;
}

// log2 of the decay of one position.  Decays down to minus infinity are decays to nothing; above 0 they count as 0, NaN stays.
DEVI float log2_decay(float l) {
  l = l > 0.f ? 0.f : l;
  return (l < -1e6f ? -1e6f : l) * kLog2e;
}

// Rows less than 2^22 elements apart are read through uniform pointers and 32-bit places of the lanes.
constexpr int64_t kNear = 1 << 22;
DEVI bool near(const LinRows &r) { return r.ls <= kNear && r.ls >= -kNear; }

// the same pointer, in scalar registers
template <typename P> DEVI P *uniform_pointer(P *p) {
  const uint64_t a = reinterpret_cast<uint64_t>(p);
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)a), hi = __builtin_amdgcn_readfirstlane((uint32_t)(a >> 32));
  return reinterpret_cast<P *>((uint64_t)hi << 32 | lo);
}

// How the head sizes lie in those that a kernel is made for: they are those; whole pieces of 16 bytes less; any number less, read
// element by element.
enum Fit { WHOLE, PIECES, ELEMENTS };

// C rows x COLS columns of a tensor on their way to LDS, in pieces of 16 bytes; rows from n on and columns from `cols` on become 0.
template <typename T, int C, int COLS, Fit FIT> struct Stage {
  using F = Frags<T>;
  static constexpr int V = F::V, PER = COLS / V, N = C * PER / kThreads, RUN = kThreads / PER;  // rows of a turn
  static_assert(C * PER % kThreads == 0 && kThreads % PER == 0, "whole pieces per thread");
  using Raw = typename F::Raw;
  Raw w[N];
  // whole blocks of near rows: where the next block's lowest row lies, bytes from a turn's rows to the next's and from block to block, the
  // thread's place
  const char *low;
  int64_t run, step;
  uint32_t place;
  int cols, lds;  // lds: of the piece in the tile
  DEVI Stage(const T *first, int64_t ls, int cols_, int tid) : cols(cols_), lds((int)sizeof(typename F::E) * F::template place<COLS>(tid / PER, tid % PER)) {
    const int row = tid / PER;
    const bool back = ls < 0;
    low = uniform_pointer(reinterpret_cast<const char *>(back ? first + (RUN - 1) * ls : first));  // a turn's rows lie from here on
    run = RUN * ls * (int64_t)sizeof(T), step = C * ls * (int64_t)sizeof(T);
    place = (uint32_t)((back ? RUN - 1 - row : row) * (int)(back ? -ls : ls) + (FIT == WHOLE ? tid % PER * V : FIT == PIECES ? min(tid % PER * V, cols - V) : 0)) * (uint32_t)sizeof(T);
  }
  DEVI void fetch_next() {
    asm("" : "+s"(low));  // (it stays a scalar: one register of offsets and no 64-bit sums in the lanes)
#pragma unroll
    for (int q = 0; q < N; ++q) w[q] = any(reinterpret_cast<const T *>(low + q * run + place));
    low += step;
  }
  // `at`: the block's first row, ls: to the next one
  DEVI void fetch(const T *at, int64_t ls, int n, int tid) {
#pragma unroll
    for (int q = 0; q < N; ++q) {
      const int id = q * kThreads + tid, row = min(id / PER, n - 1), col = id % PER * V;
      const T *src = at + (int64_t)row * ls;
      if constexpr (FIT == ELEMENTS) {
        typename F::E v[V];
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = *(const GLOBAL_AS typename F::E *)(src + min(col + e, cols - 1));
        w[q] = __builtin_bit_cast(Raw, v);
      } else {
        w[q] = any(src + min(col, cols - V));
      }
    }
  }
  template <bool FULL> DEVI void commit(char *tile, int n, int tid) const {
#pragma unroll
    for (int q = 0; q < N; ++q) {
      const int id = q * kThreads + tid, row = id / PER, col = id % PER * V;
      Raw v = w[q];
      if constexpr (FIT == ELEMENTS) {
        typename F::E e[V];
        __builtin_memcpy(e, &v, 16);
#pragma unroll
        for (int k = 0; k < V; ++k) e[k] = row < n && col + k < cols ? e[k] : typename F::E(0);
        __builtin_memcpy(&v, e, 16);
      } else if constexpr (!FULL || FIT == PIECES) {
        const bool ok = (FULL || row < n) && (FIT == WHOLE || col < cols);
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = ok ? v[k] : 0;
      }
      // (the order of a row's pieces repeats every 16 rows)
      const int at = RUN % 16 == 0 ? lds + F::size(q * RUN, COLS) : (int)sizeof(typename F::E) * F::template place<COLS>(row, id % PER);
      *reinterpret_cast<Raw *>(tile + at) = v;
    }
  }
  static DEVI Raw any(const T *at) {
    if constexpr (std::is_same_v<T, float>) return *(const GLOBAL_AS f32x4_a4 *)at;
    else return *(const GLOBAL_AS u32x4_a2 *)at;
  }
};

// A workgroup of 4 waves, DVT tiles of 16 values each: its state (KD keys) lies in their registers, the rows of a block of C positions
// and of the next one in LDS.
template <typename T, int KD, int DVT> struct Shape {
  using F = Frags<T>;
  // (16 positions of fp32 rows: two stages of 32 leave room for one workgroup or none)
  static constexpr int C = sizeof(T) == 4 ? 16 : 32;
  static constexpr int KB = KD / F::KS, JB = C / F::KS, IT = C / 16;
  static constexpr int VAL = 64 * DVT;
  static constexpr int TILES = DVT * KB * F::NT;  // tiles of a wave's state
  // blocks of 16 t and KS s that have an s <= t, row by row
  static constexpr int block_of(int ib, int jb) {
    int n = 0;
    for (int r = 0; r < ib; ++r) n += (16 * r + 15) / F::KS + 1;
    return n + jb;
  }
  static constexpr int BLOCKS = block_of(IT, 0);
  static_assert(BLOCKS * F::NT <= kWaves, "a tile of scores a wave");
  // LDS, bytes: rows a, b, c of a stage, two of them; decayed scores, twice; y
  static constexpr int B = F::size(C, KD), CC = 2 * B, STAGE = CC + F::size(C, VAL);
  static constexpr int SCORES = BLOCKS * 64 * (int)sizeof(typename F::Wide), AT_SCORES = 2 * STAGE, AT_Y = AT_SCORES + 2 * SCORES;
  static constexpr int LDS = AT_Y + F::size(C, VAL);
  // workgroups of a CU: what the LDS has room for and what the registers hold without spills (128, 256 or 512 a lane)
  static constexpr int ROOM = 160 * 1024 / LDS, MOST = TILES <= 4 ? 4 : KD <= 128 ? 2 : 1;
  static constexpr int WORKGROUPS = ROOM < 1 ? 1 : ROOM < MOST ? ROOM : MOST;
};

// f^n = 2^(n l2) of a head
struct Decay {
  float l2;
  DEVI float operator()(int n) const { return fast_exp2(l2 * (float)n); }
  DEVI float uniform(int n) const { return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, (*this)(n)))); }
};
// What the whole blocks of a walk are weighted with: products of what a lane and what an element has of f^n, neither above 1.
template <typename F, int JB, int IT> struct Weights {
  float in_lane, in_block[IT];                    // read f^(16 ib + i + late) of y's rows
  float up_lane, up_element[F::V], up_block[JB];  // write f^(last - KS jb - V g - e) of c's rows
  float keep;                                     // f^C
  DEVI Weights(const Decay &f, float read, float write, int late, int i, int g) {
    in_lane = read * f(i + late);
    up_lane = write * f(F::V * (3 - g) + (1 - late));  // last = C - late, the last block's last group: f^(C - late - (C - 4 V + V g + V - 1))
#pragma unroll
    for (int n = 0; n < IT; ++n) in_block[n] = f.uniform(16 * n);
#pragma unroll
    for (int n = 0; n < JB; ++n) up_block[n] = f.uniform(F::KS * (JB - 1 - n));
#pragma unroll
    for (int e = 0; e < F::V; ++e) up_element[e] = f.uniform(F::V - 1 - e);
    keep = f.uniform(F::KS * JB);
  }
};

// ---- the state of a wave: lane (i, g) of tile (d, kb, half) has the keys KS kb + krow(4 g + r, half) of value 16 d + i
template <typename T, int KD, int DVT> struct WaveState {
  using F = Frags<T>;
  using Sh = Shape<T, KD, DVT>;
  using Values = typename F::template ColumnLane<Sh::VAL>;
  f32x4 t[DVT][Sh::KB][F::NT];
  template <typename G> DEVI void each(G f) {
#pragma unroll
    for (int d = 0; d < DVT; ++d)
#pragma unroll
      for (int kb = 0; kb < Sh::KB; ++kb)
#pragma unroll
        for (int h = 0; h < F::NT; ++h) f(t[d][kb][h], (d * Sh::KB + kb) * F::NT + h);
  }
  DEVI void zero() {
    each([](f32x4 &v, int) { v = f32x4{0.f, 0.f, 0.f, 0.f}; });
  }
  // x = f(x, tile of values, key, whether there is such a key) for every element
  template <typename G> DEVI void each_element(int g, int key, G f) {
#pragma unroll
    for (int d = 0; d < DVT; ++d)
#pragma unroll
      for (int kb = 0; kb < Sh::KB; ++kb)
#pragma unroll
        for (int h = 0; h < F::NT; ++h)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int k = F::KS * kb + F::krow(4 * g + r, h);
            t[d][kb][h][r] = f(t[d][kb][h][r], d, k, k < key);
          }
  }
  // f^n Z + write b^T diag(f^(n - late - s)) c over the n positions of a block's rows, the weighted c in two parts or three (W)
  template <bool FULL, typename W, typename WT>
  DEVI void update(const char *b_rows, const char *c_rows, const typename F::template Lane<KD> &lanes, const Values &values, const Decay &f, const WT &weights,
                   float write, int n, int late, int g) {
    constexpr int V = F::V;
    const float keep = FULL ? weights.keep : f(n);
    each([&](f32x4 &v, int) { v *= keep; });
#pragma unroll
    for (int jb = 0; jb < Sh::JB; ++jb) {
      W wc[DVT];
#pragma unroll
      for (int d = 0; d < DVT; ++d) {
        float v[V];
        F::unpack(values.columns(c_rows + F::size(F::KS * jb, Sh::VAL), d), v);
        if constexpr (FULL) {
          const float lane = weights.up_lane * weights.up_block[jb];
#pragma unroll
          for (int e = 0; e < V; ++e) v[e] = v[e] * weights.up_element[e] * lane;
        } else {
#pragma unroll
          for (int e = 0; e < V; ++e) v[e] *= write * f(max(n - late - (F::KS * jb + V * g + e), 0));
        }
        wc[d] = F::template wide<W>(v);
      }
#pragma unroll
      for (int kb = 0; kb < Sh::KB; ++kb)
#pragma unroll
        for (int h = 0; h < F::NT; ++h) {
          const typename F::Data b = F::data(lanes.columns(b_rows + F::size(F::KS * jb, KD), kb, h));
#pragma unroll
          for (int d = 0; d < DVT; ++d) t[d][kb][h] = mma16(b, wc[d], t[d][kb][h]);
        }
    }
  }
};

// Element (first position of the segment, 0) of a tensor's head, and the step from one position of the walk to the next.
DEVI int64_t rows_at(const LinRows &r, const Item &it, int head, int reverse, int seg_len, int64_t &ls) {
  const int64_t before = (int64_t)it.before * seg_len;
  ls = reverse ? -r.ls : r.ls;
  return it.b * r.bs + (head / r.group) * r.hs + (reverse ? it.first + it.len - 1 - before : it.first + before) * r.ls;
}

}  // namespace lin
