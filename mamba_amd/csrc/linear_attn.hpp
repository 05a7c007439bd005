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
  const int xcd = blockIdx.x & 7, r = blockIdx.x >> 3;
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

// C rows x COLS columns of a tensor on their way to LDS, in pieces of 16 bytes; rows from n on and columns from `cols` on
// become 0.  RAG: `cols` may be any number.
template <typename T, int C, int COLS, bool RAG> struct Stage {
  using F = Frags<T>;
  static constexpr int V = F::V, PER = COLS / V, N = C * PER / kThreads, PITCH = COLS + F::PAD;
  static_assert(C * PER % kThreads == 0, "whole pieces per thread");
  using Raw = typename F::Raw;
  Raw w[N];
  DEVI void fetch(const T *at, int64_t ls, int n, int cols, int tid) {
#pragma unroll
    for (int q = 0; q < N; ++q) {
      const int id = q * kThreads + tid, row = min(id / PER, n - 1), col = id % PER * V;
      const T *src = at + (int64_t)row * ls;
      if constexpr (RAG) {
        typename F::E v[V];
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = *(const GLOBAL_AS typename F::E *)(src + min(col + e, cols - 1));
        w[q] = __builtin_bit_cast(Raw, v);
      } else {
        w[q] = any(src + min(col, cols - V));
      }
    }
  }
  DEVI void commit(typename F::E *lds, int n, int cols, int tid) const {
#pragma unroll
    for (int q = 0; q < N; ++q) {
      const int id = q * kThreads + tid, row = id / PER, col = id % PER * V;
      Raw v = w[q];
      if constexpr (RAG) {
        typename F::E e[V];
        __builtin_memcpy(e, &v, 16);
#pragma unroll
        for (int k = 0; k < V; ++k) e[k] = row < n && col + k < cols ? e[k] : typename F::E(0);
        __builtin_memcpy(&v, e, 16);
      } else {
        const bool ok = row < n && col < cols;
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = ok ? v[k] : 0;
      }
      *reinterpret_cast<Raw *>(lds + row * PITCH + col) = v;
    }
  }
  static DEVI Raw any(const T *at) {
    if constexpr (std::is_same_v<T, float>) return *(const GLOBAL_AS f32x4_a4 *)at;
    else return *(const GLOBAL_AS u32x4_a2 *)at;
  }
};

template <typename T, int KD, int DVT> struct Shape {
  using F = Frags<T>;
  static constexpr int C = std::is_same_v<T, float> ? 32 : 64;  // positions of a block
  static constexpr int KB = KD / F::KS, JB = C / F::KS, IT = C / 16;
  static constexpr int WV = 16 * DVT, VAL = kWaves * WV;         // values of a wave, of a workgroup
  static constexpr int TILES = KB * F::NT * DVT;                 // tiles of a wave's state
  static constexpr bool PAIR = F::NT == 2 && DVT == 2;           // a lane's 8 values lie side by side
  static constexpr int PK = KD + F::PAD, PV = VAL + F::PAD;
};

// ---- the state of a wave: tile (kb, half, d) has keys KS kb + krow(m, half) and values value(n, d)
template <typename T, int KD, int DVT> struct WaveState {
  using F = Frags<T>;
  using Sh = Shape<T, KD, DVT>;
  f32x4 t[Sh::KB][F::NT][DVT];
  static DEVI int value(int i, int d) { return Sh::PAIR ? 8 * (i >> 2) + (i & 3) + 4 * d : 16 * d + i; }
  DEVI void zero() {
    each([](f32x4 &v, int) { v = f32x4{0.f, 0.f, 0.f, 0.f}; });
  }
  template <typename G> DEVI void each(G f) {
#pragma unroll
    for (int kb = 0; kb < Sh::KB; ++kb)
#pragma unroll
      for (int h = 0; h < F::NT; ++h)
#pragma unroll
        for (int d = 0; d < DVT; ++d) f(t[kb][h][d], (kb * F::NT + h) * DVT + d);
  }
  // x = f(x, key, value, whether there is such a place in memory) for every element
  template <typename G> DEVI void each_element(int i, int g, int key, int val, int v0, G f) {
#pragma unroll
    for (int kb = 0; kb < Sh::KB; ++kb)
#pragma unroll
      for (int h = 0; h < F::NT; ++h)
#pragma unroll
        for (int d = 0; d < DVT; ++d)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int k = F::KS * kb + F::krow(4 * g + r, h), v = v0 + value(i, d);
            t[kb][h][d][r] = f(t[kb][h][d][r], k, v, k < key && v < val);
          }
  }
  DEVI void scale(float f) {
    each([&](f32x4 &v, int) { v *= f; });
  }
  // + write b^T diag(f^(n - late - s)) c over the block's positions
  DEVI void update(const typename F::E *b, const typename F::Raw (&cf)[Sh::JB][DVT], float l2, float write, int last, int i, int g) {
    constexpr int V = F::V;
#pragma unroll
    for (int jb = 0; jb < Sh::JB; ++jb) {
      float f[V];
#pragma unroll
      for (int e = 0; e < V; ++e) f[e] = write * fast_exp2(l2 * (float)max(last - (F::KS * jb + V * g + e), 0));
      typename F::Wide wc[DVT];
#pragma unroll
      for (int d = 0; d < DVT; ++d) {
        float v[V];
        F::unpack(cf[jb][d], v);
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] *= f[e];
        wc[d] = F::wide(v);
      }
#pragma unroll
      for (int kb = 0; kb < Sh::KB; ++kb)
#pragma unroll
        for (int h = 0; h < F::NT; ++h) {
          const auto bt = F::data(F::template columns<Sh::PK>(b + F::KS * jb * Sh::PK, F::KS * kb, h, i, g));
#pragma unroll
          for (int d = 0; d < DVT; ++d) t[kb][h][d] = mma16(bt, wc[d], t[kb][h][d]);
        }
    }
  }
};

// c^T fragments of the block for a wave's values
template <typename T, int KD, int DVT>
DEVI void value_frags(const typename Frags<T>::E *c, typename Frags<T>::Raw (&cf)[Shape<T, KD, DVT>::JB][DVT], int wave, int i, int g) {
  using F = Frags<T>;
  using Sh = Shape<T, KD, DVT>;
#pragma unroll
  for (int jb = 0; jb < Sh::JB; ++jb)
#pragma unroll
    for (int d = 0; d < DVT; ++d) {
      const auto *at = c + F::KS * jb * Sh::PV;
      if constexpr (Sh::PAIR) cf[jb][d] = F::template columns<Sh::PV>(at, wave * Sh::WV, d, i, g);
      else cf[jb][d] = F::template columns_in_order<Sh::PV>(at, wave * Sh::WV + 16 * d, i, g);
    }
}

// Element (first position of the segment, 0) of a tensor's head, and the step from one position of the walk to the next.
DEVI int64_t rows_at(const LinRows &r, const Item &it, int head, int reverse, int seg_len, int64_t &ls) {
  const int64_t before = (int64_t)it.before * seg_len;
  ls = reverse ? -r.ls : r.ls;
  return it.b * r.bs + (head / r.group) * r.hs + (reverse ? it.first + it.len - 1 - before : it.first + before) * r.ls;
}

}  // namespace lin
