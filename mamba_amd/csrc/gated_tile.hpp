// Tiles of the gated linear recurrence: what the forward and the backward kernel of gated_scan.hip share.
//
// A row of positions is a linear recurrence per channel, h = a h + b, and a run of positions is one such step (A, B)
// again.  The row is cut into tiles of positions and groups of 64 V channels.  A workgroup holds one tile of one group
// in registers: a wave has R positions after one another, its lanes V channels each.  The steps of the waves meet in
// LDS; the state that enters the tile comes from the workgroups of the tiles before it (`Chain`), so every tensor is
// read once and written once.
#pragma once
#include "gated_gates.hpp"

#include <type_traits>

namespace {

template <int V> struct Vec {
  float v[V];
  DEVI float &operator[](int e) { return v[e]; }
  DEVI const float &operator[](int e) const { return v[e]; }
};
template <int V> DEVI Vec<V> vec_of(float x) {
  Vec<V> r;
#pragma unroll
  for (int e = 0; e < V; ++e) r[e] = x;
  return r;
}

// W words that lie at the alignment of a 2- or 4-byte element.
template <int W, int A> struct Words;
template <int W> struct Words<W, 2> {
  typedef uint32_t type __attribute__((ext_vector_type(W), aligned(2)));
};
template <int W> struct Words<W, 4> {
  typedef uint32_t type __attribute__((ext_vector_type(W), aligned(4)));
};

// V neighbouring channels of one position as they lie in memory.
template <typename T, int V> struct Raw {
  static constexpr bool HALF = DT<T>::id != MAMBA_F32;
  static constexpr int W = HALF ? V / 2 : V;
  uint32_t w[W];
  DEVI void clear() {
#pragma unroll
    for (int i = 0; i < W; ++i) w[i] = 0;
  }
  // From here on its values are formed anew: kept since they were formed first they take twice the registers of the words.  (The
  // backward kernel of 16-bit rows spilled: 538 us at 8 x 4096 x 5120, without 512.  In 32 bits the words are the values.)
  DEVI void anew() {
    if constexpr (HALF) {
#pragma unroll
      for (int i = 0; i < W; ++i) asm("" : "+v"(w[i]));
    }
  }
  DEVI float get(int e) const {
    if constexpr (!HALF) return __builtin_bit_cast(float, w[e]);
    else if constexpr (DT<T>::id == MAMBA_BF16) return e & 1 ? bf16_hi(w[e / 2]) : bf16_lo(w[e / 2]);
    else return e & 1 ? f16_hi(w[e / 2]) : f16_lo(w[e / 2]);
  }
};

// How a lane reads and writes its channels c .. c + V - 1, in one piece at any alignment (gfx950 serves that; rows of 16-bit
// channels that begin off a word cost a quarter more).  WHOLE: the number of channels is a multiple of V, all of a lane's
// channels are there or none.  Otherwise a lane at the end reads the row's last V channels, and `get` moves its own to the
// front; rows of less than V channels (`few`) are read channel by channel.  Lanes past the last channel read the last ones
// again and write nothing.
template <typename T, int V, bool WHOLE> struct Lane {
  typedef Raw<T, V> R;
  int c, n, dim;     // the lane's first channel, how many of its channels are there, those of a row
  int shift;         // how far before c the channel read first lies
  uint32_t at, to;   // byte offsets in a row: of what is read, of c
  bool few;
  DEVI Lane(int c_, int dim_) : c(c_), dim(dim_), few(!WHOLE && dim_ < V) {
    n = min(max(dim - c, 0), V);
    const int from = max(min(c, dim - V), 0);
    shift = WHOLE ? 0 : min(c - from, V - 1);
    at = (uint32_t)from * sizeof(T);
    to = (uint32_t)c * sizeof(T);
  }
  // STREAM: past the caches' hold (the rows are read once, or written and not soon read)
  template <bool FEW = false, bool STREAM = false> DEVI R load(const T *row) const {
    R r;
    const GLOBAL_AS char *p = (const GLOBAL_AS char *)row;
    if constexpr (FEW) {
      uint32_t q[V];
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const uint32_t o = (uint32_t)min(e, dim - 1) * sizeof(T);
        if constexpr (sizeof(T) == 4) q[e] = *(const GLOBAL_AS uint32_t *)(p + o);
        else q[e] = *(const GLOBAL_AS uint16_t *)(p + o);
      }
#pragma unroll
      for (int i = 0; i < R::W; ++i) r.w[i] = R::HALF ? q[2 * i] | q[2 * i + 1] << 16 : q[i];
    } else {
      typedef typename Words<R::W, sizeof(T)>::type words;
      const GLOBAL_AS words *src = (const GLOBAL_AS words *)(p + at);
      const words v = STREAM ? __builtin_nontemporal_load(src) : *src;
#pragma unroll
      for (int i = 0; i < R::W; ++i) r.w[i] = v[i];
    }
    return r;
  }
  DEVI float get(const R &r, int e) const {
    if constexpr (WHOLE) {
      return r.get(e);
    } else {
      float v = r.get(e);
#pragma unroll
      for (int s = 1; s < V; ++s)
        if (e + s < V) v = shift == s ? r.get(e + s) : v;
      return v;
    }
  }
  // of rows of less than V channels and of others: f(rows of few channels), so that one branch stands around all loads
  template <typename F> DEVI void each_kind(F f) const {
    if constexpr (WHOLE) {
      f(std::false_type{});
    } else {
      if (few) f(std::true_type{});
      else f(std::false_type{});
    }
  }
  template <bool STREAM = false> DEVI void store(T *row, const Vec<V> &x) const {
    typedef typename Words<R::W, sizeof(T)>::type words;
    GLOBAL_AS char *p = (GLOBAL_AS char *)row;
    words v;
#pragma unroll
    for (int i = 0; i < R::W; ++i) {
      if constexpr (DT<T>::id == MAMBA_F32) v[i] = __builtin_bit_cast(uint32_t, x.v[i]);
      else if constexpr (DT<T>::id == MAMBA_BF16) v[i] = pack_bf16(x.v[2 * i], x.v[2 * i + 1]);
      else v[i] = pack_f16(x.v[2 * i], x.v[2 * i + 1]);
    }
    if (n == V) {
      GLOBAL_AS words *dst = (GLOBAL_AS words *)(p + to);
      if (STREAM) __builtin_nontemporal_store(v, dst);
      else *dst = v;
    } else if (!WHOLE) {
#pragma unroll
      for (int e = 0; e < V - 1; ++e)
        if (e < n) st1<T>(row + c + e, x[e]);
    }
  }
  DEVI Vec<V> load_state(const float *row) const {
    Vec<V> r;
#pragma unroll
    for (int e = 0; e < V; ++e) r[e] = e < n ? row[c + e] : 0.f;
    return r;
  }
  DEVI void store_state(float *row, const Vec<V> &x) const {
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (e < n) row[c + e] = x[e];
  }
};

// The step of a run of positions: h -> a h + b per channel.
// RESETS: a factor of exactly 0 marks a run in which a sequence starts; nothing before it counts, whatever it is.
template <int V> struct Step {
  Vec<V> a, b;
};
template <int V> DEVI Step<V> no_step() { return Step<V>{vec_of<V>(1.f), vec_of<V>(0.f)}; }
template <bool RESETS> DEVI float apply1(float a, float b, float h) {
  const float r = __builtin_fmaf(a, h, b);
  return RESETS && a == 0.f ? b : r;
}
template <bool RESETS> DEVI float factor1(float a, float next) {
  const float r = not_zero(a * next);
  return RESETS && (a == 0.f || next == 0.f) ? 0.f : r;
}
template <bool RESETS, int V> DEVI Vec<V> apply(const Step<V> &s, const Vec<V> &h) {
  Vec<V> r;
#pragma unroll
  for (int e = 0; e < V; ++e) r[e] = apply1<RESETS>(s.a[e], s.b[e], h[e]);
  return r;
}
// s with a position behind it that resets nothing; its factor may underflow to 0 on the way, `kept` makes that good at the end
template <int V> DEVI Step<V> with(const Step<V> &s, const Step<V> &pos) {
  Step<V> r;
#pragma unroll
  for (int e = 0; e < V; ++e) r.a[e] = s.a[e] * pos.a[e];
  r.b = apply<false>(pos, s.b);
  return r;
}
template <int V> DEVI Step<V> kept(Step<V> s) {
#pragma unroll
  for (int e = 0; e < V; ++e) s.a[e] = not_zero(s.a[e]);
  return s;
}
template <bool RESETS, int V> DEVI Step<V> then(const Step<V> &s, const Step<V> &next) {
  Step<V> r;
#pragma unroll
  for (int e = 0; e < V; ++e) r.a[e] = factor1<RESETS>(s.a[e], next.a[e]);
  r.b = apply<RESETS>(next, s.b);
  return r;
}

// The steps of a workgroup's waves in LDS.
template <int V, int NW> struct WaveSteps {
  typedef float fvec __attribute__((ext_vector_type(V)));
  fvec a[NW][64], b[NW][64];
  DEVI void put(int wave, int lane, const Step<V> &s) {
    fvec x, y;
#pragma unroll
    for (int e = 0; e < V; ++e) x[e] = s.a[e], y[e] = s.b[e];
    a[wave][lane] = x, b[wave][lane] = y;
  }
  DEVI Step<V> get(int wave, int lane) const {
    const fvec x = a[wave][lane], y = b[wave][lane];
    Step<V> s;
#pragma unroll
    for (int e = 0; e < V; ++e) s.a[e] = x[e], s.b[e] = y[e];
    return s;
  }
};

// How the tiles of one row and channel group hand the state on, always in the same order of additions.  `group` tiles
// form a group: a tile reads the steps of the tiles before it in its group and the state at the end of the group before,
// which that group's last tile leaves.  A word carries a step's factor and term, (bits of a, bits of b), and is written
// in one piece: a is not negative, so its sign bit says that the word is there.  A state's word is its bits turned by those of
// a NaN that no state has (`kNever`), so it is not 0.  (Words are 0 before the launch.)
// Every workgroup writes its step before it waits for others, and the workgroups of a chain take their tiles in the
// order in which they begin (`ticket`): whatever a tile waits for has been begun and is written without waiting, or, for
// a group's state, waits only for what lies still further ahead.  So every wait ends, in whatever order workgroups
// are started.
struct Chain {
  uint32_t *tickets;  // one per chain (row and channel group)
  uint64_t *steps;    // (chain, ntiles, 64 V), none where a group is one tile
  uint32_t *states;   // (chain, ngroups, 64 V)
  int ntiles, group, ngroups;
};
constexpr uint64_t kThere = 1ull << 63;

DEVI uint64_t word_of(float a, float b) {
  return kThere | (uint64_t)__builtin_bit_cast(uint32_t, a) << 32 | __builtin_bit_cast(uint32_t, b);
}
DEVI float word_a(uint64_t w) { return __builtin_bit_cast(float, (uint32_t)(w >> 32) & 0x7fffffffu); }
DEVI float word_b(uint64_t w) { return __builtin_bit_cast(float, (uint32_t)w); }
template <int V> DEVI void put_words(uint64_t *p, const Step<V> &s) {
#pragma unroll
  for (int e = 0; e < V; ++e) __hip_atomic_store(p + e, word_of(s.a[e], s.b[e]), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

constexpr uint32_t kNever = 0x7fc00001u;
DEVI uint32_t state_word(float h) { return (h == h ? __builtin_bit_cast(uint32_t, h) : 0x7fc00000u) ^ kNever; }
DEVI void put_state(uint32_t *p, const Vec<2> &h) {  // both in one piece
  __hip_atomic_store(reinterpret_cast<uint64_t *>(p), (uint64_t)state_word(h[1]) << 32 | state_word(h[0]), __ATOMIC_RELAXED,
                     __HIP_MEMORY_SCOPE_AGENT);
}
// Whole wave: the states of every lane, once they are there (asked for as `wait_words` does).
DEVI Vec<2> wait_state(const uint32_t *p) {
  const int lane = threadIdx.x & 63;
  const uint32_t *hint = p - lane * 2;
  while (__hip_atomic_load(hint, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == 0) __builtin_amdgcn_s_sleep(4);
  for (;;) {
    const uint64_t w = __hip_atomic_load(reinterpret_cast<const uint64_t *>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (__all(w != 0)) return Vec<2>{{__builtin_bit_cast(float, (uint32_t)w ^ kNever), __builtin_bit_cast(float, (uint32_t)(w >> 32) ^ kNever)}};
    __builtin_amdgcn_s_sleep(1);
  }
}

// Whole wave: the words of every lane for the tiles from p on, 64 V words apart, once those of the first `count` are there
// (at least one; the others repeat the last).
template <int V, int N> DEVI void wait_words(const uint64_t *p, int count, uint64_t (&w)[N][V]) {
  // Until they are there the first words of the tiles alone are asked for, a tile by each lane: whole words asked for again and
  // again by every waiting wave take the memory's paths from the tiles that still load (34 -> 45 us at 2 x 2048 x 1536).
  const int lane = threadIdx.x & 63;
  const uint64_t *hint = p - lane * V + (int64_t)min(lane, count - 1) * 64 * V;
  while (!__all((__hip_atomic_load(hint, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) & kThere) != 0)) __builtin_amdgcn_s_sleep(4);
  for (;;) {
    uint64_t all = kThere;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int e = 0; e < V; ++e)
        w[i][e] = __hip_atomic_load(p + min(i, count - 1) * 64 * V + e, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int e = 0; e < V; ++e) all &= w[i][e];
    if (__all(all != 0)) return;
    __builtin_amdgcn_s_sleep(1);
  }
}

// What lies before tile n in its chain, read by all waves of the workgroup at once: wave w composes the w-th part of the
// steps before it in its group, wave 0 reads the state at the end of the group before (`first` enters tile 0).  After the
// next barrier `enter` has the state that enters tile n.
template <int V, int NW> struct Ahead {
  WaveSteps<V, NW> steps;
  Vec<V> state[64];
  template <bool RESETS> DEVI void read(const Chain &q, int64_t chain, int n, int wave, int lane, Vec<V> first) {
    constexpr int N = 4;
    const int g = n / q.group, from = g * q.group, count = n - from, part = (count + NW - 1) / NW;
    const int lo = min(wave * part, count), hi = min(lo + part, count);
    const uint64_t *sp = q.steps + (chain * q.ntiles + from) * (64 * V) + lane * V;
    Step<V> s = no_step<V>();
    for (int i = lo; i < hi; i += N) {
      uint64_t w[N][V];
      wait_words<V, N>(sp + (int64_t)i * 64 * V, min(N, hi - i), w);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        if (i + j < hi) {
          Step<V> next;
#pragma unroll
          for (int e = 0; e < V; ++e) next.a[e] = word_a(w[j][e]), next.b[e] = word_b(w[j][e]);
          s = then<RESETS>(s, next);
        }
      }
    }
    steps.put(wave, lane, s);
    if (wave == 0) {
      if (g > 0) first = wait_state(q.states + (chain * q.ngroups + g - 1) * (64 * V) + lane * V);
      state[lane] = first;
    }
  }
  template <bool RESETS> DEVI Vec<V> enter(const Chain &q, int lane) const {
    Vec<V> h = state[lane];
    if (q.group > 1) {
#pragma unroll
      for (int w = 0; w < NW; ++w) h = apply<RESETS>(steps.get(w, lane), h);
    }
    return h;
  }
};
// What tile n leaves for the ones behind it: its step at once, the state at its end where it closes a group.
template <int V> DEVI void leave_step(const Chain &q, int64_t chain, int n, int lane, const Step<V> &s) {
  if (n + 1 < q.ntiles && (n + 1) % q.group != 0) put_words<V>(q.steps + (chain * q.ntiles + n) * (64 * V) + lane * V, s);
}
template <int V> DEVI void leave_state(const Chain &q, int64_t chain, int n, int lane, const Vec<V> &h) {
  if (n + 1 < q.ntiles && (n + 1) % q.group == 0)
    put_state(q.states + (chain * q.ngroups + n / q.group) * (64 * V) + lane * V, h);
}

// The tile of this workgroup within its chain: the number of workgroups of the chain that began before it.  (lds: one int.)
DEVI int take_tile(const Chain &q, int64_t chain, int *lds) {
  if (q.ntiles == 1) return 0;
  if (threadIdx.x == 0) *lds = (int)__hip_atomic_fetch_add(q.tickets + chain, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  lds_barrier();
  return __builtin_amdgcn_readfirstlane(*lds);
}

// Which of the R positions from t0 on start a sequence, end one, lie in one, and which one it is.  The bounds are only
// compared; taken into [0, L] they describe sequences of the row whatever they hold.
// (Read through the scalar cache: a vector load here would wait for the rows requested before it.)
DEVI int bound_at(const int32_t *cu, int s, int L) {
  const int v = ((const __attribute__((address_space(4))) int32_t *)cu)[__builtin_amdgcn_readfirstlane(s)];
  return min(max(v, 0), L);
}
template <int R> struct SeqRows {
  uint32_t start, last, in;
  int seq[R];
  DEVI bool edges() const { return (start | last) != 0 || in != (1u << R) - 1; }
  DEVI void find(const int32_t *cu, int nseq, int t0, int L) {
    start = last = in = 0;
    int lo = -1, hi = nseq + 1;  // the last bound at or before t0
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (bound_at(cu, mid, L) <= t0) lo = mid;
      else hi = mid;
    }
    int s = lo;
    int begin = s >= 0 && s < nseq ? bound_at(cu, s, L) : -1, next = s < nseq ? bound_at(cu, s + 1, L) : INT32_MAX;
#pragma unroll
    for (int j = 0; j < R; ++j) {
      const int t = t0 + j;
      while (s < nseq && t >= next) {
        ++s;
        begin = next;
        next = s < nseq ? bound_at(cu, s + 1, L) : INT32_MAX;
      }
      seq[j] = s;
      if (s >= 0 && s < nseq && t < L) {
        in |= 1u << j;
        if (t == begin) start |= 1u << j;
        if (t + 1 == next) last |= 1u << j;
      }
    }
  }
};
// Whole workgroup: f(s) for every sequence without a position, a wave at a time.
template <typename F> DEVI void empty_sequences(const int32_t *cu, int nseq, int L, F f) {
  const int lane = threadIdx.x & 63, waves = blockDim.x >> 6;
  for (int s0 = (threadIdx.x >> 6) * 64; s0 < nseq; s0 += waves * 64) {
    const int s = min(s0 + lane, nseq - 1);
    const bool empty = s0 + lane < nseq && min(max(cu[s + 1], 0), L) <= min(max(cu[s], 0), L);
    uint64_t found = __ballot(empty);
    while (found) {
      f(s0 + (int)__builtin_ctzll(found));
      found &= found - 1;
    }
  }
}

}  // namespace
