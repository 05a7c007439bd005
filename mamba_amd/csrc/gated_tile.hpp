// Tiles of the gated linear recurrence: what the forward and the backward kernel of gated_scan.hip share.
//
// A row of positions is a linear recurrence per channel, h = a h + b, and a run of positions is one such step (A, B)
// again.  The row is cut into tiles of positions and groups of 128 channels.  A workgroup holds one tile of one group
// in registers: a wave has ROWS positions after one another, its lanes two channels each (rows of 256 or 512 bytes).
// The steps of the waves meet in LDS; the state that enters the tile comes from the workgroups of the tiles before it
// (`Chain`), so every tensor is read once and written once.
#pragma once
#include "gated_gates.hpp"

namespace {

constexpr int kTileChannels = 128;

// Two neighbouring channels of one position.
template <typename T> struct Pair {
  uint32_t w;
  DEVI float lo() const { return DT<T>::id == MAMBA_BF16 ? bf16_lo(w) : f16_lo(w); }
  DEVI float hi() const { return DT<T>::id == MAMBA_BF16 ? bf16_hi(w) : f16_hi(w); }
};
template <> struct Pair<float> {
  u32x2 w;
  DEVI float lo() const { return __builtin_bit_cast(f32x2, w).x; }
  DEVI float hi() const { return __builtin_bit_cast(f32x2, w).y; }
};

// How a lane reads and writes its pair of channels c, c + 1.  EVEN: the number of channels is even, a pair is whole or
// not there.  Otherwise the last channel may stand alone: the lane reads the pair before it and takes its second half.
// Rows lie at any alignment (gfx950 serves these accesses at element alignment).  Lanes past the last channel read
// the last pair again and write nothing.
template <typename T, bool EVEN> struct Lane {
  int at;         // the channel that the lane's pair is read from
  bool two, one;  // whether both channels, or the first alone, are there
  bool half;      // the pair holds the first channel in its second half
  bool single;    // a row of one channel
  DEVI Lane(int c, int dim) {
    two = c + 1 < dim;
    one = !EVEN && c + 1 == dim;
    at = max(min(c, dim - 2), 0);
    half = !EVEN && c > dim - 2;
    single = !EVEN && dim == 1;
  }
  DEVI Pair<T> load(const T *row) const {
    Pair<T> r;
    if constexpr (DT<T>::id == MAMBA_F32) {
      typedef u32x2 a4 __attribute__((aligned(4)));
      if (!EVEN && single) {
        r.w = u32x2{*(const GLOBAL_AS uint32_t *)row, 0u};
        return r;
      }
      r.w = *(const GLOBAL_AS a4 *)(row + at);
      if (!EVEN) r.w.x = half ? r.w.y : r.w.x;
    } else {
      typedef uint32_t a2 __attribute__((aligned(2)));
      if (!EVEN && single) {
        r.w = *(const GLOBAL_AS uint16_t *)row;
        return r;
      }
      r.w = *(const GLOBAL_AS a2 *)(row + at);
      if (!EVEN) r.w = half ? r.w >> 16 : r.w;
    }
    return r;
  }
  DEVI void store(T *row, int c, float lo, float hi) const {
    if (two) {
      if constexpr (DT<T>::id == MAMBA_F32) {
        typedef f32x2 a4 __attribute__((aligned(4)));
        *(GLOBAL_AS a4 *)(row + c) = f32x2{lo, hi};
      } else {
        typedef uint32_t a2 __attribute__((aligned(2)));
        *(GLOBAL_AS a2 *)(row + c) = DT<T>::id == MAMBA_BF16 ? pack_bf16(lo, hi) : pack_f16(lo, hi);
      }
    } else if (!EVEN && one) {
      st1<T>(row + c, lo);
    }
  }
  DEVI f32x2 load_state(const float *row, int c) const {
    return f32x2{two || one ? row[c] : 0.f, two ? row[c + 1] : 0.f};
  }
  DEVI void store_state(float *row, int c, f32x2 v) const {
    if (two || one) row[c] = v.x;
    if (two) row[c + 1] = v.y;
  }
};

// The step of a run of positions for two channels: h -> a h + b.
struct Step {
  f32x2 a, b;
};
DEVI Step no_step() { return Step{f32x2{1.f, 1.f}, f32x2{0.f, 0.f}}; }
// RESETS: a factor of exactly 0 marks a run in which a sequence starts; nothing before it counts, whatever it is.  The
// decays of positions are kept from underflowing to that (a state times kTiny is gone all the same, but an infinity or a
// NaN in the sequence stays one).
constexpr float kTiny = 1.17549435e-38f;
template <bool RESETS> DEVI float apply1(float a, float b, float h) {
  const float r = __builtin_fmaf(a, h, b);
  return RESETS && a == 0.f ? b : r;
}
template <bool RESETS> DEVI float factor1(float a, float next) {
  const float r = a * next;
  if (!RESETS) return r;
  return a == 0.f || next == 0.f ? 0.f : fmaxf(r, kTiny);
}
template <bool RESETS> DEVI f32x2 apply(const Step &s, f32x2 h) {
  return f32x2{apply1<RESETS>(s.a.x, s.b.x, h.x), apply1<RESETS>(s.a.y, s.b.y, h.y)};
}
template <bool RESETS> DEVI f32x2 factor(f32x2 a, f32x2 next) {
  return f32x2{factor1<RESETS>(a.x, next.x), factor1<RESETS>(a.y, next.y)};
}
template <bool RESETS> DEVI Step then(const Step &s, const Step &next) {
  return Step{factor<RESETS>(s.a, next.a), apply<RESETS>(next, s.b)};
}

// How the tiles of one row and channel group hand the state on, always in the same order of additions.  `group` tiles
// form a group: a tile reads the steps of the tiles before it in its group and the state at the end of the group before,
// which that group's last tile leaves.  A word carries a step's factor and term, (bits of a, bits of b), and is written
// in one piece: a is not negative, so its sign bit says that the word is there.  (Words are 0 before the launch.)
// Every workgroup writes its step before it waits for others, and the workgroups of a chain take their tiles in the
// order in which they begin (`ticket`): whatever a tile waits for has been begun and is written without waiting, or, for
// a group's state, waits only for what lies still further ahead.  So every wait ends, in whatever order workgroups
// are started.
struct Chain {
  uint32_t *tickets;  // one per chain (row and channel group)
  uint64_t *steps;    // (chain, ntiles, 128)
  uint64_t *states;   // (chain, ngroups, 128)
  int ntiles, group, ngroups;
};
constexpr uint64_t kThere = 1ull << 63;

DEVI uint64_t word_of(float a, float b) {
  return kThere | (uint64_t)__builtin_bit_cast(uint32_t, a) << 32 | __builtin_bit_cast(uint32_t, b);
}
DEVI float word_a(uint64_t w) { return __builtin_bit_cast(float, (uint32_t)(w >> 32) & 0x7fffffffu); }
DEVI float word_b(uint64_t w) { return __builtin_bit_cast(float, (uint32_t)w); }
DEVI void put_words(uint64_t *p, f32x2 a, f32x2 b) {
  __hip_atomic_store(p, word_of(a.x, b.x), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __hip_atomic_store(p + 1, word_of(a.y, b.y), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
DEVI uint64_t get_word(const uint64_t *p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

// Whole wave: the two words of every lane for N tiles, `stride` words apart, once all of them are there.
template <int N> DEVI void wait_words(const uint64_t *p, int64_t stride, uint64_t (&w)[N][2]) {
  for (;;) {
    bool there = true;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      w[i][0] = get_word(p + i * stride);
      w[i][1] = get_word(p + i * stride + 1);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) there = there && (w[i][0] & w[i][1] & kThere) != 0;
    if (__all(there)) return;
    __builtin_amdgcn_s_sleep(1);
  }
}

// Whole wave: the state that enters tile n of the chain; `first` is the one that enters tile 0.  c: the lane's place in the
// channel group (0, 2, .. 126).
template <bool RESETS> DEVI f32x2 entering(const Chain &q, int64_t chain, int n, int c, f32x2 first) {
  const int g = n / q.group, from = g * q.group;
  const uint64_t *sp = q.steps + (chain * q.ntiles + from) * kTileChannels + c;
  Step s = no_step();
  int i = 0;
  constexpr int B = 4;
  auto take = [&](const uint64_t (&w)[2]) {
    s = then<RESETS>(s, Step{f32x2{word_a(w[0]), word_a(w[1])}, f32x2{word_b(w[0]), word_b(w[1])}});
  };
  for (; i + B <= n - from; i += B) {
    uint64_t w[B][2];
    wait_words<B>(sp + i * kTileChannels, kTileChannels, w);
#pragma unroll
    for (int j = 0; j < B; ++j) take(w[j]);
  }
  for (; i < n - from; ++i) {
    uint64_t w[1][2];
    wait_words<1>(sp + i * kTileChannels, kTileChannels, w);
    take(w[0]);
  }
  if (g > 0) {
    uint64_t w[1][2];
    wait_words<1>(q.states + (chain * q.ngroups + g - 1) * kTileChannels + c, 0, w);
    first = f32x2{word_b(w[0][0]), word_b(w[0][1])};
  }
  return apply<RESETS>(s, first);
}
// What tile n leaves for the ones behind it: its step at once, the state at its end where it closes a group.
DEVI void leave_step(const Chain &q, int64_t chain, int n, int c, const Step &s) {
  if (n + 1 < q.ntiles && (n + 1) % q.group != 0) put_words(q.steps + (chain * q.ntiles + n) * kTileChannels + c, s.a, s.b);
}
DEVI void leave_state(const Chain &q, int64_t chain, int n, int c, f32x2 h) {
  if (n + 1 < q.ntiles && (n + 1) % q.group == 0)
    put_words(q.states + (chain * q.ngroups + n / q.group) * kTileChannels + c, f32x2{0.f, 0.f}, h);
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
  uint32_t start = 0, last = 0, in = 0;
  int seq[R];
  DEVI SeqRows(const int32_t *cu, int nseq, int t0, int L) {
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
