// Linear attention with a decay per head (linear_attn.hpp has the formulas), gfx950.
#include "linear_attn.hpp"

#include <algorithm>
#include <initializer_list>

namespace {
using namespace lin;

// EXACT: a state is a result, in fp32, and the weighted rows that are added to it are split into three bf16 parts, 2^-25 of a value.  Else
// two, 2^-17, are more than results of 16 bits show (8 x 4096 x 20 x 128 in bf16, forward and backward: 671 us of kernels with two,
// 764 with three; 726 with both in one kernel).
template <typename F, bool EXACT> using Parts = std::conditional_t<EXACT, typename F::Wider, typename F::Wide>;

// The state of one segment alone, from zero, for the segments behind it: 81-93 us for 0.23 GB at 8 x 4096 x 20 x 128, a block's latency with
// 320 workgroups at work (of 480: the last segments' states are not asked for).
template <typename T, int KD, int DVT, Fit FIT, bool EXACT> __global__ __launch_bounds__(kThreads, (Shape<T, KD, DVT>::WORKGROUPS)) void lin_segment_kernel(const LinLaunch p) {
  using F = Frags<T>;
  using Sh = Shape<T, KD, DVT>;
  using W = Parts<F, EXACT>;
  constexpr int C = Sh::C, TURN = 2 * C, CC = F::size(TURN, KD);  // two blocks a barrier: more rows on their way
  __shared__ __align__(16) char lds[2][CC + F::size(TURN, Sh::VAL)];
  const Place at = place_of(p);
  if (at.none) return;
  const LinWalk &w = p.w[at.walk];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), i = lane & 15, g = lane >> 4;
  const int v0 = at.slice * Sh::VAL;
  const Item it = item_of(p, at.item);
  if (v0 >= w.val || it.zero || (it.before + 1) * p.seg_len >= it.len) return;  // the last segment's is not asked for
  const typename F::template Lane<KD> lanes(i, g, wave % F::NT);
  const typename F::template ColumnLane<Sh::VAL> values(wave * DVT, i, g);
  const Decay decay{log2_decay(p.log_decay[at.head])};
  int64_t b_ls, c_ls;
  const T *b = static_cast<const T *>(w.b.p) + rows_at(w.b, it, at.head, w.reverse, p.seg_len, b_ls);
  const T *c = static_cast<const T *>(w.c.p) + rows_at(w.c, it, at.head, w.reverse, p.seg_len, c_ls) + v0;
  Stage<T, TURN, KD, FIT> sb(b, b_ls, w.key, tid);
  Stage<T, TURN, Sh::VAL, FIT> sc(c, c_ls, min(w.val - v0, Sh::VAL), tid);
  WaveState<T, KD, DVT> state;
  state.zero();
  const float write = w.write;
  const int late = w.late;
  const Weights<F, Sh::JB, Sh::IT> weights(decay, 0.f, write, late, i, g);
  auto fetch = [&](int t) {
    const int n = min(it.n - t, TURN);
    sb.fetch(b + t * b_ls, b_ls, n, tid), sc.fetch(c + t * c_ls, c_ls, n, tid);
  };
  auto commit = [&](auto whole, int t, char *rows) {
    const int n = min(it.n - t, TURN);
    sb.template commit<whole.value>(rows, n, tid), sc.template commit<whole.value>(rows + CC, n, tid);
  };
  // whole: so are these two blocks and the next four
  auto turn = [&](auto whole, int t, char *now, char *next) {
    constexpr bool FULL = whole.value;
    if (FULL || t + TURN < it.n) commit(whole, t + TURN, next);
    if constexpr (FULL) sb.fetch_next(), sc.fetch_next();
    else if (t + 2 * TURN < it.n) fetch(t + 2 * TURN);
#pragma unroll
    for (int k = 0; k < 2; ++k)
      if (FULL || t + k * C < it.n)
        state.template update<FULL, W>(now + F::size(k * C, KD), now + CC + F::size(k * C, Sh::VAL), lanes, values, decay, weights, write,
                                    FULL ? C : min(it.n - t - k * C, C), late, g);
    lds_barrier();
  };
  char *now = lds[0], *next = lds[1];
  const bool steady = FIT != ELEMENTS && it.n >= 3 * TURN && near(w.b) && near(w.c);
  int t = 0;
  if (steady) {
    sb.fetch_next(), sc.fetch_next();
    commit(std::true_type{}, 0, now);
    sb.fetch_next(), sc.fetch_next();
    lds_barrier();
    for (; t + 3 * TURN <= it.n; t += TURN) {
      turn(std::true_type{}, t, now, next);
      char *const was = now;
      now = next, next = was;
    }
  } else {
    fetch(0);
    commit(std::false_type{}, 0, now);
    if (TURN < it.n) fetch(TURN);
    lds_barrier();
  }
#pragma unroll 1
  for (; t < it.n; t += TURN) {
    turn(std::false_type{}, t, now, next);
    char *const was = now;
    now = next, next = was;
  }
  f32x4 *dst = p.segs + ((((int64_t)at.walk * p.items + at.item) * p.nheads + at.head) * p.slices + at.slice) * (kWaves * Sh::TILES * 64) +
               wave * Sh::TILES * 64 + lane;
  state.each([&](f32x4 &v, int tile) { dst[tile * 64] = v; });
}

// The walk.  Blocks of 32 positions: their products with one another are 6 of a wave's 56 matrix instructions, the state's own work
// (scaling it, rounding it to operands) is shared by 32 rows.  Two tiles of values a wave use each operand read from LDS twice.  What
// bounds it at 8 x 4096 x 20 x 128 in bf16 is memory, then the latency of a block's chain of reads and products: backward 430-475 us
// for 1.28 GB read and 0.50 written, 364 with every row in L2, 336 without the products; LDS is busy 57 % of it, vector
// instructions 36 %, matrix instructions 23 %.  Forward 155-170 (three segments) after 81-93 for the segments' states.
// What is rounded for the products: the state and the scores as operands of y to what the results' type shows (F::Comp), as the
// sums of their products are rounded to that type anyhow; a second part of the state would be 16 more matrix instructions than 56.
// A score's rounding is all of its row's values': in a sequence of a few positions nothing evens it out, and 1.5 times the error of one
// rounding of the results was seen.  So the blocks at a sequence's end (all of a short one) take the scores in two parts.  (In every
// block: 450-457 / 166 us in place of 428 / 159; with the parts side by side, 102 in place of 97 for the packed forward pass.)
// PARTS: there are walks whose y is a part of a sum, in fp32.  (The loop for those beside the other one costs registers that the
// launches without them need: 8 spilled a block.)
template <typename T, int KD, int DVT, Fit FIT, bool PARTS, bool EXACT> __global__ __launch_bounds__(kThreads, (Shape<T, KD, DVT>::WORKGROUPS)) void lin_walk_kernel(const LinLaunch p) {
  using F = Frags<T>;
  using Sh = Shape<T, KD, DVT>;
  using W = Parts<F, EXACT>;
  using Raw = typename F::Raw;
  constexpr int C = Sh::C, KB = Sh::KB, JB = Sh::JB, IT = Sh::IT, NT = F::NT, KS = F::KS, V = F::V;
  __shared__ __align__(16) char lds[Sh::LDS];
  const Place at = place_of(p);
  if (at.none) return;
  const LinWalk &w = p.w[at.walk];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), i = lane & 15, g = lane >> 4;
  const int v0 = at.slice * Sh::VAL;
  const Item it = item_of(p, at.item);
  if (v0 >= w.val || it.seq < 0) return;
  const int vals = min(w.val - v0, Sh::VAL);

  // y leaves through LDS, as pieces of whole rows; sums that are still to be added to others leave in fp32 from the registers.
  // (Stores of a wave's own columns, 32 or 64 bytes a row, save a barrier and cost more: the loop without its products takes 432 us
  // and not 336 for the backward of 8 x 4096 x 20 x 128.)
  int64_t y_ls;
  const int64_t y_at = rows_at(w.y, it, at.head, w.reverse, p.seg_len, y_ls) + v0;
  constexpr int Y_PER = Sh::VAL / V, Y_RUN = kThreads / Y_PER, Y_N = C / Y_RUN;  // pieces of a row, rows of a turn, turns
  static_assert(C % Y_RUN == 0, "whole turns");
  const int y_row = tid / Y_PER, y_piece = tid % Y_PER;
  const bool y_f32 = PARTS && w.y_f32;
  auto put = [&](T *dst, Raw v) {
    if constexpr (FIT == ELEMENTS) {
      typename F::E e[V];
      __builtin_memcpy(e, &v, 16);
#pragma unroll
      for (int k = 0; k < V; ++k)
        if (y_piece * V + k < vals) *reinterpret_cast<typename F::E *>(dst + k) = e[k];
    } else if (FIT == WHOLE || y_piece * V < vals) {
      if constexpr (std::is_same_v<T, float>) *(GLOBAL_AS f32x4_a4 *)dst = v;
      else *(GLOBAL_AS u32x4_a2 *)dst = v;
    }
  };
  auto put_f32 = [&](int64_t row, f32x4 v, int d) {
    const int value = 16 * (DVT * wave + d) + 4 * g;
    float *dst = static_cast<float *>(w.y.p) + y_at + row * y_ls + value;
    if constexpr (FIT == ELEMENTS) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (value + e < vals) dst[e] = v[e];
    } else if (FIT == WHOLE || value < vals) {
      *(GLOBAL_AS f32x4_a4 *)dst = v;
    }
  };
  if (it.zero) {
    if (y_f32) {
      for (int row = i; row < it.n; row += 16)
#pragma unroll
        for (int d = 0; d < DVT; ++d) put_f32(row, f32x4{0.f, 0.f, 0.f, 0.f}, d);
    } else {
      const Raw none = {};
      for (int row = y_row; row < it.n; row += Y_RUN) put(static_cast<T *>(w.y.p) + y_at + row * y_ls + y_piece * V, none);
    }
    return;
  }

  const typename F::template Lane<KD> lanes(i, g, wave % F::NT);
  const typename F::template ColumnLane<Sh::VAL> values(wave * DVT, i, g);
  const Decay decay{log2_decay(p.log_decay[at.head])};
  int64_t a_ls, b_ls, c_ls;
  const T *a = static_cast<const T *>(w.a.p) + rows_at(w.a, it, at.head, w.reverse, p.seg_len, a_ls);
  const T *b = static_cast<const T *>(w.b.p) + rows_at(w.b, it, at.head, w.reverse, p.seg_len, b_ls);
  const T *c = static_cast<const T *>(w.c.p) + rows_at(w.c, it, at.head, w.reverse, p.seg_len, c_ls) + v0;
  Stage<T, C, KD, FIT> sa(a, a_ls, w.key, tid), sb(b, b_ls, w.key, tid);
  Stage<T, C, Sh::VAL, FIT> sc(c, c_ls, vals, tid);
  auto fetch = [&](int t) {
    const int n = min(it.n - t, C);
    sa.fetch(a + t * a_ls, a_ls, n, tid), sb.fetch(b + t * b_ls, b_ls, n, tid), sc.fetch(c + t * c_ls, c_ls, n, tid);
  };
  auto fetch_next = [&]() { sa.fetch_next(), sb.fetch_next(), sc.fetch_next(); };
  auto commit = [&](auto whole, int t, char *rows) {
    const int n = min(it.n - t, C);
    sa.template commit<whole.value>(rows, n, tid), sb.template commit<whole.value>(rows + Sh::B, n, tid);
    sc.template commit<whole.value>(rows + Sh::CC, n, tid);
  };
  const bool steady = FIT != ELEMENTS && it.n >= 3 * C && near(w.a) && near(w.b) && near(w.c) && near(w.y);
  if (steady) fetch_next();
  else if (it.n > 0) fetch(0);

  // the state that comes in
  WaveState<T, KD, DVT> state;
  const int64_t seq_head = ((int64_t)it.seq * p.nheads + at.head) * w.key * w.val;
  const int value = v0 + 16 * DVT * wave + i;
  if (w.start.p) {
    const float *src[DVT];
#pragma unroll
    for (int d = 0; d < DVT; ++d) src[d] = w.start.p + seq_head + min(value + 16 * d, w.val - 1) * w.start.vs;
    state.each_element(g, w.key, [&](float, int d, int k, bool) { return src[d][min(k, w.key - 1) * w.start.ks]; });
    state.each([](f32x4 &v, int) { asm volatile("" : "+v"(v)); });  // all of them on their way before any is looked at
    state.each_element(g, w.key, [&](float x, int d, int, bool ok) { return ok && value + 16 * d < w.val ? x : 0.f; });
  } else {
    state.zero();
  }
  if (it.before > 0) {
    const float f = decay(p.seg_len);
    const int64_t step = (int64_t)p.nheads * p.slices * (kWaves * Sh::TILES * 64);
    const f32x4 *src = p.segs + (((int64_t)at.walk * p.items + at.item - it.before) * p.nheads * p.slices + at.head * p.slices + at.slice) *
                                    (kWaves * Sh::TILES * 64) + wave * Sh::TILES * 64 + lane;
    for (int s = 0; s < it.before; ++s, src += step) state.each([&](f32x4 &v, int tile) { v = v * f + src[tile * 64]; });
  }

  const float read = w.read, write = w.write;
  const int late = w.late;
  const Weights<F, JB, IT> weights(decay, read, write, late, i, g);
  // (a_t . b_s) f^(t - s) mix: a wave has a tile of 16 t and half of KS s, of those blocks that reach the diagonal
  const int tile = wave / NT, half = wave % NT;
  int ib_of = 0, jb_of = tile;
  for (int per = 1; jb_of >= per; ++ib_of, per = (16 * ib_of + 15) / KS + 1) jb_of -= per;
  const int first = 16 * ib_of + i - (KS * jb_of + F::krow(4 * g, half));  // t - s of the lane's first s
  float pair[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) pair[r] = w.mix * decay(max(first - r, 0));
  auto scores = [&](const char *rows, char *to) {
    if (tile >= Sh::BLOCKS) return;
    const char *ar = rows + F::size(16 * ib_of, KD), *br = rows + Sh::B + F::size(KS * jb_of, KD);
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) acc = F::mma_raw(lanes.along_krow(br, kb), lanes.along(ar, kb), acc);
#pragma unroll
    for (int r = 0; r < 4; ++r) acc[r] = r <= first ? acc[r] * pair[r] : 0.f;
    F::template store_wide<Sh::BLOCKS * 64>(to, tile * 64 + lane, half, acc);
  };

  // whole blocks of near rows: the lowest row of a turn, from turn to turn, the thread's place (bytes)
  char *y_low = uniform_pointer(static_cast<char *>(w.y.p) + (y_at + (y_ls < 0 ? (Y_RUN - 1) * y_ls : 0)) * (int64_t)sizeof(T));
  const int64_t y_run = Y_RUN * y_ls * (int64_t)sizeof(T);
  const uint32_t y_place = (uint32_t)((y_ls < 0 ? Y_RUN - 1 - y_row : y_row) * (int)(y_ls < 0 ? -y_ls : y_ls) + y_piece * V) * (uint32_t)sizeof(T);
  // One block: rows in `now`, scores in `s_now`; the next one's rows are laid down, its scores formed, those of the one behind it asked
  // for.  whole: so are all three; then f32 has to be known as well: loads and stores are counted together, and where the number of
  // stores behind a block's loads depends on a branch, waiting for the loads waits for the stores too.
  auto block = [&](auto whole, auto f32, int t, char *now, char *next, const char *s_now, char *s_next) {
    constexpr bool FULL = whole.value;
    const int n = FULL ? C : min(it.n - t, C);
    if (FULL || t + C < it.n) commit(whole, t + C, next);
    if constexpr (FULL) fetch_next();
    else if (t + 2 * C < it.n) fetch(t + 2 * C);
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
        float v[V];
        F::gather(state.t[d][kb], v);
        s[d] = F::comp(v);
      }
#pragma unroll
      for (int ib = 0; ib < IT; ++ib) {
        const typename F::Data ad = F::data(lanes.along(now + F::size(16 * ib, KD), kb));
#pragma unroll
        for (int d = 0; d < DVT; ++d) y[ib][d] = mma16(s[d], ad, y[ib][d]);
      }
    }
#pragma unroll
    for (int ib = 0; ib < IT; ++ib) {
      const float in = FULL ? weights.in_lane * weights.in_block[ib] : read * decay(16 * ib + i + late);
#pragma unroll
      for (int d = 0; d < DVT; ++d) y[ib][d] *= in;
    }
#pragma unroll
    for (int jb = 0; jb < JB; ++jb) {
      typename F::Data cd[DVT];
#pragma unroll
      for (int d = 0; d < DVT; ++d) cd[d] = F::data(values.columns(now + Sh::CC + F::size(KS * jb, Sh::VAL), d));
#pragma unroll
      for (int ib = 0; ib < IT; ++ib) {
        if (jb * KS > ib * 16 + 15) continue;
        auto with = [&](const auto &s) {
#pragma unroll
          for (int d = 0; d < DVT; ++d) y[ib][d] = mma16(cd[d], s, y[ib][d]);
        };
        if constexpr (FULL) with(F::template load_comp<Sh::BLOCKS * 64>(s_now, Sh::block_of(ib, jb) * 64 + lane));
        else with(F::template load_wide<Sh::BLOCKS * 64>(s_now, Sh::block_of(ib, jb) * 64 + lane));
      }
    }
#pragma unroll
    for (int ib = 0; ib < IT; ++ib)
#pragma unroll
      for (int d = 0; d < DVT; ++d) {
        if (!f32) F::template store<Sh::VAL>(lds + Sh::AT_Y, 16 * ib + i, DVT * wave + d, g, y[ib][d]);
        else if (FULL || 16 * ib + i < n) put_f32(t + 16 * ib + i, y[ib][d], d);
      }
    lds_barrier();
    if (!f32) {
#pragma unroll
      for (int q = 0; q < Y_N; ++q) {
        const int row = q * Y_RUN + y_row;
        const Raw v = *reinterpret_cast<const Raw *>(lds + Sh::AT_Y + (int)sizeof(typename F::E) * F::template place<Sh::VAL>(row, y_piece));
        if constexpr (FULL) {
          asm("" : "+s"(y_low));
          put(reinterpret_cast<T *>(y_low + y_place), v);
          y_low += y_run;
        } else if (row < n) {
          put(static_cast<T *>(w.y.p) + y_at + (t + row) * y_ls + y_piece * V, v);
        }
      }
    }
    state.template update<FULL, W>(now + Sh::B, now + Sh::CC, lanes, values, decay, weights, write, n, late, g);
    if (FULL || t + C < it.n) scores(next, s_next);
    lds_barrier();
  };
  char *now = lds, *next = lds + Sh::STAGE, *s_now = lds + Sh::AT_SCORES, *s_next = s_now + Sh::SCORES;
  auto turn_over = [&]() {
    char *const was = now, *const s_was = s_now;
    now = next, next = was, s_now = s_next, s_next = s_was;
  };
  int t = 0;
  if (it.n > 0) {
    if (steady) {
      commit(std::true_type{}, 0, now);
      fetch_next();
    } else {
      commit(std::false_type{}, 0, now);
      if (C < it.n) fetch(C);
    }
    lds_barrier();
    scores(now, s_now);
    lds_barrier();
  }
  auto steady_blocks = [&](auto f32) {
    for (; t + 3 * C <= it.n; t += C) block(std::true_type{}, f32, t, now, next, s_now, s_next), turn_over();
  };
  if (steady) {
    if constexpr (PARTS)
      if (y_f32) steady_blocks(std::true_type{});
    steady_blocks(std::false_type{});  // (none are left behind the others)
  }
#pragma unroll 1
  for (; t < it.n; t += C) block(std::false_type{}, y_f32, t, now, next, s_now, s_next), turn_over();
  if (w.end.p && (it.before + 1) * (int64_t)p.seg_len >= it.len) {
    float *dst = w.end.p + seq_head + value * w.end.vs;
    state.each_element(g, w.key, [&](float x, int d, int k, bool ok) {
      if (ok && value + 16 * d < w.val) dst[16 * d * w.end.vs + k * w.end.ks] = x;
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

// Gradients of heads that share keys and values, added up in order: parts (rows, nheads, dim) in fp32, V columns a thread.  It reads
// group times 4 bytes for every value it writes: 124-129 us for dk and dv of 32768 x 32 heads of 64 onto
// 8, 4.7-4.9 TB/s (190 us column by column with divisions of 64 bits).
template <typename T> DEVI void store4(T *at, f32x4 v) {
  if constexpr (std::is_same_v<T, float>) {
    *(GLOBAL_AS f32x4_a4 *)at = v;
  } else {
    typedef u32x2 u32x2_a2 __attribute__((aligned(2)));
    *(GLOBAL_AS u32x2_a2 *)at = std::is_same_v<T, bf16_t> ? u32x2{pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3])} : u32x2{pack_f16(v[0], v[1]), pack_f16(v[2], v[3])};
  }
}
struct Shared {
  const float *parts;
  void *out;
  int64_t bs, ls, hs;
  int dim;
};
template <typename T, int V> __global__ __launch_bounds__(kThreads) void lin_shared_kernel(const Shared dk, const Shared dv, int64_t rows, int kv_heads, int group, int seqlen) {
  const Shared &p = blockIdx.y ? dv : dk;
  const int pieces = p.dim / V, per = kv_heads * pieces, some = max(4 * kThreads / per, 1);  // rows at a time
  for (int64_t row0 = (int64_t)blockIdx.x * some; row0 < rows; row0 += (int64_t)gridDim.x * some)
    for (int at = threadIdx.x; at < some * per; at += kThreads) {
      const int64_t row = row0 + at / per;
      const int in = at % per, h = in / pieces, x = in % pieces * V;
      if (row >= rows) break;
      const float *src = p.parts + (row * kv_heads + h) * group * p.dim + x;
      T *dst = static_cast<T *>(p.out) + row / seqlen * p.bs + row % seqlen * p.ls + h * p.hs + x;
      if constexpr (V == 4) {
        f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
        for (int m = 0; m < group; ++m) v += *reinterpret_cast<const f32x4 *>(src + m * p.dim);
        store4<T>(dst, v);
      } else {
        float v = 0.f;
        for (int m = 0; m < group; ++m) v += src[m * p.dim];
        st1<T>(dst, v);
      }
    }
}

// ------------------------------------------------------------------ host side
// How a pass is cut: the sizes that the kernels are made for, the values of a workgroup, and segments of a sequence where
// there are fewer (sequence, head, slice) walks than the chip has room for.
struct Cut {
  int kd, tiles, slices, nseg, seg_len, items;
  Fit fit;
  bool packed;
  int64_t state_bytes, plan_bytes;
};
Cut cut_of(const LinearAttnParams &p, int nwalks) {
  Cut c;
  const int most = p.headdim_k > p.headdim_v ? p.headdim_k : p.headdim_v, v = p.dtype == MAMBA_F32 ? 4 : 8;
  const int val = nwalks == 1 ? p.headdim_v : most, key = nwalks == 1 ? p.headdim_k : most;
  c.kd = key <= 64 ? 64 : key <= 128 ? 128 : 256;
  c.packed = p.nseq > 0;
  const int64_t seqs = c.packed ? p.nseq : p.batch, chains = (int64_t)p.nheads * nwalks, cus = cu_count();
  const int64_t total = (int64_t)p.batch * p.seqlen, longest = c.packed ? total : p.seqlen;
  // Segments of 128 positions at least: of 64, every segment's own state and the sum of those before it cost as much as the walk
  // (a row of 777 in bf16, 24 heads: 29 us with 128 and 30 with 64; 2048 in fp32: 38 and 48, 41 with 256).  Their number is rounded down and their
  // length up to blocks, so there can be fewer: 777 positions are five of 160.
  constexpr int64_t kLeast = 128;
  // Two tiles of 16 values a wave read a block's rows once for both (8 x 4096 x 20 x 128, backward: 454 us, 510 with one) as long as there are
  // workgroups for the chip with them (that row of 777: 38 us with two, 29 with one).
  const int64_t pieces = c.packed ? seqs + total / kLeast : seqs * std::max<int64_t>(p.seqlen / kLeast, 1);
  c.tiles = val > 64 && c.kd <= 128 && pieces * chains * ((val + 127) / 128) >= cus ? 2 : 1;
  const int values_of = 64 * c.tiles;
  c.slices = (val + values_of - 1) / values_of;
  const bool keys = p.headdim_k == c.kd && (nwalks == 1 || p.headdim_v == c.kd);
  const bool values = p.headdim_v % values_of == 0 && (nwalks == 1 || p.headdim_k % values_of == 0);
  c.fit = p.headdim_k % v != 0 || p.headdim_v % v != 0 ? ELEMENTS : keys && values ? WHOLE : PIECES;
  // Whole sequences where their walks fill the chip, as the segments' states are one more pass over half of what is read (8 x 4096 x
  // 20 x 128, backward: 454 us in one piece, 585 in two); else as many segments as fill it once (forward, 160 walks for 512 places: 250
  // us in three pieces, 264 in four, 257 in one).  Packed sequences may be of any length: segments of an even share.  (What fills the chip is
  // counted by the keys alone: two tiles of values of 64 keys have two workgroups a CU at a time, not four.)
  const int64_t walks = chains * c.slices, slots = cus * (c.kd == 256 ? 1 : c.kd == 128 ? 2 : 4);
  int64_t len = longest;
  if (seqs * walks < slots) {
    const int64_t most = std::max<int64_t>(p.seqlen / kLeast, 1), n = std::min(slots / (seqs * walks), most);
    len = c.packed ? std::max(total * walks / slots, kLeast) : (p.seqlen + n - 1) / n;
    len = (len + 31) / 32 * 32;
  }
  c.nseg = (int)std::max<int64_t>((longest + len - 1) / len, 1);
  c.seg_len = c.nseg == 1 ? INT32_MAX : (int)len;
  c.items = c.packed ? (int)(seqs + 2 + (c.nseg > 1 ? total / len : 0)) : (int)(seqs * c.nseg);
  c.plan_bytes = c.packed && c.nseg > 1 ? ((int64_t)c.items + 1) * 16 : 0;
  c.state_bytes = c.nseg > 1 ? (int64_t)nwalks * c.items * p.nheads * c.slices * c.kd * values_of * 4 : 0;
  return c;
}

template <typename T, int KD, int DVT, Fit FIT, bool PARTS, bool EXACT> int launch(const LinLaunch &l, hipStream_t st) {
  const int64_t outer = ((int64_t)l.items * l.kv_heads + 7) / 8 * 8, blocks = outer * (l.nheads / l.kv_heads) * l.nwalks * l.slices;
  if (blocks > 1 << 30) return MAMBA_E_UNSUPPORTED;
  const dim3 grid((int)std::min<int64_t>(blocks, 1 << kRowBits), (int)((blocks - 1) >> kRowBits) + 1);  // (those behind the last have nothing to do)
  if (l.nseg > 1) {
    lin_segment_kernel<T, KD, DVT, FIT, EXACT><<<grid, kThreads, 0, st>>>(l);
    if (hipGetLastError() != hipSuccess) return MAMBA_E_LAUNCH;
  }
  lin_walk_kernel<T, KD, DVT, FIT, PARTS, EXACT><<<grid, kThreads, 0, st>>>(l);
  return hipGetLastError() == hipSuccess ? MAMBA_OK : MAMBA_E_LAUNCH;
}
template <typename T, int KD, int DVT, Fit FIT> int run(const LinLaunch &l, hipStream_t st) {
  if constexpr (sizeof(T) < 4) {
    const LinWalk &last = l.w[l.nwalks - 1];  // the walk of the values: its state is the result, and heads that share are its sums too
    if constexpr (KD > 64 || DVT == 1)  // (two tiles of 64 keys are a forward pass's: backward both head sizes are keys of a walk)
      if (last.y_f32) return last.end.p ? launch<T, KD, DVT, FIT, true, true>(l, st) : launch<T, KD, DVT, FIT, true, false>(l, st);
    if (last.end.p) return launch<T, KD, DVT, FIT, false, true>(l, st);
  }
  return launch<T, KD, DVT, FIT, false, false>(l, st);
}
template <typename T, int KD, int DVT> int run_fit(const LinLaunch &l, const Cut &c, hipStream_t st) {
  switch (c.fit) {
    case WHOLE: return run<T, KD, DVT, WHOLE>(l, st);
    case PIECES: return run<T, KD, DVT, PIECES>(l, st);
    default: return run<T, KD, DVT, ELEMENTS>(l, st);
  }
}
template <typename T, int KD> int run_tiles(const LinLaunch &l, const Cut &c, hipStream_t st) {
  if constexpr (KD <= 128)
    if (c.tiles == 2) return run_fit<T, KD, 2>(l, c, st);
  return run_fit<T, KD, 1>(l, c, st);
}
template <typename T> int run_kd(const LinLaunch &l, const Cut &c, hipStream_t st) {
  switch (c.kd) {
    case 64: return run_tiles<T, 64>(l, c, st);
    case 128: return run_tiles<T, 128>(l, c, st);
    default: return run_tiles<T, 256>(l, c, st);
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
  if (p->nheads > 1 << 22) return MAMBA_E_UNSUPPORTED;  // a position's values are counted in 32 bits
  return MAMBA_OK;
}
// Workgroups write results while others still read: states that meet, or rows that begin where an operand's do, are refused.
bool apart(const LinearAttnParams &p, const float *a, const float *b) {
  const int64_t states = (int64_t)(p.nseq > 0 ? p.nseq : p.batch) * p.nheads * p.headdim_k * p.headdim_v * 4;
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return !a || !b || (x < y ? y - x : x - y) >= (uint64_t)states;
}
bool none_of(const void *result, std::initializer_list<const void *> others) { return std::find(others.begin(), others.end(), result) == others.end(); }
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
template <typename T> int shared(const LinearAttnParams &p, const Shared &dk, const Shared &dv, hipStream_t st) {
  const int64_t rows = (int64_t)p.batch * p.seqlen;
  const dim3 grid((int)std::min<int64_t>(rows, 16 * (int64_t)cu_count()), 2);
  const int group = p.nheads / p.nkvheads;
  if (p.headdim_k % 4 == 0 && p.headdim_v % 4 == 0) lin_shared_kernel<T, 4><<<grid, kThreads, 0, st>>>(dk, dv, rows, p.nkvheads, group, p.seqlen);
  else lin_shared_kernel<T, 1><<<grid, kThreads, 0, st>>>(dk, dv, rows, p.nkvheads, group, p.seqlen);
  return hipGetLastError() == hipSuccess ? MAMBA_OK : MAMBA_E_LAUNCH;
}
int shared_type(const LinearAttnParams &p, const Shared &dk, const Shared &dv, hipStream_t st) {
  switch (p.dtype) {
    case MAMBA_F32: return shared<float>(p, dk, dv, st);
    case MAMBA_BF16: return shared<bf16_t>(p, dk, dv, st);
    default: return shared<f16_t>(p, dk, dv, st);
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
  if (!apart(*p, p->final_states, p->initial_states) || !none_of(p->out, {p->q, p->k, p->v})) return MAMBA_E_BADARG;
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
  if (!apart(*p, p->dinitial_states, p->initial_states) || !apart(*p, p->dinitial_states, p->dfinal_states)) return MAMBA_E_BADARG;
  for (const void *result : {p->dq, p->dk, p->dv})
    if (!none_of(result, {p->q, p->k, p->v, p->dout})) return MAMBA_E_BADARG;
  if (p->dq == p->dk || p->dq == p->dv || p->dk == p->dv) return MAMBA_E_BADARG;
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
  return shared_type(*p, Shared{parts_k, p->dk, p->dk_bs, p->dk_ls, p->dk_hs, dk}, Shared{parts_v, p->dv, p->dv_bs, p->dv_ls, p->dv_hs, dv}, st);
}
