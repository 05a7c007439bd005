// Gated linear recurrence, one state per channel (gfx950):
//   r = sigmoid(gate_a), i = sigmoid(gate_x), k = rate softplus(decay), log a = -k r, m = sqrt(1 - a^2)
//   h_t = a_t h_{t-1} + m_t i_t x_t
// and its gradients, with g_t = dout_t + a_{t+1} g_{t+1}:
//   dx = g m i,  dgate_x = dx x (1 - i),  dgate_a = k (1 - r) e,  ddecay = rate sigmoid(decay) sum e,
//   e = g a (a i x r / m - r h_{t-1}),  dinitial = a g at the first position
// The forward pass moves 4 tensors and the backward pass 7: both are bound by memory.  8 x 4096 x 5120 bf16: forward 270 us, 5.0 TB/s,
// backward 503 us, 4.7 TB/s, where a copy of long rows reaches 6.2 and a bare pass in this pattern (tiles of 256-byte pieces of rows, 3
// tensors in and 1 out, or 4 and 3) 5.1 and 5.0.  (Three vector instructions fewer per element backward left its time as it was.)
// gated_tile.hpp says how a row is cut.  The forward pass leaves the state that enters every tile of the backward
// pass, which then forms its own states again: one float per tile and channel instead of the states in 32 bits.
#include "gated_tile.hpp"
#include "norm_common.hpp"

namespace {

constexpr int kV = 2, kTileChannels = 64 * kV;
constexpr int kSaved = 32;  // positions from one saved state to the next

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

template <typename T, int V, bool WHOLE, bool PACKED, int R, int NW, int STREAM>
__global__ __launch_bounds__(NW * 64, 4) void gated_fwd_kernel(const GatedScanParams p, const Chain q, float *ckpt, int saved) {
  __shared__ WaveSteps<V, NW> steps;
  __shared__ Ahead<V, NW> ahead;
  __shared__ int ticket;
  const int cgroups = (p.dim + 64 * V - 1) / (64 * V), nchains = cgroups * p.batch;
  const int chain = blockIdx.x % nchains, b = chain / cgroups;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), L = p.seqlen;
  const Lane<T, V, WHOLE> at((chain % cgroups) * (64 * V) + lane * V, p.dim);
  const int n = take_tile(q, chain, &ticket);
  const int t0 = (n * NW + wave) * R, rows = min(max(L - t0, 0), R);
  Rates<V> rate(p, at.c);
  Raw<T, V> x[R], ga[R], gx[R];
  at.each_kind([&](auto few) {
    const int64_t from = min(t0, L - 1);
    const T *xr = static_cast<const T *>(p.x) + b * p.x_bs + from * p.x_ls;
    const T *ar = static_cast<const T *>(p.gate_a) + b * p.gate_a_bs + from * p.gate_a_ls;
    const T *gr = static_cast<const T *>(p.gate_x) + b * p.gate_x_bs + from * p.gate_x_ls;
#pragma unroll
    for (int j = 0; j < R; ++j) {  // past the row the last position again and again
      ga[j] = at.template load<few.value, STREAM >= 1>(ar);
      gx[j] = at.template load<few.value, STREAM >= 1>(gr);
      x[j] = at.template load<few.value, STREAM >= 1>(xr);
      const bool on = t0 + j + 1 < L;
      ar += on ? p.gate_a_ls : 0, gr += on ? p.gate_x_ls : 0, xr += on ? p.x_ls : 0;
    }
  });
  SeqRows<PACKED ? R : 1> seqs;
  if constexpr (PACKED) seqs.find(p.cu_seqlens, p.nseq, t0, L);
  rate.form(p.rate);
  Step<V> pos[R], own = no_step<V>();
#pragma unroll
  for (int j = 0; j < R; ++j) {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const Gates g(at.get(ga[j], e), at.get(gx[j], e), rate.k[e], rate.k2[e]);
      pos[j].a[e] = g.a;
      pos[j].b[e] = g.m() * g.i * at.get(x[j], e);
    }
    if (!PACKED && j >= rows) pos[j] = no_step<V>();
    own = with(own, pos[j]);
  }
  own = kept(own);
  // a wave with an edge of a sequence among its positions, or with some outside of all: the others never branch
  const bool edges = PACKED && seqs.edges();
  if constexpr (PACKED) {
    if (edges) {
      own = no_step<V>();
#pragma unroll
      for (int j = 0; j < R; ++j) {
        if (!(seqs.in >> j & 1)) {
          pos[j].a = pos[j].b = vec_of<V>(0.f);
        } else if (seqs.start >> j & 1) {
          if (p.initial_states) pos[j].b = apply<false>(pos[j], at.load_state(p.initial_states + (int64_t)seqs.seq[j] * p.dim));
          pos[j].a = vec_of<V>(0.f);
        }
        own = then<true>(own, pos[j]);
      }
    }
  }
  steps.put(wave, lane, own);
  lds_barrier();
  Step<V> before = no_step<V>();
  for (int w = 0; w < wave; ++w) before = then<PACKED>(before, steps.get(w, lane));
  if (wave == NW - 1) leave_step(q, chain, n, lane, then<PACKED>(before, own));
  Vec<V> first = vec_of<V>(0.f);
  if (!PACKED && wave == 0 && p.initial_states) first = at.load_state(p.initial_states + (int64_t)b * p.dim);
  ahead.template read<PACKED>(q, chain, n, wave, lane, first);
  lds_barrier();
  Vec<V> h = apply<PACKED>(before, ahead.template enter<PACKED>(q, lane));
  if (wave == NW - 1) leave_state(q, chain, n, lane, apply<PACKED>(own, h));
  if (t0 % kSaved == 0 && rows > 0) {
    float *ck = ckpt + (((int64_t)chain * saved + t0 / kSaved) * 64 + lane) * V;
#pragma unroll
    for (int e = 0; e < V; ++e) ck[e] = h[e];
  }
  T *out = static_cast<T *>(p.out) + b * p.out_bs + (int64_t)t0 * p.out_ls;
  auto write = [&](auto with_edges) {
#pragma unroll
    for (int j = 0; j < R; ++j) {
      h = apply<with_edges.value>(pos[j], h);
      if (j < rows) at.template store<STREAM >= 2>(out, h);
      out += p.out_ls;
      if constexpr (with_edges.value) {
        if (p.final_states && (seqs.last >> j & 1)) at.store_state(p.final_states + (int64_t)seqs.seq[j] * p.dim, h);
      }
    }
  };
  if constexpr (PACKED) {
    if (edges) write(std::true_type{});
    else write(std::false_type{});
  } else {
    write(std::false_type{});
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
// Registers: 16-bit rows spill nothing.  fp32 rows take 168 to 181 at 8 x 8, one workgroup a CU (768 of them at 2 x 2048 x 1536
// are three rounds: 44 us for 28 of bytes), and spill 12 bytes a thread at 8 x 4, packed up to 68 in both forms.
template <typename T, int V, bool WHOLE, bool PACKED, int R, int NW, int STREAM>
__global__ __launch_bounds__(NW * 64, NW > 4 ? 2 : 3) void gated_bwd_kernel(const GatedScanParams p, const Chain q, const float *ckpt, int saved, float *parts) {
  __shared__ WaveSteps<V, NW> steps, back;
  __shared__ Ahead<V, NW> ahead;
  __shared__ int ticket;
  const int cgroups = (p.dim + 64 * V - 1) / (64 * V), nchains = cgroups * p.batch;
  const int chain = blockIdx.x % nchains, b = chain / cgroups;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), L = p.seqlen;
  const Lane<T, V, WHOLE> at((chain % cgroups) * (64 * V) + lane * V, p.dim);
  const int n = take_tile(q, chain, &ticket), tile = q.ntiles - 1 - n;
  const int t0 = (tile * NW + wave) * R, rows = min(max(L - t0, 0), R);
  Rates<V> rate(p, at.c);
  Vec<V> h;
  const float *ck = ckpt + (((int64_t)chain * saved + tile * (R * NW / kSaved)) * 64 + lane) * V;
#pragma unroll
  for (int e = 0; e < V; ++e) h[e] = ck[e];
  Raw<T, V> x[R], ga[R], gx[R], d[R];
  at.each_kind([&](auto few) {
    const int64_t from = min(t0, L - 1);
    const T *xr = static_cast<const T *>(p.x) + b * p.x_bs + from * p.x_ls;
    const T *ar = static_cast<const T *>(p.gate_a) + b * p.gate_a_bs + from * p.gate_a_ls;
    const T *gr = static_cast<const T *>(p.gate_x) + b * p.gate_x_bs + from * p.gate_x_ls;
    const T *dr = static_cast<const T *>(p.dout) + b * p.dout_bs + from * p.dout_ls;
#pragma unroll
    for (int j = 0; j < R; ++j) {
      ga[j] = at.template load<few.value, STREAM >= 1>(ar);
      gx[j] = at.template load<few.value, STREAM >= 1>(gr);
      x[j] = at.template load<few.value, STREAM >= 1>(xr);
      d[j] = at.template load<few.value, STREAM >= 1>(dr);
      const bool on = t0 + j + 1 < L;
      ar += on ? p.gate_a_ls : 0, gr += on ? p.gate_x_ls : 0, xr += on ? p.x_ls : 0, dr += on ? p.dout_ls : 0;
    }
  });
  SeqRows<PACKED ? R : 1> seqs;
  if constexpr (PACKED) seqs.find(p.cu_seqlens, p.nseq, t0, L);
  // a wave with an edge of a sequence among its positions, or with some outside of all: the others never branch
  const bool edges = PACKED && seqs.edges();
  auto either = [&](auto f) {  // f(whether to look at the edges)
    if constexpr (PACKED) {
      if (edges) f(std::true_type{});
      else f(std::false_type{});
    } else {
      f(std::false_type{});
    }
  };
  auto starts = [&](int j) { return (seqs.start >> (PACKED ? j : 0) & 1) != 0; };
  auto ends = [&](int j) { return (seqs.last >> (PACKED ? j : 0) & 1) != 0; };
  auto inside = [&](int j) { return (seqs.in >> (PACKED ? j : 0) & 1) != 0; };
  auto state_of = [&](int j) { return (int64_t)seqs.seq[PACKED ? j : 0] * p.dim; };
  auto initial = [&](int j) { return p.initial_states ? at.load_state(p.initial_states + state_of(j)) : vec_of<V>(0.f); };
  auto behind_end = [&](int j) { return p.dfinal_states ? at.load_state(p.dfinal_states + state_of(j)) : vec_of<V>(0.f); };
  rate.form(p.rate);
  // of every position, beside x and the gradient that arrives there as they were loaded: a, r, i, m, and f: first r / m,
  // then e / g
  Vec<V> a[R], r[R], i[R], m[R], f[R];
#pragma unroll
  for (int j = 0; j < R; ++j) {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const Gates g(at.get(ga[j], e), at.get(gx[j], e), rate.k[e], rate.k2[e]);
      const float im = g.im();
      a[j][e] = g.a;
      r[j][e] = g.r, i[j][e] = g.i, m[j][e] = g.m2 * im, f[j][e] = g.r * im;
    }
    if (!PACKED && j >= rows) {  // a position past the row hands everything on
      a[j] = vec_of<V>(1.f);
      r[j] = i[j] = m[j] = f[j] = vec_of<V>(0.f);
      x[j].clear(), d[j].clear();
    }
  }
  Step<V> own, rev;
  either([&](auto with_edges) {
    constexpr bool E = with_edges.value;
    own = rev = no_step<V>();
#pragma unroll
    for (int j = 0; j < R; ++j) {
      if constexpr (E) {
        if (!inside(j)) {  // nor does one outside of the sequences hand on anything
          a[j] = r[j] = i[j] = m[j] = f[j] = vec_of<V>(0.f);
          x[j].clear(), d[j].clear();
        }
      }
      Step<V> s;
      s.a = a[j];
#pragma unroll
      for (int e = 0; e < V; ++e) s.b[e] = m[j][e] * i[j][e] * at.get(x[j], e);
      if constexpr (E) {
        if (starts(j)) {
          s.b = apply<false>(s, initial(j));
          s.a = vec_of<V>(0.f);
        }
      }
      own = E ? then<true>(own, s) : with(own, s);
    }
#pragma unroll
    for (int j = R - 1; j >= 0; --j) {
      bool cut = false;
      if constexpr (E) {
        cut = ends(j) || !inside(j);
        if (ends(j)) rev.b = behind_end(j);
        else if (!inside(j)) rev.b = vec_of<V>(0.f);
      }
#pragma unroll
      for (int e = 0; e < V; ++e) {
        rev.a[e] = cut ? 0.f : E ? factor1<true>(rev.a[e], a[j][e]) : rev.a[e] * a[j][e];
        rev.b[e] = a[j][e] * (rev.b[e] + at.get(d[j], e));
      }
    }
    if constexpr (!E) own = kept(own), rev = kept(rev);
  });
#pragma unroll
  for (int j = 0; j < R; ++j) x[j].anew(), d[j].anew();
  steps.put(wave, lane, own);
  back.put(wave, lane, rev);
  lds_barrier();
  Step<V> behind = no_step<V>();
  for (int w = NW - 1; w > wave; --w) behind = then<PACKED>(behind, back.get(w, lane));
  if (wave == 0) leave_step(q, chain, n, lane, then<PACKED>(behind, rev));
  for (int w = 0; w < wave; ++w) h = apply<PACKED>(steps.get(w, lane), h);
  either([&](auto with_edges) {
#pragma unroll
    for (int j = 0; j < R; ++j) {
      if constexpr (with_edges.value) {
        if (starts(j)) h = initial(j);
        if (!inside(j)) h = vec_of<V>(0.f);
      }
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float ix = i[j][e] * at.get(x[j], e);
        f[j][e] = a[j][e] * __builtin_fmaf(a[j][e] * ix, f[j][e], -r[j][e] * h[e]);
        h[e] = __builtin_fmaf(a[j][e], h[e], m[j][e] * ix);
      }
    }
  });
  Vec<V> first = vec_of<V>(0.f);
  if (!PACKED && wave == 0 && p.dfinal_states) first = at.load_state(p.dfinal_states + (int64_t)b * p.dim);
  ahead.template read<PACKED>(q, chain, n, wave, lane, first);
  lds_barrier();
  Vec<V> carry = apply<PACKED>(behind, ahead.template enter<PACKED>(q, lane)), sum = vec_of<V>(0.f);
  if (wave == 0) leave_state(q, chain, n, lane, apply<PACKED>(rev, carry));
  const int64_t end = t0 + R - 1;
  T *dxr = static_cast<T *>(p.dx) + b * p.dx_bs + end * p.dx_ls;
  T *dar = static_cast<T *>(p.dgate_a) + b * p.dgate_a_bs + end * p.dgate_a_ls;
  T *dgr = static_cast<T *>(p.dgate_x) + b * p.dgate_x_bs + end * p.dgate_x_ls;
  either([&](auto with_edges) {
    constexpr bool E = with_edges.value;
#pragma unroll
    for (int j = R - 1; j >= 0; --j) {
      if constexpr (E) {
        if (ends(j)) carry = behind_end(j);
        else if (!inside(j)) carry = vec_of<V>(0.f);
      }
      Vec<V> dx, da, dg;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float g = at.get(d[j], e) + carry[e], ee = g * f[j][e];
        dx[e] = g * m[j][e] * i[j][e];
        da[e] = rate.k[e] * (1.f - r[j][e]) * ee;
        dg[e] = dx[e] * at.get(x[j], e) * (1.f - i[j][e]);
        sum[e] += PACKED || j < rows ? ee : 0.f;
        carry[e] = a[j][e] * g;
      }
      if (j < rows) {
        at.template store<STREAM >= 2>(dxr, dx);
        at.template store<STREAM >= 2>(dar, da);
        at.template store<STREAM >= 2>(dgr, dg);
      }
      dxr -= p.dx_ls, dar -= p.dgate_a_ls, dgr -= p.dgate_x_ls;
      if constexpr (E) {
        if (starts(j) && p.dinitial_states) at.store_state(p.dinitial_states + state_of(j), carry);
      }
    }
  });
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
// How a pass is cut, by its size: tiles of R positions per wave and NW waves; whether rows stream past the caches
// (0: no, 1: what is read, 2: what is written too).
//   R, NW: kernels alone, us, bf16 -- forward at 777 x 1536 (156 tiles of 64 positions) 8 x 8 11.4, 16 x 8 12.7, at 2 x 2048 x 1536
//   in fp32 (768) 34.4 and 31.4; backward there 8 x 8 52, 8 x 4 59, at 16384 x 1024 (2048 tiles) 87 and 96, at 4 x 2048 x 2560
//   (2560 tiles) 102 and 97, at 8 x 4096 x 5120 776 and 616; 4 x 9 x 1536 4 x 8 4.6, 16 x 8 6.9.
//   STREAM: with a pass over the results behind it, as a program has one -- forward and backward at 777 x 1536 0: 13.2 + 22.6, 1:
//   14.3 + 22.8, 2: 14.7 + 23.5; at 4 x 2048 x 2560 (42 MB a tensor) 60.7 + 141, 60.1 + 138, 62.7 + 135; at 4 x 4096 x 5120 (168 MB)
//   207 + 497, 197 + 486, 195 + 469.  Rows that do not lie on 64 bytes never: two groups of channels share a line, which is gone by
//   the second -- kernels alone, 0 and 2 at 4 x 4096 x 5121 190 + 386 and 205 + 423, x 5128 175 + 357 and 193 + 389, x 5152 (rows on 64
//   bytes, not 128) 152 + 306 and 153 + 287.
struct Form {
  int r, nw, stream;
};
int64_t chains_of(const GatedScanParams &p) { return (int64_t)p.batch * ((p.dim + kTileChannels - 1) / kTileChannels); }
int64_t tiles_of(const GatedScanParams &p, int rows) { return chains_of(p) * (((int64_t)p.seqlen + rows - 1) / rows); }
int streams(const GatedScanParams &p, bool bwd) {
  const int size = p.dtype == MAMBA_F32 ? 4 : 2;
  auto at = [&](const void *t, int64_t bs, int64_t ls) { return (uint64_t)reinterpret_cast<uintptr_t>(t) | (uint64_t)((bs | ls) * size); };
  uint64_t all = at(p.x, p.x_bs, p.x_ls) | at(p.gate_a, p.gate_a_bs, p.gate_a_ls) | at(p.gate_x, p.gate_x_bs, p.gate_x_ls);
  if (bwd)
    all |= at(p.dout, p.dout_bs, p.dout_ls) | at(p.dx, p.dx_bs, p.dx_ls) | at(p.dgate_a, p.dgate_a_bs, p.dgate_a_ls) |
           at(p.dgate_x, p.dgate_x_bs, p.dgate_x_ls);
  else
    all |= at(p.out, p.out_bs, p.out_ls);
  if (all % 64 != 0) return 0;
  return (int64_t)p.batch * p.seqlen * p.dim >= (int64_t)(64 << 20) / size ? 2 : 1;
}
Form fwd_form(const GatedScanParams &p) {
  if (p.seqlen <= 32) return {4, 8, 0};
  return tiles_of(p, 64) <= 512 ? Form{8, 8, 0} : Form{16, 8, streams(p, false)};
}
Form bwd_form(const GatedScanParams &p) {
  if (p.seqlen <= 32) return {4, 8, 0};
  return tiles_of(p, 64) <= 2048 ? Form{8, 8, min(streams(p, true), 1)} : Form{8, 4, streams(p, true)};
}
template <int N> using Int = std::integral_constant<int, N>;
// f(R, NW, STREAM) as compile-time values
template <typename F> int with_fwd_form(Form o, F f) {
  if (o.r == 4) return f(Int<4>{}, Int<8>{}, Int<0>{});
  if (o.r == 8) return f(Int<8>{}, Int<8>{}, Int<0>{});
  if (o.stream == 0) return f(Int<16>{}, Int<8>{}, Int<0>{});
  return o.stream == 1 ? f(Int<16>{}, Int<8>{}, Int<1>{}) : f(Int<16>{}, Int<8>{}, Int<2>{});
}
template <typename F> int with_bwd_form(Form o, F f) {
  if (o.r == 4) return f(Int<4>{}, Int<8>{}, Int<0>{});
  if (o.nw == 8) return o.stream == 0 ? f(Int<8>{}, Int<8>{}, Int<0>{}) : f(Int<8>{}, Int<8>{}, Int<1>{});
  if (o.stream == 0) return f(Int<8>{}, Int<4>{}, Int<0>{});
  return o.stream == 1 ? f(Int<8>{}, Int<4>{}, Int<1>{}) : f(Int<8>{}, Int<4>{}, Int<2>{});
}

// Tiles of one pass and what its chains need in memory: the tickets and words, cleared before the launch, lie at the
// start of the buffer, what else it holds behind them.
struct Plan {
  int ntiles, group, ngroups;
  int64_t chains, steps, head;  // words of steps, bytes of tickets, steps and states
  Plan(const GatedScanParams &p, Form o) {
    chains = chains_of(p);
    ntiles = (int)(tiles_of(p, o.r * o.nw) / chains);
    // few chains are long ones, where states from tile to tile would be the time; many have others to run meanwhile, and a state alone
    // is less to leave than a step and a state.  Forward + backward, us, in groups of 1 and of 16: 32 chains (32768 x 4096) 323 + 1007
    // and 233 + 457, 64 (16384 x 8192) 221 + 595 and 224 + 448, 160 (4 x 4096 x 5120) 145 + 266 and 156 + 287, 320 (8 x) 261 + 479 and
    // 274 + 544.  (Groups of 4: 234 + 480 at 32 chains, of 8 233 + 465, of 32 233 + 471.)
    group = min(ntiles, chains >= 128 ? 1 : 16);
    ngroups = (ntiles + group - 1) / group;
    steps = group > 1 ? chains * ntiles * kTileChannels : 0;  // a group of one tile leaves its state alone
    head = ntiles > 1 ? (chains * 4 + 15) / 16 * 16 + steps * 8 + chains * ngroups * kTileChannels * 4 : 0;
  }
  Chain chain(void *buf) const {
    Chain q;
    q.tickets = static_cast<uint32_t *>(buf);
    q.steps = reinterpret_cast<uint64_t *>(static_cast<char *>(buf) + (chains * 4 + 15) / 16 * 16);
    q.states = reinterpret_cast<uint32_t *>(q.steps + steps);
    q.ntiles = ntiles, q.group = group, q.ngroups = ngroups;
    return q;
  }
};
int saved_states(const GatedScanParams &p) { return (p.seqlen + kSaved - 1) / kSaved; }

bool shapes_ok(const GatedScanParams *p) {
  if (!p || p->batch <= 0 || p->seqlen <= 0 || p->dim <= 0 || p->nseq < 0) return false;
  if (p->nseq > 0 && p->batch != 1) return false;
  if (!(p->rate >= 0.f && p->rate <= 3.4e38f)) return false;
  return p->dtype >= MAMBA_F32 && p->dtype <= MAMBA_F16 && p->decay_dtype >= MAMBA_F32 && p->decay_dtype <= MAMBA_F16;
}
// positions and tiles are counted in 32 bits, and so are the threads of a launch
bool counts_fit(const GatedScanParams &p) {
  if (p.seqlen > 0x7fffffff - 4096 || p.nseq > 0x7fffffff - 64 || p.dim > 0x7fffffff / 8) return false;
  const Form f = fwd_form(p), b = bwd_form(p);
  return tiles_of(p, f.r * f.nw) * f.nw * 64 <= 0xffffffffll && tiles_of(p, b.r * b.nw) * b.nw * 64 <= 0xffffffffll;
}
int check(const GatedScanParams *p, bool bwd) {
  if (!shapes_ok(p)) return MAMBA_E_BADARG;
  if (!p->x || !p->gate_a || !p->gate_x || !p->decay || !p->ckpt || (p->nseq > 0) != (p->cu_seqlens != nullptr))
    return MAMBA_E_BADARG;
  if (!aligned16(p->ckpt)) return MAMBA_E_BADARG;
  if (!bwd && !p->out) return MAMBA_E_BADARG;
  if (bwd && (!p->dout || !p->dx || !p->dgate_a || !p->dgate_x || !p->ddecay || !p->ws || !aligned16(p->ws)))
    return MAMBA_E_BADARG;
  return counts_fit(*p) ? MAMBA_OK : MAMBA_E_UNSUPPORTED;
}

// f(T{}, whole, packed) with the call's types as compile-time values
template <typename F> int with_types(const GatedScanParams &p, F f) {
  auto forms = [&](auto t) {
    const bool whole = p.dim % kV == 0;
    if (p.nseq > 0) return whole ? f(t, std::true_type{}, std::true_type{}) : f(t, std::false_type{}, std::true_type{});
    return whole ? f(t, std::true_type{}, std::false_type{}) : f(t, std::false_type{}, std::false_type{});
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
  if (!counts_fit(*p)) return MAMBA_E_UNSUPPORTED;
  const Plan f(*p, fwd_form(*p));
  return f.head + f.chains * saved_states(*p) * kTileChannels * 4;
}
extern "C" int64_t gated_scan_bwd_ws_bytes(const GatedScanParams *p) {
  if (!shapes_ok(p)) return MAMBA_E_BADARG;
  if (!counts_fit(*p)) return MAMBA_E_UNSUPPORTED;
  const Plan w(*p, bwd_form(*p));
  return w.head + (int64_t)p->batch * w.ntiles * p->dim * 4;
}

extern "C" int gated_scan_fwd(const GatedScanParams *p, mamba_stream_t stream) {
  if (const int rc = check(p, false)) return rc;
  const Form o = fwd_form(*p);
  const Plan plan(*p, o);
  if (plan.head > 0)
    if (const int rc = mamba_hip_zero(p->ckpt, plan.head, stream)) return rc;
  float *saved = reinterpret_cast<float *>(static_cast<char *>(p->ckpt) + plan.head);
  return with_types(*p, [&](auto t, auto whole, auto packed) {
    return with_fwd_form(o, [&](auto r, auto nw, auto stream_rows) {
      gated_fwd_kernel<decltype(t), kV, whole.value, packed.value, r.value, nw.value, stream_rows.value>
          <<<dim3((unsigned)(plan.chains * plan.ntiles)), dim3(nw.value * 64), 0, static_cast<hipStream_t>(stream)>>>(
              *p, plan.chain(p->ckpt), saved, saved_states(*p));
      return hipGetLastError() == hipSuccess ? MAMBA_OK : MAMBA_E_LAUNCH;
    });
  });
}
extern "C" int gated_scan_bwd(const GatedScanParams *p, mamba_stream_t stream) {
  if (const int rc = check(p, true)) return rc;
  const Form o = bwd_form(*p);
  const Plan plan(*p, o);
  if (plan.head > 0)
    if (const int rc = mamba_hip_zero(p->ws, plan.head, stream)) return rc;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const float *saved = reinterpret_cast<const float *>(static_cast<const char *>(p->ckpt) + Plan(*p, fwd_form(*p)).head);
  float *parts = reinterpret_cast<float *>(static_cast<char *>(p->ws) + plan.head);
  const int rc = with_types(*p, [&](auto t, auto whole, auto packed) {
    return with_bwd_form(o, [&](auto r, auto nw, auto stream_rows) {
      gated_bwd_kernel<decltype(t), kV, whole.value, packed.value, r.value, nw.value, stream_rows.value>
          <<<dim3((unsigned)(plan.chains * plan.ntiles)), dim3(nw.value * 64), 0, st>>>(*p, plan.chain(p->ws), saved, saved_states(*p), parts);
      return hipGetLastError() == hipSuccess ? MAMBA_OK : MAMBA_E_LAUNCH;
    });
  });
  if (rc != MAMBA_OK) return rc;
  ReduceJobs jobs{};
  jobs.part[0] = parts, jobs.out[0] = p->ddecay;
  return launch_reduce(jobs, 1, p->decay_dtype, p->batch * plan.ntiles, p->dim, st);
}
