// Operand fragments of the 16 x 16 matrix instructions for kernels whose products feed one another in registers (linear
// attention, attention over a cache), for the three types of operands.
//
// D = A B^T per tile: lane (i = lane % 16, g = lane / 16) supplies row i of A and of B at the k values of its group and
// holds D[m][n] at n = i, m = 4 g + r.  So a lane that holds a result for one n and 4 consecutive m holds, read as an
// operand, row n at 4 consecutive k: results become operands where they lie.  A fragment spans KS values of k, NT = KS / 16
// tiles of results make one, and `krow` says which of the KS rows of a block the tile `half` has to take for that.
//   bf16: one instruction for 32 k.  fp16: data times data as it is (exact); where one side has been computed (a weighted
//   sum leaves fp16's range at 65504) both sides are split into two bf16 parts, 16 bits together, three instructions.
//   fp32: four instructions of 4 k, products and sums in fp32.
// Data: fragments that hold operands as they lie in memory.  Comp: a computed one in as many parts as the result's type can show.
// Wide, Wider: in two bf16 parts, 16 bits together, and in three, 24 bits.
#pragma once
#include "common.hpp"

typedef __bf16 frag_bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 frag_f16x8 __attribute__((ext_vector_type(8)));
typedef short frag_i16x4 __attribute__((ext_vector_type(4)));
typedef short frag_i16x8 __attribute__((ext_vector_type(8)));

DEVI f32x4 mma16(frag_bf16x8 a, frag_bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
DEVI f32x4 mma16(frag_f16x8 a, frag_f16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

// two bf16 parts of eight values: 8 + 8 bits
struct Split {
  frag_bf16x8 h, l;
  DEVI void set(const float (&v)[8]) {
    u32x4 hi, lo;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      hi[e] = pack_bf16(v[2 * e], v[2 * e + 1]);
      lo[e] = pack_bf16(v[2 * e] - bf16_lo(hi[e]), v[2 * e + 1] - bf16_hi(hi[e]));
    }
    h = __builtin_bit_cast(frag_bf16x8, hi);
    l = __builtin_bit_cast(frag_bf16x8, lo);
  }
};
DEVI f32x4 mma16(const Split &a, const Split &b, f32x4 c) { return mma16(a.h, b.h, mma16(a.h, b.l, mma16(a.l, b.h, c))); }
DEVI f32x4 mma16(const Split &a, frag_bf16x8 b, f32x4 c) { return mma16(a.h, b, mma16(a.l, b, c)); }
DEVI f32x4 mma16(frag_bf16x8 a, const Split &b, f32x4 c) { return mma16(a, b.h, mma16(a, b.l, c)); }

// three bf16 parts: 24 bits
struct Split3 {
  frag_bf16x8 h, m, l;
  DEVI void set(const float (&v)[8]) {
    u32x4 hi, mid, lo;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      hi[e] = pack_bf16(v[2 * e], v[2 * e + 1]);
      const float a = v[2 * e] - bf16_lo(hi[e]), b = v[2 * e + 1] - bf16_hi(hi[e]);
      mid[e] = pack_bf16(a, b);
      lo[e] = pack_bf16(a - bf16_lo(mid[e]), b - bf16_hi(mid[e]));
    }
    h = __builtin_bit_cast(frag_bf16x8, hi), m = __builtin_bit_cast(frag_bf16x8, mid), l = __builtin_bit_cast(frag_bf16x8, lo);
  }
};
DEVI f32x4 mma16(frag_bf16x8 a, const Split3 &b, f32x4 c) { return mma16(a, b.h, mma16(a, b.m, mma16(a, b.l, c))); }
DEVI f32x4 mma16(const Split &a, const Split3 &b, f32x4 c) { return mma16(a.h, b.h, mma16(a.l, b.h, mma16(a.h, b.m, mma16(a.l, b.m, mma16(a.h, b.l, c))))); }

struct Frag32 {
  f32x4 v;
};
DEVI f32x4 mma16(const Frag32 &a, const Frag32 &b, f32x4 c) {
#pragma unroll
  for (int r = 0; r < 4; ++r) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[r], b.v[r], c, 0, 0, 0);
  return c;
}

// 4 rows x 16 columns of 16-bit values, the hardware hands lane i column i of the rows: `src` is this lane's piece of 4 columns
// of row i / 4.
DEVI frag_i16x4 lds_transposed(const uint16_t *src) {
  typedef __attribute__((address_space(3))) frag_i16x4 *lds_ptr;
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)src);
}

template <typename T> struct Frags16 {
  using E = uint16_t;  // as it lies in LDS
  static constexpr int KS = 32, NT = 2, V = 8;
  static DEVI int krow(int m, int half) { return 8 * (m >> 2) + (m & 3) + 4 * half; }
  // A tile in LDS: rows of COLS values without padding, their pieces of 16 bytes permuted within the row.  A read of 16 bytes a lane is
  // served 16 lanes at a time, and those are i in 0..3, 12..15 of one group g and 4..11 of the next: along the rows they meet in no
  // bank where four rows' permutations go 0, 3, 2, 1 (0, 1, 2, 3 in order: two by two, 8 cycles an instruction and not 6).
  template <int COLS> static DEVI int swz(int row) {
    const int low = -(row >> 2) & 3;
    return COLS >= 128 ? (row & 3) << 2 | low : (row >> 1 & 1) << 2 | low;
  }
  template <int COLS> static DEVI int place(int row, int piece) { return row * COLS + (piece ^ swz<COLS>(row)) * V; }
  static constexpr int size(int rows, int cols) { return rows * cols * 2; }  // bytes
  // A lane's places (bytes) in tiles of COLS columns.  Rows and blocks of KS rows are given by where they begin (a multiple of 16
  // rows), blocks kb of KS columns by their number.
  template <int COLS> struct Lane {
    static constexpr int KB = COLS / KS;
    int row[KB], krow_row[KB], cols[KB][2];
    DEVI Lane(int i, int g, int half) {
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        row[kb] = 2 * place<COLS>(i, 4 * kb + g);
        krow_row[kb] = 2 * place<COLS>(krow(i, half), 4 * kb + g);
#pragma unroll
        for (int h = 0; h < 2; ++h) cols[kb][h] = 2 * place<COLS>(8 * g + 4 * h + (i >> 2), 4 * kb + (i & 3));
      }
    }
    // row i, or row krow(i, half) with the half that the lane was made with: k = KS kb + V g .. + 7
    DEVI u32x4 along(const char *at, int kb) const { return *reinterpret_cast<const u32x4 *>(at + row[kb]); }
    DEVI u32x4 along_krow(const char *at, int kb) const { return *reinterpret_cast<const u32x4 *>(at + krow_row[kb]); }
    // the rows of a block are k: the columns of kb, for tile `half` of them in the order of krow
    DEVI u32x4 columns(const char *block, int kb, int half) const { return both(block + cols[kb][0] + 8 * half, block + cols[kb][1] + 8 * half); }
  };
  // the same for the columns 16 (n + d) .. in order, n a multiple of the number of tiles d
  template <int COLS> struct ColumnLane {
    int cols[2];
    DEVI ColumnLane(int n, int i, int g) {
#pragma unroll
      for (int h = 0; h < 2; ++h) cols[h] = 2 * (place<COLS>(8 * g + 4 * h + (i >> 2), 2 * n + (i >> 1 & 1)) + 4 * (i & 1));
    }
    DEVI u32x4 columns(const char *block, int d = 0) const { return both(block + (cols[0] ^ 32 * d), block + (cols[1] ^ 32 * d)); }
  };
  static DEVI u32x4 both(const char *rows, const char *rows4) {
    const frag_i16x4 lo = lds_transposed(reinterpret_cast<const uint16_t *>(rows)), hi = lds_transposed(reinterpret_cast<const uint16_t *>(rows4));
    return __builtin_bit_cast(u32x4, (frag_i16x8)__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  }
  // Computed fragments of N lanes in LDS, the first parts of all of them before the second ones: what a lane holds of a tile of results
  // becomes the tile `half` of fragment n.
  template <int N> static DEVI void store_wide(char *at, int n, int half, f32x4 v) {
    const u32x2 hi = {pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3])};
    reinterpret_cast<u32x2 *>(at + 16 * n)[half] = hi;
    reinterpret_cast<u32x2 *>(at + 16 * (N + n))[half] = u32x2{pack_bf16(v[0] - bf16_lo(hi[0]), v[1] - bf16_hi(hi[0])), pack_bf16(v[2] - bf16_lo(hi[1]), v[3] - bf16_hi(hi[1]))};
  }
  template <int N> static DEVI Split load_wide(const char *at, int n) {
    const frag_bf16x8 *of = reinterpret_cast<const frag_bf16x8 *>(at);
    return Split{of[n], of[N + n]};
  }
  static DEVI void gather(const f32x4 (&t)[2], float (&v)[8]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = t[0][e], v[4 + e] = t[1][e];
  }
};

template <typename T> struct Frags;
template <> struct Frags<bf16_t> : Frags16<bf16_t> {
  using Raw = u32x4;
  using Data = frag_bf16x8;
  using Comp = frag_bf16x8;
  using Wide = Split;
  using Wider = Split3;
  static DEVI Data data(u32x4 w) { return __builtin_bit_cast(frag_bf16x8, w); }
  static DEVI f32x4 mma_raw(u32x4 a, u32x4 b, f32x4 c) { return mma16(data(a), data(b), c); }
  static DEVI void unpack(u32x4 w, float (&v)[8]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[2 * e] = bf16_lo(w[e]), v[2 * e + 1] = bf16_hi(w[e]);
  }
  // what a lane holds of a tile of results, into row `row` of a tile in LDS as the columns 16 n + 4 g ..
  template <int COLS> static DEVI void store(char *tile, int row, int n, int g, f32x4 v) {
    *reinterpret_cast<u32x2 *>(tile + 2 * (place<COLS>(row, 2 * n + (g >> 1)) + 4 * (g & 1))) = u32x2{pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3])};
  }
  static DEVI u32x4 pack(const float (&v)[8]) {
    return u32x4{pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7])};
  }
  static DEVI Comp comp(const float (&v)[8]) { return data(pack(v)); }
  template <int N> static DEVI Comp load_comp(const char *at, int n) { return reinterpret_cast<const frag_bf16x8 *>(at)[n]; }
  template <typename W> static DEVI W wide(const float (&v)[8]) {
    W s;
    s.set(v);
    return s;
  }
};
template <> struct Frags<f16_t> : Frags16<f16_t> {
  using Raw = u32x4;
  using Data = Split;
  using Comp = Split;
  using Wide = Split;
  using Wider = Split3;
  static DEVI void unpack(u32x4 w, float (&v)[8]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[2 * e] = f16_lo(w[e]), v[2 * e + 1] = f16_hi(w[e]);
  }
  template <int COLS> static DEVI void store(char *tile, int row, int n, int g, f32x4 v) {
    *reinterpret_cast<u32x2 *>(tile + 2 * (place<COLS>(row, 2 * n + (g >> 1)) + 4 * (g & 1))) = u32x2{pack_f16(v[0], v[1]), pack_f16(v[2], v[3])};
  }
  static DEVI u32x4 pack(const float (&v)[8]) {
    return u32x4{pack_f16(v[0], v[1]), pack_f16(v[2], v[3]), pack_f16(v[4], v[5]), pack_f16(v[6], v[7])};
  }
  static DEVI Data data(u32x4 w) {
    float v[8];
    unpack(w, v);
    return comp(v);
  }
  static DEVI f32x4 mma_raw(u32x4 a, u32x4 b, f32x4 c) {
    return mma16(__builtin_bit_cast(frag_f16x8, a), __builtin_bit_cast(frag_f16x8, b), c);
  }
  template <typename W> static DEVI W wide(const float (&v)[8]) {
    W s;
    s.set(v);
    return s;
  }
  static DEVI Comp comp(const float (&v)[8]) {
    Split s;
    s.set(v);
    return s;
  }
  template <int N> static DEVI Comp load_comp(const char *at, int n) { return load_wide<N>(at, n); }
};
template <> struct Frags<float> {
  using E = float;
  using Raw = f32x4;
  using Data = Frag32;
  using Comp = Frag32;
  using Wide = Frag32;
  using Wider = Frag32;
  static constexpr int KS = 16, NT = 1, V = 4;
  static DEVI int krow(int m, int) { return m; }
  // (columns are read element by element here: 4 elements of padding a row keep them and the rows apart)
  template <int COLS> static DEVI int place(int row, int piece) { return row * (COLS + 4) + piece * V; }
  static constexpr int size(int rows, int cols) { return rows * (cols + 4) * 4; }  // bytes
  template <int COLS> struct ColumnLane {
    int col;
    DEVI ColumnLane(int n, int i, int g) { col = 4 * (4 * g * (COLS + 4) + 16 * n + i); }
    DEVI f32x4 columns(const char *block, int d = 0) const {
      f32x4 v;
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] = *reinterpret_cast<const float *>(block + col + 4 * (r * (COLS + 4) + 16 * d));
      return v;
    }
  };
  template <int COLS> struct Lane {
    int row;
    ColumnLane<COLS> cols;
    DEVI Lane(int i, int g, int) : cols(0, i, g) { row = 4 * (i * (COLS + 4) + V * g); }
    DEVI f32x4 along(const char *at, int kb) const { return *reinterpret_cast<const f32x4 *>(at + row + 4 * KS * kb); }
    DEVI f32x4 along_krow(const char *at, int kb) const { return along(at, kb); }
    DEVI f32x4 columns(const char *block, int kb, int) const { return cols.columns(block + 4 * KS * kb); }
  };
  static DEVI void gather(const f32x4 (&t)[1], float (&v)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = t[0][e];
  }
  static DEVI Data data(f32x4 w) { return Frag32{w}; }
  static DEVI f32x4 mma_raw(f32x4 a, f32x4 b, f32x4 c) { return mma16(Frag32{a}, Frag32{b}, c); }
  static DEVI void unpack(f32x4 w, float (&v)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = w[e];
  }
  template <int COLS> static DEVI void store(char *tile, int row, int n, int g, f32x4 v) { *reinterpret_cast<f32x4 *>(tile + 4 * place<COLS>(row, 4 * n + g)) = v; }
  template <int N> static DEVI void store_wide(char *at, int n, int, f32x4 v) { reinterpret_cast<f32x4 *>(at)[n] = v; }
  template <int N> static DEVI Frag32 load_wide(const char *at, int n) { return Frag32{reinterpret_cast<const f32x4 *>(at)[n]}; }
  template <int N> static DEVI Frag32 load_comp(const char *at, int n) { return load_wide<N>(at, n); }
  static DEVI f32x4 pack(const float (&v)[4]) { return f32x4{v[0], v[1], v[2], v[3]}; }
  static DEVI Frag32 comp(const float (&v)[4]) { return Frag32{f32x4{v[0], v[1], v[2], v[3]}}; }
  template <typename W> static DEVI W wide(const float (&v)[4]) { return comp(v); }
};
