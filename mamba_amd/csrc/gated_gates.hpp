// The terms of one position of the gated linear recurrence (gated_scan.hip has the formulas).
#pragma once
#include "common.hpp"

namespace {

// softplus to 2e-7 of its value at every size.  (An error in k repeats at every position, and a long memory adds it up;
// softplus_f's 2e-6 near e^x = 0.05 would show in fp32 results.)  e = exp(x) with the rounding of its argument made good;
// log(1 + e) = 2 atanh(e / (2 + e)) by its series below e = 0.5 (next term 1e-8 of the sum), the logarithm beyond.  It is 0 in
// 32 bits from x = -104 down; further down x log2(e) leaves their range, and its rounding is no number.
DEVI float softplus_exact(float x) {
  x = __builtin_elementwise_maximum(x, -200.f);  // (a NaN stays one)
  const float t = x * kLog2e, lo = __builtin_fmaf(x, kLog2e, -t) + x * 1.9259629911e-8f;  // log2(e) = kLog2e + 1.93e-8
  const float e = __builtin_amdgcn_exp2f(t) * __builtin_fmaf(lo, kLn2, 1.f);
  const float s = e * fast_rcp(2.f + e), s2 = s * s;
  float q = __builtin_fmaf(s2, 1.f / 9.f, 1.f / 7.f);
  q = __builtin_fmaf(s2, q, 1.f / 5.f);
  q = __builtin_fmaf(s2, q, 1.f / 3.f);
  q = __builtin_fmaf(s2, q, 1.f);
  const float r = e < 0.5f ? 2.f * s * q : fast_log(1.f + e);
  return x <= 20.f ? r : x;
}

// Factors of a state are positive; one that underflows is taken as the least normal number, so that an infinite state stays infinite
// and 0 is free as a mark.  A finite state then keeps kTiny of itself instead of nothing, and dgate_a k kTiny of it: 1e-8 where
// they are 1e30, not worth a word below.  (A NaN stays one.)
constexpr float kTiny = 1.17549435e-38f;
DEVI float not_zero(float a) { return __builtin_elementwise_maximum(a, kTiny); }

// One position's gates from kr's factor k and k2 = -k log2(e): r, i, a and m^2 = 1 - a^2.
//   1 - exp(-2 w) = 2 exp(-w) sinh(w), w = k r: no cancellation where a is near 1, and its series needs two terms below
// w = 0.25 (the next one is 5e-8 of the sum); from there on 1 - a^2 as it stands.
// Five of a position's six quarter-rate instructions (two exponentials and two reciprocals for the sigmoids, the
// exponential of the decay), with the root of m^2 the sixth.
struct Gates {
  float r, i, a, m2;
  DEVI Gates(float ga, float gx, float k, float k2) {
    r = sigmoid_f(ga);
    i = sigmoid_f(gx);
    const float w = k * r, w2 = w * w;
    a = not_zero(__builtin_amdgcn_exp2f(k2 * r));
    const float s = __builtin_fmaf(w2, __builtin_fmaf(w2, 1.f / 60.f, 1.f / 3.f), 2.f);
    const float near1 = a * w * s, else_ = __builtin_fmaf(-a, a, 1.f);  // both are formed: no branch
    m2 = w < 0.25f ? near1 : else_;
  }
  DEVI float m() const { return __builtin_amdgcn_sqrtf(m2); }
  // 1 / m, 0 where m is 0 (a gate shut to the last bit, a decay of 0): r / m tends to 0 there like sqrt(r).  Both roots take
  // an m2 below the least normal number for 0, and the reciprocal of that is an infinity.
  DEVI float im() const {
    const float root = __builtin_amdgcn_rsqf(m2);  // (of a NaN one)
    return m2 < kTiny ? 0.f : root;
  }
};

}  // namespace
