// The terms of one position of the gated linear recurrence (gated_scan.hip has the formulas).
#pragma once
#include "common.hpp"

namespace {

// softplus and its slope to the last bits: once per channel, not per position.  (An error in k repeats at every
// position, and a long memory adds it up; softplus_f's 2e-6 near e^x = 0.05 would show in fp32 results.)
DEVI float softplus_exact(float x) { return x > 20.f ? x : log1pf(expf(x)); }
template <typename P> DEVI float decay_rate(const P &p, int c) {
  return p.rate * softplus_exact(ld_param(p.decay, p.decay_dtype, c));
}
template <typename P> DEVI float decay_slope(const P &p, int c) {  // dk / ddecay
  return p.rate / (1.f + expf(-ld_param(p.decay, p.decay_dtype, c)));
}

// 1 - exp(-v) for v >= 0 without cancellation: the series up to v^7 (next term below 2e-7 of the sum at v = 0.5),
// beyond it the difference, with ev = exp(-v).
DEVI float one_minus_exp(float v, float ev) {
  float s = __builtin_fmaf(v, 1.f / 5040.f, -1.f / 720.f);
  s = __builtin_fmaf(v, s, 1.f / 120.f);
  s = __builtin_fmaf(v, s, -1.f / 24.f);
  s = __builtin_fmaf(v, s, 1.f / 6.f);
  s = __builtin_fmaf(v, s, -0.5f);
  s = __builtin_fmaf(v, s, 1.f) * v;
  return v < 0.5f ? s : 1.f - ev;
}

// One position: six instructions at quarter rate (two exponentials and two reciprocals of the sigmoids, the exponential
// of the decay, one reciprocal square root) and ~20 others.
struct Gates {
  float r, i, a, m, im;  // im = 1 / m, 0 where m is 0
  DEVI Gates(float ga, float gx, float k) {
    r = sigmoid_f(ga);
    i = sigmoid_f(gx);
    const float kr = k * r;
    a = fast_exp(-kr);
    const float m2 = one_minus_exp(2.f * kr, a * a);
    im = m2 > 0.f ? __builtin_amdgcn_rsqf(m2) : 0.f * m2;  // (a NaN stays one)
    m = m2 * im;
  }
  // Gradients of one position from g, the gradient of h, and h of the position before.  Where m is 0 (a gate shut to
  // the last bit, a decay of 0) r / m tends to 0 like sqrt(r), which im = 0 gives.
  DEVI void grads(float g, float hprev, float x, float k, float &dx, float &dga, float &dgx, float &e) const {
    const float gm = g * m;
    dx = gm * i;
    dgx = dx * x * (1.f - i);
    e = g * a * (a * i * x * (r * im) - hprev * r);
    dga = k * (1.f - r) * e;
  }
};

}  // namespace
