// exponent.h -- exponents of a row's softmax, for the device and for a host
// build that tests them (tests/test_code_exponent_cpu.py).  The caller defines
// GS_HD as the function qualifiers of its compiler.
#pragma once

namespace gs {

// Exponents (x - m) c - l of a row's elements in one fused multiply-add: t(x) =
// x c - k with k = m c + l rounded, and what the rounding of k took, the same
// for all the row's elements: the exponent is t + shift.  That holds as long as
// shift is small beside the powers' range: t is off by as much, and from |k| of
// 2^31 on 2^t would be infinite or 0 in every element.  So rows whose k reaches
// kPlainLimit (a largest logit far from zero over a small temperature, or no
// probabilities at all) are not `plain` and take slow(x), one instruction more,
// whose shift is 0.  Below it |shift| <= 1.
constexpr float kPlainLimit = 16777216.0f;  // 2^24
struct Exponent {
  float m, l, c, k, shift;
  bool plain;
  GS_HD Exponent(float m_, float l_, float c_) : m(m_), l(l_), c(c_) {
#ifdef __clang__
#pragma clang fp contract(off)
#endif
    const float hi = m * c;
    const float lo = __builtin_fmaf(m, c, -hi);
    k = hi + l;
    const float back = k - hi;
    const float rest = (hi - (k - back)) + (l - back);
    plain = __builtin_fabsf(k) < kPlainLimit;
    shift = plain ? -(lo + rest) : l == l ? 0.0f : l;  // (a NaN row's is NaN)
  }
  GS_HD float fast(float x) const { return __builtin_fmaf(x, c, -k); }
  GS_HD float slow(float x) const { return (x - m) * c - l; }
};

}  // namespace gs
