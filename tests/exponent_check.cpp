// Host build of the exponents of a row's softmax (fast-mac-gsplat_amd/csrc/
// exponent.h) for tests/test_code_exponent_cpu.py.
#define GS_HD inline
#include "../fast-mac-gsplat_amd/csrc/exponent.h"

// The exponents of n elements x of a row, without the row's shift; returns
// whether the row is plain.
extern "C" int exponent_check(float m, float l, float c, const float* x, int n, float* t, float* shift) {
  const gs::Exponent e(m, l, c);
  for (int i = 0; i < n; ++i) t[i] = e.plain ? e.fast(x[i]) : e.slow(x[i]);
  *shift = e.shift;
  return e.plain;
}
