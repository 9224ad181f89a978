// block128_check.h — host checks of the block-scaled e4m3 operators' outputs,
// from the definition of the form: one power-of-two scale byte for each block,
// values rounded once to the nearest e4m3.
#pragma once

#include <algorithm>
#include <cmath>
#include <cstdint>

namespace cmb {
namespace check {

// The value of an e4m3 code; 0x7F and 0xFF are NaN.
inline double e4m3_value(uint8_t code) {
  const int e = (code >> 3) & 15, m = code & 7;
  if ((code & 0x7F) == 0x7F) return NAN;
  const double v = e == 0 ? std::ldexp(m, -9) : std::ldexp(8 + m, e - 10);
  return code & 0x80 ? -v : v;
}

// The nearest code (ties to the even one) of |x| <= 448.
inline uint8_t e4m3_nearest(double x) {
  const double a = std::fabs(x);
  int code = 0;
  while (code < 0x7E && e4m3_value(code + 1) <= a) ++code;
  if (code < 0x7E) {
    const double down = a - e4m3_value(code), up = e4m3_value(code + 1) - a;
    if (up < down || (up == down && (code & 1))) ++code;
  }
  return static_cast<uint8_t>(std::signbit(x) ? code | 0x80 : code);
}

// E8M0 byte of the smallest power of two s >= 2^-127 with top / s <= 448; 127 (a
// scale of 1) for a block of zeros.
inline int scale_byte(double top) {
  if (top == 0.0) return 127;
  int byte = 0;
  while (top > 448.0 * std::ldexp(1.0, byte - 127)) ++byte;
  return byte;
}

// Whether q(r, c) and the scale byte are x(r, c) (finite) in this form, rows x cols
// values under one scale.
template <class FX, class FQ>
bool block_holds(FX x, FQ q, int scale, int rows, int cols) {
  double top = 0.0;
  for (int r = 0; r < rows; ++r)
    for (int c = 0; c < cols; ++c) top = std::max(top, std::fabs(static_cast<double>(x(r, c))));
  if (scale != scale_byte(top)) return false;
  const double s = std::ldexp(1.0, scale - 127);
  for (int r = 0; r < rows; ++r)
    for (int c = 0; c < cols; ++c)
      if (q(r, c) != e4m3_nearest(x(r, c) / s)) return false;
  return true;
}

// Whether `got` is the sum of term(0) .. term(n - 1) in fp32, of which no term meets
// more than `depth` roundings: each is off by at most 2^-24 of the magnitudes' sum.
template <class F>
bool sum_holds(double got, F term, int n, int depth) {
  double sum = 0.0, size = 0.0;
  for (int i = 0; i < n; ++i) {
    const double t = term(i);
    sum += t;
    size += std::fabs(t);
  }
  return std::fabs(got - sum) <= std::ldexp(depth * size, -24) * 1.001;  // false for NaN
}

}  // namespace check
}  // namespace cmb
