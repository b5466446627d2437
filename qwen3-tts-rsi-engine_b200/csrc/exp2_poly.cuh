// 2^x by a polynomial. Any C++ compiler takes it, so that it is checked on the host: include it behind a two-element
// type with `fma2` and `add2` in namespace q3t (common.cuh has them for the GPU).
#pragma once

#include <math.h>
#include <stdint.h>
#include <string.h>

#include "paged.cuh"

namespace q3t {

// p * 2^n, where n is the low bits of `shifted`.
Q3T_HD float add_exponent(float p, float shifted) {
  uint32_t bits, n;
  memcpy(&bits, &p, 4);
  memcpy(&n, &shifted, 4);
  bits += n << 23;
  memcpy(&p, &bits, 4);
  return p;
}

// 2^x of two values up to 127 without the special-function unit, whose 16 results a cycle and SM a softmax is short of:
// x = n + f with n the nearest integer (adding 1.5 * 2^23 leaves n in the low bits), then 2^f on [-1/2, 1/2] as
// 1 + a polynomial of degree 4 (fitted here for the least maximal relative error: 2^-18.4) and n added to the exponent.
// Results below 2^-126 are off by less than 2^-126. From x = -127 down the result is exactly 0: f is 0 there, and 1.0's
// exponent becomes 0. NaN gives 0 too: the caller has to see it elsewhere.
template <class Float2>
Q3T_HD Float2 exp2_poly(Float2 x) {
  x.x = fmaxf(x.x, -127.f);
  x.y = fmaxf(x.y, -127.f);
  const Float2 n = add2(x, Float2{12582912.f, 12582912.f});
  const Float2 f = add2(x, fma2(n, Float2{-1.f, -1.f}, Float2{12582912.f, 12582912.f}));
  Float2 p = fma2(Float2{0.009585323743522167f, 0.009585323743522167f}, f, Float2{0.05590662732720375f, 0.05590662732720375f});
  p = fma2(p, f, Float2{0.24024039506912231f, 0.24024039506912231f});
  p = fma2(p, f, Float2{0.6931241750717163f, 0.6931241750717163f});
  p = fma2(p, f, Float2{1.f, 1.f});
  return Float2{add_exponent(p.x, n.x), add_exponent(p.y, n.y)};
}

}  // namespace q3t
