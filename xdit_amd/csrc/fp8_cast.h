// Division by a scale in front of a cast to fp8 (OCP e4m3fn), shared by the quantisers.
#pragma once
#include "common.h"

namespace xdit {

constexpr float kFp8Max = 448.0f;
constexpr int kFiniteNonZero = 0x198;  // class mask: normal and subnormal numbers of either sign

// x / scale to the fp8 byte of a true fp32 division, in three instructions instead of the dozen of the
// compiler's sequence: with r the correctly rounded 1 / scale, y = q + r (x - q scale) with q = x r
// (Markstein, "Computation of elementary functions on the IBM RISC System/6000 processor", 1990).  q is
// within 1.5 units of the quotient (one from r, for quotients near two, and half from its own rounding), the
// remainder in one fused multiply-add has at most 25 bits and so is off by at most 2^-23 units of the quotient, and
// the sum before its last rounding is within 1.75 * 2^-23 units of it.  What can round to another byte than the
// division are thus only quotients that close to the middle between an fp8 rounding point and a neighbouring fp32
// number, a few hundred pairs of mantissas that a host test enumerates: none does.  (The fp32 quotient was the
// division's in 4 * 10^9 random cases as well.)  The bounds need the remainder's and the reciprocal's exponents in range:
// scales outside [2^-80, 2^80] take the division itself, and where q is a zero, an infinity or a NaN it
// is the quotient already (the remainder would cost a negative zero its sign and make an infinity a NaN).
struct Divider {
  float scale, r;
  bool plain;
  __device__ __forceinline__ explicit Divider(float s) : scale(s), r(1.0f / s), plain(!(s >= 0x1p-80f && s <= 0x1p80f)) {}
  __device__ __forceinline__ float operator()(float x) const {
    const float q = x * r;
    const float y = __builtin_fmaf(__builtin_fmaf(-q, scale, x), r, q);
    return __builtin_amdgcn_classf(q, kFiniteNonZero) ? y : q;
  }
};

}  // namespace xdit
