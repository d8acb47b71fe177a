// Pieces of the row-wise kernels (norms, rotations, block quantiser): 8-element loads and stores, sums over a
// wavefront, the scale and cast of a 1 x 128 fp8 block.
#pragma once
#include "common.h"
#include "fp8_cast.h"

namespace xdit {

// Eight consecutive elements as they are in memory (16 bytes, or 32 in fp32).
template <typename T> struct Raw8 {
  static constexpr int N = sizeof(T) / 2;
  typedef __attribute__((ext_vector_type(8 / N))) T vec;
  vec x[N];
  __device__ __forceinline__ float operator[](int i) const { return (float)x[i / (8 / N)][i % (8 / N)]; }
};
template <typename T>
__device__ __forceinline__ void get8(const Raw8<T>& r, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; i++) v[i] = r[i];
}
template <typename T>
__device__ __forceinline__ Raw8<T> load_raw8(const void* p, int64_t off) { return *(const Raw8<T>*)((const T*)p + off); }
template <typename T>
__device__ __forceinline__ void store8(void* p, int64_t off, const float (&v)[8]) {
  Raw8<T> r;
#pragma unroll
  for (int i = 0; i < 8; i++) r.x[i / (8 / Raw8<T>::N)][i % (8 / Raw8<T>::N)] = (T)v[i];
  *(Raw8<T>*)((T*)p + off) = r;
}
// Eight parameters held as T or as fp32 (`wide`, uniform).
template <typename T>
__device__ __forceinline__ void load_param8(const void* p, int64_t off, bool wide, float (&v)[8]) {
  if (wide) get8(load_raw8<float>(p, off), v);
  else get8(load_raw8<T>(p, off), v);
}
template <typename T>
__device__ __forceinline__ void store_param8(void* p, int64_t off, bool wide, const float (&v)[8]) {
  if (wide) store8<float>(p, off, v);
  else store8<T>(p, off, v);
}

template <int CTRL>
__device__ __forceinline__ unsigned dpp_bits(unsigned x) {
  return (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xf, 0xf, true);
}
template <int CTRL>
__device__ __forceinline__ float dpp_plus(float x) { return x + __uint_as_float(dpp_bits<CTRL>(__float_as_uint(x))); }
// Sum over the 16 lanes of a DPP row, to all of them: quad permutes, then the half-row and row mirrors.
__device__ __forceinline__ float row16_sum(float x) {
  x = dpp_plus<0xB1>(x);
  x = dpp_plus<0x4E>(x);
  x = dpp_plus<0x141>(x);
  return dpp_plus<0x140>(x);
}
// Sum over the 64 lanes, to all of them, in a fixed order.
__device__ __forceinline__ float wave_sum(float x) {
  x = row16_sum(x);
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  return sum_halves(x);
}
// Largest of the 16 lanes' values, as bit patterns of non-negative floats: infinities above numbers, NaN above all.
__device__ __forceinline__ unsigned row16_max(unsigned x) {
  x = max(x, dpp_bits<0xB1>(x));
  x = max(x, dpp_bits<0x4E>(x));
  x = max(x, dpp_bits<0x141>(x));
  return max(x, dpp_bits<0x140>(x));
}

// Scale of an fp8 block from the bits of its abs-max: absmax / 448, at least the smallest normal number, 1 for a block
// of zeros; NaN and infinities pass through (a block with one of them has no finite scale).
__device__ __forceinline__ float block_scale(unsigned amax_bits) {
  const float s = __uint_as_float(amax_bits) / kFp8Max;
  return amax_bits == 0 ? 1.0f : (s < 0x1p-126f ? 0x1p-126f : s);
}
// The largest absolute value of 8 elements, as bits; NaN where one of them is (v_maximum3_f32: four instructions).
__device__ __forceinline__ unsigned absmax8(const float (&v)[8]) {
  float m = __builtin_fabsf(v[0]);
#pragma unroll
  for (int i = 1; i < 8; i++) m = __builtin_elementwise_maximum(m, __builtin_fabsf(v[i]));
  return __float_as_uint(m) & 0x7fffffffu;
}
// 1 / sqrt(x) within a unit: the hardware's estimate and one Newton step; numbers too small for that by division, and
// infinity (the step would make its zero a NaN), which one comparison of the bits finds with them.
__device__ __forceinline__ float inv_sqrt(float x) {
  constexpr unsigned kLow = 0x0d800000u, kInf = 0x7f800000u;   // 2^-100, infinity
  if (__float_as_uint(x) - kLow >= kInf - kLow) return 1.0f / sqrtf(x);
  const float r = __builtin_amdgcn_rsqf(x);
  return r * __builtin_fmaf(-0.5f * x * r, r, 1.5f);
}
// Eight numbers as e4m3 bytes.
__device__ __forceinline__ i32x2 to_fp8(const float (&q)[8]) {
  i32x2 w;
  w[0] = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
  w[0] = __builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], w[0], true);
  w[1] = __builtin_amdgcn_cvt_pk_fp8_f32(q[4], q[5], 0, false);
  w[1] = __builtin_amdgcn_cvt_pk_fp8_f32(q[6], q[7], w[1], true);
  return w;
}
// Eight quotients as the bytes of a true division.
__device__ __forceinline__ i32x2 cast8(const float (&v)[8], const Divider& div) {
  float q[8];
  if (div.plain) {
#pragma unroll
    for (int j = 0; j < 8; j++) q[j] = v[j] / div.scale;
  } else {
#pragma unroll
    for (int j = 0; j < 8; j++) q[j] = div(v[j]);
  }
  return to_fp8(q);
}

}  // namespace xdit
