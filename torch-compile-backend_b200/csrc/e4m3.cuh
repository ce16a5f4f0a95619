// Device helpers shared by the kernels with an e4m3 output: conversions, and
// the scale of a group of values.
#pragma once

#include "common.cuh"

namespace b200k {

constexpr float kE4m3Max = 448.0f;
constexpr float kMinAmax = 1e-12f;  // the smallest largest magnitude that a scale is made of

__device__ __forceinline__ uint16_t e4m3x2(float lo, float hi) {
  uint16_t u;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(u) : "f"(hi), "f"(lo));
  return u;
}
// 8 fp32 values as e4m3, times inv.
__device__ __forceinline__ uint2 e4m3x8(const float (&v)[8], float inv) {
  uint16_t q[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) q[j] = e4m3x2(v[2 * j] * inv, v[2 * j + 1] * inv);
  return make_uint2(q[0] | (static_cast<uint32_t>(q[1]) << 16), q[2] | (static_cast<uint32_t>(q[3]) << 16));
}
// 8 16-bit values as fp32.
template <bool BF16>
__device__ __forceinline__ void unpack16(const uint4& u, float (&f)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (BF16) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    } else {
      const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      f[2 * i] = v.x;
      f[2 * i + 1] = v.y;
    }
  }
}
// |v| as an unsigned pattern: ordered as the magnitudes are, infinity above
// every number and NaN above infinity, so a row's NaN reaches its scale.
__device__ __forceinline__ uint32_t mag(float v) { return __float_as_uint(v) & 0x7fffffffu; }
// The largest magnitude of 8 values, NaN above all.
__device__ __forceinline__ uint32_t top8(const float (&v)[8]) {
  float m = fabsf(v[0]);
#pragma unroll
  for (int j = 1; j < 7; j += 2)
    asm("max.NaN.f32 %0, %0, %1, %2;" : "+f"(m) : "f"(fabsf(v[j])), "f"(fabsf(v[j + 1])));
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(m) : "f"(fabsf(v[7])));
  return __float_as_uint(m);
}
// Scale of the largest magnitude `top`, and inv = 448 / it, rounded once: the
// codes' product with it moves only values next to the border of two e4m3
// numbers.  (The fast division gives 0 for divisors above 2^126.)
__device__ __forceinline__ float scale_of(uint32_t top, float& inv) {
  const float a = __uint_as_float(max(top, __float_as_uint(kMinAmax)));
  inv = __fdiv_rn(kE4m3Max, a);
  return a * (1.0f / kE4m3Max);
}

// The same with the reciprocal in two parts, inv + rest = 448 / max to 2^-48, so that
// y * inv + y * rest is y * 448 / max rounded once: half way between two e4m3 numbers
// where the quotient is (of 16-bit values 3 in 10000; the product with inv alone
// missed most of them).  Beside a largest magnitude of infinity both are 0.
__device__ __forceinline__ float scale_of(uint32_t top, float& inv, float& rest) {
  const float s = scale_of(top, inv);
  const float a = __uint_as_float(max(top, __float_as_uint(kMinAmax)));
  rest = inv > 0.0f ? fmaf(-inv, a, kE4m3Max) * (1.0f / kE4m3Max) * inv : 0.0f;
  return s;
}
// 8 fp32 values as e4m3, times inv + rest: packed, so as many instructions as one product each.
__device__ __forceinline__ uint2 e4m3x8(const float (&v)[8], float inv, float rest) {
  uint16_t q[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 y = make_float2(v[2 * j], v[2 * j + 1]);
    const float2 z = __ffma2_rn(y, make_float2(inv, inv), __fmul2_rn(y, make_float2(rest, rest)));
    q[j] = e4m3x2(z.x, z.y);
  }
  return make_uint2(q[0] | (static_cast<uint32_t>(q[1]) << 16), q[2] | (static_cast<uint32_t>(q[3]) << 16));
}
// One value.
__device__ __forceinline__ uint8_t e4m3(float y, float inv, float rest) {
  return static_cast<uint8_t>(e4m3x2(fmaf(y, inv, y * rest), 0.0f) & 0xff);
}

}  // namespace b200k
