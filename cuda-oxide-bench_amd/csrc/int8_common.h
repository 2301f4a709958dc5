// int8 codes of a row of bf16 / f16 values with one scale: shared by the quantiser and the
// linear layer for few rows, which quantises in its product's kernel.
//
//     s = amax |x| / 127   (fp32; 1.0 for a zero row, NaN for one with an infinity or a NaN)
//     q = RNE(x / s)       (of the exact quotient, -127..127; 0 where s is NaN)
//
// The amax is a max of the 15 magnitude bits as integers, two values an instruction,
// and an infinity or NaN shows as a maximum past the largest finite one.
//
// Rounding: q = RNE(x * (1/s)) may miss the nearest integer only where the
// quotient lies next to a half.  e = x - q s is exact in one FMA (x and q s are
// multiples of the unit in the last place of s, and |e| <= s), so 2|e| < s
// proves q, and the rest (a vote per wave) takes the neighbour, or the even one
// of a tie.  Rows whose scale is below 2^-100 (its reciprocal could
// overflow) divide in 64 bits.
#pragma once

#include "mx_common.h"

namespace mx {
namespace quant8 {

template <typename T>
__device__ __forceinline__ constexpr uint32_t first_nonfinite() {
  return std::is_same<T, BF16>::value ? 0x7f80u : 0x7c00u;
}

// max of the two 16-bit halves, each as an unsigned integer
__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
  typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
}

__device__ __forceinline__ uint32_t pack_i8(float a, float b, float c, float d) {
  const uint32_t lo = __builtin_amdgcn_perm((uint32_t)(int)b, (uint32_t)(int)a, 0x0c0c0400u);
  const uint32_t hi = __builtin_amdgcn_perm((uint32_t)(int)d, (uint32_t)(int)c, 0x04000c0cu);
  return lo | hi;
}

template <typename T>
__device__ __forceinline__ u32x4 encode16(const u32x4& lo, const u32x4& hi, float s, float r) {
  float x[16], q[16];
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    x[2 * w] = T::to_f32(lo[w] & 0xffffu);
    x[2 * w + 1] = T::to_f32(lo[w] >> 16);
    x[8 + 2 * w] = T::to_f32(hi[w] & 0xffffu);
    x[8 + 2 * w + 1] = T::to_f32(hi[w] >> 16);
  }
  bool edge = false;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    q[i] = rintf(x[i] * r);
    const float e = __builtin_fmaf(-q[i], s, x[i]);
    edge |= fabsf(e) + fabsf(e) >= s;
  }
  if (__any(edge)) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float e = __builtin_fmaf(-q[i], s, x[i]);
      const float d = fabsf(e) + fabsf(e);
      if (d > s || (d == s && ((int)q[i] & 1))) q[i] += copysignf(1.0f, e);
    }
  }
  return u32x4{pack_i8(q[0], q[1], q[2], q[3]), pack_i8(q[4], q[5], q[6], q[7]), pack_i8(q[8], q[9], q[10], q[11]),
               pack_i8(q[12], q[13], q[14], q[15])};
}

template <typename T>
__device__ u32x4 encode16_tiny(const u32x4& lo, const u32x4& hi, float s) {
  u32x4 out;
  for (int w = 0; w < 4; ++w) {
    uint32_t p = 0;
    for (int i = 0; i < 4; ++i) {
      const int e = 4 * w + i;
      const uint32_t word = e < 8 ? lo[e >> 1] : hi[(e - 8) >> 1];
      const float x = T::to_f32((e & 1) ? word >> 16 : word & 0xffffu);
      p |= ((uint32_t)(int)rint((double)x / (double)s) & 0xffu) << (8 * i);
    }
    out[w] = p;
  }
  return out;
}

template <typename T>
__device__ __forceinline__ void take_magnitudes(uint32_t& mx, const u32x4& v) {
#pragma unroll
  for (int w = 0; w < 4; ++w) mx = max_u16x2(mx, v[w] & 0x7fff7fffu);
}
// The row's scale from the largest magnitude of its values' bits.
template <typename T>
__device__ __forceinline__ float scale_of(uint32_t mx) {
  return mx >= first_nonfinite<T>() ? __builtin_nanf("") : mx == 0 ? 1.0f : T::to_f32(mx) / 127.0f;
}
template <typename T>
__device__ __forceinline__ u32x4 encode(const u32x4& lo, const u32x4& hi, float s, float r) {
  return s != s ? u32x4{} : s < 0x1p-100f ? encode16_tiny<T>(lo, hi, s) : encode16<T>(lo, hi, s, r);
}

}  // namespace quant8
}  // namespace mx
