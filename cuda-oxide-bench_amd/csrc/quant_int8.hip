// int8 quantisation of the rows of a matrix, one scale per row, for gfx950.
//
// For every row m of X[M,K] (bf16 or f16):
//     s[m]   = amax_k |X[m,k]| / 127        (fp32; 1.0 for an all-zero row)
//     Q[m,k] = RNE(X[m,k] / s[m])           (of the exact quotient, -127..127)
// A row with an infinity or a NaN gets s = NaN and codes 0, so that every
// product with it is NaN: int8 has no code that could carry it.
// Rows of activations give a scale per token, rows of an [N,K] weight one per
// output channel: both operands of mx_gemm_int8.
//
// One workgroup per row.  A lane owns units of 16 values (two 128-bit loads,
// one 128-bit store) and keeps them in registers between the two passes
// (the row's amax, then the codes), so X is read once.  The amax is a max
// of the 15 magnitude bits as integers, two values an instruction, and an
// infinity or NaN shows as a maximum past the largest finite one.
//
// Rounding: q = RNE(x * (1/s)) may miss the nearest integer only where the
// quotient lies next to a half.  e = x - q s is exact in one FMA (x and q s are
// multiples of the unit in the last place of s, and |e| <= s), so 2|e| < s
// proves q, and the rest (a vote per wave) takes the neighbour, or the even one
// of a tie.  Rows whose scale is below 2^-100 (its reciprocal could
// overflow) divide in 64 bits.
#include "mx_common.h"

namespace mx {
namespace quant8 {

constexpr int NT = 256;

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

// U units of 16 values per thread stay in registers (K <= 16 NT U); U = 0:
// rows of any length, read twice.
template <typename T, int U>
__global__ __launch_bounds__(NT) void quant_int8_kernel(const uint16_t* __restrict__ X, uint8_t* __restrict__ Q,
                                                       float* __restrict__ S, int K, int ldx) {
  __shared__ uint32_t red[NT / 64];
  const int t = threadIdx.x;
  const uint16_t* row = X + (size_t)blockIdx.x * ldx;
  uint8_t* out = Q + (size_t)blockIdx.x * K;
  const int units = K / 16;
  u32x4 a[U > 0 ? U : 1], b[U > 0 ? U : 1];
  uint32_t mx = 0;
  auto take = [&](const u32x4& v) {
#pragma unroll
    for (int w = 0; w < 4; ++w) mx = max_u16x2(mx, v[w] & 0x7fff7fffu);
  };
  if constexpr (U > 0) {
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int u = t + i * NT;
      a[i] = b[i] = u32x4{};
      if (u < units) {
        a[i] = ld128(row + 16 * u);
        b[i] = ld128(row + 16 * u + 8);
      }
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      take(a[i]);
      take(b[i]);
    }
  } else {
    for (int u = t; u < units; u += NT) {
      take(ld128(row + 16 * (size_t)u));
      take(ld128(row + 16 * (size_t)u + 8));
    }
  }
  mx = max(mx & 0xffffu, mx >> 16);
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) mx = max(mx, (uint32_t)__shfl_xor((int)mx, off, 64));
  if ((t & 63) == 0) red[t >> 6] = mx;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) mx = max(mx, red[w]);

  const bool finite = mx < first_nonfinite<T>();
  const float s = !finite ? __builtin_nanf("") : mx == 0 ? 1.0f : T::to_f32(mx) / 127.0f;
  if (t == 0) S[blockIdx.x] = s;
  const bool tiny = s < 0x1p-100f;  // false for NaN
  const float r = 1.0f / s;
  auto encode = [&](const u32x4& lo, const u32x4& hi) {
    return !finite ? u32x4{} : tiny ? encode16_tiny<T>(lo, hi, s) : encode16<T>(lo, hi, s, r);
  };
  if constexpr (U > 0) {
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int u = t + i * NT;
      if (u < units) st128(out + 16 * (size_t)u, encode(a[i], b[i]));
    }
  } else {
    for (int u = t; u < units; u += NT)
      st128(out + 16 * (size_t)u, encode(ld128(row + 16 * (size_t)u), ld128(row + 16 * (size_t)u + 8)));
  }
}

template <typename T>
static int launch(const void* X, void* Q, float* S, int M, int K, int ldx, hipStream_t s) {
  const int per = (K / 16 + NT - 1) / NT;
  auto go = [&](auto kern) {
    hipLaunchKernelGGL(kern, dim3((unsigned)M), dim3(NT), 0, s, (const uint16_t*)X, (uint8_t*)Q, S, K, ldx);
  };
  if (per <= 1) go(quant_int8_kernel<T, 1>);
  else if (per <= 2) go(quant_int8_kernel<T, 2>);
  else if (per <= 4) go(quant_int8_kernel<T, 4>);
  else go(quant_int8_kernel<T, 0>);
  MX_RETURN_IF_HIP(hipGetLastError());
  return MX_OK;
}

}  // namespace quant8
}  // namespace mx

extern "C" int mx_quant_int8(const void* X, void* Q, float* scales, int M, int K, int ldx, int dtype, void* stream) {
  if (!X || !Q || !scales) return MX_ERR_NULL;
  if (M <= 0 || K <= 0 || K % 16 || ldx < K) return MX_ERR_SHAPE;
  if (ldx % 8 || (((uintptr_t)X | (uintptr_t)Q) & 15) || ((uintptr_t)scales & 3)) return MX_ERR_ALIGN;
  if (dtype == MX_DTYPE_BF16) return mx::quant8::launch<mx::BF16>(X, Q, scales, M, K, ldx, (hipStream_t)stream);
  if (dtype == MX_DTYPE_F16) return mx::quant8::launch<mx::F16>(X, Q, scales, M, K, ldx, (hipStream_t)stream);
  return MX_ERR_DTYPE;
}
