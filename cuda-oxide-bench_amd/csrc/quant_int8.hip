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
// One workgroup or wave per row.  A lane owns units of 16 values (two 128-bit loads,
// one 128-bit store) and keeps them in registers between the two passes
// (the row's amax, then the codes), so X is read once.
#include "int8_common.h"

namespace mx {
namespace quant8 {

constexpr int NT = 256;

// LANES lanes per row (64 or NT).  U units of 16 values per lane stay in registers (K <= 16
// LANES U); U = 0: rows of any length, read twice.
template <typename T, int LANES, int U>
__global__ __launch_bounds__(NT) void quant_int8_kernel(const uint16_t* __restrict__ X, uint8_t* __restrict__ Q,
                                                       float* __restrict__ S, int M, int K, int ldx) {
  __shared__ uint32_t red[NT / 64];
  const int t = threadIdx.x % LANES;
  const int m = blockIdx.x * (NT / LANES) + __builtin_amdgcn_readfirstlane(threadIdx.x / LANES);
  if (LANES < NT && m >= M) return;  // a wave of its own, which meets no other
  const uint16_t* row = X + (size_t)m * ldx;
  uint8_t* out = Q + (size_t)m * K;
  const int units = K / 16;
  u32x4 a[U > 0 ? U : 1], b[U > 0 ? U : 1];
  uint32_t mx = 0;
  auto take = [&](const u32x4& v) { take_magnitudes<T>(mx, v); };
  if constexpr (U > 0) {
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int u = t + i * LANES;
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
    for (int u = t; u < units; u += LANES) {
      take(ld128(row + 16 * (size_t)u));
      take(ld128(row + 16 * (size_t)u + 8));
    }
  }
  mx = max(mx & 0xffffu, mx >> 16);
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) mx = max(mx, (uint32_t)__shfl_xor((int)mx, off, 64));
  if constexpr (LANES > 64) {
    if ((t & 63) == 0) red[t >> 6] = mx;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) mx = max(mx, red[w]);
  }

  const float s = scale_of<T>(mx);
  if (t == 0) S[m] = s;
  const float r = 1.0f / s;
  if constexpr (U > 0) {
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int u = t + i * LANES;
      if (u < units) st128(out + 16 * (size_t)u, encode<T>(a[i], b[i], s, r));
    }
  } else {
    for (int u = t; u < units; u += LANES)
      st128(out + 16 * (size_t)u, encode<T>(ld128(row + 16 * (size_t)u), ld128(row + 16 * (size_t)u + 8), s, r));
  }
}

template <typename T>
static int launch(const void* X, void* Q, float* S, int M, int K, int ldx, hipStream_t s) {
  constexpr int MOST = 1 << 23;  // rows of a launch: fewer than 2^32 threads
  const int units = K / 16;
  for (long long m = 0; m < M; m += MOST) {
    auto go = [&](auto kern, int rows) {
      const int n = (int)(M - m < MOST ? M - m : MOST);
      hipLaunchKernelGGL(kern, dim3((unsigned)((n + rows - 1) / rows)), dim3(NT), 0, s, (const uint16_t*)X + m * ldx,
                         (uint8_t*)Q + m * K, S + m, n, K, ldx);
    };
    // many short rows: a wave each, no meeting in LDS (16384 rows of 128, 512, 1024: 9.2, 10.5, 12.7 us,
    // a workgroup each 15.3, 16.1, 18.9; below some 1000 rows no faster, from 2064 values on slower)
    if (units <= 64 && M >= 2048) go(quant_int8_kernel<T, 64, 1>, NT / 64);
    else if (units <= NT) go(quant_int8_kernel<T, NT, 1>, 1);
    else if (units <= 2 * NT) go(quant_int8_kernel<T, NT, 2>, 1);
    else if (units <= 4 * NT) go(quant_int8_kernel<T, NT, 4>, 1);
    else go(quant_int8_kernel<T, NT, 0>, 1);
    MX_RETURN_IF_HIP(hipGetLastError());
  }
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
