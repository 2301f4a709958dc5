// int8 matrix product with a scale per token and per channel, for gfx950.
//
//   C[m,n] = (sum_k A[m,k] * B[n,k]) * sA[m] * sB[n]
//
// A[M,K] holds activations, B[N,K] a weight as a linear layer stores it (one
// row per output channel): K is contiguous in both, which is what the int8
// MFMAs take (16 consecutive k of a row per lane), so no operand is
// transposed.  The sum is exact in int32 (K <= 131071); it is converted to
// fp32 once (half a unit in the last place past 2^24), scaled by sA, then by
// sB, and rounded to bf16 / f16: three fp32 roundings of 2^-24 against the output's
// 2^-9 / 2^-12.
//
// Both kernels compute C^T = B . A^T with 16x16x64 MFMAs: a lane of the result
// then holds one row m and 4 consecutive n per fragment, its sA is one value
// and its stores run along C's rows.
#include "mx_common.h"

namespace mx {
namespace gemmi8 {

typedef int i32x4 __attribute__((ext_vector_type(4)));

// A: lane l holds row l%16, k = 16 (l/16) .. +15; B: column l%16, same k;
// D: lane l holds column l%16, rows 4 (l/16) .. +3.
__device__ __forceinline__ i32x4 mfma_i8(const u32x4& a, const u32x4& b, const i32x4& c) {
  return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, a), __builtin_bit_cast(i32x4, b), c, 0, 0, 0);
}

template <typename T>
__device__ __forceinline__ u32x2 scaled4(const i32x4& c, float sa, const f32x4& sb) {
  return u32x2{T::pack2((float)c[0] * sa * sb[0], (float)c[1] * sa * sb[1]),
               T::pack2((float)c[2] * sa * sb[2], (float)c[3] * sa * sb[3])};
}
__device__ __forceinline__ void store4(uint16_t* p, const u32x2& v, int left) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (i < left) p[i] = (uint16_t)(v[i >> 1] >> (16 * (i & 1)));
}
// sB of 4 channels from n, those past N as 0
__device__ __forceinline__ f32x4 scales4(const float* sB, int n, int N) {
  f32x4 s{};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (n + i < N) s[i] = sB[n + i];
  return s;
}

// ---------------------------------------------------------------------------
// Tiles for many rows: WM x WN waves, each TM rows of A by 64 rows of B.  Whole
// 128-byte lines of both operands go HBM -> LDS with direct loads into two
// slots, one K step of 128 ahead of the MFMAs.
// ---------------------------------------------------------------------------
constexpr int KS = 128;  // bytes of K per slot
constexpr int TN = 64;   // B rows of a wave: 4 fragments
constexpr int FN = 4;
constexpr int GROUP_M = 8;

template <int BM, int BN, int NW>
struct Cfg {
  static constexpr int WN = BN / TN, WM = NW / WN;
  static constexpr int TM = BM / WM, FM = TM / 16;
  static constexpr int SLOT = (BM + BN) * KS;
  static constexpr int LDS = 2 * SLOT;
  static constexpr int A_LPW = BM * KS / 1024 / NW, B_LPW = BN * KS / 1024 / NW;
  static_assert(WM * WN == NW && FM >= 1 && A_LPW >= 1 && B_LPW >= 1 && LDS <= 160 * 1024, "tile");
};

// Swizzles of the eight 16-byte chunks of a row: the 16 lanes that LDS serves
// together then read 16 different 16-byte slots of two rows (256 bytes).  An A
// fragment is 16 consecutive rows, a B fragment rows 16 i + 4 f + 0..3 (i = 0..3).
__device__ __forceinline__ int swz_a(int r) { return (r >> 1) & 7; }
__device__ __forceinline__ int swz_b(int r) { return ((r >> 1) & 1) | (((r >> 4) & 3) << 1); }

template <int BM, int BN, int NW, typename T>
__global__ __launch_bounds__(64 * NW, NW == 8 ? 1 : 2) void gemm_int8_kernel(
    const uint8_t* __restrict__ A, const float* __restrict__ sA, const uint8_t* __restrict__ B,
    const float* __restrict__ sB, uint16_t* __restrict__ C, int M, int N, int K) {
  using CF = Cfg<BM, BN, NW>;
  constexpr int FM = CF::FM;
  extern __shared__ __align__(1024) unsigned char smem[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / CF::WN, wn = wave % CF::WN;

  const int tiles_m = (M + BM - 1) / BM, tiles_n = (N + BN - 1) / BN;
  const int id = xcd_remap(blockIdx.x, tiles_m * tiles_n);
  const int per_group = GROUP_M * tiles_n;
  const int first_m = id / per_group * GROUP_M;
  const int gsz = min(tiles_m - first_m, GROUP_M);
  const int m0 = (first_m + (id % per_group) % gsz) * BM, n0 = (id % per_group) / gsz * BN;
  const int steps = (K + KS - 1) / KS;

  // Load n of a wave: 8 rows of 128 bytes, lane i row i/8, chunk (i%8) ^ swizzle.
  // Rows past M or N repeat the last one (never stored).  In a last step of fewer
  // than 128 the chunks past K repeat the row's last one; their products are
  // dropped by zeros in A's fragments.
  const uint32_t lds0 = lds_addr(smem);
  uint32_t a_off[CF::A_LPW], b_off[CF::B_LPW];
  int a_ch[CF::A_LPW], b_ch[CF::B_LPW];
#pragma unroll
  for (int n = 0; n < CF::A_LPW; ++n) {
    const int r = 8 * (wave * CF::A_LPW + n) + (lane >> 3);
    a_ch[n] = (lane & 7) ^ swz_a(r);
    a_off[n] = (uint32_t)(min(m0 + r, M - 1) - m0) * (uint32_t)K;
  }
#pragma unroll
  for (int n = 0; n < CF::B_LPW; ++n) {
    const int r = 8 * (wave * CF::B_LPW + n) + (lane >> 3);
    b_ch[n] = (lane & 7) ^ swz_b(r);
    b_off[n] = (uint32_t)(min(n0 + r, N - 1) - n0) * (uint32_t)K;
  }
  const uint8_t* a_tile = A + (size_t)m0 * K;
  const uint8_t* b_tile = B + (size_t)n0 * K;
  auto issue = [&](int j) {
    const uint32_t slot = lds0 + (j & 1) * CF::SLOT;
    const int most = (K - j * KS) / 16 - 1;  // the step's last chunk
#pragma unroll
    for (int n = 0; n < CF::A_LPW; ++n)
      dma16(a_tile + (size_t)j * KS, a_off[n] + 16 * min(a_ch[n], most), slot + (wave * CF::A_LPW + n) * 1024);
#pragma unroll
    for (int n = 0; n < CF::B_LPW; ++n)
      dma16(b_tile + (size_t)j * KS, b_off[n] + 16 * min(b_ch[n], most),
            slot + BM * KS + (wave * CF::B_LPW + n) * 1024);
  };

  const int r16 = lane & 15, g = lane >> 4;
  const int ar = wm * CF::TM + r16;                          // plus 16 f
  const int br = wn * TN + 16 * (r16 >> 2) + (r16 & 3);      // plus 4 f: swz_b the same for every f
  uint32_t a_at[2], b_at[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    a_at[h] = lds0 + ar * KS + 16 * ((4 * h + g) ^ swz_a(ar));
    b_at[h] = lds0 + BM * KS + br * KS + 16 * ((4 * h + g) ^ swz_b(br));
  }

  i32x4 acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) acc[i][j] = i32x4{};
  land_args(C, sA, sB);

  issue(0);
  for (int j = 0; j < steps; ++j) {
    wait_vmcnt<0>();
    lds_barrier();  // step j is in LDS, and every wave is done with step j-1
    if (j + 1 < steps) issue(j + 1);
    const uint32_t so = (j & 1) * CF::SLOT;
    const int left = K - j * KS;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      u32x4 a[FM], b[FN];
#pragma unroll
      for (int f = 0; f < FN; ++f) b[f] = lds_ld128(b_at[h] + so + 4 * f * KS);
#pragma unroll
      for (int f = 0; f < FM; ++f) a[f] = lds_ld128(a_at[h] + so + 16 * f * KS);
      if (left < KS) {  // the last step of a K that is no multiple of 128
#pragma unroll
        for (int f = 0; f < FM; ++f)
          if (64 * h + 16 * g >= left) a[f] = u32x4{};
      }
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int f = 0; f < FN; ++f) acc[i][f] = mfma_i8(b[f], a[i], acc[i][f]);
    }
    __builtin_amdgcn_sched_barrier(0);  // the step's reads have arrived before the next barrier
  }

  // Lane: row m = .. + 16 i + r16, columns 16 g + 4 f + 0..3: 16 consecutive ones,
  // 32 bytes, and the four lanes of a row a whole 128-byte line.
  const int n = n0 + wn * TN + 16 * g;
  f32x4 sb[FN];
#pragma unroll
  for (int f = 0; f < FN; ++f) sb[f] = scales4(sB, n + 4 * f, N);
  const bool wide = (N & 7) == 0;
#pragma unroll
  for (int i = 0; i < FM; ++i) {
    const int m = m0 + wm * CF::TM + 16 * i + r16;
    if (m < M && n < N) {
      const float sa = sA[m];
      uint16_t* out = C + (size_t)m * N + n;
#pragma unroll
      for (int f = 0; f < FN; f += 2) {
        const u32x2 lo = scaled4<T>(acc[i][f], sa, sb[f]), hi = scaled4<T>(acc[i][f + 1], sa, sb[f + 1]);
        if (wide) {
          if (n + 4 * f < N) st128(out + 4 * f, u32x4{lo[0], lo[1], hi[0], hi[1]});
        } else {
          store4(out + 4 * f, lo, N - n - 4 * f);
          store4(out + 4 * f + 4, hi, N - n - 4 * f - 4);
        }
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Few rows: the weight is streamed once from HBM into registers.  A workgroup
// takes 16 rows of B and all rows of A (16 NM at most); its waves split K and
// meet in LDS (exact integer sums).  A lane reads 32 consecutive bytes of its
// row, a quarter of the line that its group of four lanes reads together.
// ---------------------------------------------------------------------------
template <int NM, int NW, typename T>
__global__ __launch_bounds__(64 * NW) void gemm_int8_rows_kernel(
    const uint8_t* __restrict__ A, const float* __restrict__ sA, const uint8_t* __restrict__ B,
    const float* __restrict__ sB, uint16_t* __restrict__ C, int M, int N, int K) {
  __shared__ i32x4 red[NW][NM][64];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r16 = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * 16;
  const int m0 = blockIdx.y * 16 * NM;
  const int steps = (K + KS - 1) / KS;
  const int k0 = (int)((long long)steps * wave / NW), k1 = (int)((long long)steps * (wave + 1) / NW);
  const uint8_t* brow = B + (size_t)min(n0 + r16, N - 1) * K;
  const uint8_t* arow[NM];
#pragma unroll
  for (int i = 0; i < NM; ++i) arow[i] = A + (size_t)min(m0 + 16 * i + r16, M - 1) * K;
  i32x4 acc[NM];
#pragma unroll
  for (int i = 0; i < NM; ++i) acc[i] = i32x4{};
  auto step = [&](int k, bool whole) {
    u32x4 b[2], a[NM][2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int at = k * KS + 32 * g + 16 * h;
      const bool in = whole || at < K;
      b[h] = in ? ld128(brow + at) : u32x4{};
#pragma unroll
      for (int i = 0; i < NM; ++i) a[i][h] = in ? ld128(arow[i] + at) : u32x4{};
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < NM; ++i) acc[i] = mfma_i8(b[h], a[i][h], acc[i]);
  };
  const int whole = min(k1, K / KS);
  int k = k0;
  constexpr int UN = NM <= 2 ? 4 : 2;
#pragma unroll UN
  for (; k < whole; ++k) step(k, true);
  if (k < k1) step(k, false);
#pragma unroll
  for (int i = 0; i < NM; ++i) red[wave][i][lane] = acc[i];
  __syncthreads();
  for (int i = wave; i < NM; i += NW) {
    i32x4 c = red[0][i][lane];
#pragma unroll
    for (int w = 1; w < NW; ++w) c += red[w][i][lane];
    const int m = m0 + 16 * i + r16, n = n0 + 4 * g;
    if (m < M && n < N) {
      const u32x2 v = scaled4<T>(c, sA[m], scales4(sB, n, N));
      uint16_t* out = C + (size_t)m * N + n;
      if ((N & 3) == 0)
        st64(out, v);
      else
        store4(out, v, N - n);
    }
  }
}

template <int BM, int BN, int NW, typename T>
static int launch_tile(const uint8_t* A, const float* sA, const uint8_t* B, const float* sB, uint16_t* C, int M, int N,
                       int K, hipStream_t s) {
  using CF = Cfg<BM, BN, NW>;
  const long long grid = (long long)((M + BM - 1) / BM) * ((N + BN - 1) / BN);
  if (grid > 0x7fffffffLL) return MX_ERR_SHAPE;
  constexpr auto kern = gemm_int8_kernel<BM, BN, NW, T>;
  MX_RETURN_IF_HIP(lds_limit_once<kern>(CF::LDS));
  hipLaunchKernelGGL(kern, dim3((unsigned)grid), dim3(64 * NW), CF::LDS, s, A, sA, B, sB, C, M, N, K);
  MX_RETURN_IF_HIP(hipGetLastError());
  return MX_OK;
}

template <int NM, int NW, typename T>
static int launch_rows(const uint8_t* A, const float* sA, const uint8_t* B, const float* sB, uint16_t* C, int M, int N,
                       int K, hipStream_t s) {
  const dim3 grid((unsigned)((N + 15) / 16), (unsigned)((M + 16 * NM - 1) / (16 * NM)));
  hipLaunchKernelGGL((gemm_int8_rows_kernel<NM, NW, T>), grid, dim3(64 * NW), 0, s, A, sA, B, sB, C, M, N, K);
  MX_RETURN_IF_HIP(hipGetLastError());
  return MX_OK;
}

template <typename T>
static int dispatch(const uint8_t* A, const float* sA, const uint8_t* B, const float* sB, uint16_t* C, int M, int N,
                    int K, hipStream_t s) {
  if (M <= 16) return launch_rows<1, 8, T>(A, sA, B, sB, C, M, N, K, s);
  if (M <= 32) return launch_rows<2, 8, T>(A, sA, B, sB, C, M, N, K, s);
  if (M <= 64) return launch_rows<4, 8, T>(A, sA, B, sB, C, M, N, K, s);
  const long long big = (long long)((M + 255) / 256) * ((N + 255) / 256);
  if (big >= 200) return launch_tile<256, 256, 8, T>(A, sA, B, sB, C, M, N, K, s);
  return launch_tile<128, 128, 4, T>(A, sA, B, sB, C, M, N, K, s);
}

static int check(const void* A, const float* sA, const void* B, const float* sB, const void* C, int M, int N, int K,
                 int dtype) {
  if (!A || !sA || !B || !sB || !C) return MX_ERR_NULL;
  if (M <= 0 || N <= 0 || K <= 0 || K % 16 || K > 131071) return MX_ERR_SHAPE;
  if (((uintptr_t)A | (uintptr_t)B | (uintptr_t)C) & 15) return MX_ERR_ALIGN;
  if (((uintptr_t)sA | (uintptr_t)sB) & 3) return MX_ERR_ALIGN;
  if (dtype != MX_DTYPE_BF16 && dtype != MX_DTYPE_F16) return MX_ERR_DTYPE;
  if ((long long)((M + 63) / 64) * ((N + 63) / 64) > 0x7fffffffLL) return MX_ERR_SHAPE;
  return MX_OK;
}

}  // namespace gemmi8
}  // namespace mx

extern "C" int mx_gemm_int8(const void* A, const float* sA, const void* B, const float* sB, void* C, int M, int N,
                            int K, int dtype, void* stream) {
  using namespace mx::gemmi8;
  const int rc = check(A, sA, B, sB, C, M, N, K, dtype);
  if (rc != MX_OK) return rc;
  const uint8_t *a = (const uint8_t*)A, *b = (const uint8_t*)B;
  if (dtype == MX_DTYPE_BF16) return dispatch<mx::BF16>(a, sA, b, sB, (uint16_t*)C, M, N, K, (hipStream_t)stream);
  return dispatch<mx::F16>(a, sA, b, sB, (uint16_t*)C, M, N, K, (hipStream_t)stream);
}

// Workspace of the linear layer: the codes (256-byte multiple), then the scales.
static size_t linear_codes(int M, int K) { return ((size_t)M * K + 255) / 256 * 256; }

extern "C" size_t mx_linear_int8_workspace(int M, int K) {
  if (M <= 0 || K <= 0 || K % 16) return 0;
  return linear_codes(M, K) + (size_t)M * sizeof(float);
}

extern "C" int mx_linear_int8(const void* X, const void* W, const float* sW, void* C, int M, int N, int K, int ldx,
                              int dtype, void* workspace, size_t ws_bytes, void* stream) {
  if (!X || !workspace) return MX_ERR_NULL;
  float* sx = (float*)((unsigned char*)workspace + linear_codes(M > 0 ? M : 1, K > 0 ? K : 1));
  const int rc = mx::gemmi8::check(workspace, sx, W, sW, C, M, N, K, dtype);
  if (rc != MX_OK) return rc;
  if (ldx < K) return MX_ERR_SHAPE;
  if (ldx % 8 || ((uintptr_t)X & 15)) return MX_ERR_ALIGN;
  if (ws_bytes < mx_linear_int8_workspace(M, K)) return MX_ERR_WORKSPACE;
  const int q = mx_quant_int8(X, workspace, sx, M, K, ldx, dtype, stream);
  if (q != MX_OK) return q;
  return mx_gemm_int8(workspace, sx, W, sW, C, M, N, K, dtype, stream);
}
