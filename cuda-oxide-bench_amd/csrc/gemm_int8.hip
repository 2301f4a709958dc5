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
#include "int8_common.h"

namespace mx {
namespace gemmi8 {

typedef int i32x4 __attribute__((ext_vector_type(4)));

// A: lane l holds row l%16, k = 16 (l/16) .. +15; B: column l%16, same k;
// D: lane l holds column l%16, rows 4 (l/16) .. +3.
__device__ __forceinline__ i32x4 mfma_i8(const u32x4& a, const u32x4& b, const i32x4& c) {
  return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, a), __builtin_bit_cast(i32x4, b), c, 0, 0, 0);
}

// c sa sb, rounded.  c sa may leave fp32's normal range where the result does not: FAR takes an sa that far
// from one in two parts.
__device__ __forceinline__ bool far_from_one(float sa) { return fabsf(sa) >= 0x1p96f || fabsf(sa) < 0x1p-96f; }
template <typename T, bool FAR>
__device__ __forceinline__ u32x2 scaled4(const i32x4& c, float sa, const f32x4& sb) {
  f32x4 y;
  if constexpr (FAR) {
    const bool large = fabsf(sa) >= 0x1p96f, small = fabsf(sa) < 0x1p-96f;
    const float part = large ? 0x1p64f : small ? 0x1p-64f : 1.f, rest = sa * (large ? 0x1p-64f : small ? 0x1p64f : 1.f);
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = (float)c[i] * rest * sb[i] * part;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = (float)c[i] * sa * sb[i];
  }
  return u32x2{T::pack2(y[0], y[1]), T::pack2(y[2], y[3])};
}
template <typename T>
__device__ __forceinline__ u32x2 scaled4(const i32x4& c, float sa, const f32x4& sb) {
  return __any(far_from_one(sa)) ? scaled4<T, true>(c, sa, sb) : scaled4<T, false>(c, sa, sb);
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
// 128-byte lines of both operands go HBM -> LDS with direct loads into a ring of
// NS slots, NS - 1 K steps of 128 ahead of the MFMAs.
// ---------------------------------------------------------------------------
constexpr int KS = 128;  // bytes of K per slot
constexpr int TN = 64;   // B rows of a wave: 4 fragments
constexpr int FN = 4;
constexpr int GROUP_M = 8;

template <int BM, int BN, int NW, int NS>
struct Tile {
  static constexpr int WN = BN / TN, WM = NW / WN;
  static constexpr int TM = BM / WM, FM = TM / 16;
  static constexpr int SLOT = (BM + BN) * KS;
  static constexpr int LDS = NS * SLOT;
  static constexpr int A_LPW = BM * KS / 1024 / NW, B_LPW = BN * KS / 1024 / NW;
  static constexpr int LPW = A_LPW + B_LPW;
  static constexpr int PER_CU = LDS <= 80 * 1024 ? 2 : 1;  // workgroups
  static_assert((NS - 2) * LPW < 64, "vmcnt");
  static_assert(WM * WN == NW && FM >= 1 && A_LPW >= 1 && B_LPW >= 1 && LDS <= 160 * 1024, "tile");
};

// Swizzles of the eight 16-byte chunks of a row: the 16 lanes that LDS serves
// together then read 16 different 16-byte slots of two rows (256 bytes).  An A
// fragment is 16 consecutive rows, a B fragment rows 16 i + 4 f + 0..3 (i = 0..3).
__device__ __forceinline__ int swz_a(int r) { return (r >> 1) & 7; }
__device__ __forceinline__ int swz_b(int r) { return ((r >> 1) & 1) | (((r >> 4) & 3) << 1); }

template <int BM, int BN, int NW, int NS, typename T>
__global__ __launch_bounds__(64 * NW, (NW / 4 * Tile<BM, BN, NW, NS>::PER_CU)) void gemm_int8_kernel(
    const uint8_t* __restrict__ A, const float* __restrict__ sA, const uint8_t* __restrict__ B,
    const float* __restrict__ sB, uint16_t* __restrict__ C, int M, int N, int K) {
  using CF = Tile<BM, BN, NW, NS>;
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
    const uint32_t slot = lds0 + (j % NS) * CF::SLOT;
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

#pragma unroll
  for (int j = 0; j < NS - 1; ++j)
    if (j < steps) issue(j);
  for (int j = 0; j < steps; ++j) {
    if (j + NS - 2 < steps)
      wait_vmcnt<(NS - 2) * CF::LPW>();
    else
      wait_vmcnt<0>();
    lds_barrier();  // step j is in LDS, and every wave is done with step j-1
    if (j + NS - 1 < steps) issue(j + NS - 1);
    const uint32_t so = (j % NS) * CF::SLOT;
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
  // 32 bytes, and the four lanes of a row a whole 128-byte line.  Where C's rows
  // are no multiple of 16 bytes the 16 x 64 results of a fragment row go through
  // LDS, and out along the rows, 4 bytes a lane (2 for an odd N): stores of a
  // lane's own columns, 2 bytes each, took 68 us for 2197x7908x336, this way 25.
  const int nw = n0 + wn * TN, n = nw + 16 * g;
  f32x4 sb[FN];
#pragma unroll
  for (int f = 0; f < FN; ++f) sb[f] = scales4(sB, n + 4 * f, N);
  const bool wide = (N & 7) == 0;
  if (!wide) __syncthreads();  // the rings are free
  unsigned char* stage = smem + wave * 2048;
  float sa[FM];
  bool far = false;
#pragma unroll
  for (int i = 0; i < FM; ++i) {
    sa[i] = sA[min(m0 + wm * CF::TM + 16 * i + r16, M - 1)];
    far |= far_from_one(sa[i]);
  }
  far = __any(far);
#pragma unroll
  for (int i = 0; i < FM; ++i) {
    const int m = m0 + wm * CF::TM + 16 * i + r16;
    u32x4 row[2];
    auto scale = [&](auto far_tag) {
#pragma unroll
      for (int f = 0; f < 2; ++f) {
        const u32x2 lo = scaled4<T, decltype(far_tag)::value>(acc[i][2 * f], sa[i], sb[2 * f]);
        const u32x2 hi = scaled4<T, decltype(far_tag)::value>(acc[i][2 * f + 1], sa[i], sb[2 * f + 1]);
        row[f] = u32x4{lo[0], lo[1], hi[0], hi[1]};
      }
    };
    if (far)
      scale(std::true_type{});
    else
      scale(std::false_type{});
    if (wide) {
      uint16_t* out = C + (size_t)m * N + n;
#pragma unroll
      for (int f = 0; f < 2; ++f)
        if (m < M && n + 8 * f < N) st128(out + 8 * f, row[f]);
    } else {
      const int mw = m - r16;  // the fragment's first row
#pragma unroll
      for (int f = 0; f < 2; ++f) st128(stage + r16 * 128 + 16 * ((2 * g + f) ^ (r16 & 7)), row[f]);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the wave's own stage: no barrier
      if ((N & 1) == 0) {
#pragma unroll
        for (int s = 0; s < 8; ++s) {
          const int r = 2 * s + (lane >> 5), c = lane & 31;  // a dword: columns 2 c, 2 c + 1
          const uint32_t v = *reinterpret_cast<const uint32_t*>(stage + r * 128 + 16 * ((c >> 2) ^ (r & 7)) + 4 * (c & 3));
          if (mw + r < M && nw + 2 * c < N) *reinterpret_cast<uint32_t*>(C + (size_t)(mw + r) * N + nw + 2 * c) = v;
        }
      } else {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const uint16_t v =
              *reinterpret_cast<const uint16_t*>(stage + r * 128 + 16 * ((lane >> 3) ^ (r & 7)) + 2 * (lane & 7));
          if (mw + r < M && nw + lane < N) C[(size_t)(mw + r) * N + nw + lane] = v;
        }
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
  }
}

// ---------------------------------------------------------------------------
// Few rows: the weight is streamed once.  A workgroup takes 16 FB rows of B and 16
// FM rows of A; its four waves split K and meet in LDS (exact integer sums).
// Each wave fills a ring of its own with direct loads of whole 128-byte lines and
// waits for nobody: no barrier before the sums.  Loading the fragments straight
// into registers needs no LDS, but neighbouring lanes then read different rows,
// which the L1 takes one at a time (64x4096x7168: 21 us, and 11.5 this way).
// ---------------------------------------------------------------------------
constexpr int RW = 4;  // waves
template <int FM, int FB>
struct Rows {
  static constexpr int SLOT = 16 * (FM + FB) * KS;
  static constexpr int LPW = 2 * (FM + FB);  // 1 KB loads of a step
  static constexpr int FIT = 80 * 1024 / RW / SLOT;  // two workgroups on a CU
  static constexpr int NS = FIT > 8 ? 8 : FIT;
  static constexpr int LDS = RW * NS * SLOT;
  static_assert(NS >= 2 && (NS - 1) * LPW < 64, "vmcnt");
  static_assert(FM * FB * 64 * 16 <= NS * SLOT, "the sums meet in the rings");
};

template <int FM, int FB, typename T>
__global__ __launch_bounds__(64 * RW) void gemm_int8_rows_kernel(
    const uint8_t* __restrict__ A, const float* __restrict__ sA, const uint8_t* __restrict__ B,
    const float* __restrict__ sB, uint16_t* __restrict__ C, int M, int N, int K) {
  using R = Rows<FM, FB>;
  extern __shared__ __align__(1024) unsigned char smem[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r16 = lane & 15, g = lane >> 4;
  // workgroups of the same rows of B side by side: one XCD's L2 then reads them once
  const int tiles_m = (M + 16 * FM - 1) / (16 * FM);
  const int id = xcd_remap(blockIdx.x, gridDim.x);
  const int n0 = id / tiles_m * 16 * FB, m0 = id % tiles_m * 16 * FM;
  const int steps = (K + KS - 1) / KS;
  const int k0 = steps * wave / RW, k1 = steps * (wave + 1) / RW;

  // rows of a slot: A's 16 FM, then B's 16 FB; lane i of load n: row 8 n + i/8, chunk
  // (i%8) ^ swizzle.  Past M, N or K: the last row or chunk again.
  const uint32_t ring = lds_addr(smem) + wave * R::NS * R::SLOT;
  const int lr = lane >> 3;
  uint32_t off[R::LPW];
#pragma unroll
  for (int n = 0; n < R::LPW; ++n) {
    const int r = 8 * n + lr;
    off[n] = (uint32_t)(n < 2 * FM ? min(m0 + r, M - 1) - m0 : min(n0 + r - 16 * FM, N - 1) - n0) * (uint32_t)K;
  }
  const uint8_t *a_rows = A + (size_t)m0 * K, *b_rows = B + (size_t)n0 * K;
  const int ch[2] = {(lane & 7) ^ swz_a(lr), (lane & 7) ^ swz_a(8 + lr)};
  auto issue = [&](int k, int slot) {
    const int most = (K - k * KS) / 16 - 1;
#pragma unroll
    for (int n = 0; n < R::LPW; ++n)
      dma16((n < 2 * FM ? a_rows : b_rows) + (size_t)k * KS, off[n] + 16 * min(ch[n & 1], most),
            ring + slot * R::SLOT + n * 1024);
  };
  uint32_t at[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) at[h] = ring + r16 * KS + 16 * ((4 * h + g) ^ swz_a(r16));

  i32x4 acc[FM][FB];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int f = 0; f < FB; ++f) acc[i][f] = i32x4{};
  land_args(C, sA, sB);

#pragma unroll
  for (int s = 0; s < R::NS; ++s)
    if (k0 + s < k1) issue(k0 + s, s);
  int slot = 0;
  for (int k = k0; k < k1; ++k) {
    if (k + R::NS <= k1)
      wait_vmcnt<(R::NS - 1) * R::LPW>();
    else
      wait_vmcnt<0>();
    asm volatile("" ::: "memory");  // no read before the wait
    const uint32_t so = slot * R::SLOT;
    const int left = K - k * KS;
    u32x4 a[2][FM], b[2][FB];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int f = 0; f < FB; ++f) b[h][f] = lds_ld128(at[h] + so + 16 * (FM + f) * KS);
#pragma unroll
      for (int f = 0; f < FM; ++f) {
        a[h][f] = lds_ld128(at[h] + so + 16 * f * KS);
        if (64 * h + 16 * g >= left) a[h][f] = u32x4{};  // past K
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int f = 0; f < FB; ++f) acc[i][f] = mfma_i8(b[h][f], a[h][i], acc[i][f]);
    __builtin_amdgcn_sched_barrier(0);  // the slot's reads have arrived: it can be filled again
    if (k + R::NS < k1) issue(k + R::NS, slot);
    slot = slot + 1 == R::NS ? 0 : slot + 1;
  }

  __syncthreads();
  i32x4* red = reinterpret_cast<i32x4*>(smem);  // [RW][FM * FB][64]
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int f = 0; f < FB; ++f) red[(wave * FM * FB + i * FB + f) * 64 + lane] = acc[i][f];
  __syncthreads();
  for (int i = wave; i < FM * FB; i += RW) {
    i32x4 c = red[i * 64 + lane];
#pragma unroll
    for (int w = 1; w < RW; ++w) c += red[(w * FM * FB + i) * 64 + lane];
    const int m = m0 + 16 * (i / FB) + r16, n = n0 + 16 * (i % FB) + 4 * g;
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

// ---------------------------------------------------------------------------
// A linear layer for one to a few rows in one kernel: every workgroup quantises the rows
// for itself (in LDS, while its rows of B are on the way), and the second launch, the codes'
// way through memory and the workspace fall away.  Otherwise as the kernel above.
// ---------------------------------------------------------------------------
constexpr int FEW_ROWS = 8, FEW_VALUES = 8192;  // the most rows, the most rows times K
template <int FB>
struct Few {
  static constexpr int X = FEW_VALUES * 2;  // the rows as they come, then their codes
  static constexpr int SCALES = X, RING = X + 1024;
  static constexpr int SLOT = 16 * FB * KS, LPW = 2 * FB;
  static constexpr int NS = (80 * 1024 - RING) / RW / SLOT;  // two workgroups on a CU
  static constexpr int LDS = RING + RW * NS * SLOT;
  static_assert(NS >= 2 && NS * LPW < 64 && FB * 64 * 16 <= NS * SLOT, "rings");
};

template <int FB, typename T>
__global__ __launch_bounds__(64 * RW, 2) void linear_int8_few_kernel(
    const uint16_t* __restrict__ X, const uint8_t* __restrict__ B, const float* __restrict__ sB, uint16_t* __restrict__ C,
    int M, int N, int K, int ldx) {
  using F = Few<FB>;
  constexpr int NT = 64 * RW;
  extern __shared__ __align__(1024) unsigned char smem[];
  const int t = threadIdx.x, lane = t & 63;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int r16 = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * 16 * FB;
  const int steps = (K + KS - 1) / KS;
  const int k0 = steps * wave / RW, k1 = steps * (wave + 1) / RW;
  const uint32_t x0 = lds_addr(smem);

  // X's rows, 8 values a lane and load, one behind the other in LDS
  const uint32_t eighths = K / 8, pieces = M * eighths;
  for (uint32_t i = 64 * wave; i < pieces; i += NT) {
    const uint32_t p = min(i + lane, pieces - 1);
    dma16(X, (p / eighths * ldx + p % eighths * 8) * 2, x0 + 16 * i);
  }
  // the wave's ring of B's rows
  const uint32_t ring = x0 + F::RING + wave * F::NS * F::SLOT;
  const int lr = lane >> 3;
  uint32_t off[F::LPW];
#pragma unroll
  for (int n = 0; n < F::LPW; ++n) off[n] = (uint32_t)(min(n0 + 8 * n + lr, N - 1) - n0) * (uint32_t)K;
  const uint8_t* b_rows = B + (size_t)n0 * K;
  const int ch[2] = {(lane & 7) ^ swz_a(lr), (lane & 7) ^ swz_a(8 + lr)};
  auto issue = [&](int k, int slot) {
    const int last = (K - k * KS) / 16 - 1;
#pragma unroll
    for (int n = 0; n < F::LPW; ++n)
      dma16(b_rows + (size_t)k * KS, off[n] + 16 * min(ch[n & 1], last), ring + slot * F::SLOT + n * 1024);
  };
#pragma unroll
  for (int s = 0; s < F::NS; ++s)
    if (k0 + s < k1) issue(k0 + s, s);
  land_args(C, sB);

  uint32_t* most = reinterpret_cast<uint32_t*>(smem + F::SCALES);  // the rows' maxima, then their scales
  if (t < FEW_ROWS) most[t] = 0;
  auto meet = [] {  // LDS reads and writes done, B's loads still on the way
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    lds_barrier();
  };
  if (k1 - k0 >= F::NS)
    wait_vmcnt<F::NS * F::LPW>();  // X is there, B may be on the way
  else
    wait_vmcnt<0>();
  meet();

  // ---- codes: units of 16 values, those of a row are K / 16 ----
  constexpr int U = FEW_VALUES / 16 / NT;
  const uint32_t per = K / 16, units = M * per;
  u32x4 lo[U], hi[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t i = t + u * NT;
    if (i - lane >= units) break;  // the wave's units all lie behind the last
    lo[u] = hi[u] = u32x4{};
    if (i < units) {
      lo[u] = lds_ld128(x0 + 32 * i);
      hi[u] = lds_ld128(x0 + 32 * i + 16);
    }
    uint32_t v = 0;
    quant8::take_magnitudes<T>(v, lo[u]);
    quant8::take_magnitudes<T>(v, hi[u]);
    v = max(v & 0xffffu, v >> 16);
    const uint32_t m = min(i, units - 1) / per;
    if (__all(m == (uint32_t)__builtin_amdgcn_readfirstlane((int)m))) {  // one row: one lane for all
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) v = max(v, (uint32_t)__shfl_xor((int)v, o, 64));
      if (lane == 0) atomicMax(most + m, v);
    } else {
      atomicMax(most + m, v);
    }
  }
  meet();  // the maxima are whole, and X is in registers: the codes take its place
  float* scales = reinterpret_cast<float*>(most);
  const float own = t < M ? quant8::scale_of<T>(most[t]) : 0.f;
  if (t < M) scales[t] = own;  // a thread reads and writes its own row's
  meet();
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t i = t + u * NT;
    if (i < units) {
      const float s = scales[i / per];
      st128(smem + 16 * i, quant8::encode<T>(lo[u], hi[u], s, 1.0f / s));
    }
  }
  meet();

  // ---- the product: lane's row of A r16 (the last one again past M: never stored) ----
  const uint32_t a_at = x0 + min(r16, M - 1) * K + 16 * g;
  uint32_t b_at[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) b_at[h] = ring + r16 * KS + 16 * ((4 * h + g) ^ swz_a(r16));
  i32x4 acc[FB];
#pragma unroll
  for (int f = 0; f < FB; ++f) acc[f] = i32x4{};
  int slot = 0;
  for (int k = k0; k < k1; ++k) {
    if (k + F::NS <= k1)
      wait_vmcnt<(F::NS - 1) * F::LPW>();
    else
      wait_vmcnt<0>();
    asm volatile("" ::: "memory");  // no read before the wait
    const uint32_t so = slot * F::SLOT;
    u32x4 a[2], b[2][FB];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      a[h] = u32x4{};
      if (k * KS + 64 * h + 16 * g < K) a[h] = lds_ld128(a_at + k * KS + 64 * h);
#pragma unroll
      for (int f = 0; f < FB; ++f) b[h][f] = lds_ld128(b_at[h] + so + 16 * f * KS);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int f = 0; f < FB; ++f) acc[f] = mfma_i8(b[h][f], a[h], acc[f]);
    __builtin_amdgcn_sched_barrier(0);  // the slot's reads have arrived: it can be filled again
    if (k + F::NS < k1) issue(k + F::NS, slot);
    slot = slot + 1 == F::NS ? 0 : slot + 1;
  }
  __syncthreads();
  i32x4* red = reinterpret_cast<i32x4*>(smem + F::RING);  // [RW][FB][64]
#pragma unroll
  for (int f = 0; f < FB; ++f) red[(wave * FB + f) * 64 + lane] = acc[f];
  __syncthreads();
  for (int f = wave; f < FB; f += RW) {
    i32x4 c = red[f * 64 + lane];
#pragma unroll
    for (int w = 1; w < RW; ++w) c += red[(w * FB + f) * 64 + lane];
    const int n = n0 + 16 * f + 4 * g;
    if (r16 < M && n < N) {
      const u32x2 v = scaled4<T>(c, scales[r16], scales4(sB, n, N));
      uint16_t* out = C + (size_t)r16 * N + n;
      if ((N & 3) == 0)
        st64(out, v);
      else
        store4(out, v, N - n);
    }
  }
}

// ---------------------------------------------------------------------------
// Launch choice.  What bounds every variant short of the largest products is the rate
// at which a CU takes operand lines in (44 to 82 GB/s with one workgroup on the CU, 58 to 71
// with more; the 256x256 tile, whose ring holds two slots, 40), and where K is short a
// workgroup's begin and end.  So a variant costs
//     start + next * (n - 1) + n * (rows of A and B of a workgroup) * K / rate
// for n workgroups on a CU.  The constants are fits to the times of all variants over 158 products
// (1x64x16 to 8192^3); over these and 84 others the choice loses 1.5% on average against the best
// variant of each, and 27% at most (3034x964x4480: 33 us, 26 with 64x128 tiles).  Without `next` it
// lost 8%, and 5267x830x16 took 27.9 us in place of 7.6.  Rows kernels of 64x32 and 32x64 gained
// 0.2% where they were best, and are not kept.
// ---------------------------------------------------------------------------
struct Variant {
  int bm, bn;
  float start, next, one, many;  // us; bytes per us with one workgroup on a CU, with more
};
constexpr Variant kVariants[] = {
    {16, 16, 2.6f, 0.5f, 68e3f, 65e3f},    {16, 32, 2.7f, 0.6f, 64e3f, 71e3f},   {32, 16, 2.7f, 0.6f, 82e3f, 68e3f},
    {32, 32, 2.9f, 0.8f, 71e3f, 68e3f},    {64, 64, 3.8f, 1.4f, 51e3f, 71e3f},   {128, 64, 4.6f, 1.8f, 55e3f, 70e3f},
    {64, 128, 4.8f, 1.9f, 51e3f, 71e3f},   {128, 128, 5.1f, 2.8f, 44e3f, 61e3f}, {256, 256, 11.8f, 10.4f, 47e3f, 40e3f},
};
constexpr int kNumVariants = sizeof(kVariants) / sizeof(kVariants[0]);

static int pick(int M, int N, int K) {
  int best = 0;
  double least = 1e30;
  for (int i = 0; i < kNumVariants; ++i) {
    const Variant& v = kVariants[i];
    const double wgs = (double)((M + v.bm - 1) / v.bm) * ((N + v.bn - 1) / v.bn);
    const double n = wgs <= 256 ? 1 : wgs <= 8192 ? (double)(((long long)wgs + 255) / 256) : wgs / 256;
    const double us = v.start + v.next * (n - 1) + n * (v.bm + v.bn) * K / (n > 1 ? v.many : v.one);
    if (us < least) least = us, best = i;
  }
  return best;
}

template <typename Kern>
static int launch(Kern kern, hipError_t ready, int lds, int threads, dim3 grid, const uint8_t* A, const float* sA,
                  const uint8_t* B, const float* sB, uint16_t* C, int M, int N, int K, hipStream_t s) {
  MX_RETURN_IF_HIP(ready);
  hipLaunchKernelGGL(kern, grid, dim3(threads), lds, s, A, sA, B, sB, C, M, N, K);
  MX_RETURN_IF_HIP(hipGetLastError());
  return MX_OK;
}

template <typename T>
static int run(int variant, const uint8_t* A, const float* sA, const uint8_t* B, const float* sB, uint16_t* C, int M,
               int N, int K, hipStream_t s) {
  const Variant& v = kVariants[variant];
  const long long tm = (M + v.bm - 1) / v.bm, tn = (N + v.bn - 1) / v.bn;
  if (tm * tn >= (1 << 23)) return MX_ERR_SHAPE;  // fewer than 2^32 threads
#define ROWS(FM, FB)                                                                                               \
  launch(gemm_int8_rows_kernel<FM, FB, T>, lds_limit_once<gemm_int8_rows_kernel<FM, FB, T>>(Rows<FM, FB>::LDS),    \
         Rows<FM, FB>::LDS, 64 * RW, dim3((unsigned)(tm * tn)), A, sA, B, sB, C, M, N, K, s)
#define TILE(BM, BN, NW, NS)                                                                                      \
  launch(gemm_int8_kernel<BM, BN, NW, NS, T>, lds_limit_once<gemm_int8_kernel<BM, BN, NW, NS, T>>(Tile<BM, BN, NW, NS>::LDS), \
         Tile<BM, BN, NW, NS>::LDS, 64 * NW, dim3((unsigned)(tm * tn)), A, sA, B, sB, C, M, N, K, s)
  switch (variant) {
    case 0: return ROWS(1, 1);
    case 1: return ROWS(1, 2);
    case 2: return ROWS(2, 1);
    case 3: return ROWS(2, 2);
    case 4: return TILE(64, 64, 4, 4);
    case 5: return TILE(128, 64, 4, 3);
    case 6: return TILE(64, 128, 4, 3);
    case 7: return TILE(128, 128, 8, 2);
    default: return TILE(256, 256, 8, 2);
  }
#undef ROWS
#undef TILE
}

// One kernel where the codes that every workgroup makes again cost less than the launch and
// the codes' way that it saves, against the quantiser and the best product (K x N, us):
//   rows  512x4096  1024x4096  2048x4096  4096x4096  4096x16384  8192x4096
//   1      4.3/5.3    4.8/5.8    5.8/6.8    6.3/8.0   15.3/18.1  10.3/11.5
//   2      4.2/5.7    5.2/6.2    6.6/7.4    7.8/8.5   15.9/18.7  13.5/12.9
//   4      4.4/5.8    5.6/6.4    7.6/7.4   10.6/8.8   17.7/18.7
//   8      5.1/6.2    7.3/6.6   10.4/7.7
static bool few(int M, int K) {
  const long long values = (long long)M * K;
  return M <= 2 ? values <= FEW_VALUES : M <= FEW_ROWS && values <= FEW_VALUES / 2;
}

template <int FB, typename T>
static int launch_few(const void* X, const void* B, const float* sB, void* C, int M, int N, int K, int ldx, hipStream_t s) {
  using F = Few<FB>;
  constexpr auto kern = linear_int8_few_kernel<FB, T>;
  MX_RETURN_IF_HIP(lds_limit_once<kern>(F::LDS));
  hipLaunchKernelGGL(kern, dim3((unsigned)((N + 16 * FB - 1) / (16 * FB))), dim3(64 * RW), F::LDS, s, (const uint16_t*)X,
                     (const uint8_t*)B, sB, (uint16_t*)C, M, N, K, ldx);
  MX_RETURN_IF_HIP(hipGetLastError());
  return MX_OK;
}

static int check(const void* A, const float* sA, const void* B, const float* sB, const void* C, int M, int N, int K,
                 int dtype) {
  if (!A || !sA || !B || !sB || !C) return MX_ERR_NULL;
  if (M <= 0 || N <= 0 || K <= 0 || K % 16 || K > 131071) return MX_ERR_SHAPE;
  if (((uintptr_t)A | (uintptr_t)B | (uintptr_t)C) & 15) return MX_ERR_ALIGN;
  if (((uintptr_t)sA | (uintptr_t)sB) & 3) return MX_ERR_ALIGN;
  if (dtype != MX_DTYPE_BF16 && dtype != MX_DTYPE_F16) return MX_ERR_DTYPE;
  if (M > 0x7fffff00 || N > 0x7fffff00) return MX_ERR_SHAPE;
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
  const int v = pick(M, N, K);
  if (dtype == MX_DTYPE_BF16) return run<mx::BF16>(v, a, sA, b, sB, (uint16_t*)C, M, N, K, (hipStream_t)stream);
  return run<mx::F16>(v, a, sA, b, sB, (uint16_t*)C, M, N, K, (hipStream_t)stream);
}

// Workspace of the linear layer: the codes (256-byte multiple), then the scales.
static size_t linear_codes(int M, int K) { return ((size_t)M * K + 255) / 256 * 256; }

extern "C" size_t mx_linear_int8_workspace(int M, int K) {
  if (M <= 0 || K <= 0 || K % 16 || mx::gemmi8::few(M, K)) return 0;
  return linear_codes(M, K) + (size_t)M * sizeof(float);
}

extern "C" int mx_linear_int8(const void* X, const void* W, const float* sW, void* C, int M, int N, int K, int ldx,
                              int dtype, void* workspace, size_t ws_bytes, void* stream) {
  using namespace mx::gemmi8;
  if (!X) return MX_ERR_NULL;
  // X, the scales sW in place of the rows' own, for the checks that the product makes
  const int rc = check(X, sW, W, sW, C, M, N, K, dtype);
  if (rc != MX_OK) return rc;
  if (ldx < K) return MX_ERR_SHAPE;
  if (ldx % 8) return MX_ERR_ALIGN;
  hipStream_t s = (hipStream_t)stream;
  if (few(M, K)) {
    if (M == 1) ldx = K;
    if ((long long)M * ldx >= (1LL << 30) || N >= (1 << 27)) return MX_ERR_SHAPE;  // 32-bit offsets; threads
    // 16 rows of B a workgroup while two on every CU hold all of N
    const bool one = N <= 8192;
    if (dtype == MX_DTYPE_BF16)
      return one ? launch_few<1, mx::BF16>(X, W, sW, C, M, N, K, ldx, s) : launch_few<2, mx::BF16>(X, W, sW, C, M, N, K, ldx, s);
    return one ? launch_few<1, mx::F16>(X, W, sW, C, M, N, K, ldx, s) : launch_few<2, mx::F16>(X, W, sW, C, M, N, K, ldx, s);
  }
  if (!workspace) return MX_ERR_NULL;
  if ((uintptr_t)workspace & 15) return MX_ERR_ALIGN;
  if (ws_bytes < linear_codes(M, K) + (size_t)M * sizeof(float)) return MX_ERR_WORKSPACE;
  float* sx = (float*)((unsigned char*)workspace + linear_codes(M, K));
  const int q = mx_quant_int8(X, workspace, sx, M, K, ldx, dtype, stream);
  if (q != MX_OK) return q;
  return mx_gemm_int8(workspace, sx, W, sW, C, M, N, K, dtype, stream);
}
