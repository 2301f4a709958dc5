// The paged 8-bit cache: new keys and values quantised into it, pages copied.
//
// A page of a head has one scale for K and one for V, a power of two s, and holds
// e4m3 codes with value = code * s.  When new tokens reach a page, with a = their
// largest finite magnitude,
//     s = max(s_old, 2^ceil(log2(a / 448)), 2^-32)   (s_old only if the page holds
//                                                    tokens before them)
//     kept codes = e4m3(code * s_old / s),   new codes = e4m3(x / s)
// Both quotients are by powers of two, so they are exact in fp32 and each code is
// rounded once, to nearest even.  e4m3 has 18 binades: a scale between two
// powers of two would place the largest value better in its last binade, and
// lose or gain nothing else.
#include "kv8_common.h"

namespace mx {
namespace kv8 {

constexpr float kLeast = 0x1p-32f;

// 2^ceil(log2(a / 448)) for the magnitude bits of a finite bf16 / f16: 448 = 1.75 * 2^8.
template <typename T>
__device__ __forceinline__ float scale_for(uint32_t magnitude) {
  const uint32_t b = __float_as_uint(T::to_f32(magnitude));
  const int e = (int)(b >> 23) - 127 - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);  // 1.75 = 1 + 0x600000 / 2^23
  return fmaxf(__uint_as_float((uint32_t)(max(e, -32) + 127) << 23), kLeast);
}

template <typename T>
__device__ __forceinline__ constexpr uint32_t first_nonfinite() {
  return std::is_same<T, BF16>::value ? 0x7f80u : 0x7c00u;
}

// Two codes of finite values or NaN (|x| <= 448).
__device__ __forceinline__ uint32_t codes2(float a, float b) {
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false) & 0xffffu;
}

// Four codes of packed values x, y of the 16-bit type, divided by s = a power of two: one
// instruction for two (all finite values of both types at scales from 2^-32 to 2^127 give
// the codes of the exact quotient).
template <typename T>
__device__ __forceinline__ uint32_t codes4(uint32_t x, uint32_t y, float s);
typedef short i16x2_t __attribute__((ext_vector_type(2)));
template <>
__device__ __forceinline__ uint32_t codes4<BF16>(uint32_t x, uint32_t y, float s) {
  const i16x2_t lo = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(i16x2_t{}, __builtin_bit_cast(bf16x2_t, x), s, false);
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(lo, __builtin_bit_cast(bf16x2_t, y), s, true));
}
template <>
__device__ __forceinline__ uint32_t codes4<F16>(uint32_t x, uint32_t y, float s) {
  const i16x2_t lo = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(i16x2_t{}, __builtin_bit_cast(f16x2_t, x), s, false);
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(lo, __builtin_bit_cast(f16x2_t, y), s, true));
}
// The same for any values and any scale: infinities and NaN become NaN.
template <typename T>
__device__ uint32_t codes4_any(uint32_t x, uint32_t y, float r) {
  float v[4] = {T::to_f32(x & 0xffffu) * r, T::to_f32(x >> 16) * r, T::to_f32(y & 0xffffu) * r, T::to_f32(y >> 16) * r};
  const uint32_t bits[4] = {x & 0x7fffu, (x >> 16) & 0x7fffu, y & 0x7fffu, (y >> 16) & 0x7fffu};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (bits[i] >= first_nonfinite<T>()) v[i] = __builtin_nanf("");
  return codes2(v[0], v[1]) | codes2(v[2], v[3]) << 16;
}

// max of the two 16-bit halves, each as an unsigned integer
__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
  typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
}
// The magnitudes of x's halves, 0 for one that is not finite.
template <typename T>
__device__ __forceinline__ uint32_t finite_magnitudes(uint32_t x) {
  const uint32_t lo = x & 0x7fffu, hi = (x >> 16) & 0x7fffu;
  return (lo < first_nonfinite<T>() ? lo : 0u) | (hi < first_nonfinite<T>() ? hi << 16 : 0u);
}

// One code at another scale; NaN stays the NaN that it is.
__device__ __forceinline__ uint8_t moved(uint8_t code, float ratio) {
  if ((code & 0x7f) == 0x7f) return code;
  return (uint8_t)codes2(__builtin_amdgcn_cvt_f32_fp8(code, 0) * ratio, 0.f);
}

// Rows i of four words become columns: out[c] holds byte c of w[0] .. w[3].
__device__ __forceinline__ void transpose4(const uint32_t (&w)[4], uint32_t (&out)[4]) {
  const uint32_t a = __builtin_amdgcn_perm(w[1], w[0], 0x05010400u), b = __builtin_amdgcn_perm(w[3], w[2], 0x05010400u);
  const uint32_t c = __builtin_amdgcn_perm(w[1], w[0], 0x07030602u), d = __builtin_amdgcn_perm(w[3], w[2], 0x07030602u);
  out[0] = __builtin_amdgcn_perm(b, a, 0x05040100u);
  out[1] = __builtin_amdgcn_perm(b, a, 0x07060302u);
  out[2] = __builtin_amdgcn_perm(d, c, 0x05040100u);
  out[3] = __builtin_amdgcn_perm(d, c, 0x07060302u);
}

// One workgroup per (page that new tokens reach, head): it reads them once, 4 tokens
// by 8 channels a thread, and keeps them in registers from the maximum to the
// codes.  K's codes go out 8 bytes a token; V's pass through LDS, 4 tokens
// packed in a dword, so that its transposed rows are written 16 bytes (16
// tokens) at a time where they are all new.
template <typename T, int D, int LP>
__global__ __launch_bounds__(256) void append_kernel(const uint16_t* __restrict__ knew, const uint16_t* __restrict__ vnew,
                                                     uint8_t* __restrict__ kc, uint8_t* __restrict__ vc,
                                                     float* __restrict__ ks, float* __restrict__ vs,
                                                     const int* __restrict__ table, const int* __restrict__ lens,
                                                     const int* __restrict__ cu, int n_kv, int T_, int pages,
                                                     int max_pages, int k_stride, int v_stride) {
  constexpr int P = 1 << LP;
  constexpr int UNITS = P * D / 32;  // 4 tokens x 8 channels
  constexpr int NT = UNITS < 64 ? 64 : UNITS < 256 ? UNITS : 256;
  constexpr int U = (UNITS + NT - 1) / NT;
  constexpr int VROW = P + 4;  // bytes of a V row in LDS
  __shared__ __align__(16) uint8_t vt[D * VROW];
  __shared__ uint32_t red[2][NT / 64];

  const int t = threadIdx.x;
  const int h = blockIdx.x % n_kv, b = blockIdx.x / n_kv;
  const int len = cut_len(lens[b], max_pages, LP);
  const Rows rows = rows_of(cu, b, T_);
  const int n = rows.last - rows.first;
  if (n == 0) return;
  const int start = len - n;  // position of the first new token; below 0 where there are more rows than tokens
  const int j_end = (len - 1) >> LP;
  for (int j = (max(start, 0) >> LP) + blockIdx.y; j <= j_end; j += gridDim.y) {
    const int lo = max(start - (j << LP), 0), hi = min(len - (j << LP), P);  // the new tokens' slots
    const int row0 = rows.first + (j << LP) - start;                       // the row of slot 0

    u32x4 x[2][U][4];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int unit = t + u * NT, s0 = unit / (D / 8) * 4, c0 = unit % (D / 8) * 8;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[0][u][i] = x[1][u][i] = u32x4{};
        if (unit < UNITS && s0 + i >= lo && s0 + i < hi) {
          x[0][u][i] = ld128(knew + (size_t)(row0 + s0 + i) * k_stride + h * D + c0);
          x[1][u][i] = ld128(vnew + (size_t)(row0 + s0 + i) * v_stride + h * D + c0);
        }
      }
    }
    const int page = page_of(table + (size_t)b * max_pages, j << LP, LP, max_pages, pages);
    if (page < 0) continue;
    const size_t at = (size_t)page * n_kv + h;
    const float was[2] = {lo > 0 ? ks[at] : 0.f, lo > 0 ? vs[at] : 0.f};  // no tokens before: a scale of any size

    // the largest magnitudes, an infinity or NaN the largest of all
    uint32_t mx[2] = {0, 0};
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int w = 0; w < 4; ++w) mx[kv] = max_u16x2(mx[kv], x[kv][u][i][w] & 0x7fff7fffu);
    }
    auto meet = [&] {  // the maxima of all threads
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        mx[kv] = max(mx[kv] & 0xffffu, mx[kv] >> 16);
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) mx[kv] = max(mx[kv], (uint32_t)__shfl_xor((int)mx[kv], off, 64));
        if ((t & 63) == 0) red[kv][t >> 6] = mx[kv];
      }
      __syncthreads();  // also: every thread has read the page's scales
#pragma unroll
      for (int kv = 0; kv < 2; ++kv)
#pragma unroll
        for (int w = 0; w < NT / 64; ++w) mx[kv] = max(mx[kv], red[kv][w]);
    };
    meet();
    const bool finite = max(mx[0], mx[1]) < first_nonfinite<T>();
    if (!finite) {
      mx[0] = mx[1] = 0;
#pragma unroll
      for (int kv = 0; kv < 2; ++kv)
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int w = 0; w < 4; ++w) mx[kv] = max_u16x2(mx[kv], finite_magnitudes<T>(x[kv][u][i][w]));
      __syncthreads();  // red has been read
      meet();
    }
    float now[2];
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      now[kv] = scale_for<T>(mx[kv]);
      if (lo > 0) now[kv] = fmaxf(now[kv], was[kv]);
    }
    if (t == 0) {
      ks[at] = now[0];
      vs[at] = now[1];
    }
    uint8_t* kp = kc + at * (P * D);
    uint8_t* vp = vc + at * (P * D);

    // codes before the new ones, where the scale grew, a byte a thread (single tokens of 64 sequences, 8 heads,
    // pages of 64 tokens: 25 us where every scale grows, 6 where none does)
    if (lo > 0 && now[0] != was[0]) {
      const float ratio = was[0] / now[0];
      for (int i = t; i < lo * D; i += NT) kp[i] = moved(kp[i], ratio);
    }
    if (lo > 0 && now[1] != was[1]) {
      const float ratio = was[1] / now[1];
      for (int i = t; i < lo * D; i += NT) {
        uint8_t* p = vp + (size_t)(i % D) * P + i / D;
        *p = moved(*p, ratio);
      }
    }

    const bool plain = finite && ((__float_as_uint(now[0]) | __float_as_uint(now[1])) & 0x7fffffu) == 0;  // powers of two
    const float r[2] = {1.0f / now[0], 1.0f / now[1]};
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int unit = t + u * NT, s0 = unit / (D / 8) * 4, c0 = unit % (D / 8) * 8;
      if (unit >= UNITS || s0 >= hi || s0 + 4 <= lo) continue;
      uint32_t code[2][2][4];  // [K, V][4 channels][token]
#pragma unroll
      for (int kv = 0; kv < 2; ++kv)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            const u32x4& v = x[kv][u][i];
            code[kv][w][i] = plain ? codes4<T>(v[2 * w], v[2 * w + 1], now[kv]) : codes4_any<T>(v[2 * w], v[2 * w + 1], r[kv]);
          }
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (s0 + i >= lo && s0 + i < hi) st64(kp + (s0 + i) * D + c0, u32x2{code[0][0][i], code[0][1][i]});
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        uint32_t four[4];
        transpose4(code[1][w], four);
#pragma unroll
        for (int c = 0; c < 4; ++c) *reinterpret_cast<uint32_t*>(vt + (c0 + 4 * w + c) * VROW + s0) = four[c];
      }
    }
    __syncthreads();
    for (int i = t; i < D * (P / 16); i += NT) {
      const int c = i / (P / 16), s0 = i % (P / 16) * 16;
      if (s0 >= hi || s0 + 16 <= lo) continue;
      const uint32_t* src = reinterpret_cast<const uint32_t*>(vt + c * VROW + s0);
      uint8_t* dst = vp + c * P + s0;
      if (s0 >= lo && s0 + 16 <= hi) {
        st128(dst, u32x4{src[0], src[1], src[2], src[3]});
      } else {
        for (int k = max(lo - s0, 0); k < min(hi - s0, 16); ++k) dst[k] = (uint8_t)(src[k >> 2] >> (8 * (k & 3)));
      }
    }
    __syncthreads();  // vt and red serve the next page
  }
}

// Pairs of pages: PIECE bytes of a page's K or V codes per workgroup, 16 bytes a thread; the
// first of a page's workgroups takes the scales too.  Stores past the caches, and one
// load a thread: 2500 pages of 128 KB move in 113 us (5.8 TB/s); with cached stores
// 123, with 4 loads a thread 119, with both 136.
constexpr int COPY_NT = 256, PIECE = COPY_NT * 16;
__global__ __launch_bounds__(COPY_NT) void copy_kernel(uint8_t* kc, uint8_t* vc, float* ks, float* vs,
                                                       const int* __restrict__ src, const int* __restrict__ dst,
                                                       int n_kv, uint32_t bytes, int pieces, int pages) {
  const int i = blockIdx.x / (2 * pieces), part = blockIdx.x % (2 * pieces);
  const int from = src[i], to = dst[i];
  if (from < 0 || from >= pages || to < 0 || to >= pages || from == to) return;
  const bool v = part >= pieces;
  const uint32_t at = (uint32_t)(v ? part - pieces : part) * PIECE + threadIdx.x * 16;
  uint8_t* codes = v ? vc : kc;
  if (at < bytes) st128_nt(codes + (size_t)to * bytes + at, ld128(codes + (size_t)from * bytes + at));
  if (part == 0)
    for (int h = threadIdx.x; h < n_kv; h += COPY_NT) {
      ks[(size_t)to * n_kv + h] = ks[(size_t)from * n_kv + h];
      vs[(size_t)to * n_kv + h] = vs[(size_t)from * n_kv + h];
    }
}

template <typename T, int D, int LP>
static int launch_append(const void* k, const void* v, void* kc, void* vc, float* ks, float* vs, const int* table,
                         const int* lens, const int* cu, int B, int T_, int reach, int n_kv, int pages, int max_pages,
                         int k_stride, int v_stride, hipStream_t s) {
  constexpr int UNITS = (D << LP) / 32;
  constexpr int NT = UNITS < 64 ? 64 : UNITS < 256 ? UNITS : 256;
  hipLaunchKernelGGL((append_kernel<T, D, LP>), dim3((unsigned)(B * n_kv), (unsigned)reach), dim3(NT), 0, s,
                     (const uint16_t*)k, (const uint16_t*)v, (uint8_t*)kc, (uint8_t*)vc, ks, vs, table, lens, cu, n_kv,
                     T_, pages, max_pages, k_stride, v_stride);
  MX_RETURN_IF_HIP(hipGetLastError());
  return MX_OK;
}

}  // namespace kv8
}  // namespace mx

extern "C" int mx_kv8_append(const void* k, const void* v, void* k_cache, void* v_cache, float* k_scale, float* v_scale,
                             const int* page_table, const int* kv_lens, const int* cu, int B, int T, int max_q, int n_kv,
                             int d, int page, int pages, int max_pages, int k_stride, int v_stride, int dtype,
                             void* stream) {
  using namespace mx::kv8;
  if (!k || !v || !page_table || !kv_lens) return MX_ERR_NULL;
  const int rc = check_cache(k_cache, v_cache, k_scale, v_scale, n_kv, d, page, pages);
  if (rc != MX_OK) return rc;
  if (B <= 0 || T <= 0 || max_q <= 0 || (!cu && T != B)) return MX_ERR_SHAPE;
  if (max_pages <= 0 || (long long)max_pages * page > kMostTokens) return MX_ERR_SHAPE;
  if ((long long)B * n_kv > (1 << 22)) return MX_ERR_SHAPE;  // fewer than 2^32 threads in x
  if (k_stride < (long long)n_kv * d || v_stride < (long long)n_kv * d) return MX_ERR_SHAPE;
  if (k_stride % 8 || v_stride % 8 || (((uintptr_t)k | (uintptr_t)v) & 15)) return MX_ERR_ALIGN;
  if (dtype != MX_DTYPE_BF16 && dtype != MX_DTYPE_F16) return MX_ERR_DTYPE;
  const int lp = log2_page(page);
  // pages that max_q consecutive tokens can reach
  const long long most = ((long long)(max_q < T ? max_q : T) + page - 2) / page + 1;
  const int reach = (int)(most < 65535 ? most : 65535);
  hipStream_t s = (hipStream_t)stream;
#define KV8_APPEND(TT, DD, LL)                                                                                      \
  launch_append<TT, DD, LL>(k, v, k_cache, v_cache, k_scale, v_scale, page_table, kv_lens, cu, B, T, reach, n_kv, pages, \
                            max_pages, k_stride, v_stride, s)
#define KV8_APPEND_P(TT, DD) \
  (lp == 4 ? KV8_APPEND(TT, DD, 4) : lp == 5 ? KV8_APPEND(TT, DD, 5) : lp == 6 ? KV8_APPEND(TT, DD, 6) : KV8_APPEND(TT, DD, 7))
  if (dtype == MX_DTYPE_BF16) return d == 64 ? KV8_APPEND_P(mx::BF16, 64) : KV8_APPEND_P(mx::BF16, 128);
  return d == 64 ? KV8_APPEND_P(mx::F16, 64) : KV8_APPEND_P(mx::F16, 128);
}

extern "C" int mx_kv8_copy_pages(void* k_cache, void* v_cache, float* k_scale, float* v_scale, const int* src,
                                 const int* dst, int n, int n_kv, int d, int page, int pages, void* stream) {
  using namespace mx::kv8;
  const int rc = check_cache(k_cache, v_cache, k_scale, v_scale, n_kv, d, page, pages);
  if (rc != MX_OK) return rc;
  if (!src || !dst) return MX_ERR_NULL;
  if (n <= 0) return MX_ERR_SHAPE;
  const long long bytes = (long long)n_kv * page * d;
  const long long pieces = (bytes + PIECE - 1) / PIECE;
  if (bytes > 0x7fffffffLL || 2 * pieces * n > (1 << 23)) return MX_ERR_SHAPE;  // fewer than 2^32 threads
  hipLaunchKernelGGL(copy_kernel, dim3((unsigned)(2 * pieces * n)), dim3(COPY_NT), 0, (hipStream_t)stream,
                     (uint8_t*)k_cache, (uint8_t*)v_cache, k_scale, v_scale, src, dst, n_kv, (uint32_t)bytes, (int)pieces,
                     pages);
  MX_RETURN_IF_HIP(hipGetLastError());
  return MX_OK;
}
