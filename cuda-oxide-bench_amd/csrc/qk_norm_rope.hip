// RMS norm of every query and key head and the position rotation, in one pass, for gfx950.
//
// For head x of token t, with weights w of its kind and position p = positions[t]:
//     y = x * rsqrt(mean(x^2) + eps) * w
//     (y_a, y_b) <- (y_a cos - y_b sin, y_b cos + y_a sin)   for each pair i < rot / 2
// with cos = table[p][i], sin = table[p][rot / 2 + i]; the pairs are (i, i + rot / 2) or the
// neighbours (2 i, 2 i + 1), channels from rot on are not turned.  All of it in fp32, rounded once.
//
// Memory bounds it: each head is read and written once.  A lane holds 8 channels (one 128-bit
// load and store), LPH lanes a head, 64 / LPH heads a wave at a time.  A wave stays with its
// token, whose cosines and sines it keeps in registers, and with halves as pairs a lane gets the
// other half's channels from the lane that loaded them.  Stores pass the caches (16384 tokens of 40 heads of 128
// 60.3 us, 5.7 TB/s; with cached ones 68.4, 1024 tokens 7.5 and not 6.5.  The append and the attention behind it read the
// outputs at once, and the three together take as long either way: 1024 tokens 54.8 us and 55.6 with cached stores, 4096
// 117.3 and 114.6, 16384 422 and 420).
#include <algorithm>

#include "mx_common.h"

namespace mx {
namespace rope {

constexpr int NT = 256;
constexpr int U = 5;  // groups of heads that a wave has under way together

// Heads whose mean square with eps is below kSmall are normed kUp times as large, eps with them: the squares of either
// type's least values (2^-133, 2^-24) then are normal numbers, those of the largest of such heads below 2^117.  (The look
// at each group of heads costs 0.5% where memory bounds: 16384 tokens 51.4 and 51.6 us in a graph.)
constexpr float kSmall = 0x1p-100f, kUp = 0x1p100f;

struct Args {
  const uint16_t *q, *k, *wq, *wk;
  const float* table;
  const int* positions;
  uint16_t *qo, *ko;
  int T, n_q, n_kv, d, rot, rows, q_stride, k_stride, qo_stride, ko_stride;
  int parts, per;  // a token's groups of heads go to `parts` waves, `per` to each
  float eps;
};

template <typename T>
__device__ __forceinline__ void widen(const u32x4& v, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = T::to_f32(v[i] & 0xffffu);
    x[2 * i + 1] = T::to_f32(v[i] >> 16);
  }
}

template <typename T, int LPH, bool NEIGHBOURS>
__global__ __launch_bounds__(NT) void rope_kernel(const Args a) {
  constexpr int HPW = 64 / LPH;  // heads of a wave at a time
  const int lane = threadIdx.x & 63, c = lane % LPH, sub = lane / LPH;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const bool there = c < a.d / 8;  // heads of other than 8 LPH channels leave lanes idle
  const int gq = (a.n_q + HPW - 1) / HPW, groups = gq + (a.n_kv + HPW - 1) / HPW;
  const int rc = a.rot / 16;  // lanes of half the turned channels
  const bool turned = c < 2 * rc;
  const int partner = turned && !NEIGHBOURS ? (c < rc ? lane + rc : lane - rc) : lane;
  const int pairs = NEIGHBOURS ? 4 * c : c < rc ? 8 * c : 8 * (c - rc);  // the lane's first pair
  const float inv_d = 1.0f / (float)a.d;

  float w[2][8];
  {
    const u32x4 none{};
    widen<T>(there ? ld128(a.wq + 8 * c) : none, w[0]);
    widen<T>(there ? ld128(a.wk + 8 * c) : none, w[1]);
  }

  const uint32_t items = (uint32_t)a.T * (uint32_t)a.parts, step = gridDim.x * (NT / 64);  // below 2^31, 2^22
  for (uint32_t item = blockIdx.x * (NT / 64) + wave; item < items; item += step) {
    const int t = (int)(item / (uint32_t)a.parts), part = (int)(item % (uint32_t)a.parts);
    const int pos = a.positions[t];
    if ((uint32_t)pos >= (uint32_t)a.rows) continue;  // no row of the table: left as it is
    constexpr int N = NEIGHBOURS ? 4 : 8;
    float cs[N], sn[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
      cs[j] = 1.f;
      sn[j] = 0.f;
    }
    if (turned) {
      const float* row = a.table + (size_t)pos * a.rot + pairs;
#pragma unroll
      for (int j = 0; j < N; j += 4) {
        const f32x4 x = *reinterpret_cast<const f32x4*>(row + j), y = *reinterpret_cast<const f32x4*>(row + a.rot / 2 + j);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          cs[j + i] = x[i];
          sn[j + i] = !NEIGHBOURS && c < rc ? -y[i] : y[i];
        }
      }
    }
    const int last = min((part + 1) * a.per, groups);
    for (int g0 = part * a.per; g0 < last; g0 += U) {
      u32x4 raw[U];
      uint16_t* to[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const bool key = g0 + u >= gq;
        const int head = (g0 + u - (key ? gq : 0)) * HPW + sub;
        const bool live = there && g0 + u < last && head < (key ? a.n_kv : a.n_q);
        const uint16_t* from = key ? a.k + (size_t)t * a.k_stride : a.q + (size_t)t * a.q_stride;
        uint16_t* out = key ? a.ko + (size_t)t * a.ko_stride : a.qo + (size_t)t * a.qo_stride;
        to[u] = live ? out + head * a.d + 8 * c : nullptr;
        raw[u] = live ? ld128(from + head * a.d + 8 * c) : u32x4{};
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (g0 + u >= last) break;
        const bool key = g0 + u >= gq;
        float x[8], sum = 0.f;
        widen<T>(raw[u], x);
#pragma unroll
        for (int j = 0; j < 8; ++j) sum = __builtin_fmaf(x[j], x[j], sum);
#pragma unroll
        for (int off = 1; off < LPH; off <<= 1) sum += __shfl_xor(sum, off, 64);
        const float mean = __builtin_fmaf(sum, inv_d, a.eps);
        float r = __builtin_amdgcn_rsqf(mean);
        if (__builtin_expect(__any(mean < kSmall), 0)) {  // (the root takes no subnormal numbers, and the squares may have lost theirs)
          float big = 0.f;
#pragma unroll
          for (int j = 0; j < 8; ++j) big = __builtin_fmaf(x[j] * kUp, x[j] * kUp, big);
#pragma unroll
          for (int off = 1; off < LPH; off <<= 1) big += __shfl_xor(big, off, 64);
          const float up = mean < kSmall ? kUp : 1.f;
          if (mean < kSmall) r = __builtin_amdgcn_rsqf(__builtin_fmaf(big, inv_d, a.eps * kUp * kUp));
#pragma unroll
          for (int j = 0; j < 8; ++j) x[j] *= up;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] *= r * (key ? w[1][j] : w[0][j]);
        float y[8];
        if constexpr (NEIGHBOURS) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            y[2 * j] = x[2 * j] * cs[j] - x[2 * j + 1] * sn[j];
            y[2 * j + 1] = x[2 * j + 1] * cs[j] + x[2 * j] * sn[j];
          }
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float other = __shfl(x[j], partner, 64);
            y[j] = turned ? x[j] * cs[j] + other * sn[j] : x[j];
          }
        }
        if (to[u])
          st128_nt(to[u], u32x4{T::pack2(y[0], y[1]), T::pack2(y[2], y[3]), T::pack2(y[4], y[5]), T::pack2(y[6], y[7])});
      }
    }
  }
}

// Whether rows of `an` elements at a, as apart, meet those of `bn` elements at b, bs apart (T rows each, 2 bytes
// an element).  The same rows are no meeting: a head is read whole before it is written.
static bool meets(const void* a, long long an, long long as, const void* b, long long bn, long long bs, long long T) {
  const long long x = (long long)(uintptr_t)a / 2, y = (long long)(uintptr_t)b / 2;
  if (x + (T - 1) * as + an <= y || y + (T - 1) * bs + bn <= x) return false;
  if (T == 1) return true;
  if (as != bs) return true;  // rows of two strides in one range: taken to meet
  const long long off = ((y - x) % as + as) % as;  // rows of one stride, one beside the other
  return off < an || off + bn > as;
}

template <typename T, int LPH>
static int launch(Args a, int neighbours, hipStream_t s) {
  constexpr int HPW = 64 / LPH;
  const int groups = (a.n_q + HPW - 1) / HPW + (a.n_kv + HPW - 1) / HPW;
  // few tokens: their heads side by side, for 4096 waves; many: a wave's groups all under way at once (16384 tokens of 10
  // groups: 59.2 us with 5 to a wave, 63.9 with all of them in turn, 61.6 with 4)
  const long long want = (4096 + a.T - 1) / a.T;
  a.per = (int)std::min<long long>((groups + want - 1) / want, U);
  a.parts = (groups + a.per - 1) / a.per;
  a.per = (groups + a.parts - 1) / a.parts;
  const long long waves = (long long)a.T * a.parts, blocks = (waves + NT / 64 - 1) / (NT / 64);
  const dim3 grid((unsigned)(blocks < (1 << 20) ? blocks : 1 << 20));
  if (neighbours)
    hipLaunchKernelGGL((rope_kernel<T, LPH, true>), grid, dim3(NT), 0, s, a);
  else
    hipLaunchKernelGGL((rope_kernel<T, LPH, false>), grid, dim3(NT), 0, s, a);
  MX_RETURN_IF_HIP(hipGetLastError());
  return MX_OK;
}

template <typename T>
static int run(const Args& a, int neighbours, hipStream_t s) {
  return a.d <= 64    ? launch<T, 8>(a, neighbours, s)
         : a.d <= 128 ? launch<T, 16>(a, neighbours, s)
                      : launch<T, 32>(a, neighbours, s);
}

}  // namespace rope
}  // namespace mx

extern "C" int mx_qk_norm_rope(const void* q, const void* k, const void* q_weight, const void* k_weight,
                               const float* table, const int* positions, void* q_out, void* k_out, int T, int n_q,
                               int n_kv, int d, int rot, int rows, int q_stride, int k_stride, int qo_stride,
                               int ko_stride, float eps, int neighbours, int dtype, void* stream) {
  using namespace mx::rope;
  if (!q || !k || !q_weight || !k_weight || !table || !positions || !q_out || !k_out) return MX_ERR_NULL;
  if (T <= 0 || n_q <= 0 || n_kv <= 0 || rows <= 0 || d < 16 || d > 256 || d % 16 || rot < 16 || rot > d || rot % 16)
    return MX_ERR_SHAPE;
  const long long nq = (long long)n_q * d, nk = (long long)n_kv * d;
  if ((long long)T * ((long long)n_q + n_kv) > 0x7fffffffLL) return MX_ERR_SHAPE;
  if (nq > 0x7fffffffLL || nk > 0x7fffffffLL || q_stride < nq || qo_stride < nq || k_stride < nk || ko_stride < nk)
    return MX_ERR_SHAPE;
  if ((q_stride | k_stride | qo_stride | ko_stride) % 8) return MX_ERR_ALIGN;
  if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)q_weight | (uintptr_t)k_weight | (uintptr_t)table | (uintptr_t)q_out |
       (uintptr_t)k_out) & 15)
    return MX_ERR_ALIGN;
  if ((uintptr_t)positions & 3) return MX_ERR_ALIGN;
  if (dtype != MX_DTYPE_BF16 && dtype != MX_DTYPE_F16) return MX_ERR_DTYPE;
  const bool same_q = q_out == q && qo_stride == q_stride, same_k = k_out == k && ko_stride == k_stride;
  if ((!same_q && meets(q_out, nq, qo_stride, q, nq, q_stride, T)) || meets(q_out, nq, qo_stride, k, nk, k_stride, T) ||
      (!same_k && meets(k_out, nk, ko_stride, k, nk, k_stride, T)) || meets(k_out, nk, ko_stride, q, nq, q_stride, T) ||
      meets(q_out, nq, qo_stride, k_out, nk, ko_stride, T))
    return MX_ERR_ALIAS;
  const Args a{(const uint16_t*)q, (const uint16_t*)k, (const uint16_t*)q_weight, (const uint16_t*)k_weight, table,
               positions, (uint16_t*)q_out, (uint16_t*)k_out, T, n_q, n_kv, d, rot, rows, q_stride, k_stride, qo_stride,
               ko_stride, 0, 0, eps};
  if (dtype == MX_DTYPE_BF16) return run<mx::BF16>(a, neighbours, (hipStream_t)stream);
  return run<mx::F16>(a, neighbours, (hipStream_t)stream);
}
