// Grouped-query attention over the paged 8-bit cache, for gfx950.
//
//   O[i,h] = softmax_t(scale * q[i,h] . K[t]) . V[t],   K[t] = k8[t] ks, V[t] = v8[t] vs,
// the scales ks, vs those of t's page and head.  The codes go through the 16-bit
// MFMAs (e4m3 -> bf16 / f16 is exact), the scales around them:
//     y[t]  = scale log2(e) ks (q . k8[t]) + log2(vs)
//     P'[t] = 2^(y[t] - m),   m = the running maximum of y
//     O     = (sum_t P'[t] v8[t]) / (sum_t P'[t] / vs)
// so a page's two scales cost one FMA constant per score and one product per page in
// the denominator, P' carries vs and stays within 0..1 in either 16-bit type, and any positive
// scales serve.  (m - max y of a page is at most the spread of log2 vs, so the
// denominator's terms stay in fp32's range while the vs of a sequence lie within 2^100.)
//
// S^T = K . Q^T and O^T = V^T . P'^T: a lane of the score tile holds one query and its
// keys, which is the layout that the second product takes P' in.
#include <algorithm>

#include "kv8_common.h"

namespace mx {
namespace kv8 {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNoScore = -3.0e38f;  // m of a partial whose visible keys all score -inf

struct Args {
  const uint16_t* q;
  const uint8_t *kc, *vc;
  const float *ks, *vs;
  const int *table, *lens, *cu;
  uint16_t* out;
  float* part;  // [splits][T * Hq][D] unnormalised, then [splits][T * Hq][2]: m and the denominator
  int B, T, n_q, n_kv, pages, max_pages, q_stride, lp, causal, splits, chunk;
  float c;  // scale * log2(e)
};

// Two codes (byte pair HI of x) as packed bf16 / f16.
template <typename T, bool HI>
__device__ __forceinline__ uint32_t widen2(uint32_t x);
template <>
__device__ __forceinline__ uint32_t widen2<BF16, false>(uint32_t x) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, 1.0f, false));
}
template <>
__device__ __forceinline__ uint32_t widen2<BF16, true>(uint32_t x) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, 1.0f, true));
}
template <>
__device__ __forceinline__ uint32_t widen2<F16, false>(uint32_t x) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, 1.0f, false));
}
template <>
__device__ __forceinline__ uint32_t widen2<F16, true>(uint32_t x) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, 1.0f, true));
}
template <typename T>
__device__ __forceinline__ u32x4 widen8(uint32_t a, uint32_t b) {
  return u32x4{widen2<T, false>(a), widen2<T, true>(a), widen2<T, false>(b), widen2<T, true>(b)};
}

template <typename T>
__device__ __forceinline__ constexpr uint32_t one_bits() {
  return std::is_same<T, BF16>::value ? 0x3f80u : 0x3c00u;
}

// A dword with 0x80 in each byte of x that is a NaN code.
__device__ __forceinline__ uint32_t nan_bytes(uint32_t x) { return ((x & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }
// 0xff for each byte of a nan_bytes() dword that is set.
__device__ __forceinline__ uint32_t spread(uint32_t m) { return (m >> 7) * 0xffu; }

// ---------------------------------------------------------------------------
// Few rows per sequence (decode, a few speculated tokens): the cache is read once
// from HBM into registers.  A workgroup takes one KV head of a sequence and one
// chunk of its tokens; its waves take 64-key tiles in turn and meet in LDS.
//
// 16x16x32 MFMAs on 16 NR rows (row = token * G + head of the group).  Row r of
// score subtile t is key 16 (r / 4) + 4 t + r % 4 of the tile: lane group g = lane / 16
// then owns keys 16 g .. 16 g + 15, which are 16 consecutive bytes of V's transposed
// page, one load per 16 channels.  Pages of 16 tokens and more never split
// them, so a lane has one page, one ks and one vs per tile whatever the page.
// K's rows are read 32 bytes a lane at d = 128 (16 at 64), the contraction's order
// of channels permuted alike in Q.
// ---------------------------------------------------------------------------
constexpr int NW = 4;  // waves of a workgroup

template <typename T, int D, int NR>
__global__ __launch_bounds__(64 * NW, NR == 1 ? 2 : 1) void rows_kernel(const Args a) {
  constexpr int KC = D / 32;   // contraction steps
  constexpr int KL = D / 64;   // 16-byte loads of a K row per lane
  constexpr int DT = D / 16;   // output fragments
  extern __shared__ __align__(16) unsigned char smem[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r16 = lane & 15, g = lane >> 4;
  const int G = a.n_q / a.n_kv;
  const int h = blockIdx.x % a.n_kv, b = blockIdx.x / a.n_kv;
  const int split = blockIdx.y;
  const int P = 1 << a.lp;

  const Rows rw = rows_of(a.cu, b, a.T);
  const int n = rw.last - rw.first;
  if (n == 0) return;
  const int len = cut_len(a.lens[b], a.max_pages, a.lp);
  const int t0 = min((long long)split * a.chunk, (long long)len);
  const int t1 = split + 1 == a.splits ? len : min(len, t0 + a.chunk);
  const int* row_pages = a.table + (size_t)b * a.max_pages;
  const int tiles = (t1 - t0 + 63) / 64;
  const float c = fabsf(a.c);
  const uint32_t flip = a.c < 0.f ? 0x80008000u : 0u;  // a negative scale turns q, so that larger scores stay larger

  for (int r0 = 0; r0 < n * G; r0 += 16 * NR) {
    // ---- this block's rows ----
    u32x4 qf[NR][KC];
    int limit[NR];  // keys that the lane's row sees: t < limit
    int low = len;  // ... that every row of the block sees
#pragma unroll
    for (int i = 0; i < NR; ++i) {
      const int r = min(r0 + 16 * i + r16, n * G - 1);
      const int tok = r / G;
      const uint16_t* src = a.q + (size_t)(rw.first + tok) * a.q_stride + (h * G + r % G) * D + g * (D / 4);
#pragma unroll
      for (int k = 0; k < KC; ++k) qf[i][k] = ld128(src + 8 * k) ^ u32x4{flip, flip, flip, flip};
      limit[i] = a.causal ? max(len - n + tok + 1, 0) : len;
    }
    if (a.causal) low = max(len - n + r0 / G + 1, 0);

    f32x4 acc[NR][DT];
    float m[NR], l[NR];
    bool seen[NR];
#pragma unroll
    for (int i = 0; i < NR; ++i) {
      m[i] = -INFINITY;
      l[i] = 0.f;
      seen[i] = false;
#pragma unroll
      for (int d = 0; d < DT; ++d) acc[i][d] = f32x4{};
    }

    // ---- a tile's pages: of the lane's K rows and of its V keys ----
    struct Ids {
      int k, v;
    };
    auto ids_of = [&](int tile) {
      const int at = t0 + 64 * tile;
      const bool in = tile < tiles;
      return Ids{in ? page_of(row_pages, at + 16 * (r16 >> 2), a.lp, a.max_pages, a.pages) : -1,
                 in ? page_of(row_pages, at + 16 * g, a.lp, a.max_pages, a.pages) : -1};
    };
    u32x4 kx[4][KL], vx[DT];
    float ks = 1.f, vs = 1.f;
    auto load_k = [&](int tile, Ids id) {
      const int at = t0 + 64 * tile + 16 * (r16 >> 2) + (r16 & 3);
      const size_t page = (size_t)max(id.k, 0) * a.n_kv + h;  // a page that is none reads page 0 and is masked
      const uint8_t* p = a.kc + page * (size_t)(D * P) + (size_t)(at & (P - 1)) * D + g * (D / 4);
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int u = 0; u < KL; ++u) kx[t][u] = ld128(p + 4 * t * D + 16 * u);
      ks = a.ks[(size_t)max(id.v, 0) * a.n_kv + h];
    };
    auto load_v = [&](int tile, Ids id) {
      const int at = t0 + 64 * tile + 16 * g;
      const size_t page = (size_t)max(id.v, 0) * a.n_kv + h;
      const uint8_t* p = a.vc + page * (size_t)(D * P) + (size_t)r16 * P + (at & (P - 1));
#pragma unroll
      for (int d = 0; d < DT; ++d) vx[d] = ld128(p + (size_t)16 * d * P);
      vs = a.vs[page];
    };

    int tile = wave;
    Ids now = ids_of(tile), next = ids_of(tile + NW);
    if (tile < tiles) {
      load_k(tile, now);
      load_v(tile, now);
    }
    for (; tile < tiles; tile += NW) {
      const int key0 = t0 + 64 * tile + 16 * g;  // the lane's keys: key0 .. key0 + 15
      const bool bad = now.v < 0;
      const bool masked = t0 + 64 * tile + 64 > min(low, t1) || __any(bad);
      // ---- scores ----
      f32x4 s[NR][4];
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int k = 0; k < KC; ++k) {
          const u32x4 kf = widen8<T>(kx[t][k >> 1][2 * (k & 1)], kx[t][k >> 1][2 * (k & 1) + 1]);
#pragma unroll
          for (int i = 0; i < NR; ++i) s[i][t] = mfma16<T>(kf, qf[i][k], k ? s[i][t] : f32x4{});
        }
      const float cs = c * ks, lv = __builtin_amdgcn_logf(vs), iv = 1.0f / vs;
      const Ids after = ids_of(tile + 2 * NW);
      if (tile + NW < tiles) load_k(tile + NW, next);

      // ---- P' ----
      u32x4 pf[NR][2];
#pragma unroll
      for (int i = 0; i < NR; ++i) {
        float y[16];
        float mx = -INFINITY;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          y[e] = __builtin_fmaf(s[i][e >> 2][e & 3], cs, lv);
          if (masked) {
            const bool in = !bad && key0 + e < min(limit[i], t1);
            seen[i] |= in;
            y[e] = in ? y[e] : -INFINITY;
          }
          mx = fmaxf(mx, y[e]);
        }
        if (!masked) seen[i] = true;
        const float top = fmaxf(m[i], max_xor32(max_xor16(mx)));
        const float base = top == -INFINITY ? 0.f : top;
        const float corr = m[i] == top ? 1.f : __builtin_amdgcn_exp2f(m[i] - top);
        m[i] = top;
        float sum = 0.f;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          y[e] = __builtin_amdgcn_exp2f(y[e] - base);
          sum += y[e];
        }
        // masked keys of a page that is none have its vs of garbage
        l[i] = l[i] * corr + (bad ? 0.f : sum * iv);
#pragma unroll
        for (int d = 0; d < DT; ++d) acc[i][d] *= corr;
#pragma unroll
        for (int u = 0; u < 2; ++u)
          pf[i][u] = u32x4{T::pack2(y[8 * u], y[8 * u + 1]), T::pack2(y[8 * u + 2], y[8 * u + 3]),
                           T::pack2(y[8 * u + 4], y[8 * u + 5]), T::pack2(y[8 * u + 6], y[8 * u + 7])};
      }

      // ---- codes of V that a row does not see must not reach it: 0 * NaN ----
      if (masked) {
        uint32_t any_nan = 0;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int w = 0; w < 4; ++w) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (bad || key0 + 4 * w + j >= t1) vx[d][w] &= ~(0xffu << (8 * j));
            any_nan |= nan_bytes(vx[d][w]);
          }
        if (a.causal && __any(any_nan != 0)) {
          // some row may not see it: count, for every row and channel, the NaNs it does
          // see, and take them out of the product
#pragma unroll
          for (int i = 0; i < NR; ++i) {
            u32x4 vis[2];
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
              for (int w = 0; w < 4; ++w) {
                const int e = 8 * u + 2 * w;
                vis[u][w] = (key0 + e < limit[i] ? one_bits<T>() : 0u) | (key0 + e + 1 < limit[i] ? one_bits<T>() << 16 : 0u);
              }
#pragma unroll
            for (int d = 0; d < DT; ++d) {
              f32x4 cnt{};
#pragma unroll
              for (int u = 0; u < 2; ++u) {
                u32x4 x;
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                  const uint32_t two = nan_bytes(vx[d][2 * u + (w >> 1)]) >> (16 * (w & 1));
                  x[w] = ((two & 0x80u) ? one_bits<T>() : 0u) | ((two & 0x8000u) ? one_bits<T>() << 16 : 0u);
                }
                cnt = mfma16<T>(x, vis[u], cnt);
              }
#pragma unroll
              for (int j = 0; j < 4; ++j)
                if (cnt[j] > 0.f) acc[i][d][j] = __builtin_nanf("");
            }
          }
#pragma unroll
          for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int w = 0; w < 4; ++w) vx[d][w] &= ~spread(nan_bytes(vx[d][w]));
        }
      }

      // ---- O^T += V^T P'^T ----
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const u32x4 vf = widen8<T>(vx[d][2 * u], vx[d][2 * u + 1]);
#pragma unroll
          for (int i = 0; i < NR; ++i) acc[i][d] = mfma16<T>(vf, pf[i][u], acc[i][d]);
        }
      if (tile + NW < tiles) load_v(tile + NW, next);
      now = next;
      next = after;
    }

    // ---- the waves' states meet: m and the denominator, then the sums ----
    float* ml = reinterpret_cast<float*>(smem);                         // [NW][NR][16][2]
    f32x4* red = reinterpret_cast<f32x4*>(smem + NW * NR * 16 * 2 * 4);  // [NW][NR][DT][64]
#pragma unroll
    for (int i = 0; i < NR; ++i) {
      l[i] = sum_xor32(sum_xor16(l[i]));
      const bool met = __shfl_xor((int)seen[i], 16, 64) | __shfl_xor((int)seen[i], 32, 64) |
                       __shfl_xor((int)seen[i], 48, 64) | (int)seen[i];
      if (g == 0) {
        ml[((wave * NR + i) * 16 + r16) * 2] = met && m[i] == -INFINITY ? kNoScore : m[i];
        ml[((wave * NR + i) * 16 + r16) * 2 + 1] = l[i];
      }
#pragma unroll
      for (int d = 0; d < DT; ++d) red[((wave * NR + i) * DT + d) * 64 + lane] = acc[i][d];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NR; ++i) {
      const int r = r0 + 16 * i + r16;
      float top = -INFINITY, w[NW], total = 0.f;
#pragma unroll
      for (int k = 0; k < NW; ++k) top = fmaxf(top, ml[((k * NR + i) * 16 + r16) * 2]);
#pragma unroll
      for (int k = 0; k < NW; ++k) {
        const float mk = ml[((k * NR + i) * 16 + r16) * 2];
        w[k] = mk == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mk - top);
        if (mk != -INFINITY) total += w[k] * ml[((k * NR + i) * 16 + r16) * 2 + 1];
      }
      if (r >= n * G) continue;
      const size_t orow = (size_t)(rw.first + r / G) * a.n_q + h * G + r % G;
      const bool none = top == -INFINITY;
      const float inv = none ? 0.f : 1.0f / total;
      for (int d = wave; d < DT; d += NW) {
        f32x4 o{};
#pragma unroll
        for (int k = 0; k < NW; ++k) {
          o += w[k] * red[((k * NR + i) * DT + d) * 64 + lane];
        }
        if (a.splits == 1) {
          o = none ? f32x4{} : o * inv;
          st64(a.out + orow * D + 16 * d + 4 * g, u32x2{T::pack2(o[0], o[1]), T::pack2(o[2], o[3])});
        } else {
          *reinterpret_cast<f32x4*>(a.part + ((size_t)split * a.T * a.n_q + orow) * D + 16 * d + 4 * g) = o;
        }
      }
      if (a.splits > 1 && wave == 0 && g == 0) {
        float* p = a.part + (size_t)a.splits * a.T * a.n_q * D + ((size_t)split * a.T * a.n_q + orow) * 2;
        p[0] = top;
        p[1] = total;
      }
    }
    __syncthreads();  // smem serves the next rows
  }
}

// ---------------------------------------------------------------------------
// Many rows per sequence (prompts and their chunks): a workgroup of 8 waves takes 256
// rows (row = token * G + head of the group) of one KV head, 32 a wave, and walks
// the keys in tiles of 64.  A tile's codes go HBM -> registers one tile ahead, are
// widened to 16 bits once per workgroup and written to one of two LDS stages; every
// wave then reads its 32x32x16 MFMA operands from there: K as stored, V from its
// transposed page, in the order of keys that a score tile leaves in a lane's
// registers, so that P' is the second product's operand as it is.
// ---------------------------------------------------------------------------
constexpr int TW = 8;           // waves
constexpr int TR = 32 * TW;     // rows of a workgroup
constexpr int BN = 64;          // keys of a tile
constexpr float kLazy = 8.0f;   // log2 units that a score may pass the running maximum by before it moves

template <int D>
struct Stage {
  static constexpr int K = BN * D * 2, V = D * BN * 2;
  static constexpr int BYTES = K + V;
  static constexpr int CONSTS = 2 * BYTES;            // [2][4 groups of 16 keys] x {cs, lv, iv, 0}
  static constexpr int FLAGS = CONSTS + 2 * 4 * 16;   // [2][TW] a NaN among V's codes
  static constexpr int LDS = FLAGS + 2 * TW * 4;
};
// 16-byte slot of a row, swizzled so that the 16 lanes LDS serves together hit different
// slots of its 256-byte window.
template <int ROW>
__device__ __forceinline__ int slot_at(int row, int slot) {
  return ROW == 256 ? slot ^ (row & 15) : slot ^ ((row >> 1) & 7);
}

template <typename T, int D>
__global__ __launch_bounds__(64 * TW, 1) void tile_kernel(const Args a) {
  using L = Stage<D>;
  constexpr int DC = D / 16, DT = D / 32;
  constexpr int NT = 64 * TW;
  constexpr int U = D * 8 / NT;  // 16-byte units of a tile (K, then V) per thread
  static_assert(U >= 1 && U * NT == D * 8, "units");
  extern __shared__ __align__(1024) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int ql = lane & 31, g = lane >> 5;
  const int G = a.n_q / a.n_kv;
  const int h = blockIdx.x % a.n_kv, b = blockIdx.x / a.n_kv;
  const int split = blockIdx.z;
  const int P = 1 << a.lp;

  const Rows rw = rows_of(a.cu, b, a.T);
  const int n = rw.last - rw.first;
  const int len = cut_len(a.lens[b], a.max_pages, a.lp);
  const int s0 = min((long long)split * a.chunk, (long long)len);
  const int s1 = split + 1 == a.splits ? len : min(len, s0 + a.chunk);
  const int* row_pages = a.table + (size_t)b * a.max_pages;
  const float c = fabsf(a.c);
  const uint32_t flip = a.c < 0.f ? 0x80008000u : 0u;
  const uint32_t lds0 = lds_addr(smem);

  // later rows first: with a causal mask they have the most keys
  const uint32_t all_rows = (uint32_t)n * G;
  for (uint32_t r0 = (gridDim.y - 1 - blockIdx.y) * TR; r0 < all_rows; r0 += gridDim.y * TR) {
    const int rows = (int)min((uint32_t)TR, all_rows - r0);
    auto sees = [&](int r) {  // keys t < sees(r) are those of row r0 + r
      return a.causal ? max(len - n + (int)((r0 + r) / (uint32_t)G) + 1, 0) : len;
    };
    const int low = sees(0), high = min(sees(rows - 1), s1);
    const int tiles = high > s0 ? (high - s0 + BN - 1) / BN : 0;
    const int r = 32 * wave + ql;
    const int rr = min(r, rows - 1);
    const int limit = min(sees(rr), s1);
    const int w_low = sees(min(32 * wave, rows - 1)), w_high = min(sees(min(32 * wave + 31, rows - 1)), s1);
    const bool idle = 32 * wave >= rows;
    const int tok = (int)((r0 + rr) / (uint32_t)G), head = h * G + (int)((r0 + rr) % (uint32_t)G);

    u32x4 qf[DC];
    {
      const uint16_t* src = a.q + (size_t)(rw.first + tok) * a.q_stride + head * D + 8 * g;
#pragma unroll
      for (int k = 0; k < DC; ++k) qf[k] = ld128(src + 16 * k) ^ u32x4{flip, flip, flip, flip};
    }

    // ---- a tile's codes: unit id < 4 D: K, row id / (D/16); else V, channel ----
    u32x4 raw[U];
    float rks = 0.f, rvs = 0.f;
    int page_n[U], page_s;  // pages of the next tile to load
    auto key_of = [&](int u) {
      const int id = tid + u * NT;
      return id < 4 * D ? id / (D / 16) : (id - 4 * D) % 4 * 16;
    };
    auto find = [&](int tile) {
      const int at = s0 + BN * tile;
#pragma unroll
      for (int u = 0; u < U; ++u)
        page_n[u] = at + key_of(u) < high ? page_of(row_pages, at + key_of(u), a.lp, a.max_pages, a.pages) : -1;
      page_s = tid < 4 && at + 16 * tid < high ? page_of(row_pages, at + 16 * tid, a.lp, a.max_pages, a.pages) : -1;
    };
    bool bad[U], bad_s;
    auto load = [&](int tile) {
      const int at = s0 + BN * tile;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int id = tid + u * NT, key = (at + key_of(u)) & (P - 1);
        bad[u] = page_n[u] < 0;
        const size_t page = ((size_t)max(page_n[u], 0) * a.n_kv + h) * (size_t)(D * P);
        raw[u] = ld128(id < 4 * D ? a.kc + page + (size_t)key * D + id % (D / 16) * 16
                                  : a.vc + page + (size_t)((id - 4 * D) / 4) * P + key);
      }
      bad_s = page_s < 0;
      rks = a.ks[(size_t)max(page_s, 0) * a.n_kv + h];
      rvs = a.vs[(size_t)max(page_s, 0) * a.n_kv + h];
    };
    auto store = [&](int tile) {
      const int at = s0 + BN * tile;
      const uint32_t st = (tile & 1) * L::BYTES;
      bool nan = false;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int id = tid + u * NT;
        u32x4 x = bad[u] ? u32x4{} : raw[u];
        if (id < 4 * D) {
          const int row = id / (D / 16), slot = id % (D / 16) * 2;
          st128(smem + st + row * (2 * D) + 16 * slot_at<2 * D>(row, slot), widen8<T>(x[0], x[1]));
          st128(smem + st + row * (2 * D) + 16 * slot_at<2 * D>(row, slot + 1), widen8<T>(x[2], x[3]));
        } else {
          const int row = (id - 4 * D) / 4, slot = (id - 4 * D) % 4 * 2;
          if (at + BN > low) {  // some row does not see every key of the tile
            const int left = high - at - 8 * slot;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
#pragma unroll
              for (int j = 0; j < 4; ++j)
                if (4 * w + j >= left) x[w] &= ~(0xffu << (8 * j));
              const uint32_t bits = a.causal ? nan_bytes(x[w]) : 0u;
              nan |= bits != 0;
              x[w] &= ~spread(bits);
            }
          }
          st128(smem + st + L::K + row * (2 * BN) + 16 * slot_at<2 * BN>(row, slot), widen8<T>(x[0], x[2]));
          st128(smem + st + L::K + row * (2 * BN) + 16 * slot_at<2 * BN>(row, slot + 1), widen8<T>(x[1], x[3]));
        }
      }
      if (tid < 4)
        *reinterpret_cast<f32x4*>(smem + L::CONSTS + ((tile & 1) * 4 + tid) * 16) =
            bad_s ? f32x4{0.f, -INFINITY, 0.f, 0.f} : f32x4{c * rks, __builtin_amdgcn_logf(rvs), 1.0f / rvs, 0.f};
      const bool any = __any(nan);
      if (lane == 0) *reinterpret_cast<int*>(smem + L::FLAGS + ((tile & 1) * TW + wave) * 4) = any;
    };

    f32x16 acc[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d) acc[d] = f32x16{};
    float m = 0.f, l = 0.f;
    bool open = true, seen = false;

    __syncthreads();  // the stages are free
    if (tiles > 0) {
      find(0);
      load(0);
      find(1);
      store(0);
      if (tiles > 1) load(1);
      find(2);
    }
    for (int tile = 0; tile < tiles; ++tile) {
      __syncthreads();  // the tile's stage is written, the other one read
      if (tile + 1 < tiles) {
        store(tile + 1);
        if (tile + 2 < tiles) load(tile + 2);
        find(tile + 3);
      }
      const int at = s0 + BN * tile;
      if (idle || at >= w_high) continue;
      const uint32_t st = lds0 + (tile & 1) * L::BYTES;

      // ---- S^T ----
      f32x16 s[2];
#pragma unroll
      for (int k = 0; k < DC; ++k)
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const u32x4 kf = lds_ld128(st + (32 * t + ql) * (2 * D) + 16 * slot_at<2 * D>(ql, 2 * k + g));
          s[t] = mfma32<T>(kf, qf[k], k ? s[t] : f32x16{});
        }
      f32x4 cst[4];
#pragma unroll
      for (int u = 0; u < 4; ++u)
        cst[u] = *reinterpret_cast<const f32x4*>(smem + L::CONSTS + ((tile & 1) * 4 + u) * 16);

      // ---- y - m, the running maximum ----
      float mx = -INFINITY;
      const bool masked = at + BN > min(w_low, s1);
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const f32x4& k = cst[2 * t + (e >> 3)];
          s[t][e] = __builtin_fmaf(s[t][e], k[0], k[1] - m);
          if (masked) s[t][e] = at + 32 * t + 8 * (e >> 2) + 4 * g + (e & 3) < limit ? s[t][e] : -INFINITY;
          mx = fmaxf(mx, s[t][e]);
        }
      mx = max_xor32(mx);
      const bool moved = __any(mx > kLazy);
      if (moved || open) {
        const bool empty = open && sum_xor32(l) == 0.f, met = mx > -INFINITY;
        const float shift = empty ? (met ? mx : 0.f) : moved ? fmaxf(mx, 0.f) : 0.f;
        open = __any(empty && !met);
#pragma unroll
        for (int u = 0; u < 4; ++u) seen |= cst[u][1] > -INFINITY && at + 16 * u < limit;
        m += shift;
        const float corr = empty ? 1.f : __builtin_amdgcn_exp2f(-shift);
        l *= corr;
#pragma unroll
        for (int d = 0; d < DT; ++d) acc[d] *= corr;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int e = 0; e < 16; ++e) s[t][e] -= shift;
      }

      // ---- a NaN among V's codes that some row does not see: see rows_kernel ----
      if (at + BN > low && a.causal) {
        int any = 0;
#pragma unroll
        for (int w = 0; w < TW; ++w) any |= *reinterpret_cast<const int*>(smem + L::FLAGS + ((tile & 1) * TW + w) * 4);
        if (any) {
          for (int k = 0; k < 4; ++k) {
            const int page = at + 16 * k < high ? page_of(row_pages, at + 16 * k, a.lp, a.max_pages, a.pages) : -1;
            if (page < 0) continue;
            const int key = at + 16 * k + 4 * g;
            u32x4 vis, x;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              const int e = key + 8 * (w >> 1) + 2 * (w & 1);
              vis[w] = (e < limit ? one_bits<T>() : 0u) | (e + 1 < limit ? one_bits<T>() << 16 : 0u);
            }
#pragma unroll
            for (int d = 0; d < DT; ++d) {
              const uint8_t* p = a.vc + ((size_t)page * a.n_kv + h) * (size_t)(D * P) + (size_t)(32 * d + ql) * P + (key & (P - 1));
#pragma unroll
              for (int w = 0; w < 4; ++w) {
                const int e = 8 * (w >> 1) + 2 * (w & 1);
                x[w] = ((p[e] & 0x7f) == 0x7f && key + e < high ? one_bits<T>() : 0u) |
                       ((p[e + 1] & 0x7f) == 0x7f && key + e + 1 < high ? one_bits<T>() << 16 : 0u);
              }
              const f32x16 cnt = mfma32<T>(x, vis, f32x16{});
#pragma unroll
              for (int e = 0; e < 16; ++e)
                if (cnt[e] > 0.f) acc[d][e] = __builtin_nanf("");
            }
          }
        }
      }

      // ---- P', O^T += V^T P'^T ----
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        f32x16& x = s[k >> 1];
        const int o = 8 * (k & 1);
        float sum = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          x[o + e] = __builtin_amdgcn_exp2f(x[o + e]);
          sum += x[o + e];
        }
        l = __builtin_fmaf(sum, cst[k][2], l);
        const u32x4 pf{T::pack2(x[o], x[o + 1]), T::pack2(x[o + 2], x[o + 3]), T::pack2(x[o + 4], x[o + 5]),
                       T::pack2(x[o + 6], x[o + 7])};
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          const u32x4 vf = lds_ld128(st + L::K + (32 * d + ql) * (2 * BN) + 16 * slot_at<2 * BN>(ql, 2 * k + g));
          acc[d] = mfma32<T>(vf, pf, acc[d]);
        }
      }
    }

    // ---- store: the lane's query, d = 32 dt + 8 i + 4 g + j ----
    const float total = sum_xor32(l);
    seen = __shfl_xor((int)seen, 32, 64) | (int)seen;
    if (r < rows) {
      const size_t orow = (size_t)(rw.first + tok) * a.n_q + head;
      const bool none = total == 0.f && !seen;
      if (a.splits == 1) {
        const float inv = none ? 0.f : 1.0f / total;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            st64(a.out + orow * D + 32 * d + 8 * i + 4 * g,
                 u32x2{T::pack2(acc[d][4 * i] * inv, acc[d][4 * i + 1] * inv),
                       T::pack2(acc[d][4 * i + 2] * inv, acc[d][4 * i + 3] * inv)});
      } else {
        const size_t all = (size_t)a.T * a.n_q;
        float* p = a.part + ((size_t)split * all + orow) * D;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            *reinterpret_cast<f32x4*>(p + 32 * d + 8 * i + 4 * g) =
                f32x4{acc[d][4 * i], acc[d][4 * i + 1], acc[d][4 * i + 2], acc[d][4 * i + 3]};
        if (g == 0) {
          float* ml = a.part + (size_t)a.splits * all * D + ((size_t)split * all + orow) * 2;
          ml[0] = none ? -INFINITY : total == 0.f ? kNoScore : m;
          ml[1] = total;
        }
      }
    }
  }
}

// ---------------------------------------------------------------------------
// The splits' partial results of a row meet: one wave per row.
// ---------------------------------------------------------------------------
template <typename T, int D>
__global__ __launch_bounds__(256) void combine_kernel(const Args a) {
  const int lane = threadIdx.x & 63;
  const long long r = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  const size_t rows = (size_t)a.T * a.n_q;
  if (r >= (long long)rows) return;
  if (a.cu) {
    const int tok = (int)(r / a.n_q);
    if (tok < a.cu[0] || tok >= a.cu[a.B]) return;  // no sequence's row
  }
  const float* ml = a.part + (size_t)a.splits * rows * D;
  float top = -INFINITY;
  for (int s = lane; s < a.splits; s += 64) top = fmaxf(top, ml[((size_t)s * rows + r) * 2]);
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) top = fmaxf(top, __shfl_xor(top, off, 64));
  constexpr int V = D / 64;  // channels of a lane
  float o[V] = {}, total = 0.f;
  for (int s = 0; s < a.splits; ++s) {
    const float m = ml[((size_t)s * rows + r) * 2];
    if (m == -INFINITY) continue;
    const float w = __builtin_amdgcn_exp2f(m - top);
    total += w * ml[((size_t)s * rows + r) * 2 + 1];
    const float* p = a.part + ((size_t)s * rows + r) * D + lane * V;
#pragma unroll
    for (int v = 0; v < V; ++v) o[v] += w * p[v];
  }
  const float inv = top == -INFINITY ? 0.f : 1.0f / total;
  uint16_t* out = a.out + (size_t)r * D + lane * V;
  if constexpr (V == 2)
    *reinterpret_cast<uint32_t*>(out) = top == -INFINITY ? 0u : T::pack2(o[0] * inv, o[1] * inv);
  else
    *out = top == -INFINITY ? (uint16_t)0 : (uint16_t)T::pack2(o[0] * inv, 0.f);
}

// ---------------------------------------------------------------------------
// Launch choice
// ---------------------------------------------------------------------------
struct Plan {
  int nr;       // 16-row blocks of the rows kernel; 0: the tile kernel
  int tiles;    // 256-row tiles of the tile kernel
  int splits, chunk;
};

static Plan plan(int B, int T, int max_q, int max_kv, int n_q, int n_kv) {
  const int G = n_q / n_kv;
  const long long rows = (long long)max_q * G;
  Plan p;
  p.nr = rows <= 16 ? 1 : rows <= 32 ? 2 : 0;
  p.tiles = (int)std::min((rows + TR - 1) / TR, 65535LL);
  const long long units = (long long)B * n_kv * (p.nr ? 1 : p.tiles);
  const long long want = ((p.nr ? 2048 : 256) + units - 1) / units;
  long long chunk = (max_kv + want - 1) / want;
  chunk = (chunk + 255) / 256 * 256;
  p.splits = (int)((max_kv + chunk - 1) / chunk);
  p.chunk = (int)chunk;
  return p;
}

template <typename T, int D, int NR>
static int launch_rows(const Args& a, hipStream_t s) {
  constexpr int lds = NW * NR * (16 * 2 * 4 + (D / 16) * 64 * 16);
  MX_RETURN_IF_HIP((lds_limit_once<rows_kernel<T, D, NR>>(lds)));
  hipLaunchKernelGGL((rows_kernel<T, D, NR>), dim3((unsigned)(a.B * a.n_kv), (unsigned)a.splits), dim3(64 * NW), lds, s, a);
  MX_RETURN_IF_HIP(hipGetLastError());
  return MX_OK;
}

template <typename T, int D>
static int launch_tiles(const Args& a, const Plan& p, hipStream_t s) {
  constexpr int lds = Stage<D>::LDS;
  MX_RETURN_IF_HIP((lds_limit_once<tile_kernel<T, D>>(lds)));
  hipLaunchKernelGGL((tile_kernel<T, D>), dim3((unsigned)(a.B * a.n_kv), (unsigned)p.tiles, (unsigned)a.splits), dim3(64 * TW),
                     lds, s, a);
  MX_RETURN_IF_HIP(hipGetLastError());
  return MX_OK;
}

template <typename T, int D>
static int run(const Args& a, const Plan& p, hipStream_t s) {
  const int rc = p.nr == 1 ? launch_rows<T, D, 1>(a, s) : p.nr == 2 ? launch_rows<T, D, 2>(a, s) : launch_tiles<T, D>(a, p, s);
  if (rc != MX_OK || p.splits == 1) return rc;
  const long long rows = (long long)a.T * a.n_q;
  hipLaunchKernelGGL((combine_kernel<T, D>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, s, a);
  MX_RETURN_IF_HIP(hipGetLastError());
  return MX_OK;
}

static bool sizes_ok(int B, int T, int max_q, int max_kv, int n_q, int n_kv, int d) {
  return B > 0 && T > 0 && max_q > 0 && max_kv > 0 && n_q > 0 && n_kv > 0 && n_q % n_kv == 0 && (d == 64 || d == 128) &&
         (long long)B * n_kv <= (1 << 24) && (long long)T * n_q <= 0x7fffffffLL;
}

}  // namespace kv8
}  // namespace mx

extern "C" size_t mx_gqa_kv8_workspace(int B, int T, int max_q, int max_kv, int n_q, int n_kv, int d) {
  using namespace mx::kv8;
  if (!sizes_ok(B, T, max_q, max_kv, n_q, n_kv, d)) return 0;
  const Plan p = plan(B, T, max_q, max_kv, n_q, n_kv);
  return p.splits == 1 ? 0 : (size_t)p.splits * T * n_q * (d + 2) * sizeof(float);
}

extern "C" int mx_gqa_kv8(const void* q, const void* k_cache, const void* v_cache, const float* k_scale,
                          const float* v_scale, const int* page_table, const int* kv_lens, const int* cu, void* O, int B,
                          int T, int max_q, int max_kv, int n_q, int n_kv, int d, int page, int pages, int max_pages,
                          int q_stride, float scale, int causal, int dtype, void* workspace, size_t ws_bytes,
                          void* stream) {
  using namespace mx::kv8;
  if (!q || !O || !page_table || !kv_lens) return MX_ERR_NULL;
  const int rc = check_cache(k_cache, v_cache, k_scale, v_scale, n_kv, d, page, pages);
  if (rc != MX_OK) return rc;
  if (!sizes_ok(B, T, max_q, max_kv, n_q, n_kv, d) || max_pages <= 0 || (!cu && T != B)) return MX_ERR_SHAPE;
  if (q_stride < n_q * d) return MX_ERR_SHAPE;
  if (q_stride % 8 || (((uintptr_t)q | (uintptr_t)O) & 15)) return MX_ERR_ALIGN;
  if (dtype != MX_DTYPE_BF16 && dtype != MX_DTYPE_F16) return MX_ERR_DTYPE;
  const Plan p = plan(B, T, max_q, max_kv, n_q, n_kv);
  if (p.splits > 1) {
    if (!workspace || ws_bytes < mx_gqa_kv8_workspace(B, T, max_q, max_kv, n_q, n_kv, d)) return MX_ERR_WORKSPACE;
    if ((uintptr_t)workspace & 15) return MX_ERR_ALIGN;
  }
  const Args a{(const uint16_t*)q, (const uint8_t*)k_cache, (const uint8_t*)v_cache, k_scale, v_scale, page_table, kv_lens,
               cu, (uint16_t*)O, (float*)workspace, B, T, n_q, n_kv, pages, max_pages, q_stride, log2_page(page),
               causal ? 1 : 0, p.splits, p.chunk, scale * kLog2e};
  hipStream_t s = (hipStream_t)stream;
  if (dtype == MX_DTYPE_BF16) return d == 64 ? run<mx::BF16, 64>(a, p, s) : run<mx::BF16, 128>(a, p, s);
  return d == 64 ? run<mx::F16, 64>(a, p, s) : run<mx::F16, 128>(a, p, s);
}
