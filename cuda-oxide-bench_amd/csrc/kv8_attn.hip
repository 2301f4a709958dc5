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
  const int len = cut_len(a.lens[b], a.max_pages, a.lp);
  if (n == 0) return;
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
  static constexpr int FLAGS = CONSTS + 2 * 4 * 16;   // tiles with a NaN among V's codes
  static constexpr int LDS = FLAGS + 16;
};
// 16-byte slot of a row, swizzled so that the 16 lanes LDS serves together hit different
// slots of its 256-byte window.
template <int ROW>
__device__ __forceinline__ int slot_at(int row, int slot) {
  return ROW == 256 ? slot ^ (row & 15) : slot ^ ((row >> 1) & 7);
}

// WIDE: pages of 64 tokens and more, one page and one set of scales per tile.
template <typename T, int D, bool WIDE>
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

    // ---- a tile's codes: unit id < 4 D: K, row id / (D/16); else V, channel.  Page
    // numbers are looked up a tile before the codes are loaded, those a tile before
    // they are widened.  Past the last tile: page -1, zeros into a stage nobody reads. ----
    u32x4 raw[U];
    float rks = 0.f, rvs = 0.f;
    int page_n[U], page_s;
    bool bad[U], bad_s = true;
    auto key_of = [&](int u) {
      const int id = tid + u * NT;
      return id < 4 * D ? id / (D / 16) : (id - 4 * D) % 4 * 16;
    };
    const int last_col = a.max_pages - 1;
    auto find = [&](int tile) {
      const int at = s0 + BN * tile;
#pragma unroll
      for (int u = 0; u < U; ++u) page_n[u] = row_pages[min((at + key_of(u)) >> a.lp, last_col)];
      page_s = row_pages[min((at + 16 * (tid & 3)) >> a.lp, last_col)];
    };
    auto load = [&](int tile) {
      const int at = s0 + BN * tile;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int id = tid + u * NT, key = at + key_of(u);
        bad[u] = key >= high || (uint32_t)page_n[u] >= (uint32_t)a.pages;
        const size_t page = ((size_t)(uint32_t)(bad[u] ? 0 : page_n[u]) * a.n_kv + h) * (size_t)(D * P);
        raw[u] = ld128(id < 4 * D ? a.kc + page + (size_t)(key & (P - 1)) * D + id % (D / 16) * 16
                                  : a.vc + page + (size_t)((id - 4 * D) / 4) * P + (key & (P - 1)));
      }
      bad_s = at + 16 * (tid & 3) >= high || (uint32_t)page_s >= (uint32_t)a.pages;
      const size_t page = (size_t)(uint32_t)(bad_s ? 0 : page_s) * a.n_kv + h;
      rks = a.ks[page];
      rvs = a.vs[page];
    };
    // Tiles from first_masked on are not seen whole by every row: at most 6, bits of *flags.
    int* flags = reinterpret_cast<int*>(smem + L::FLAGS);
    const int first_masked = low > s0 ? (low - s0) / BN : 0;
    // A tile that some row does not see whole: V's codes of tokens past the last become 0,
    // and so do NaNs, which are flagged (with a causal mask: without one every row sees
    // every token that is there).
    auto clean = [&](int tile) {
      const int at = s0 + BN * tile;
      bool nan = false;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int id = tid + u * NT;
        if (id >= 4 * D) {
          const int left = high - at - (id - 4 * D) % 4 * 16;
#pragma unroll
          for (int w = 0; w < 4; ++w) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (bad[u] || 4 * w + j >= left) raw[u][w] &= ~(0xffu << (8 * j));
            const uint32_t bits = a.causal ? nan_bytes(raw[u][w]) : 0u;
            nan |= bits != 0;
            raw[u][w] &= ~spread(bits);
          }
        }
      }
      if (__any(nan) && lane == 0) atomicOr(flags, 1 << (tile - first_masked));
    };
    // unit u of the loaded tile into the stage at byte st
    auto store = [&](int u, int st) {
      const int id = tid + u * NT;
      const u32x4 x = bad[u] ? u32x4{} : raw[u];
      if (id < 4 * D) {
        const int row = id / (D / 16), slot = id % (D / 16) * 2;
        st128(smem + st + row * (2 * D) + 16 * slot_at<2 * D>(row, slot), widen8<T>(x[0], x[1]));
        st128(smem + st + row * (2 * D) + 16 * slot_at<2 * D>(row, slot + 1), widen8<T>(x[2], x[3]));
      } else {
        const int row = (id - 4 * D) / 4, slot = (id - 4 * D) % 4 * 2;
        st128(smem + st + L::K + row * (2 * BN) + 16 * slot_at<2 * BN>(row, slot), widen8<T>(x[0], x[2]));
        st128(smem + st + L::K + row * (2 * BN) + 16 * slot_at<2 * BN>(row, slot + 1), widen8<T>(x[1], x[3]));
      }
    };
    auto store_consts = [&](int stage) {
      if (tid < 4)
        *reinterpret_cast<f32x4*>(smem + L::CONSTS + (stage * 4 + tid) * 16) =
            bad_s ? f32x4{0.f, -INFINITY, 0.f, 0.f} : f32x4{c * rks, __builtin_amdgcn_logf(rvs), 1.0f / rvs, 0.f};
    };

    // K fragment: key row 32 t + ql, slot 2 k + g; V fragment: channel row 32 d + ql, slot
    // 2 k + g of the tile's 16-key chunk k.  The swizzle is an xor, so slot 2 k is an xor away
    // from slot 0: one register each, made opaque in every tile lest all of them be kept.
    const uint32_t k_base = lds0 + ql * (2 * D) + 16 * slot_at<2 * D>(ql, g);
    const uint32_t v_base = lds0 + L::K + ql * (2 * BN) + 16 * slot_at<2 * BN>(ql, g);

    f32x16 acc[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d) acc[d] = f32x16{};
    float m = 0.f, l = 0.f;
    bool open = true, seen = false;

    // LDS writes done, then the barrier: no wait for the loads that are under way
    auto meet = [&] {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      lds_barrier();
    };
    __syncthreads();  // the stages and flags are free
    if (tid == 0) *flags = 0;
    if (a.causal) __syncthreads();
    if (tiles > 0) {
      find(0);
      load(0);
      find(1);
      if (s0 + BN > low) clean(0);
#pragma unroll
      for (int u = 0; u < U; ++u) store(u, 0);
      store_consts(0);
      load(1);
      find(2);
    }
    auto step = [&](int tile, auto stage_tag) {
      constexpr int STG = decltype(stage_tag)::value;
      constexpr uint32_t st = STG * L::BYTES, other = (1 - STG) * L::BYTES;
      meet();  // the tile's stage is written, the other one read
      const int at = s0 + BN * tile;
      if (at + 2 * BN > low) clean(tile + 1);
      if (idle || at >= w_high) {  // nothing to compute: the wave's share of the next tile
#pragma unroll
        for (int u = 0; u < U; ++u) store(u, other);
        store_consts(1 - STG);
        load(tile + 2);
        find(tile + 3);
        return;
      }

      // ---- S^T, the next tile's codes widened and stored beside its MFMAs ----
      __builtin_amdgcn_s_setprio(1);
      f32x16 s[2];
      u32x4 kb[3][2];
      uint32_t kb0 = k_base;
      asm volatile("" : "+v"(kb0));
      auto kread = [&](int t, int k) { return lds_ld128((kb0 ^ (32 * k)) + st + 32 * t * (2 * D)); };
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        kb[i][0] = kread(0, i);
        kb[i][1] = kread(1, i);
      }
#pragma unroll
      for (int k = 0; k < DC; ++k) {
        if (k + 2 < DC) {
          kb[(k + 2) % 3][0] = kread(0, k + 2);
          kb[(k + 2) % 3][1] = kread(1, k + 2);
        }
#pragma unroll
        for (int t = 0; t < 2; ++t) s[t] = mfma32<T>(kb[k % 3][t], qf[k], k ? s[t] : f32x16{});
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (k == 1 + u * 2) store(u, other);
        if (k == DC - 1) {
          store_consts(1 - STG);
          load(tile + 2);
          find(tile + 3);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      f32x4 cst[WIDE ? 1 : 4];
#pragma unroll
      for (int u = 0; u < (WIDE ? 1 : 4); ++u) cst[u] = *reinterpret_cast<const f32x4*>(smem + L::CONSTS + (STG * 4 + u) * 16);
      uint32_t vb0 = v_base;
      asm volatile("" : "+v"(vb0));
      auto vread = [&](int k, int d) { return lds_ld128((vb0 ^ (32 * k)) + st + 32 * d * (2 * BN)); };
      u32x4 vb[2][DT];
#pragma unroll
      for (int d = 0; d < DT; ++d) vb[0][d] = vread(0, d);
      __builtin_amdgcn_s_setprio(0);

      // ---- y - m, the running maximum ----
      float mx = -INFINITY;
      const bool masked = at + BN > min(w_low, s1);
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const f32x4& k = cst[WIDE ? 0 : 2 * t + (e >> 3)];
          s[t][e] = __builtin_fmaf(s[t][e], k[0], k[1] - m);
        }
      if (masked) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            s[t][e] = at + 32 * t + 8 * (e >> 2) + 4 * g + (e & 3) < limit ? s[t][e] : -INFINITY;
      }
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e) mx = fmaxf(mx, s[t][e]);
      mx = max_xor32(mx);
      const bool moved = __any(mx > kLazy);
      if (moved || open) {
        const bool empty = open && sum_xor32(l) == 0.f, met = mx > -INFINITY;
        const float shift = empty ? (met ? mx : 0.f) : moved ? fmaxf(mx, 0.f) : 0.f;
        open = __any(empty && !met);
#pragma unroll
        for (int u = 0; u < (WIDE ? 1 : 4); ++u) seen |= cst[u][1] > -INFINITY && at + 16 * u < limit;
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

      // ---- P', O^T += V^T P'^T by chunks of 16 keys: the next chunk's exponentials and
      // V reads run beside a chunk's MFMAs ----
#pragma unroll
      for (int e = 0; e < 8; ++e) s[0][e] = __builtin_amdgcn_exp2f(s[0][e]);
      __builtin_amdgcn_s_setprio(1);
      float sum = 0.f;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        f32x16& x = s[k >> 1];
        const int o = 8 * (k & 1);
        const u32x4 pf{T::pack2(x[o], x[o + 1]), T::pack2(x[o + 2], x[o + 3]), T::pack2(x[o + 4], x[o + 5]),
                       T::pack2(x[o + 6], x[o + 7])};
        const float part = ((x[o] + x[o + 1]) + (x[o + 2] + x[o + 3])) + ((x[o + 4] + x[o + 5]) + (x[o + 6] + x[o + 7]));
        if constexpr (WIDE)
          sum += part;
        else
          l = __builtin_fmaf(part, cst[WIDE ? 0 : k][2], l);
        if (k + 1 < 4) {
#pragma unroll
          for (int d = 0; d < DT; ++d) vb[(k + 1) & 1][d] = vread(k + 1, d);
          const int o1 = 8 * ((k + 1) & 1);
#pragma unroll
          for (int e = 0; e < 8; ++e) s[(k + 1) >> 1][o1 + e] = __builtin_amdgcn_exp2f(s[(k + 1) >> 1][o1 + e]);
        }
#pragma unroll
        for (int d = 0; d < DT; ++d) acc[d] = mfma32<T>(vb[k & 1][d], pf, acc[d]);
        if (k + 1 < 4) {
          __builtin_amdgcn_sched_group_barrier(0x002, 4, 0);
#pragma unroll
          for (int d = 0; d < DT; ++d) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x400, 8 / DT, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x002, 8 / DT, 0);
          }
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      if constexpr (WIDE) l = __builtin_fmaf(sum, cst[0][2], l);
      __builtin_amdgcn_s_setprio(0);
    };
    for (int tile = 0; tile < tiles; tile += 2) {
      step(tile, std::integral_constant<int, 0>{});
      if (tile + 1 < tiles) step(tile + 1, std::integral_constant<int, 1>{});
    }

    // ---- a NaN among V's codes that some row does not see: those that it does see are
    // counted, by channel and row, with the products' own layout ----
    if (a.causal) {
      meet();
      for (int flagged = *flags; flagged; flagged &= flagged - 1) {
        const int at = s0 + BN * (first_masked + __builtin_ctz(flagged));
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
              x[w] = ((p[e] & 0x7f) == 0x7f ? one_bits<T>() : 0u) | ((p[e + 1] & 0x7f) == 0x7f ? one_bits<T>() << 16 : 0u);
            }
            const f32x16 cnt = mfma32<T>(x, vis, f32x16{});
#pragma unroll
            for (int e = 0; e < 16; ++e)
              if (cnt[e] > 0.f) acc[d][e] = __builtin_nanf("");
          }
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

template <typename T, int D, bool WIDE>
static int launch_tiles(const Args& a, const Plan& p, hipStream_t s) {
  constexpr int lds = Stage<D>::LDS;
  MX_RETURN_IF_HIP((lds_limit_once<tile_kernel<T, D, WIDE>>(lds)));
  hipLaunchKernelGGL((tile_kernel<T, D, WIDE>), dim3((unsigned)(a.B * a.n_kv), (unsigned)p.tiles, (unsigned)a.splits), dim3(64 * TW),
                     lds, s, a);
  MX_RETURN_IF_HIP(hipGetLastError());
  return MX_OK;
}

template <typename T, int D>
static int run(const Args& a, const Plan& p, hipStream_t s) {
  const int rc = p.nr == 1 ? launch_rows<T, D, 1>(a, s) : p.nr == 2 ? launch_rows<T, D, 2>(a, s) : a.lp >= 6 ? launch_tiles<T, D, true>(a, p, s) : launch_tiles<T, D, false>(a, p, s);
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
