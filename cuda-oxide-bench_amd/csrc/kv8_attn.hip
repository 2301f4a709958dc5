// Grouped-query attention over the paged 8-bit cache, for gfx950.
//
//   O[i,h] = softmax_t(scale * q[i,h] . K[t]) . V[t],   K[t] = k8[t] ks, V[t] = v8[t] vs,
// the scales ks, vs those of t's page and head.  The codes go through the 16-bit
// MFMAs (e4m3 -> bf16 / f16 is exact), the scales around them:
//     y[t]  = scale log2(e) ks (q . k8[t]) + log2(vs)
//     P'[t] = 2^(y[t] - m),   m = the running maximum of y (f16: less a constant)
//     O     = (sum_t P'[t] v8[t]) / (sum_t P'[t] / vs)
// so a page's two scales cost one FMA constant per score and one product per page in
// the denominator, and P' carries vs and stays within either 16-bit type's range.  (m - max y of a
// page is at most the spread of log2 vs, so no term of the denominator that counts is lost in fp32
// while the vs of a sequence lie within 2^100; a term is at most 2^8 / vs (f16: 2^15, where a vs
// below 2^-40 gives outputs of 0 anyway), so that the sum of 2^30 stays finite from vs = 2^-90 on.)
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

// log2 of the largest P'.  f16 has no more than 24 binades below one, and a page whose vs is that
// far below the largest may hold all of a channel: P' then fills the range up to 2^15.
// tile_kernel, whose maximum may lag by lazy(), leaves room for that.
template <typename T>
__device__ __forceinline__ constexpr float lift() {
  return std::is_same<T, BF16>::value ? 0.f : 15.f;
}

// A dword with 0x80 in each byte of x that is a NaN code.
__device__ __forceinline__ uint32_t nan_bytes(uint32_t x) { return ((x & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }
// 0xff for each byte of a nan_bytes() dword that is set.
__device__ __forceinline__ uint32_t spread(uint32_t m) { return (m >> 7) * 0xffu; }

// MFMA operands of ones and zeros, their product counts the NaNs that a row sees: which of keys
// at .. at + 7 lie below limit, and which of 8 codes are NaN.
template <typename T>
__device__ __forceinline__ u32x4 visible8(int at, int limit) {
  u32x4 v;
#pragma unroll
  for (int w = 0; w < 4; ++w)
    v[w] = (at + 2 * w < limit ? one_bits<T>() : 0u) | (at + 2 * w + 1 < limit ? one_bits<T>() << 16 : 0u);
  return v;
}
template <typename T>
__device__ __forceinline__ u32x4 nans8(uint32_t lo, uint32_t hi) {
  u32x4 v;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const uint32_t two = nan_bytes(w < 2 ? lo : hi) >> (16 * (w & 1));
    v[w] = ((two & 0x80u) ? one_bits<T>() : 0u) | ((two & 0x8000u) ? one_bits<T>() << 16 : 0u);
  }
  return v;
}
// The NaNs among a tile's V codes that rows see, into their sums.  The lane's 16 keys begin
// at `key`, p points at their codes of channel r16 (`there`: on a page that is one), and the
// products have the layout of the kernels' own.
template <typename T, int D, int NR>
__device__ __forceinline__ void add_nans(f32x4 (&acc)[NR][D / 16], const int (&limit)[NR], const uint8_t* p, bool there,
                                         int key, int P) {
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    u32x4 vis[NR];
#pragma unroll
    for (int i = 0; i < NR; ++i) vis[i] = visible8<T>(key + 8 * u, limit[i]);
#pragma unroll
    for (int d = 0; d < D / 16; ++d) {
      const u32x2 v = there ? ld64(p + (size_t)16 * d * P + 8 * u) : u32x2{};
      const u32x4 x = nans8<T>(v[0], v[1]);
#pragma unroll
      for (int i = 0; i < NR; ++i) {
        const f32x4 cnt = mfma16<T>(x, vis[i], f32x4{});
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (cnt[j] > 0.f) acc[i][d][j] = __builtin_nanf("");
      }
    }
  }
}
// x of any of the lanes l, l ^ 16, l ^ 32, l ^ 48
__device__ __forceinline__ bool any_group(bool x) {
  const int v = (int)x | __shfl_xor((int)x, 16, 64);
  return v | __shfl_xor(v, 32, 64);
}

// ---------------------------------------------------------------------------
// Few rows per sequence (decode, a few speculated tokens): the cache is read once
// from HBM into registers.  A workgroup takes one KV head of a sequence and one
// chunk of its tokens; its NW waves take 64-key tiles in turn and meet in LDS.
//
// 16x16x32 MFMAs on 16 NR rows (row = token * G + head of the group).  Row r of
// score subtile t is key 16 (r / 4) + 4 t + r % 4 of the tile: lane group g = lane / 16
// then owns keys 16 g .. 16 g + 15, which are 16 consecutive bytes of V's transposed
// page, one load per 16 channels.  Pages of 16 tokens and more never split
// them, so a lane has one page, one ks and one vs per tile whatever the page.
// K's rows are read 32 bytes a lane at d = 128 (16 at 64), the contraction's order
// of channels permuted alike in Q.
//
// WIDE: pages of 64 tokens and more, where a tile has one page.  Its address is the
// scalar unit's work, and a lane adds an offset that never changes.
// ---------------------------------------------------------------------------
constexpr int NW = 4;
// Workgroups on a CU.  32 rows of 128 channels need some 430 registers a lane: with two workgroups
// they spill (32 rows on 4096 tokens, B4 26.6 and 19.6 us, B16 47 and 36).
constexpr int rows_per_cu(int nr, int d) { return nr * d == 256 ? 1 : 2; }
template <typename T, int D, int NR, bool WIDE>
__global__ __launch_bounds__(64 * NW, rows_per_cu(NR, D)) void rows_kernel(const Args a) {
  constexpr int KC = D / 32;   // contraction steps
  constexpr int KL = D / 64;   // 16-byte loads of a K row per lane
  constexpr int DT = D / 16;   // output fragments
  constexpr int LD = D == 128 ? 7 : 6;
  extern __shared__ __align__(16) unsigned char smem[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r16 = lane & 15, g = lane >> 4;
  const int G = a.n_q / a.n_kv;
  const int h = blockIdx.x % a.n_kv, b = blockIdx.x / a.n_kv;
  const int split = blockIdx.y;
  const int P = 1 << a.lp;

  // ---- page numbers: of the lane's K rows and of its V keys (WIDE: of the tile), raw.  Their
  // columns do not wait for the sequence's length. ----
  struct Ids {
    int k, v;
  };
  const int* row_pages = a.table + (size_t)b * a.max_pages;
  const int last_col = a.max_pages - 1;
  const long long begin = (long long)split * a.chunk;
  auto ids_of = [&](int tile) {
    const int at = (int)min(begin + 64LL * tile, 0x7fffffc0LL);
    if constexpr (WIDE) {
      const int p = row_pages[min(at >> a.lp, last_col)];
      return Ids{p, p};
    } else {
      return Ids{row_pages[min((at + 16 * (r16 >> 2)) >> a.lp, last_col)], row_pages[min((at + 16 * g) >> a.lp, last_col)]};
    }
  };
  Ids now = ids_of(wave), next = ids_of(wave + NW);
  const Rows rw = rows_of(a.cu, b, a.T);
  const int n = rw.last - rw.first;
  const int len = cut_len(a.lens[b], a.max_pages, a.lp);
  if (n == 0) return;
  const int t0 = (int)min(begin, (long long)len);
  const int t1 = split + 1 == a.splits ? len : (int)min(begin + a.chunk, (long long)len);
  const float c = fabsf(a.c);
  const uint32_t flip = a.c < 0.f ? 0x80008000u : 0u;  // a negative scale turns q, so that larger scores stay larger

  // lane offsets in a page: of K row 16 (r16 / 4) + r16 % 4, of V's channel r16
  const int k_key = 16 * (r16 >> 2) + (r16 & 3);
  const uint32_t k_off = (uint32_t)(k_key * D + g * (D / 4)), v_off = (uint32_t)(r16 * P + 16 * g);

  for (int r0 = 0; r0 < n * G; r0 += 16 * NR) {
    // ---- this block's rows ----
    u32x4 qf[NR][KC];
    int limit[NR];  // keys that the lane's row sees: t < limit
#pragma unroll
    for (int i = 0; i < NR; ++i) {
      const int r = min(r0 + 16 * i + r16, n * G - 1);
      const int tok = r / G;
      const uint16_t* src = a.q + (size_t)(rw.first + tok) * a.q_stride + (h * G + r % G) * D + g * (D / 4);
#pragma unroll
      for (int k = 0; k < KC; ++k) qf[i][k] = ld128(src + 8 * k) ^ u32x4{flip, flip, flip, flip};
      limit[i] = min(a.causal ? max(len - n + tok + 1, 0) : len, t1);
    }
    // keys that every row of the block sees, and those that any does
    const int low = min(a.causal ? max(len - n + r0 / G + 1, 0) : len, t1);
    const int high = min(a.causal ? max(len - n + min(r0 + 16 * NR - 1, n * G - 1) / G + 1, 0) : len, t1);
    const int tiles = high > t0 ? (high - t0 + 63) / 64 : 0;

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

    // tiles that not every row of the block sees whole start here: at most 3, with a causal mask
    const int first_partial = low > t0 ? (low - t0) / 64 : 0;
    int flagged = 0;
    u32x4 kx[4][KL], vx[DT];
    float ks = 1.f, vs = 1.f;
    // a page that is none reads page 0 and is masked
    auto valid = [&](int p) { return (uint32_t)p < (uint32_t)a.pages; };
    auto load_k = [&](int tile, Ids id) {
      const int at = t0 + 64 * tile;
      const uint8_t* p;
      uint32_t ph;
      if constexpr (WIDE) {
        const int page = __builtin_amdgcn_readfirstlane(id.k);
        ph = (uint32_t)((valid(page) ? page : 0) * a.n_kv + h);
        p = a.kc + ((uint64_t)ph << (a.lp + LD)) + (at & (P - 1)) * D + k_off;
      } else {
        const uint64_t pk = (uint32_t)((valid(id.k) ? id.k : 0) * a.n_kv + h);
        ph = (uint32_t)((valid(id.v) ? id.v : 0) * a.n_kv + h);
        p = a.kc + (pk << (a.lp + LD)) + (uint32_t)(((at + k_key) & (P - 1)) * D + g * (D / 4));
      }
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int u = 0; u < KL; ++u) kx[t][u] = ld128(p + 4 * t * D + 16 * u);
      ks = a.ks[ph];
    };
    auto load_v = [&](int tile, Ids id) {
      const int at = t0 + 64 * tile;
      const uint8_t* p;
      uint32_t ph;
      if constexpr (WIDE) {
        const int page = __builtin_amdgcn_readfirstlane(id.v);
        ph = (uint32_t)((valid(page) ? page : 0) * a.n_kv + h);
        p = a.vc + ((uint64_t)ph << (a.lp + LD)) + (at & (P - 1)) + v_off;
      } else {
        ph = (uint32_t)((valid(id.v) ? id.v : 0) * a.n_kv + h);
        p = a.vc + ((uint64_t)ph << (a.lp + LD)) + (uint32_t)(r16 * P + ((at + 16 * g) & (P - 1)));
      }
#pragma unroll
      for (int d = 0; d < DT; ++d) vx[d] = ld128(p + (size_t)16 * d * P);
      vs = a.vs[ph];
    };

    int tile = wave;
    if (r0 > 0) {
      now = ids_of(tile);
      next = ids_of(tile + NW);
    }
    if (tile < tiles) {
      load_k(tile, now);
      load_v(tile, now);
    }
    // (as a lambda the compiler schedules it better than in the loop: 33 sequences of up to
    // 2000 tokens, d = 64: 25.0 -> 23.5 us)
    auto step = [&](int tile) {
      const int key0 = t0 + 64 * tile + 16 * g;  // the lane's keys: key0 .. key0 + 15
      // also bad: a page behind the sequence's last, whose scales may be anything (WIDE: a tile's
      // one page always holds a token)
      const bool bad = !valid(now.v) || (!WIDE && key0 >= t1);
      const bool masked = t0 + 64 * tile + 64 > low || __any(bad);
      // ---- scores ----
      f32x4 s[NR][4];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
#pragma unroll
        for (int k = 0; k < KC; ++k) {
          const u32x4 kf = widen8<T>(kx[t][k >> 1][2 * (k & 1)], kx[t][k >> 1][2 * (k & 1) + 1]);
#pragma unroll
          for (int i = 0; i < NR; ++i) s[i][t] = mfma16<T>(kf, qf[i][k], k ? s[i][t] : f32x4{});
        }
        __builtin_amdgcn_sched_barrier(0);  // or every fragment is widened before the first product
      }
      const float cs = c * ks, lv = __builtin_amdgcn_logf(vs), iv = 1.0f / vs;
      const Ids after = ids_of(tile + 2 * NW);
      if (tile + NW < tiles) load_k(tile + NW, next);

      // ---- P' ----
      u32x4 pf[NR][2];
#pragma unroll
      for (int i = 0; i < NR; ++i) {
        float mx = -INFINITY;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          float y = __builtin_fmaf(s[i][e >> 2][e & 3], cs, lv);
          if (masked) {
            const bool in = !bad && key0 + e < limit[i];
            seen[i] |= in;
            y = in ? y : -INFINITY;
          }
          s[i][e >> 2][e & 3] = y;
          mx = fmaxf(mx, y);
        }
        if (!masked) seen[i] = true;
        const float top = fmaxf(m[i], max_xor32(max_xor16(mx)));
        const float base = top == -INFINITY ? 0.f : top - lift<T>();
        if (__any(m[i] != top)) {
          const float corr = m[i] == top ? 1.f : __builtin_amdgcn_exp2f(m[i] - top);
          l[i] *= corr;
#pragma unroll
          for (int d = 0; d < DT; ++d) acc[i][d] *= corr;
          m[i] = top;
        }
        float sum = 0.f;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          f32x4 p;
#pragma unroll
          for (int j = 0; j < 4; ++j) p[j] = __builtin_amdgcn_exp2f(s[i][t][j] - base);
          sum += (p[0] + p[1]) + (p[2] + p[3]);
          pf[i][t >> 1][2 * (t & 1)] = T::pack2(p[0], p[1]);
          pf[i][t >> 1][2 * (t & 1) + 1] = T::pack2(p[2], p[3]);
        }
        l[i] += bad ? 0.f : sum * iv;  // 0 * inf: such a page has no scale
      }

      // ---- codes of V that a row does not see must not reach it: 0 * NaN.  Those past the
      // last token or of no page become 0; so do NaNs that only some rows see, which are
      // looked at again behind the loop. ----
      if (masked) {
        const bool partial = a.causal && t0 + 64 * tile + 64 > low;
        bool nan = false;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int w = 0; w < 4; ++w) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (bad || key0 + 4 * w + j >= t1) vx[d][w] &= ~(0xffu << (8 * j));
            if (partial) {
              const uint32_t bits = nan_bytes(vx[d][w]);
              nan |= bits != 0;
              vx[d][w] &= ~spread(bits);
            }
          }
        if (__any(nan)) flagged |= 1 << (tile - first_partial);
      }

      // ---- O^T += V^T P'^T ----
#pragma unroll
      for (int d = 0; d < DT; ++d) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const u32x4 vf = widen8<T>(vx[d][2 * u], vx[d][2 * u + 1]);
#pragma unroll
          for (int i = 0; i < NR; ++i) acc[i][d] = mfma16<T>(vf, pf[i][u], acc[i][d]);
        }
        if (d & 1) __builtin_amdgcn_sched_barrier(0);
      }
      if (tile + NW < tiles) load_v(tile + NW, next);
      now = next;
      next = after;
    };
    for (; tile < tiles; tile += NW) step(tile);

    for (; flagged; flagged &= flagged - 1) {
      const int key = t0 + 64 * (first_partial + __builtin_ctz(flagged)) + 16 * g;
      const int page = key < t1 ? page_of(row_pages, key, a.lp, a.max_pages, a.pages) : -1;
      add_nans<T, D, NR>(acc, limit, a.vc + ((size_t)max(page, 0) * a.n_kv + h) * (size_t)(D * P) + r16 * P + (key & (P - 1)),
                         page >= 0, key, P);
    }

    // ---- the waves' states meet: m and the denominator, then the sums ----
    float* ml = reinterpret_cast<float*>(smem);                         // [NW][NR][16][2]
    f32x4* red = reinterpret_cast<f32x4*>(smem + NW * NR * 16 * 2 * 4);  // [NW][NR][DT][64]
#pragma unroll
    for (int i = 0; i < NR; ++i) {
      l[i] = sum_xor32(sum_xor16(l[i]));
      const bool met = any_group(seen[i]);
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
// Many rows per sequence (prompts and their chunks): a workgroup of TW waves takes 32 TW
// rows (row = token * G + head of the group) of one KV head, 32 a wave, and walks
// the keys in tiles of 64.  A tile's codes go HBM -> registers one tile ahead, are
// widened to 16 bits once per workgroup and written to one of two LDS stages; every
// wave reads its MFMA operands from there.  Rows, keys and channels sit in the lanes as in
// rows_kernel: a lane's 16 keys are a piece of one page, with one set of scales.
//
// 16x16x32 MFMAs: for the same products 32x32x16 ones read and write twice the
// accumulator registers, and the power that takes costs clock.
// ---------------------------------------------------------------------------
constexpr int TW = 8;           // waves
constexpr int TR = 32 * TW;     // rows of a workgroup
constexpr int BN = 64;          // keys of a tile
constexpr int kOdd = 1 << 30;   // in a row's token number: its query holds an infinity or a NaN
// Log2 units that a score may pass the running maximum by before it moves.  f16: what P' has of its
// range above 2^10, so that weights 2^24 below the row's largest are still normal numbers.
template <typename T>
__device__ __forceinline__ constexpr float lazy() {
  return std::is_same<T, BF16>::value ? 8.f : 5.f;
}

template <int D>
struct Stage {
  static constexpr int K = BN * D * 2, V = D * BN * 2;
  static constexpr int V_OFF = 2 * K;                 // two stages of K, three of V
  static constexpr int CONSTS = V_OFF + 3 * V;        // [2][4 groups of 16 keys] x {cs, lv, iv, 0}
  static constexpr int FLAGS = CONSTS + 2 * 4 * 16;   // tiles with a NaN among V's codes
  static constexpr int LDS = FLAGS + 16;
};
// 16-byte slots of a row, swizzled so that the 16 lanes that LDS serves together hit
// different slots of its 256-byte window.  K: a fragment's rows are 16 i + 4 t + 0..3, i = 0..3;
// V: 16 consecutive ones.
template <int D>
__device__ __forceinline__ int k_slot(int row, int slot) {
  return D == 128 ? slot ^ ((row & 3) | ((row >> 4) & 3) << 2) : slot ^ (((row >> 1) & 1) | ((row >> 4) & 3) << 1);
}
__device__ __forceinline__ int v_slot(int row, int slot) { return slot ^ ((row >> 1) & 7); }

// WIDE: pages of 64 tokens and more.  A tile then has one page, whose address the scalar unit
// works out; its threads add an offset that never changes (3 x 2048 rows on 4096 tokens 281 us,
// 290 with pages of 16).  For d = 64 the other form serves every page: 209..212 us, 216..219 this way.
template <typename T, int D, bool WIDE>
__global__ __launch_bounds__(64 * TW, 2) void tile_kernel(const Args a) {
  using L = Stage<D>;
  constexpr int KC = D / 32, DT = D / 16;
  constexpr int NT = 64 * TW;
  constexpr int U = D * 8 / NT;  // 16-byte units of a tile (K, then V) per thread
  constexpr float TOP = lift<T>() > 0.f ? lift<T>() : lazy<T>();  // a larger log2 P' moves the maximum,
  constexpr float LEVEL = TOP - lazy<T>();                        // to here
  static_assert(U >= 1 && U * NT == D * 8, "units");
  extern __shared__ __align__(1024) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r16 = lane & 15, g = lane >> 4;
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
  const int last_col = a.max_pages - 1;
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
    const int w_low = min(sees(min(32 * wave, rows - 1)), s1), w_high = min(sees(min(32 * wave + 31, rows - 1)), s1);
    const bool idle = 32 * wave >= rows;
    int limit[2], tok[2], head[2];
    u32x4 qf[2][KC];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int rr = min(32 * wave + 16 * i + r16, rows - 1);
      limit[i] = min(sees(rr), s1);
      tok[i] = (int)((r0 + rr) / (uint32_t)G);
      head[i] = h * G + (int)((r0 + rr) % (uint32_t)G);
      const uint16_t* src = a.q + (size_t)(rw.first + tok[i]) * a.q_stride + head[i] * D + 8 * g;
#pragma unroll
      for (int k = 0; k < KC; ++k) qf[i][k] = ld128(src + 32 * k) ^ u32x4{flip, flip, flip, flip};
    }

    // ---- a tile's codes: unit id < 4 D: K, row id / (D/16); else V, channel.  Page
    // numbers are looked up a tile before the codes are loaded, those a tile before
    // they are widened.  Past the last tile: zeros into a stage nobody reads. ----
    u32x4 raw[U];
    float rks = 0.f, rvs = 0.f;
    int page_n[U], page_s;
    bool bad[U], bad_s = true;
    auto is_k = [&](int u) { return (u + 1) * NT <= 4 * D ? true : u * NT >= 4 * D ? false : tid + u * NT < 4 * D; };
    auto key_of = [&](int u) {
      const int id = tid + u * NT;
      return is_k(u) ? id / (D / 16) : id % 4 * 16;
    };
    auto offset_of = [&](int u, int slot) {  // of unit u in its page, slot: the token of its first byte
      const int id = tid + u * NT;
      return (uint32_t)(is_k(u) ? slot * D + id % (D / 16) * 16 : (id - 4 * D) / 4 * P + slot);
    };
    uint32_t wide_off[U];
#pragma unroll
    for (int u = 0; u < U; ++u) wide_off[u] = offset_of(u, key_of(u));
    auto find = [&](int tile) {
      const int at = s0 + BN * tile;
      if constexpr (WIDE) {
        page_s = row_pages[min(at >> a.lp, last_col)];
      } else {
#pragma unroll
        for (int u = 0; u < U; ++u) page_n[u] = row_pages[min((at + key_of(u)) >> a.lp, last_col)];
        page_s = row_pages[min((at + 16 * (tid & 3)) >> a.lp, last_col)];
      }
    };
    auto load = [&](int tile) {
      const int at = s0 + BN * tile;
      constexpr int LD = D == 128 ? 7 : 6;
      if constexpr (WIDE) {
        const int page = __builtin_amdgcn_readfirstlane(page_s);
        bad_s = at >= high || (uint32_t)page >= (uint32_t)a.pages;
        const uint32_t ph = (uint32_t)((bad_s ? 0 : page) * a.n_kv + h);
        const uint64_t base = (uint64_t)ph << (a.lp + LD);
        const uint32_t half = at & (P - 1);  // 64 in the second tile of a page of 128
        const uint8_t *kp = a.kc + base + half * D, *vp = a.vc + base + half;
#pragma unroll
        for (int u = 0; u < U; ++u) {
          bad[u] = bad_s || at + key_of(u) >= high;
          raw[u] = ld128((is_k(u) ? kp : vp) + wide_off[u]);
        }
        rks = a.ks[ph];
        rvs = a.vs[ph];
        bad_s |= at + 16 * (tid & 3) >= high;
      } else {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int key = at + key_of(u);
          bad[u] = key >= high || (uint32_t)page_n[u] >= (uint32_t)a.pages;
          const uint64_t page = (uint64_t)(uint32_t)((bad[u] ? 0 : page_n[u]) * a.n_kv + h) << (a.lp + LD);
          raw[u] = ld128((is_k(u) ? a.kc : a.vc) + page + offset_of(u, key & (P - 1)));
        }
        bad_s = at + 16 * (tid & 3) >= high || (uint32_t)page_s >= (uint32_t)a.pages;
        const uint32_t page = (uint32_t)((bad_s ? 0 : page_s) * a.n_kv + h);
        rks = a.ks[page];
        rvs = a.vs[page];
      }
    };
    // Before a loaded tile is stored: the codes of pages that are none become 0.  Tiles from
    // first_masked on are not seen whole by every row: at most TR / 64 + 2 with a causal
    // mask, bits of *flags.  There V's codes of tokens past the last become 0, and so do
    // NaNs, which are flagged (without a causal mask every row sees every token that is
    // there).
    int* flags = reinterpret_cast<int*>(smem + L::FLAGS);
    const int first_masked = low > s0 ? (low - s0) / BN : 0;
    auto clean = [&](int tile) {
      const int at = s0 + BN * tile;
      const bool partial = at + BN > low;
      bool none = false;  // a tile that is seen whole has no keys past the last
      if constexpr (WIDE) {
        none = bad_s;
      } else {
#pragma unroll
        for (int u = 0; u < U; ++u) none |= bad[u];
      }
      if (!partial && !__any(none)) return;
      bool nan = false;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (bad[u]) raw[u] = u32x4{};
        if (partial && !is_k(u)) {
          const int left = high - at - key_of(u);
#pragma unroll
          for (int w = 0; w < 4; ++w) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (4 * w + j >= left) raw[u][w] &= ~(0xffu << (8 * j));
            const uint32_t bits = a.causal ? nan_bytes(raw[u][w]) : 0u;
            nan |= bits != 0;
            raw[u][w] &= ~spread(bits);
          }
        }
      }
      if (__any(nan) && lane == 0) atomicOr(flags, 1 << (tile - first_masked));
    };
    // unit u of the loaded tile into its stage: 16 channels of a K row are its slots 2 i,
    // 2 i + 1, 16 keys of a V row (a lane group's) slots g (keys 0..7) and 4 + g
    uint32_t put[U][2];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int v = 0; v < 2; ++v) {
        const int id = tid + u * NT;
        const int kr = id / (D / 16), vr = (id - 4 * D) / 4;
        put[u][v] = is_k(u) ? kr * (2 * D) + 16 * k_slot<D>(kr, id % (D / 16) * 2 + v)
                            : L::V_OFF + vr * (2 * BN) + 16 * v_slot(vr, id % 4 + 4 * v);
      }
    auto store = [&](int u, int k_st, int v_st) {
      const int st = is_k(u) ? k_st : v_st;
      st128(smem + put[u][0] + st, widen8<T>(raw[u][0], raw[u][1]));
      st128(smem + put[u][1] + st, widen8<T>(raw[u][2], raw[u][3]));
    };
    auto store_consts = [&](int stage) {
      if (tid < 4)
        *reinterpret_cast<f32x4*>(smem + L::CONSTS + (stage * 4 + tid) * 16) =
            f32x4{bad_s ? 0.f : c * rks, bad_s ? -INFINITY : __builtin_amdgcn_logf(rvs),
                  bad_s ? 0.f : __builtin_amdgcn_rcpf(rvs), 0.f};
    };

    // K fragment t: key row 16 (r16 / 4) + 4 t + r16 % 4, slot 4 k + g; V fragment d:
    // channel row 16 d + r16, slot 4 u + g.  The swizzle is an xor, so slot 4 k is an xor away
    // from slot 0.
    const int k_row = 16 * (r16 >> 2) + (r16 & 3);
    const uint32_t k_base = lds0 + k_row * (2 * D) + 16 * k_slot<D>(k_row, g);
    const uint32_t v_base = lds0 + L::V_OFF + r16 * (2 * BN) + 16 * v_slot(r16, g);

    f32x4 acc[2][DT];
    float m[2] = {0.f, 0.f}, l[2] = {0.f, 0.f};
    bool open = true, seen[2] = {false, false};
    u32x4 pf[2][2];  // P' of the tile before, 8 keys of a lane each
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      pf[i][0] = pf[i][1] = u32x4{};
#pragma unroll
      for (int d = 0; d < DT; ++d) acc[i][d] = f32x4{};
    }

    // LDS writes done, then the barrier: no wait for the loads that are under way
    auto meet = [&] {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      lds_barrier();
    };
    __syncthreads();  // the stages and flags are free
    if (tid == 0) *flags = 0;
    if (tiles > 0) {
      // V's last stage, the first tile's "tile before": zeros
      for (int i = tid; i < L::V / 16; i += NT) st128(smem + L::V_OFF + 2 * L::V + 16 * i, u32x4{});
      find(0);
      load(0);
      // A query with an infinity or a NaN: all its scores are infinite or NaN, and its output is NaN if it
      // sees a token, 0 if not.  A page that is none does not hold such scores back (0 * inf), so zeros
      // take the query's place, and kOdd in tok tells the store.  0 times the query, summed, is NaN in
      // each of the row's four lanes.  (Here the tile's codes are waited for anyway: up to 0.4% of a
      // large prompt's time, behind find(1) up to 1.8%.)
      f32x4 x[2] = {};
#pragma unroll
      for (int k = 0; k < KC; ++k)
#pragma unroll
        for (int i = 0; i < 2; ++i) x[i] = mfma16<T>(u32x4{}, qf[i][k], x[i]);
      if (__any(x[0][0] + x[1][0] != 0.f)) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const bool odd = x[i][0] != 0.f;
          tok[i] |= odd ? kOdd : 0;
#pragma unroll
          for (int k = 0; k < KC; ++k) qf[i][k] = odd ? u32x4{} : qf[i][k];
        }
      }
      find(1);
    }
    if (a.causal) __syncthreads();
    if (tiles > 0) {
      clean(0);
#pragma unroll
      for (int u = 0; u < U; ++u) store(u, 0, 0);
      store_consts(0);
      load(1);
      find(2);
    }
    const int mine = idle ? 0 : w_high > s0 ? (w_high - s0 + BN - 1) / BN : 0;  // tiles that the wave's rows see

    // V fragment e: half u = e / DT of the keys, channels d = e % DT
    auto vread = [&](uint32_t vb0, int e) { return lds_ld128((vb0 ^ (64 * (e / DT))) + 16 * (e % DT) * (2 * BN)); };
    // One tile: S^T beside the next tile's widening, then the product of the tile before beside
    // this tile's exponents and their maximum.
    // P' is taken with the maximum as it was: a tile that moves it (or meets a row's first
    // keys) is seen at the vote behind, and its scores are then computed once more.  The
    // exponentials stand before the vote here, but both ways out of it set pn and sum, and the compiler
    // moves them behind it, where the SIMD's other wave covers them with its MFMAs.  That is
    // the faster place: held before the vote, beside the product, with 3, 5 or 6 VALU
    // instructions to an MFMA, three prompts of 2048 on 4096 take 17, 11 or 5% longer, d = 64 1%.
    auto step = [&](int tile, int v_old, int v_new, auto masked_tag) {
      constexpr bool MASKED = decltype(masked_tag)::value;
      const int at = s0 + BN * tile;
      const uint32_t kb0 = k_base + (tile & 1) * L::K, vb0 = v_base + v_old * L::V;
      auto kread = [&](int k, int t) { return lds_ld128((kb0 ^ (64 * k)) + 4 * t * (2 * D)); };

      f32x4 s[2][4];
      u32x4 kb[2][4], vb[DT];
#pragma unroll
      for (int t = 0; t < 4; ++t) kb[0][t] = kread(0, t);
#pragma unroll
      for (int k = 0; k < KC; ++k) {
        if (k + 1 < KC) {
#pragma unroll
          for (int t = 0; t < 4; ++t) kb[(k + 1) & 1][t] = kread(k + 1, t);
        } else {
#pragma unroll
          for (int d = 0; d < DT; ++d) vb[d] = vread(vb0, d);
        }
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int i = 0; i < 2; ++i) s[i][t] = mfma16<T>(kb[k & 1][t], qf[i][k], k ? s[i][t] : f32x4{});
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (k == u * KC / U) store(u, ((tile + 1) & 1) * L::K, v_new * L::V);
        if (k == KC - 1) {
          store_consts((tile + 1) & 1);
          load(tile + 2);
          find(tile + 3);
        }
        __builtin_amdgcn_sched_barrier(0);
      }

      // from here to the vote a wave goes before the other one of its SIMD, which then stages and
      // computes scores meanwhile (512 rows on 4096 tokens 59 -> 57 us; 3 VALU instructions to an MFMA
      // at d = 128 and 8 at 64, with 4 each 1-2% slower)
      __builtin_amdgcn_s_setprio(1);
      const f32x4 cst = *reinterpret_cast<const f32x4*>(smem + L::CONSTS + ((tile & 1) * 4 + g) * 16);
      auto exponents = [&](int i) {  // y - m, masked; the lane's maximum
        const float off = cst[1] - m[i];
        float mx = -INFINITY;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          float x = __builtin_fmaf(s[i][e >> 2][e & 3], cst[0], off);
          if constexpr (MASKED) x = at + 16 * g + e < limit[i] ? x : -INFINITY;
          s[i][e >> 2][e & 3] = x;
          mx = fmaxf(mx, x);
        }
        return mx;
      };
      u32x4 pn[2][2];
      float sum[2];
      auto expo = [&](int i) {
        sum[i] = 0.f;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          f32x4 p;
#pragma unroll
          for (int j = 0; j < 4; ++j) p[j] = __builtin_amdgcn_exp2f(s[i][t][j]);
          sum[i] += (p[0] + p[1]) + (p[2] + p[3]);
          pn[i][t >> 1][2 * (t & 1)] = T::pack2(p[0], p[1]);
          pn[i][t >> 1][2 * (t & 1) + 1] = T::pack2(p[2], p[3]);
        }
      };
      float mx[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        mx[i] = exponents(i);
        expo(i);
      }
#pragma unroll
      for (int e = 0; e < 2 * DT; ++e) {
#pragma unroll
        for (int i = 0; i < 2; ++i) acc[i][e % DT] = mfma16<T>(vb[e % DT], pf[i][e / DT], acc[i][e % DT]);
        if (e + DT < 2 * DT) vb[e % DT] = vread(vb0, e + DT);
      }
#pragma unroll
      for (int e = 0; e < 4 * DT; ++e) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        if (e & 1) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x002, D == 128 ? 3 : 8, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_setprio(0);

      const bool moved = __any(fmaxf(mx[0], mx[1]) > TOP);
      if (moved || open) {
#pragma unroll
        for (int k = 0; k < KC; ++k)
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            const u32x4 kf = kread(k, t);
#pragma unroll
            for (int i = 0; i < 2; ++i) s[i][t] = mfma16<T>(kf, qf[i][k], k ? s[i][t] : f32x4{});
            __builtin_amdgcn_sched_barrier(0);
          }
        bool still = false;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          mx[i] = exponents(i);
          mx[i] = max_xor32(max_xor16(mx[i]));
          const bool empty = open && sum_xor32(sum_xor16(l[i])) == 0.f, met = mx[i] > -INFINITY;
          const float shift = empty ? (met ? mx[i] - LEVEL : 0.f) : mx[i] > TOP ? mx[i] - LEVEL : 0.f;
          still |= empty && !met;
          seen[i] |= cst[1] > -INFINITY && at + 16 * g < limit[i];
          m[i] += shift;
          const float corr = empty ? 1.f : __builtin_amdgcn_exp2f(-shift);
          l[i] *= corr;
#pragma unroll
          for (int d = 0; d < DT; ++d) acc[i][d] *= corr;
#pragma unroll
          for (int e = 0; e < 16; ++e) s[i][e >> 2][e & 3] -= shift;
          expo(i);
        }
        open = __any(still);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        l[i] = __builtin_fmaf(sum[i], cst[2], l[i]);
        pf[i][0] = pn[i][0];
        pf[i][1] = pn[i][1];
      }
    };
    auto last = [&](int v_old) {  // the product of the wave's last tile
      const uint32_t vb0 = v_base + v_old * L::V;
#pragma unroll
      for (int e = 0; e < 2 * DT; ++e) {
        const u32x4 vf = vread(vb0, e);
#pragma unroll
        for (int i = 0; i < 2; ++i) acc[i][e % DT] = mfma16<T>(vf, pf[i][e / DT], acc[i][e % DT]);
      }
    };
    // tiles that every row of the wave sees whole, those that some rows see in part, and
    // those that only other waves need: three loops, so that each has one path
    int v_old = 2, v_now = 0, v_new = 1;  // V's stages of the tile before, this one and the next
    auto next = [&] {
      const int v = v_old;
      v_old = v_now;
      v_now = v_new;
      v_new = v;
    };
    const int whole = w_low > s0 ? min((w_low - s0) / BN, mine) : 0;
    int tile = 0;
    for (; tile < whole; ++tile, next()) {
      meet();  // the tile's stages are written; K's other one and V's next are read
      clean(tile + 1);
      step(tile, v_old, v_new, std::false_type{});
    }
    for (; tile < mine; ++tile, next()) {
      meet();
      clean(tile + 1);
      step(tile, v_old, v_new, std::true_type{});
    }
    if (mine > 0) last(v_old);
    for (; tile < tiles; ++tile, next()) {
      meet();
      clean(tile + 1);
#pragma unroll
      for (int u = 0; u < U; ++u) store(u, ((tile + 1) & 1) * L::K, v_new * L::V);
      store_consts((tile + 1) & 1);
      load(tile + 2);
      find(tile + 3);
    }

    // ---- a NaN among V's codes that some row does not see: those that it does see are
    // counted, by channel and row, with the products' own layout ----
    if (a.causal) {
      meet();
      for (int flagged = *flags; flagged; flagged &= flagged - 1) {
        const int key = s0 + BN * (first_masked + __builtin_ctz(flagged)) + 16 * g;  // the lane's keys
        const int page = key < high ? page_of(row_pages, key, a.lp, a.max_pages, a.pages) : -1;
        add_nans<T, D, 2>(acc, limit, a.vc + ((size_t)max(page, 0) * a.n_kv + h) * (size_t)(D * P) + r16 * P + (key & (P - 1)),
                          page >= 0, key, P);
      }
    }

    // ---- store: the lane's query, d = 16 dt + 4 g + j ----
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float total = sum_xor32(sum_xor16(l[i]));
      const bool met = any_group(seen[i]);
      if (32 * wave + 16 * i + r16 >= rows) continue;
      const size_t orow = (size_t)(rw.first + (tok[i] & ~kOdd)) * a.n_q + head[i];
      const bool none = total == 0.f && !met;
      if ((tok[i] & kOdd) && !none) total = __builtin_nanf("");
      if (a.splits == 1) {
        const float inv = none ? 0.f : 1.0f / total;
#pragma unroll
        for (int d = 0; d < DT; ++d)
          st64(a.out + orow * D + 16 * d + 4 * g, u32x2{T::pack2(acc[i][d][0] * inv, acc[i][d][1] * inv),
                                                        T::pack2(acc[i][d][2] * inv, acc[i][d][3] * inv)});
      } else {
        const size_t all = (size_t)a.T * a.n_q;
        float* p = a.part + ((size_t)split * all + orow) * D;
#pragma unroll
        for (int d = 0; d < DT; ++d) *reinterpret_cast<f32x4*>(p + 16 * d + 4 * g) = acc[i][d];
        if (g == 0) {
          float* ml = a.part + (size_t)a.splits * all * D + ((size_t)split * all + orow) * 2;
          ml[0] = none ? -INFINITY : total == 0.f ? kNoScore : m[i];
          ml[1] = total;
        }
      }
    }
  }
}

// ---------------------------------------------------------------------------
// The splits' partial results of a row meet: WAVES waves per row, D / 4 lanes per split, so
// that the splits' loads are under way together.
// ---------------------------------------------------------------------------
constexpr int CT = 256;  // threads
template <typename T, int D, int WAVES>
__global__ __launch_bounds__(CT) void combine_kernel(const Args a) {
  constexpr int LANES = D / 4, GROUPS = 64 * WAVES / LANES, ROWS = CT / 64 / WAVES;
  __shared__ f32x4 sums[ROWS][GROUPS][LANES];
  __shared__ float2 state[ROWS][GROUPS];  // m and the denominator
  const int own = threadIdx.x / (64 * WAVES), grp = threadIdx.x / LANES % GROUPS, c = threadIdx.x % LANES;
  const size_t rows = (size_t)a.T * a.n_q, at = (size_t)blockIdx.x * ROWS + own;
  const size_t r = at < rows ? at : rows - 1;
  bool live = at < rows;
  if (a.cu) {  // else no sequence's row
    const int tok = (int)(r / a.n_q);
    live = live && tok >= a.cu[0] && tok < a.cu[a.B];
  }
  const float2* ml = reinterpret_cast<const float2*>(a.part + (size_t)a.splits * rows * D);
  float top = -INFINITY, total = 0.f;
  f32x4 o{};
  if (live) {
#pragma unroll 4
    for (int s = grp; s < a.splits; s += GROUPS) {
      const float2 x = ml[(size_t)s * rows + r];
      const f32x4 v = *reinterpret_cast<const f32x4*>(a.part + ((size_t)s * rows + r) * D + 4 * c);
      if (x.x == -INFINITY) continue;  // no visible token: nothing was summed
      const float up = fmaxf(top, x.x);
      const float w0 = top == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(top - up), w1 = __builtin_amdgcn_exp2f(x.x - up);
      total = total * w0 + x.y * w1;
      o = o * w0 + v * w1;
      top = up;
    }
  }
  sums[own][grp][c] = o;
  if (c == 0) state[own][grp] = float2{top, total};
  __syncthreads();
  if (grp > 0 || !live) return;
  float most = -INFINITY;
#pragma unroll
  for (int k = 0; k < GROUPS; ++k) most = fmaxf(most, state[own][k].x);
  total = 0.f;
  o = f32x4{};
#pragma unroll
  for (int k = 0; k < GROUPS; ++k) {
    const float2 x = state[own][k];
    if (x.x == -INFINITY) continue;
    const float w = __builtin_amdgcn_exp2f(x.x - most);
    total += w * x.y;
    o += w * sums[own][k][c];
  }
  o *= most == -INFINITY ? 0.f : 1.0f / total;
  st64(a.out + r * D + 4 * c, u32x2{T::pack2(o[0], o[1]), T::pack2(o[2], o[3])});
}

// ---------------------------------------------------------------------------
// Launch choice
// ---------------------------------------------------------------------------
struct Plan {
  int nr;       // 16-row blocks of the rows kernel; 0: the tile kernel
  int tiles;    // 256-row tiles of the tile kernel
  int splits, chunk;
};

static long long up(long long x, long long to) { return (x + to - 1) / to; }

// The rows kernel up to 32 rows a KV head, else the tile kernel.  The keys are split
// where there are fewer workgroups than CUs.  A split costs its workgroup's start and
// end, some 250 tokens' worth, and the combine's launch, so chunks are as long as the GPU
// stays filled: rows kernel, one workgroup per CU while sequences times KV heads are
// few, two from 128 on (chunks of 256, 512, 1024, 2048 and 4096 tokens: B4 of 4096 tokens 14.6, 13.8,
// 16.8, 23.1, 33.8 us; B32 59, 47, 42, 38, 41), and at most 4096 tokens, which keeps sequences of
// different lengths apart (B64 of up to 8192: 218, 174, 154, 147, 149).  Up to 512 tokens of
// 128, 1024 of 64, one workgroup is as fast as two and the combine (B1..16, us: d = 128, 512
// tokens 9.1..10.9 and 10.0..12.0, 768 tokens 10.7..12.6 and 10.0..14.0; d = 64, 512 tokens
// 6.4..7.5 and 8.3..9.6, 1001 tokens 9.3..9.5 and 9.2..10.5).  Tile kernel: one per
// CU, chunks a multiple of 128 (256: 512 rows on 4096 tokens 63.6 us, not 61.7; 64 on 1024
// 25.8, not 23.4; 64: as 128).
static Plan plan(int B, int T, int max_q, int max_kv, int n_q, int n_kv, int d) {
  const long long rows = (long long)(max_q < T ? max_q : T) * (n_q / n_kv), heads = (long long)B * n_kv;
  Plan p;
  p.nr = rows <= 16 ? 1 : rows <= 32 ? 2 : 0;
  p.tiles = (int)std::min(up(rows, TR), 65535LL);
  long long chunk;
  if (p.nr) {
    chunk = up(up(heads * max_kv, heads >= 128 && rows_per_cu(p.nr, d) == 2 ? 512 : 256), 256) * 256;
    chunk = std::min(chunk, 4096LL);
    if ((long long)max_kv * d <= 65536) chunk = max_kv;
  } else {
    chunk = up(max_kv, up(256, heads * p.tiles));
    chunk = up(chunk, 128) * 128;
  }
  p.splits = (int)std::min(up(max_kv, chunk), 65535LL);
  p.chunk = (int)std::min(chunk, 0x40000000LL);
  return p;
}

template <typename T, int D, int NR, bool WIDE>
static int launch_rows(const Args& a, hipStream_t s) {
  constexpr int lds = NW * NR * (16 * 2 * 4 + (D / 16) * 64 * 16);
  MX_RETURN_IF_HIP((lds_limit_once<rows_kernel<T, D, NR, WIDE>>(lds)));
  hipLaunchKernelGGL((rows_kernel<T, D, NR, WIDE>), dim3((unsigned)(a.B * a.n_kv), (unsigned)a.splits), dim3(64 * NW), lds, s, a);
  MX_RETURN_IF_HIP(hipGetLastError());
  return MX_OK;
}

template <typename T, int D, bool WIDE>
static int launch_tiles(const Args& a, const Plan& p, hipStream_t s) {
  constexpr int lds = Stage<D>::LDS;
  MX_RETURN_IF_HIP((lds_limit_once<tile_kernel<T, D, WIDE>>(lds)));
  hipLaunchKernelGGL((tile_kernel<T, D, WIDE>), dim3((unsigned)(a.B * a.n_kv), (unsigned)p.tiles, (unsigned)a.splits),
                     dim3(64 * TW), lds, s, a);
  MX_RETURN_IF_HIP(hipGetLastError());
  return MX_OK;
}

template <typename T, int D>
static int run(const Args& a, const Plan& p, hipStream_t s) {
  const bool wide = a.lp >= 6;
  const int rc = p.nr == 1   ? (wide ? launch_rows<T, D, 1, true>(a, s) : launch_rows<T, D, 1, false>(a, s))
                 : p.nr == 2 ? (wide ? launch_rows<T, D, 2, true>(a, s) : launch_rows<T, D, 2, false>(a, s))
                 : wide && D == 128 ? launch_tiles<T, D, D == 128>(a, p, s)
                                    : launch_tiles<T, D, false>(a, p, s);
  if (rc != MX_OK || p.splits == 1) return rc;
  const long long rows = (long long)a.T * a.n_q;
  // few rows: the splits of a row side by side; many: few splits each (of 16384 rows in 2
  // splits 17 us with 4 waves a row, 8.8 with one)
  if (rows < 2048)
    hipLaunchKernelGGL((combine_kernel<T, D, 4>), dim3((unsigned)rows), dim3(CT), 0, s, a);
  else
    hipLaunchKernelGGL((combine_kernel<T, D, 1>), dim3((unsigned)up(rows, 4)), dim3(CT), 0, s, a);
  MX_RETURN_IF_HIP(hipGetLastError());
  return MX_OK;
}

// A launch has fewer than 2^32 threads in x: 512 a workgroup here, 64 a row in the combine.
static bool sizes_ok(int B, int T, int max_q, int max_kv, int n_q, int n_kv, int d) {
  return B > 0 && T > 0 && max_q > 0 && max_kv > 0 && n_q > 0 && n_kv > 0 && n_q % n_kv == 0 && (d == 64 || d == 128) &&
         (long long)B * n_kv <= (1 << 22) && (long long)T * n_q <= (1 << 25) && (long long)n_q * d <= 0x7fffffffLL;
}

}  // namespace kv8
}  // namespace mx

extern "C" size_t mx_gqa_kv8_workspace(int B, int T, int max_q, int max_kv, int n_q, int n_kv, int d) {
  using namespace mx::kv8;
  if (!sizes_ok(B, T, max_q, max_kv, n_q, n_kv, d)) return 0;
  const Plan p = plan(B, T, max_q, max_kv, n_q, n_kv, d);
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
  if (!sizes_ok(B, T, max_q, max_kv, n_q, n_kv, d) || (!cu && T != B)) return MX_ERR_SHAPE;
  if (max_pages <= 0 || (long long)max_pages * page > kMostTokens) return MX_ERR_SHAPE;
  if (q_stride < n_q * d) return MX_ERR_SHAPE;
  if (q_stride % 8 || (((uintptr_t)q | (uintptr_t)O) & 15)) return MX_ERR_ALIGN;
  if (dtype != MX_DTYPE_BF16 && dtype != MX_DTYPE_F16) return MX_ERR_DTYPE;
  const Plan p = plan(B, T, max_q, max_kv, n_q, n_kv, d);
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
