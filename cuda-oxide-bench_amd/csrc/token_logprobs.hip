// Log probabilities of given tokens, the entropy and the top alternatives of rows of logits, for gfx950.
//
//     y[v] = x[v] - m,  m = the row's largest
//     S = sum exp(y),  E = sum exp(y) y
//     log p[v] = y[v] - log S,  entropy = -sum p log p = log S - E / S
// in one pass: each thread holds m, S and E of what it has read, in fp32, and rescales them where its maximum
// moves (S by f = exp(m - m'), E by f and by f S (m - m')).  The threads', waves' and slices' states meet by the
// same rule.  (x - m first, then log2(e): with x log2(e) - m log2(e) in one FMA the rounding of the second
// product, 2^-24 of it, would pass every exponent's range for masks like -1e30.)
//
// The alternatives: a key per logit orders them (the value's bits, made to rise with it, above the complement of
// its place, so that ties go to the lowest id).  A wave keeps its best 64 keys sorted across its lanes.  A logit that
// reaches the bar, a bound on the k-th best that only rises, waits in LDS by its place; 64 of them are
// sorted and merged in at a time, and raise the bar.  It is the k-th of the wave's list (before there is one, of its
// lanes' maxima), or what the workgroup's W waves know together: the largest k-th of theirs, the least
// (k/W)-th.  -inf never reaches it: a row with fewer than k others has its lowest ids of -inf behind them.
//
// A workgroup takes a row, one of 16 waves where there are few; where those few are long a row is cut into slices, which
// a second kernel joins.
#include <algorithm>

#include "mx_common.h"

namespace mx {
namespace logprobs {

constexpr int kMostTop = 32;
constexpr int kMostSlices = 16;
constexpr float kLog2e = 1.4426950408889634f;

struct Args {
  const void* x;
  const int* tokens;
  float *logprob, *entropy;
  int* ids;
  float* top_logprob;
  float4* states;  // [T][slices]: m, S, E
  uint64_t* keys;  // [T][slices][top]
  int V, given, top, slices, per;  // per: 16-byte blocks of a slice
  long long stride;
};

struct F32 {};
template <typename T>
constexpr int kBytes = std::is_same<T, F32>::value ? 4 : 2;

// A dword of -inf.
template <typename T>
constexpr uint32_t kNone = std::is_same<T, F32>::value ? 0xff800000u : std::is_same<T, BF16>::value ? 0xff80ff80u : 0xfc00fc00u;

template <typename T>
__device__ __forceinline__ float at(const void* row, int v) {
  if constexpr (std::is_same<T, F32>::value) return ((const float*)row)[v];
  else return T::to_f32(((const uint16_t*)row)[v]);
}

// ---- lanes ----
template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, CTRL, 0xf, 0xf, false);
}
// v of lane l ^ J
template <int J>
__device__ __forceinline__ uint32_t lane_xor(uint32_t v, int lane) {
  if constexpr (J == 1) return dpp<0xB1>(v);
  else if constexpr (J == 2) return dpp<0x4E>(v);
  else if constexpr (J == 4) return dpp<0x1B>(dpp<0x141>(v));  // 7 - l of 8, then 3 - l of 4
  else if constexpr (J == 8) return dpp<0x128>(v);
  else if constexpr (J == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return lane & 16 ? r[0] : r[1];
  } else {
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return lane & 32 ? r[0] : r[1];
  }
}
template <int J>
__device__ __forceinline__ uint64_t lane_xor64(uint64_t v, int lane) {
  return (uint64_t)lane_xor<J>((uint32_t)(v >> 32), lane) << 32 | lane_xor<J>((uint32_t)v, lane);
}
template <int J>
__device__ __forceinline__ float lane_xorf(float v, int lane) {
  return __uint_as_float(lane_xor<J>(__float_as_uint(v), lane));
}

// Sorted across the lanes, the largest first.  A bitonic network: a stage J meets the lane J away, and keeps the larger
// where both its bit J and the direction of its block of SIZE say so.
constexpr uint64_t lanes_of_larger(int size, int j) {
  uint64_t m = 0;
  for (int l = 0; l < 64; ++l)
    if (((l & j) == 0) == ((l & size) == 0)) m |= 1ull << l;
  return m;
}
template <int SIZE, int J>
__device__ __forceinline__ bool keeps_larger() {  // a constant per lane: scalar registers, not kept between stages
  constexpr uint64_t m = lanes_of_larger(SIZE, J);
  return __builtin_amdgcn_inverse_ballot_w64(m);
}
template <int SIZE, int J>
__device__ __forceinline__ void stage(uint64_t& v, int lane) {
  const uint64_t o = lane_xor64<J>(v, lane);
  v = (o > v) == keeps_larger<SIZE, J>() ? o : v;
}
template <int SIZE, int J = SIZE / 2>
__device__ __forceinline__ void merge(uint64_t& v, int lane) {
  stage<SIZE, J>(v, lane);
  if constexpr (J > 1) merge<SIZE, J / 2>(v, lane);
}
template <int SIZE = 2>
__device__ __forceinline__ void sort(uint64_t& v, int lane) {
  merge<SIZE>(v, lane);
  if constexpr (SIZE < 64) sort<2 * SIZE>(v, lane);
}
// The same of plain floats.
template <int SIZE = 2, int J = 1>
__device__ __forceinline__ void sort_floats(float& v, int lane) {
  const float o = lane_xorf<J>(v, lane);
  v = keeps_larger<SIZE, J>() ? fmaxf(v, o) : fminf(v, o);
  if constexpr (J > 1) sort_floats<SIZE, J / 2>(v, lane);
  else if constexpr (SIZE < 64) sort_floats<2 * SIZE, SIZE>(v, lane);
}
// v of lane 63 - l
__device__ __forceinline__ uint64_t reversed(uint64_t v, int lane) {
  const uint32_t hi = (uint32_t)__shfl((int)(v >> 32), 63 - lane, 64), lo = (uint32_t)__shfl((int)v, 63 - lane, 64);
  return (uint64_t)hi << 32 | lo;
}
// The best 64 of two sorted lists, sorted.
__device__ __forceinline__ void take_best(uint64_t& list, uint64_t other, int lane) {
  const uint64_t o = reversed(other, lane);
  list = o > list ? o : list;
  merge<64>(list, lane);
}

__device__ __forceinline__ uint64_t key_of(float x, int v) {
  const uint32_t bits = __float_as_uint(x + 0.f);  // -0 as 0
  return (uint64_t)(bits & 0x80000000u ? ~bits : bits | 0x80000000u) << 32 | (uint32_t)~v;
}
__device__ __forceinline__ float value_of(uint64_t key) {
  const uint32_t bits = (uint32_t)(key >> 32);
  return __uint_as_float(bits & 0x80000000u ? bits & 0x7fffffffu : ~bits);
}
__device__ __forceinline__ uint64_t broadcast(uint64_t v, int lane) {
  return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32 |
         (uint32_t)__builtin_amdgcn_readlane((int)v, lane);
}

// What the wave's lanes wrote to LDS, before other lanes of it read that: the LDS serves a wave in order, and the
// compiler is held to that order here.
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

__device__ __forceinline__ float uniform(float v) {
  return __uint_as_float((uint32_t)__builtin_amdgcn_readfirstlane((int)__float_as_uint(v)));
}

// ---- the softmax's state ----
struct State {
  float m, s, e;
};
// With a maximum of m: what was summed below another one.
__device__ __forceinline__ void move_to(State& st, float m) {
  if (st.m == m || m == -INFINITY) return;
  const float shift = st.m - m;  // -inf where nothing was summed
  const float f = __builtin_amdgcn_exp2f(shift * kLog2e);
  st.e = f == 0.f ? 0.f : f * __builtin_fmaf(st.s, shift, st.e);
  st.s *= f;
  st.m = m;
}
__device__ __forceinline__ void join(State& st, State o) {
  const float m = fmaxf(st.m, o.m);
  move_to(st, m);
  move_to(o, m);
  st.s += o.s;
  st.e += o.e;
}
template <int J = 32>
__device__ __forceinline__ float lanes_max(float v, int lane) {
  v = fmaxf(v, lane_xorf<J>(v, lane));
  if constexpr (J > 1) return lanes_max<J / 2>(v, lane);
  else return v;
}
template <int J = 32>
__device__ __forceinline__ float lanes_sum(float v, int lane) {
  v += lane_xorf<J>(v, lane);
  if constexpr (J > 1) return lanes_sum<J / 2>(v, lane);
  else return v;
}
// The lanes' states in every lane: each moves to the largest maximum once.
__device__ __forceinline__ void join_lanes(State& st, int lane) {
  move_to(st, lanes_max(st.m, lane));
  st.s = lanes_sum(st.s, lane);
  st.e = lanes_sum(st.e, lane);
}

// What a wave has of the alternatives.
constexpr float kLowest = -3.402823466e38f;
struct Best {
  uint64_t list = 0;    // sorted across the lanes; 0: none
  float bar = kLowest;  // logits below it cannot be among them
  int waiting = 0;      // places in LDS that are not merged yet, below 64
};
// In LDS, of each wave: places that wait, and what it knows: its k-th and its (k/NW)-th value, or values below them.
template <int NW>
struct Shared {
  int wait[NW][128];
  uint64_t known[NW];  // the k-th's bits above the (k/NW)-th's
};
template <int NW>
__device__ __forceinline__ void tell(Shared<NW>& sh, int wave, float kth, float part, int lane) {
  if (lane == 0)
    __hip_atomic_store(&sh.known[wave], (uint64_t)__float_as_uint(kth) << 32 | __float_as_uint(part), __ATOMIC_RELAXED,
                       __HIP_MEMORY_SCOPE_WORKGROUP);
}

template <typename T, int NW>
__device__ __forceinline__ void merge_in(Best& best, Shared<NW>& sh, int wave, int n, int top, const void* row, int lane) {
  wave_sync();
  uint64_t v = 0;
  if (lane < n) {
    const int place = sh.wait[wave][lane];
    v = key_of(at<T>(row, place), place);
  }
  sort(v, lane);
  if (__any(best.list != 0)) take_best(best.list, v, lane);
  else best.list = v;
  const uint64_t kth = broadcast(best.list, top - 1);
  if (!kth) return;
  tell(sh, wave, value_of(kth), value_of(broadcast(best.list, (top - 1) / NW)), lane);
  // what comes has larger ids than the list: it must be above the k-th's value
  best.bar = uniform(fmaxf(best.bar, value_of((kth | 0xffffffffu) + 1)));
}
// The others may know more.
template <int NW>
__device__ __forceinline__ void raise_bar(Best& best, Shared<NW>& sh, int lane) {
  const uint64_t k = __hip_atomic_load(&sh.known[lane % NW], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
  const float most = lanes_max<NW / 2>(__uint_as_float((uint32_t)(k >> 32)), lane);
  const float least = -lanes_max<NW / 2>(-__uint_as_float((uint32_t)k), lane);
  best.bar = uniform(fmaxf(best.bar, fmaxf(most, least)));
}

// The lane's logits of a chunk that reach the bar are `good`, bit j the place first + j / EB * apart + j % EB.
template <typename T, int EB, int NW>
__device__ __forceinline__ void offer(Best& best, Shared<NW>& sh, uint32_t good, int first, int apart, int top, const void* row,
                                      int wave, int lane) {
  for (;; good &= good - 1) {  // each lane's first, then its second
    const uint64_t who = __ballot(good != 0);
    if (!who) break;
    const int j = __builtin_ctz(good | 0x80000000u);
    if (good)
      sh.wait[wave][best.waiting + __builtin_amdgcn_mbcnt_hi((uint32_t)(who >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0))] =
          first + j / EB * apart + j % EB;
    best.waiting += __popcll(who);
    if (best.waiting >= 64) {
      merge_in<T>(best, sh, wave, 64, top, row, lane);
      const int rest = sh.wait[wave][64 + lane];
      best.waiting -= 64;
      wave_sync();
      sh.wait[wave][lane] = rest;
    }
  }
}

// One chunk, x[u] the EB logits from place first + u * apart on (-inf where there are none), into the state and the
// alternatives.
template <typename T, bool TOP, int U, int EB, int NW>
__device__ __forceinline__ void take(State& st, Best& best, Shared<NW>& sh, const float (&x)[U][EB], int first, int apart, int top,
                                     const void* row, int wave, int lane) {
  float block[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    block[u] = x[u][0];
#pragma unroll
    for (int j = 1; j < EB; ++j) block[u] = fmaxf(block[u], x[u][j]);
  }
  float most = block[0];
#pragma unroll
  for (int u = 1; u < U; ++u) most = fmaxf(most, block[u]);
  if (__any(most > st.m)) move_to(st, fmaxf(most, st.m));
  const float off = st.m == -INFINITY ? 0.f : st.m;
  float s[4] = {}, e[4] = {};
#pragma unroll
  for (int u = 0; u < U; ++u) {
#pragma unroll
    for (int j = 0; j < EB; ++j) {
      const float y = x[u][j] - off;
      const float p = __builtin_amdgcn_exp2f(y * kLog2e);
      s[j % 4] += p;
      e[j % 4] = __builtin_fmaf(p, fmaxf(y, kLowest), e[j % 4]);  // not 0 times -inf
    }
    __builtin_amdgcn_sched_barrier(0);  // or the exponentials of all blocks are held at once, in registers that cost a wave
  }
  st.s += (s[0] + s[1]) + (s[2] + s[3]);
  st.e += (e[0] + e[1]) + (e[2] + e[3]);
  if constexpr (TOP) {
    if (best.bar == kLowest) {  // at least `top` logits reach the k-th of the lanes' maxima
      float v = most;
      sort_floats(v, lane);
      const float kth = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), top - 1));
      tell(sh, wave, kth, __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), (top - 1) / NW)), lane);
      best.bar = uniform(fmaxf(best.bar, kth));
    }
    if (__any(most >= best.bar)) {
      uint32_t good = 0;
#pragma unroll
      for (int u = U - 1; u >= 0; --u) {
        if (__any(block[u] >= best.bar)) {
#pragma unroll
          for (int j = EB - 1; j >= 0; --j) good = good << 1 | (x[u][j] >= best.bar ? 1u : 0u);
        } else {
          good <<= EB;
        }
      }
      offer<T, EB>(best, sh, good, first, apart, top, row, wave, lane);
    }
  }
}

// A given token's logit, read ahead of its use: NaN where the number is no token.
template <typename T>
__device__ __forceinline__ float given_logit(const Args& a, const void* x, size_t row, int i) {
  const int v = a.tokens[row * a.given + i];
  return (uint32_t)v < (uint32_t)a.V ? at<T>(x, v) : __builtin_nanf("");
}

// A row's answers, by one wave, from its state (in every lane), its best keys and the lane's given token's logit.
template <typename T>
__device__ __forceinline__ void answer(const Args& a, const State& st, uint64_t key, float asked, const void* x, size_t row,
                                       int lane) {
  const bool none = !(st.s > 0.f && st.s < INFINITY);  // a NaN, +inf, nothing but -inf: no distribution
  const float log_s = logf(st.s), nan = __builtin_nanf("");
  for (int i = lane; i < a.given; i += 64) {
    if (i >= 64) asked = given_logit<T>(a, x, row, i);
    a.logprob[row * a.given + i] = none ? nan : (asked - st.m) - log_s;
  }
  if (lane == 0) a.entropy[row] = none ? nan : log_s - st.e / st.s;
  int n = __popcll(__ballot(key != 0));
  if (n < a.top && !none) {  // the rest are -inf: their lowest ids, which are among the first 64
    uint64_t who = __ballot(lane < a.V && at<T>(x, min(lane, a.V - 1)) == -INFINITY);
    for (; n < a.top; ++n, who &= who - 1)
      if (lane == n) key = key_of(-INFINITY, __builtin_ctzll(who));
  }
  if (lane < a.top) {
    a.ids[row * a.top + lane] = none ? -1 : (int)~(uint32_t)key;
    a.top_logprob[row * a.top + lane] = none ? nan : (value_of(key) - st.m) - log_s;
  }
}

template <int J, bool MOST>
__device__ __forceinline__ uint64_t extreme(uint64_t v, int lane) {
  const uint64_t o = lane_xor64<J>(v, lane);
  v = (o > v) == MOST ? o : v;
  if constexpr (J > 1) return extreme<J / 2, MOST>(v, lane);
  else return v;
}
// The best of `lists` sorted lists of `top` keys each (up to 64 lists), by one wave; wait: 128 keys of LDS.
__device__ __forceinline__ uint64_t join_lists(const uint64_t* keys, int lists, int top, uint64_t* wait, int lane) {
  const int all = lists * top;
  constexpr int N = 8;  // reads under way
  uint64_t key[N], list = 0;
  auto load = [&](int i) {
#pragma unroll
    for (int n = 0; n < N; ++n) key[n] = keys[min(i + 64 * n + lane, all - 1)];
  };
  // no key below the largest of the lists' last ones counts, nor below the least of their (top / lists)-th
  const uint64_t last = lane < lists ? keys[lane * top + top - 1] : 0;
  const uint64_t part = lane < lists ? keys[lane * top + (top - 1) / lists] : ~0ull;
  load(0);
  uint64_t bar = extreme<32, true>(last, lane);
  const uint64_t least = extreme<32, false>(part, lane);
  bar = least > bar ? least : bar;
  int waiting = 0;
  auto merge_some = [&](int n) {
    wave_sync();
    uint64_t v = lane < n ? wait[lane] : 0;
    sort(v, lane);
    if (__any(list != 0)) take_best(list, v, lane);
    else list = v;
  };
  for (int i = 0; i < all; i += 64 * N) {
    if (i) load(i);
#pragma unroll 1
    for (int n = 0; n < N && i + 64 * n < all; ++n) {
      const bool good = i + 64 * n + lane < all && key[0] && key[0] >= bar;
      const uint64_t who = __ballot(good);
      if (good)
        wait[waiting + __builtin_amdgcn_mbcnt_hi((uint32_t)(who >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0))] = key[0];
      waiting += __popcll(who);
      if (waiting >= 64) {
        merge_some(64);
        const uint64_t rest = wait[64 + lane];
        waiting -= 64;
        wave_sync();
        wait[lane] = rest;
      }
#pragma unroll
      for (int m = 0; m + 1 < N; ++m) key[m] = key[m + 1];
    }
  }
  if (waiting) merge_some(waiting);
  return list;
}

template <typename T, bool TOP, int NT>
__global__ __launch_bounds__(NT) void rows_kernel(const Args a) {
  constexpr int NW = NT / 64;
  constexpr int EB = 16 / kBytes<T>;  // logits of a block
  constexpr int U = 4;                // blocks of a chunk and thread
  __shared__ Shared<NW> sh;
  __shared__ uint64_t lists[NW * kMostTop], joined[NW > 4 ? 128 : 1];
  __shared__ State states[NW];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const size_t row = blockIdx.x / (unsigned)a.slices;
  const int slice = (int)(blockIdx.x % (unsigned)a.slices);
  const char* x = (const char*)a.x + row * a.stride * kBytes<T>;
  // 16-byte blocks, and the logits before the first and behind the last of them
  const int head = min((int)((16 - ((uintptr_t)x & 15)) & 15) / kBytes<T>, a.V);
  const int blocks = (a.V - head) / EB, tail = (a.V - head) % EB;
  const u32x4* body = (const u32x4*)(x + head * kBytes<T>);

  State st{-INFINITY, 0.f, 0.f};
  Best best;
  if constexpr (TOP) {
    if (threadIdx.x < NW) tell(sh, threadIdx.x, kLowest, kLowest, 0);
    __syncthreads();
  }
  const int begin = (int)min((long long)slice * a.per, (long long)blocks);
  const int end = (int)min((long long)(slice + 1) * a.per, (long long)blocks);
  u32x4 raw[U] = {};
  auto load = [&](int at0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      raw[u] = body[min(at0 + u * NT + (int)threadIdx.x, end - 1)];  // behind the end: a line that was read
    }
  };
  if (begin < end) load(begin);
  const float asked = a.slices == 1 && wave == 0 && lane < a.given ? given_logit<T>(a, x, row, lane) : 0.f;
  for (int at0 = begin; at0 < end; at0 += U * NT) {
    float v[U][EB];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool there = at0 + u * NT + (int)threadIdx.x < end;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        raw[u][i] = there ? raw[u][i] : kNone<T>;
        if constexpr (std::is_same<T, F32>::value) {
          v[u][i] = __uint_as_float(raw[u][i]);
        } else {
          v[u][2 * i] = T::to_f32(raw[u][i] & 0xffffu);
          v[u][2 * i + 1] = T::to_f32(raw[u][i] >> 16);
        }
      }
    }
    load(at0 + U * NT);
    if constexpr (TOP) raise_bar(best, sh, lane);
    take<T, TOP, U, EB>(st, best, sh, v, head + (at0 + (int)threadIdx.x) * EB, NT * EB, a.top, x, wave, lane);
  }
  // the logits outside the blocks: the first wave of the first slice takes those before them, of the last one those behind
  for (int side = 0; wave == 0 && side < 2; ++side) {
    const int n = side ? tail : head, v = side ? a.V - tail + lane : lane;
    if (n == 0 || slice != (side ? a.slices - 1 : 0)) continue;
    const float x1[1][1] = {{lane < n ? at<T>(x, v) : -INFINITY}};
    if constexpr (TOP) {
      // (those before the blocks have smaller ids than the list: they may be as large as the k-th)
      const uint64_t kth = broadcast(best.list, a.top - 1);
      if (kth) best.bar = uniform(fminf(best.bar, value_of(kth)));
    }
    take<T, TOP, 1, 1>(st, best, sh, x1, v, 0, a.top, x, wave, lane);
  }

  join_lanes(st, lane);
  if (lane == 0) states[wave] = st;
  if constexpr (TOP) {
    if (best.waiting) merge_in<T>(best, sh, wave, best.waiting, a.top, x, lane);
    if (lane < a.top) lists[wave * a.top + lane] = best.list;
  }
  __syncthreads();
  if (wave != 0) return;
  st = states[lane % NW];
  if (lane >= NW) st.s = st.e = 0.f;
  join_lanes(st, lane);
  if constexpr (TOP && NW > 4) {
    best.list = join_lists(lists, NW, a.top, joined, lane);
  } else if constexpr (TOP) {  // (so few one after the other: 4096 rows of 32000 62 us, 66 the other way)
#pragma unroll
    for (int w = 1; w < NW; ++w) take_best(best.list, lane < a.top ? lists[w * a.top + lane] : 0, lane);
  }
  if (a.slices == 1) {
    answer<T>(a, st, best.list, asked, x, row, lane);
    return;
  }
  const size_t at = row * a.slices + slice;
  if (lane == 0) a.states[at] = float4{st.m, st.s, st.e, 0.f};
  if (TOP && lane < a.top) a.keys[at * a.top + lane] = best.list;
}

// The slices of a row meet in a wave.
template <typename T>
__global__ __launch_bounds__(64) void join_kernel(const Args a) {
  __shared__ uint64_t wait[128];
  const int lane = threadIdx.x;
  const size_t row = blockIdx.x;
  const char* x = (const char*)a.x + row * a.stride * kBytes<T>;
  const float asked = lane < a.given ? given_logit<T>(a, x, row, lane) : 0.f;
  State st{-INFINITY, 0.f, 0.f};
  if (lane < a.slices) {
    const float4 s = a.states[row * a.slices + lane];
    st = State{s.x, s.y, s.z};
  }
  const uint64_t list = a.top ? join_lists(a.keys + row * a.slices * a.top, a.slices, a.top, wait, lane) : 0;
  join_lanes(st, lane);
  answer<T>(a, st, list, asked, x, row, lane);
}

struct Plan {
  int threads, slices, per;
};

// Few rows of up to 64 KB: one workgroup of 16 waves each, and no second launch (one row of 32000 bf16 9.5 us, as in 15
// slices; one of 50000 fp32 13.8, in 12 slices 9.5).  Longer ones: 512 workgroups of 4 waves, up to 16 a row: the join takes longer
// with more (with 20 alternatives, us: one row of 200000 bf16 12.0, with 64 slices 16.2; 16 rows of 128000 11.7 and
// 14.2; 64 rows of 128000 fp32 17.9, with 256 workgroups 18.5, 1024 19.3; 256 rows of 100003 bf16 23.9, 23.5, 25.7).
static Plan plan(int T, int V, int dtype) {
  constexpr int THREADS = 256;
  const int eb = dtype == MX_DTYPE_F32 ? 4 : 8;
  const long long blocks = V / eb;
  const bool one = T >= 512 || blocks <= 4096;
  Plan p;
  p.threads = T <= 256 && blocks > THREADS && one ? 1024 : THREADS;
  long long slices = one ? 1 : std::min((512LL + T - 1) / T, blocks / THREADS);  // a block a thread at least
  slices = std::min<long long>(slices, kMostSlices);
  p.per = (int)std::max(1LL, (blocks + slices - 1) / slices);
  p.slices = (int)std::max(1LL, (blocks + p.per - 1) / p.per);
  return p;
}

static bool sizes_ok(int T, int V, int given, int top, int dtype) {
  return T > 0 && V > 0 && V <= (1 << 30) && given >= 0 && top >= 0 && top <= kMostTop && top <= V &&
         (long long)T * (given > top ? given : top) <= 0x7fffffffLL &&
         (dtype == MX_DTYPE_BF16 || dtype == MX_DTYPE_F16 || dtype == MX_DTYPE_F32);
}

template <typename T>
static int run(Args a, int rows, int threads, hipStream_t s) {
  const int most = (1 << 21) / a.slices;  // rows of a launch: fewer than 2^32 threads
  for (long long first = 0; first < rows; first += most) {
    const int n = (int)std::min<long long>(rows - first, most);
    const dim3 grid((unsigned)(n * a.slices));
    Args b = a;
    b.x = (const char*)a.x + (size_t)first * a.stride * kBytes<T>;
    b.tokens = a.tokens + (size_t)first * a.given;
    b.logprob = a.logprob + (size_t)first * a.given;
    b.entropy = a.entropy + first;
    b.ids = a.ids + (size_t)first * a.top;
    b.top_logprob = a.top_logprob + (size_t)first * a.top;
    if (threads == 1024) {
      if (a.top) hipLaunchKernelGGL((rows_kernel<T, true, 1024>), grid, dim3(1024), 0, s, b);
      else hipLaunchKernelGGL((rows_kernel<T, false, 1024>), grid, dim3(1024), 0, s, b);
    } else {
      if (a.top) hipLaunchKernelGGL((rows_kernel<T, true, 256>), grid, dim3(256), 0, s, b);
      else hipLaunchKernelGGL((rows_kernel<T, false, 256>), grid, dim3(256), 0, s, b);
    }
    MX_RETURN_IF_HIP(hipGetLastError());
    if (a.slices > 1) {
      hipLaunchKernelGGL(join_kernel<T>, dim3((unsigned)n), dim3(64), 0, s, b);
      MX_RETURN_IF_HIP(hipGetLastError());
    }
  }
  return MX_OK;
}

}  // namespace logprobs
}  // namespace mx

extern "C" size_t mx_token_logprobs_workspace(int T, int V, int top, int dtype) {
  using namespace mx::logprobs;
  if (!sizes_ok(T, V, 0, top, dtype)) return 0;
  const Plan p = plan(T, V, dtype);
  return p.slices == 1 ? 0 : (size_t)T * p.slices * (sizeof(float4) + (size_t)top * sizeof(uint64_t));
}

extern "C" int mx_token_logprobs(const void* logits, const int* tokens, float* logprob, float* entropy, int* top_ids,
                                 float* top_logprob, int T, int V, long long stride, int given, int top, int dtype,
                                 void* workspace, size_t ws_bytes, void* stream) {
  using namespace mx::logprobs;
  if (!logits || !entropy) return MX_ERR_NULL;
  if (given > 0 && (!tokens || !logprob)) return MX_ERR_NULL;
  if (top > 0 && (!top_ids || !top_logprob)) return MX_ERR_NULL;
  if (dtype != MX_DTYPE_BF16 && dtype != MX_DTYPE_F16 && dtype != MX_DTYPE_F32) return MX_ERR_DTYPE;
  if (!sizes_ok(T, V, given, top, dtype) || stride < V || stride > 0x7fffffffLL) return MX_ERR_SHAPE;
  const int size = dtype == MX_DTYPE_F32 ? 4 : 2;
  if ((uintptr_t)logits % size || (((uintptr_t)tokens | (uintptr_t)logprob | (uintptr_t)entropy | (uintptr_t)top_ids |
                                    (uintptr_t)top_logprob) & 3))
    return MX_ERR_ALIGN;
  const Plan p = plan(T, V, dtype);
  if (p.slices > 1) {
    if (!workspace || ws_bytes < mx_token_logprobs_workspace(T, V, top, dtype)) return MX_ERR_WORKSPACE;
    if ((uintptr_t)workspace & 15) return MX_ERR_ALIGN;
  }
  const Args a{logits, tokens, logprob, entropy, top_ids, top_logprob, (float4*)workspace,
               (uint64_t*)((float4*)workspace + (size_t)T * p.slices), V, given, top, p.slices, p.per, stride};
  hipStream_t s = (hipStream_t)stream;
  if (dtype == MX_DTYPE_BF16) return run<mx::BF16>(a, T, p.threads, s);
  if (dtype == MX_DTYPE_F16) return run<mx::F16>(a, T, p.threads, s);
  return run<F32>(a, T, p.threads, s);
}
