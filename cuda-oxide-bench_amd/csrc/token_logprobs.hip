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
// its place, so that ties go to the lowest id).  A wave keeps its best 64 keys sorted across its lanes, and only a
// chunk in which a lane's maximum reaches the k-th of them is looked at again.  What it has there is gathered
// in LDS, sorted 64 at a time and merged in.  The first chunk would all qualify: there the k-th largest of the 64
// lanes' maxima is the bar, which at least k logits reach.
//
// A row is cut into slices, a workgroup each, where there are few rows; a second kernel joins them.
#include <algorithm>

#include "mx_common.h"

namespace mx {
namespace logprobs {

constexpr int NT = 256, NW = NT / 64;
constexpr int kMostTop = 32;
constexpr int kMostSlices = 64;
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
template <int SIZE, int J>
__device__ __forceinline__ void stage(uint64_t& v, int lane) {
  const uint64_t o = lane_xor64<J>(v, lane);
  const bool larger = ((lane & J) == 0) == ((lane & SIZE) == 0);
  v = (o > v) == larger ? o : v;
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
  const bool larger = ((lane & J) == 0) == ((lane & SIZE) == 0);
  v = larger ? fmaxf(v, o) : fminf(v, o);
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
template <int J>
__device__ __forceinline__ void join_lanes(State& st, int lane) {
  join(st, State{lane_xorf<J>(st.m, lane), lane_xorf<J>(st.s, lane), lane_xorf<J>(st.e, lane)});
  if constexpr (J > 1) join_lanes<J / 2>(st, lane);
}

// What a wave has of the alternatives.
struct Best {
  uint64_t list = 0;    // sorted across the lanes; 0: none
  uint64_t kth = 0;     // the k-th of them
  float bar = -INFINITY;  // its value
  int waiting = 0;      // keys in LDS that are not merged yet, below 64
};

__device__ __forceinline__ void merge_in(Best& best, uint64_t* buf, int n, int top, int lane) {
  wave_sync();
  uint64_t v = lane < n ? buf[lane] : 0;
  sort(v, lane);
  take_best(best.list, v, lane);
  best.kth = broadcast(best.list, top - 1);
  best.bar = best.kth ? value_of(best.kth) : -INFINITY;
}

// x[j], by a tree of selections: registers have no index.
template <int N>
__device__ __forceinline__ float pick(const float (&x)[N], int j) {
  if constexpr (N == 1) {
    return x[0];
  } else {
    float half[N / 2];
#pragma unroll
    for (int i = 0; i < N / 2; ++i) half[i] = j & 1 ? x[2 * i + 1] : x[2 * i];
    return pick<N / 2>(half, j >> 1);
  }
}

// The logits x of a chunk, x[j] the token first + (j / EB) * apart + j % EB of the lane where it is there.
template <int N, int EB>
__device__ __forceinline__ void offer(Best& best, const float (&x)[N], const bool (&there)[N / EB], float most, int first,
                                      int apart, int top, uint64_t* buf, int lane) {
  float bar = best.bar;
  if (!best.kth) {  // fewer than `top` so far
    float v = most;
    sort_floats(v, lane);
    bar = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), top - 1));
  }
  uint32_t good = 0;  // of the lane's
#pragma unroll
  for (int j = 0; j < N; ++j) good |= there[j / EB] && x[j] >= bar ? 1u << j : 0u;
  for (; __any(good != 0); good &= good - 1) {
    const int j = good ? __builtin_ctz(good) : 0;
    const uint64_t key = key_of(pick<N>(x, j), first + j / EB * apart + j % EB);
    const uint64_t who = __ballot(good && key > best.kth);
    if (who >> lane & 1)
      buf[best.waiting + __builtin_amdgcn_mbcnt_hi((uint32_t)(who >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0))] = key;
    best.waiting += __popcll(who);
    if (best.waiting >= 64) {
      merge_in(best, buf, 64, top, lane);
      const uint64_t rest = buf[64 + lane];
      best.waiting -= 64;
      wave_sync();
      buf[lane] = rest;
    }
  }
  if (best.waiting) {
    merge_in(best, buf, best.waiting, top, lane);
    best.waiting = 0;
  }
}

// One chunk into the state and the alternatives.
template <bool TOP, int N, int EB>
__device__ __forceinline__ void take(State& st, Best& best, const float (&x)[N], const bool (&there)[N / EB], int first,
                                     int apart, int top, uint64_t* buf, int lane) {
  float most = x[0];
#pragma unroll
  for (int j = 1; j < N; ++j) most = fmaxf(most, x[j]);
  if (__any(most > st.m)) move_to(st, fmaxf(most, st.m));
  const float off = st.m == -INFINITY ? 0.f : st.m;
  float s[4] = {}, e[4] = {};
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const float y = x[j] - off;
    const float p = __builtin_amdgcn_exp2f(y * kLog2e);
    s[j % 4] += p;
    e[j % 4] = __builtin_fmaf(p, y, e[j % 4]);
  }
  float more = (e[0] + e[1]) + (e[2] + e[3]);
  if (__any(more != more)) {  // 0 times -inf: such logits add nothing (a NaN is in S)
    more = 0.f;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const float y = x[j] - off;
      more += y > -INFINITY ? __builtin_amdgcn_exp2f(y * kLog2e) * y : 0.f;
    }
  }
  st.s += (s[0] + s[1]) + (s[2] + s[3]);
  st.e += more;
  if constexpr (TOP) {
    if (__any(most >= best.bar)) offer<N, EB>(best, x, there, most, first, apart, top, buf, lane);
  }
}

// A row's answers from its state (in every thread) and its best keys (a lane's of one wave).
template <typename T>
__device__ __forceinline__ void answer(const Args& a, const State& st, uint64_t key, size_t row, int tid, int threads) {
  const void* x = (const char*)a.x + row * a.stride * kBytes<T>;
  const bool none = !(st.s > 0.f && st.s < INFINITY);  // a NaN, +inf, nothing but -inf: no distribution
  const float log_s = logf(st.s), nan = __builtin_nanf("");
  auto log_p = [&](float v) { return (v - st.m) - log_s; };
  for (int i = tid; i < a.given; i += threads) {
    const int v = a.tokens[row * a.given + i];
    const bool token = (uint32_t)v < (uint32_t)a.V;
    a.logprob[row * a.given + i] = none || !token ? nan : log_p(at<T>(x, v));
  }
  if (tid == 0) a.entropy[row] = none ? nan : log_s - st.e / st.s;
  if (tid < a.top) {
    a.ids[row * a.top + tid] = none ? -1 : (int)~(uint32_t)key;
    a.top_logprob[row * a.top + tid] = none ? nan : log_p(value_of(key));
  }
}

template <typename T, bool TOP>
__global__ __launch_bounds__(NT) void rows_kernel(const Args a) {
  constexpr int EB = 16 / kBytes<T>;  // logits of a block
  constexpr int UB = 4;               // blocks of a chunk and thread
  __shared__ uint64_t bufs[NW][128];
  __shared__ uint64_t lists[NW][kMostTop];
  __shared__ State states[NW];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const size_t row = blockIdx.x / (unsigned)a.slices;
  const int slice = (int)(blockIdx.x % (unsigned)a.slices);
  uint64_t* buf = bufs[wave];
  const char* x = (const char*)a.x + row * a.stride * kBytes<T>;
  // 16-byte blocks, and the logits before the first and behind the last of them
  const int head = min((int)((16 - ((uintptr_t)x & 15)) & 15) / kBytes<T>, a.V);
  const int blocks = (a.V - head) / EB, tail = (a.V - head) % EB;
  const u32x4* body = (const u32x4*)(x + head * kBytes<T>);

  State st{-INFINITY, 0.f, 0.f};
  Best best;
  auto widen = [&](const u32x4& r, float* v) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same<T, F32>::value) {
        v[i] = __uint_as_float(r[i]);
      } else {
        v[2 * i] = T::to_f32(r[i] & 0xffffu);
        v[2 * i + 1] = T::to_f32(r[i] >> 16);
      }
    }
  };
  const int end = min((int)min((long long)(slice + 1) * a.per, (long long)blocks), blocks);
  for (int at0 = slice * a.per; at0 < end; at0 += UB * NT) {
    u32x4 raw[UB];
    bool there[UB];
    float v[UB * EB];
#pragma unroll
    for (int u = 0; u < UB; ++u) {
      const int i = at0 + u * NT + (int)threadIdx.x;
      there[u] = i < end;
      raw[u] = there[u] ? body[i] : u32x4{};
    }
#pragma unroll
    for (int u = 0; u < UB; ++u) {
      widen(raw[u], v + u * EB);
      if (!there[u]) {
#pragma unroll
        for (int j = 0; j < EB; ++j) v[u * EB + j] = -INFINITY;
      }
    }
    take<TOP, UB * EB, EB>(st, best, v, there, head + (at0 + (int)threadIdx.x) * EB, NT * EB, a.top, buf, lane);
  }
  // the logits outside the blocks: the first wave of the first slice takes those before them, of the last one those behind
  for (int side = 0; wave == 0 && side < 2; ++side) {
    const int n = side ? tail : head, v = side ? a.V - tail + lane : lane;
    if (n == 0 || slice != (side ? a.slices - 1 : 0)) continue;
    const bool there[1] = {lane < n};
    const float x1[1] = {lane < n ? at<T>(x, v) : -INFINITY};
    take<TOP, 1, 1>(st, best, x1, there, v, 0, a.top, buf, lane);
  }

  join_lanes<32>(st, lane);
  if (lane == 0) states[wave] = st;
  if constexpr (TOP) {
    if (lane < kMostTop) lists[wave][lane] = best.list;
  }
  __syncthreads();
  if (wave != 0) return;
#pragma unroll
  for (int w = 1; w < NW; ++w) {
    join(st, states[w]);
    if constexpr (TOP) take_best(best.list, lane < kMostTop ? lists[w][lane] : 0, lane);
  }
  if (a.slices == 1) {
    answer<T>(a, st, best.list, row, lane, 64);
    return;
  }
  const size_t at = row * a.slices + slice;
  if (lane == 0) a.states[at] = float4{st.m, st.s, st.e, 0.f};
  if (TOP && lane < a.top) a.keys[at * a.top + lane] = best.list;
}

// The slices of a row meet in a wave.
template <typename T>
__global__ __launch_bounds__(64) void join_kernel(const Args a) {
  const int lane = threadIdx.x;
  const size_t row = blockIdx.x;
  State st{-INFINITY, 0.f, 0.f};
  if (lane < a.slices) {
    const float4 s = a.states[row * a.slices + lane];
    st = State{s.x, s.y, s.z};
  }
  join_lanes<32>(st, lane);
  // the lanes' lists are sorted: the slices' best first, then their second, until none is good enough
  uint64_t list = 0, kth = 0;
  const uint64_t* keys = a.keys + (row * a.slices + lane) * a.top;
  for (int j = 0; j < a.top; ++j) {
    uint64_t v = lane < a.slices ? keys[j] : 0;
    if (!__any(v > kth)) break;
    sort(v, lane);
    take_best(list, v, lane);
    kth = broadcast(list, a.top - 1);
  }
  answer<T>(a, st, list, row, lane, 64);
}

struct Plan {
  int slices, per;
};

// A workgroup takes at least a block a thread.
static Plan plan(int T, int V, int dtype) {
  const int eb = dtype == MX_DTYPE_F32 ? 4 : 8;
  const long long blocks = V / eb;
  long long slices = T >= 512 ? 1 : (1024 + T - 1) / T;
  const long long most = blocks / NT > 0 ? blocks / NT : 1;
  slices = slices < most ? slices : most;
  slices = slices < kMostSlices ? slices : kMostSlices;
  Plan p;
  const long long per = (blocks + slices - 1) / slices;
  p.per = (int)(per > 0 ? per : 1);
  p.slices = (int)((blocks + p.per - 1) / p.per);
  if (p.slices < 1) p.slices = 1;
  return p;
}

static bool sizes_ok(int T, int V, int given, int top, int dtype) {
  return T > 0 && V > 0 && V <= (1 << 30) && given >= 0 && top >= 0 && top <= kMostTop && top <= V &&
         (long long)T * (given > top ? given : top) <= 0x7fffffffLL &&
         (dtype == MX_DTYPE_BF16 || dtype == MX_DTYPE_F16 || dtype == MX_DTYPE_F32);
}

template <typename T>
static int run(Args a, int rows, hipStream_t s) {
  const int most = (1 << 23) / a.slices;  // rows of a launch: fewer than 2^32 threads
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
    if (a.top)
      hipLaunchKernelGGL((rows_kernel<T, true>), grid, dim3(NT), 0, s, b);
    else
      hipLaunchKernelGGL((rows_kernel<T, false>), grid, dim3(NT), 0, s, b);
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
  if (dtype == MX_DTYPE_BF16) return run<mx::BF16>(a, T, s);
  if (dtype == MX_DTYPE_F16) return run<mx::F16>(a, T, s);
  return run<F32>(a, T, s);
}
