// experts.cu — routing of tokens to experts, and the weighted sum of the experts' rows.
//
// Routing: a warp holds a token's logits as order-preserving 32-bit keys. The k-th largest of the lanes' own maxima is a bound that at
// least k keys reach, and few more; those that do are collected in the experts' order, and each counts how many come before it, which is its
// rank. (k rounds of a maximum over lanes that held their keys sorted took 29 us for 16384 tokens of 256 experts, where this took 25.) Then the pairs
// are counted and placed by expert. A pair's place is the number of pairs of lower experts plus that of the same
// expert's earlier tokens, so it does not depend on the order in which anything runs: within 128 tokens the earlier
// ones are the lower bits of a mask that each expert has (set by atomicOr, which commutes), before them the counts of earlier blocks.
// Bound by instructions, not by the 19 MB: 530 a token in the choice, 215 in the placing. Measured: 1 token of 128 experts 3.5 us, 64 of 256
// 7.0, 2048 9.4, 16384 22.9. (With 513 to 1024 experts a lane holds 32 keys, and some 40 to 90 words of a thread's are kept in memory.)
// The operator's other sources, which its revision hash covers through this line (build.py --sources):
// FNV-1a 64 of divide.cuh, launch.cuh: 2e2d27af524d7113
#include "common.cuh"
#include "divide.cuh"
#include "launch.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace up {
namespace experts {

constexpr int kMaxExperts = 1024;
constexpr int kMaxK = 32;
constexpr int kTile = 128;            // tokens a tile at most: four words of mask an expert
constexpr int kOne = 64;              // tokens that one block takes in one launch: 7.0 us of 256 experts, where two launches take 7.6 (96: 8.0, 7.4)
constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxBlocks = 256;       // each block of the placing kernel reads every block's counts

struct Route {
  const void* logits;
  int64_t stride;
  int tokens, experts, k, score, renormalise;
  int span, per;                      // tokens a tile, tiles a block
  float gain;
  int32_t *ids, *rows, *slots, *offsets;
  float* weights;
  uint32_t* counts;                   // [blocks][experts]
};

__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ float as_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float as_float(__nv_bfloat16 v) { return __bfloat162float(v); }

// Order-preserving key: larger logits have larger keys. Adding 0 makes every NaN the canonical one, whose key is the largest, and -0 equal to 0.
// Keys up to that of -inf are never taken.
constexpr uint32_t kMasked = 0x007fffffu;
__device__ __forceinline__ uint32_t key_of(float v) {
  const uint32_t u = __float_as_uint(v + 0.f);
  return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float((key & 0x80000000u) ? key & 0x7fffffffu : ~key);
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// One token's choice by one warp, lane l holding the keys of experts l, l + 32, ...: up to k of its lanes get a rank (below k), an expert
// and its weight; the others' rank is kMaxK.
struct Choice {
  int rank, id;
  float weight;
};
struct Candidate {
  uint32_t key;
  int id;
};
template <int PER>
__device__ __forceinline__ Choice choose(const uint32_t (&key)[PER], const Route& a, int lane, Candidate* found) {
  uint32_t own = key[0];
#pragma unroll
  for (int i = 1; i < PER; ++i) own = max(own, key[i]);
  // after r rounds at least r lanes have a maximum that reaches the bound (equal ones leave together)
  uint32_t left = own, top = 0, bound = 0;
  for (int j = 0; j < a.k; ++j) {
    bound = __reduce_max_sync(0xffffffffu, left);
    if (j == 0) top = bound;
    if (left == bound) left = 0;
  }
  bound = max(bound, kMasked + 1);
  int n = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const bool is = key[i] >= bound;
    const unsigned who = __ballot_sync(0xffffffffu, is);
    const int at = n + __popc(who & ((1u << lane) - 1u));
    if (is && at < 32) found[at] = Candidate{key[i], i * 32 + lane};
    n += __popc(who);
  }
  Choice c{kMaxK, -1, 0.f};
  uint32_t mine = 0;
  if (n <= 32) {
    __syncwarp();
    if (lane < n) mine = found[lane].key, c.id = found[lane].id;
    int before = 0;  // candidates stand in the order of their experts: of equal ones the earlier comes first
    for (int j = 0; j < n; ++j) {
      const uint32_t other = __shfl_sync(0xffffffffu, mine, j);
      before += other > mine || (other == mine && j < lane) ? 1 : 0;
    }
    if (lane < n && before < a.k) c.rank = before;
    __syncwarp();  // before the next token's are written
  } else {
    // many equal ones: a round for each, of the largest key left and the lowest expert that has it
    uint32_t rest[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) rest[i] = key[i];
    for (int j = 0; j < a.k; ++j) {
      uint32_t best = rest[0];
      int e = lane;
#pragma unroll
      for (int i = 1; i < PER; ++i)
        if (rest[i] > best) best = rest[i], e = i * 32 + lane;
      const uint32_t high = __reduce_max_sync(0xffffffffu, best);
      if (high <= kMasked) break;
      e = (int)__reduce_min_sync(0xffffffffu, best == high ? (unsigned)e : 0x7fffffffu);
      if (lane == j) mine = high, c.id = e, c.rank = j;
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (e == i * 32 + lane) rest[i] = 0;
    }
  }
  const bool taken = c.rank < kMaxK;
  const float l = value_of(mine);
  float w = 0.f, total = 1.f;
  if (a.score == UP_EXPERT_SOFTMAX) {
    const float m = value_of(top);
    if (taken) w = expf(l - m);
    if (!a.renormalise) {
      total = 0.f;
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (key[i] > kMasked) total += expf(value_of(key[i]) - m);
      total = warp_sum(total);
    }
  } else {
    const float m = value_of(top);
    // Shares of scores that are no normal numbers: exp(-m) times as large, which no quotient changes. None where the largest score is 0 in f32.
    if (a.renormalise && m < 0.f && __any_sync(0xffffffffu, taken && l < -64.f)) {
      if (taken && expf(m) > 0.f) w = expf(l - m) / (1.f + expf(l));
    } else if (taken) {
      const float d = 1.f + expf(-l);
      w = d < __uint_as_float(0x7f800000u) ? 1.f / d : expf(l);  // below -88.7 they are one number
    }
  }
  if (a.renormalise) total = warp_sum(w);
  c.weight = taken && !(total == 0.f) ? w / total * a.gain : 0.f;
  return c;
}

// Chooses for the tile's tokens; marks them in the experts' masks. A warp's tokens' logits are all on their way at once where
// they leave it the registers.
template <int PER, typename T>
__device__ __forceinline__ void choose_tile(const Route& a, int first, uint32_t (*mask)[kTile / 32], int16_t* held, Candidate* found) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int end = min(first + a.span, a.tokens);
  constexpr int kEach = kTile / kWarps, kAtOnce = PER <= 4 ? kEach : PER <= 8 ? 2 : 1;
#pragma unroll 1
  for (int t0 = first + warp; t0 < end; t0 += kAtOnce * kWarps) {
    uint32_t key[kAtOnce][PER];
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      const int t = t0 + u * kWarps;
      const T* row = static_cast<const T*>(a.logits) + (int64_t)t * a.stride;
#pragma unroll
      for (int i = 0; i < PER; ++i)
        key[u][i] = t < end && i * 32 + lane < a.experts ? key_of(as_float(row[i * 32 + lane])) : 0u;
    }
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      const int t = t0 + u * kWarps;
      if (t >= end) break;
      const Choice c = choose<PER>(key[u], a, lane, found + 32 * warp);
      const int64_t at = (int64_t)t * a.k;
      const int in = t - first, n = __popc(__ballot_sync(0xffffffffu, c.rank < kMaxK));
      if (c.rank < kMaxK) {
        a.ids[at + c.rank] = c.id;
        a.weights[at + c.rank] = c.weight;
        if (held) held[in * a.k + c.rank] = (int16_t)c.id;
        atomicOr(&mask[c.id][in >> 5], 1u << (in & 31));
      }
      if (lane >= n && lane < a.k) {  // the ranks that no expert has
        a.ids[at + lane] = -1;
        a.weights[at + lane] = 0.f;
        if (held) held[in * a.k + lane] = -1;
      }
    }
  }
}

__device__ __forceinline__ uint32_t count_of(const uint32_t (&m)[kTile / 32]) {
  uint32_t n = 0;
#pragma unroll
  for (int i = 0; i < kTile / 32; ++i) n += __popc(m[i]);
  return n;
}

__device__ __forceinline__ void clear(uint32_t (*mask)[kTile / 32], int experts) {
  for (int i = threadIdx.x; i < experts * (kTile / 32); i += kThreads) (&mask[0][0])[i] = 0;
}

// start[e] becomes the sum of the totals before e, by all warps: each scans 32 experts, then adds the warps before. Returns the sum of all.
// Ends and begins with the block in step.
__device__ __forceinline__ uint32_t scan_experts(const uint32_t* total, uint32_t* start, int experts) {
  __shared__ uint32_t of_warp[kWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, e = threadIdx.x;  // kMaxExperts threads
  const uint32_t n = e < experts ? total[e] : 0u;
  uint32_t s = n;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t v = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += v;
  }
  if (lane == 31) of_warp[warp] = s;
  __syncthreads();
  uint32_t w = of_warp[lane];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t v = __shfl_up_sync(0xffffffffu, w, o);
    if (lane >= o) w += v;
  }
  const uint32_t all = __shfl_sync(0xffffffffu, w, 31);
  const uint32_t before = warp > 0 ? __shfl_sync(0xffffffffu, w, warp - 1) : 0u;
  if (e < experts) start[e] = before + s - n;
  __syncthreads();
  return all;
}
static_assert(kThreads == kMaxExperts && kWarps == 32, "a thread an expert, a lane a warp");

// Places the tile's pairs: next[e] is the place of expert e's first pair in it.
__device__ __forceinline__ void place_tile(const Route& a, int first, const uint32_t (*mask)[kTile / 32], const uint32_t* next,
                                           const int16_t* held) {
  const int pairs = (min(first + a.span, a.tokens) - first) * a.k;
  for (int p = threadIdx.x; p < pairs; p += kThreads) {
    const int in = p / a.k, id = held[p];
    int slot = -1;
    if (id >= 0) {
      uint32_t before = __popc(mask[id][in >> 5] & ((1u << (in & 31)) - 1u));
      for (int i = 0; i < (in >> 5); ++i) before += __popc(mask[id][i]);
      slot = (int)(next[id] + before);
      a.rows[slot] = first + in;
    }
    a.slots[(int64_t)first * a.k + p] = slot;
  }
}

// All of it in one block, for at most kOne tokens.
template <int PER, typename T>
__global__ void __launch_bounds__(kThreads) route_one_kernel(const Route a) {
  __shared__ uint32_t mask[PER * 32][kTile / 32];
  __shared__ uint32_t total[PER * 32], start[PER * 32];
  __shared__ int16_t held[kTile * kMaxK];
  __shared__ Candidate found[kThreads];
  clear(mask, a.experts);
  after_previous();
  let_next_begin();
  __syncthreads();
  choose_tile<PER, T>(a, 0, mask, held, found);
  __syncthreads();
  for (int e = threadIdx.x; e < a.experts; e += kThreads) total[e] = count_of(mask[e]);
  __syncthreads();
  const uint32_t all = scan_experts(total, start, a.experts);
  for (int e = threadIdx.x; e <= a.experts; e += kThreads) a.offsets[e] = (int32_t)(e < a.experts ? start[e] : all);
  place_tile(a, 0, mask, start, held);
  for (int i = (int)all + threadIdx.x; i < a.tokens * a.k; i += kThreads) a.rows[i] = -1;
}

// First of two launches: choice, and each block's counts.
template <int PER, typename T>
__global__ void __launch_bounds__(kThreads) choose_kernel(const Route a) {
  __shared__ uint32_t mask[PER * 32][kTile / 32];
  __shared__ uint32_t total[PER * 32];
  __shared__ Candidate found[kThreads];
  for (int e = threadIdx.x; e < a.experts; e += kThreads) total[e] = 0;
  after_previous();
  let_next_begin();
  for (int i = 0; i < a.per; ++i) {
    const int first = (blockIdx.x * a.per + i) * a.span;
    if (first >= a.tokens) break;
    clear(mask, a.experts);
    __syncthreads();
    choose_tile<PER, T>(a, first, mask, nullptr, found);
    __syncthreads();
    for (int e = threadIdx.x; e < a.experts; e += kThreads) total[e] += count_of(mask[e]);
    __syncthreads();
  }
  for (int e = threadIdx.x; e < a.experts; e += kThreads) a.counts[(int64_t)blockIdx.x * a.experts + e] = total[e];
}

// Second: where each block's pairs begin, and the places.
__global__ void __launch_bounds__(kThreads) place_kernel(const Route a) {
  __shared__ uint32_t mask[kMaxExperts][kTile / 32];
  __shared__ uint32_t total[kMaxExperts], next[kMaxExperts], before[kMaxExperts];
  __shared__ int16_t held[kTile * kMaxK];
  for (int e = threadIdx.x; e < a.experts; e += kThreads) total[e] = before[e] = 0;
  clear(mask, a.experts);
  after_previous();
  let_next_begin();
  // The choice of a tile, marked in its masks. The first one's is on its way beside the counts.
  auto mark = [&](int first) {
    const int pairs = (min(first + a.span, a.tokens) - first) * a.k;
    for (int p = threadIdx.x; p < pairs; p += kThreads) {
      const int id = a.ids[(int64_t)first * a.k + p], in = p / a.k;
      held[p] = (int16_t)id;
      if (id >= 0) atomicOr(&mask[id][in >> 5], 1u << (in & 31));
    }
  };
  const int first0 = blockIdx.x * a.per * a.span;
  __syncthreads();
  // warps take columns of 32 experts, and where these are fewer than the warps share a column's blocks
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int wide = (a.experts + 31) / 32;
  const int c = warp % wide, e = c * 32 + lane, parts = (kWarps - c + wide - 1) / wide;  // wide is at most kWarps
  uint32_t n = 0, m = 0;
  if (e < a.experts) {
#pragma unroll 16
    for (int b = warp / wide; b < (int)gridDim.x; b += parts) {
      const uint32_t v = a.counts[(int64_t)b * a.experts + e];
      n += v;
      if (b < (int)blockIdx.x) m += v;
    }
  }
  mark(first0);
  if (e < a.experts) {
    atomicAdd(&total[e], n);
    atomicAdd(&before[e], m);
  }
  __syncthreads();
  const uint32_t all = scan_experts(total, next, a.experts);
  if (blockIdx.x == 0)
    for (int i = threadIdx.x; i <= a.experts; i += kThreads) a.offsets[i] = (int32_t)(i < a.experts ? next[i] : all);
  __syncthreads();
  for (int i = threadIdx.x; i < a.experts; i += kThreads) next[i] += before[i];
  __syncthreads();
  for (int i = 0; i < a.per; ++i) {
    const int first = first0 + i * a.span;
    if (first >= a.tokens) break;
    if (i > 0) {
      clear(mask, a.experts);
      __syncthreads();
      mark(first);
      __syncthreads();
    }
    place_tile(a, first, mask, next, held);
    __syncthreads();
    for (int x = threadIdx.x; x < a.experts; x += kThreads) next[x] += count_of(mask[x]);
    __syncthreads();
  }
  const int64_t pairs = (int64_t)a.tokens * a.k;
  for (int64_t i = (int64_t)all + blockIdx.x * kThreads + threadIdx.x; i < pairs; i += (int64_t)gridDim.x * kThreads)
    a.rows[i] = -1;
}

// Blocks of the two launches, their tiles and a tile's tokens: whole warps of them, as few as give every SM a block (2048 tokens of 256 experts:
// 16.7 us in tiles of 128 on 16 SMs, 9.4 in tiles of 32 on 64).
static int split(int64_t tokens, int* span, int* per) {
  const int64_t each = ((tokens + sm_count() - 1) / sm_count() + kWarps - 1) / kWarps * kWarps;
  *span = (int)(each < kTile ? each : kTile);
  const int64_t tiles = (tokens + *span - 1) / *span;
  *per = (int)((tiles + kMaxBlocks - 1) / kMaxBlocks);
  return (int)((tiles + *per - 1) / *per);
}

template <int PER, typename T>
int route(Route& a, cudaStream_t s) {
  if (a.tokens <= kOne) {
    const cudaError_t e = launch_early(route_one_kernel<PER, T>, 1, kThreads, 0, s, a);
    if (e != cudaSuccess) return cuda_status(e);
    note_launch();
    return check_launch();
  }
  const int blocks = split(a.tokens, &a.span, &a.per);
  cudaError_t e = launch_early(choose_kernel<PER, T>, blocks, kThreads, 0, s, a);
  if (e == cudaSuccess) e = launch_early(place_kernel, blocks, kThreads, 0, s, a);
  if (e != cudaSuccess) return cuda_status(e);
  note_launch(2);
  return check_launch();
}
template <typename T>
int route_sized(Route& a, cudaStream_t s) {
  const int per = (a.experts + 31) / 32;
  if (per <= 1) return route<1, T>(a, s);
  if (per <= 2) return route<2, T>(a, s);
  if (per <= 4) return route<4, T>(a, s);
  if (per <= 8) return route<8, T>(a, s);
  if (per <= 16) return route<16, T>(a, s);
  return route<32, T>(a, s);
}

// ---- the weighted sum ----
constexpr int kSumThreads = 256;

template <typename T, int V>
struct Vec;
template <>
struct Vec<float, 4> {
  using Raw = uint4;
  static __device__ __forceinline__ void widen(const Raw& r, float (&f)[4]) {
    f[0] = __uint_as_float(r.x), f[1] = __uint_as_float(r.y), f[2] = __uint_as_float(r.z), f[3] = __uint_as_float(r.w);
  }
  static __device__ __forceinline__ Raw narrow(const float (&f)[4]) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
};
template <>
struct Vec<__half, 8> {
  using Raw = uint4;
  static __device__ __forceinline__ void widen(const Raw& r, float (&f)[8]) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      f[2 * i] = v.x, f[2 * i + 1] = v.y;
    }
  }
  static __device__ __forceinline__ Raw narrow(const float (&f)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};
template <>
struct Vec<__nv_bfloat16, 8> {
  using Raw = uint4;
  static __device__ __forceinline__ void widen(const Raw& r, float (&f)[8]) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) f[2 * i] = __uint_as_float(w[i] << 16), f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
  static __device__ __forceinline__ Raw narrow(const float (&f)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};
template <typename T>
struct Vec<T, 1> {
  using Raw = T;
  static __device__ __forceinline__ void widen(const T& r, float (&f)[1]) { f[0] = as_float(r); }
  static __device__ __forceinline__ T narrow(const float (&f)[1]);
};
template <>
__device__ __forceinline__ float Vec<float, 1>::narrow(const float (&f)[1]) { return f[0]; }
template <>
__device__ __forceinline__ __half Vec<__half, 1>::narrow(const float (&f)[1]) { return __float2half_rn(f[0]); }
template <>
__device__ __forceinline__ __nv_bfloat16 Vec<__nv_bfloat16, 1>::narrow(const float (&f)[1]) { return __float2bfloat16_rn(f[0]); }

// A thread sums U pieces of V values (16 bytes each) over their token's slots. Bound by HBM: every chosen row once. With U pieces of up to
// kAtOnce slots about 8 loads are on their way a thread. Measured: 8192 tokens' 8 rows of 4096 bf16 values 104 us (5.8 TB/s).
template <typename T, int V, int U, typename Div>
__global__ void __launch_bounds__(kSumThreads)
    combine_kernel(const T* y, int64_t rows, int64_t ys, const int32_t* slots, const float* weights, int k, const T* add, int64_t as,
                   T* out, int64_t os, typename Div::Int pieces, typename Div::Int row_pieces, Div by_row) {
  using Int = typename Div::Int;
  using W = Vec<T, V>;
  constexpr int kAtOnce = 8 / U;
  const Int p0 = (Int)blockIdx.x * (kSumThreads * U) + threadIdx.x;
  after_previous();
  let_next_begin();
  float sum[U][V];
  int64_t at[U], tk[U], out_at[U];
  bool in[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const Int p = p0 + u * kSumThreads;
    in[u] = p < pieces;
    const Int t = in[u] ? by_row(p) : 0;
    at[u] = in[u] ? (int64_t)(p - t * row_pieces) * V : 0;
    tk[u] = (int64_t)t * k, out_at[u] = (int64_t)t * os + at[u];
#pragma unroll
    for (int i = 0; i < V; ++i) sum[u][i] = 0.f;
    if (add && in[u]) W::widen(*reinterpret_cast<const typename W::Raw*>(add + (int64_t)t * as + at[u]), sum[u]);
  }
  for (int j0 = 0; j0 < k; j0 += kAtOnce) {
    typename W::Raw raw[U][kAtOnce];
    float w[U][kAtOnce];
    bool there[U][kAtOnce];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j) {
        const int64_t s = in[u] && j0 + j < k ? (int64_t)slots[tk[u] + j0 + j] : -1;
        there[u][j] = (uint64_t)s < (uint64_t)rows;
        w[u][j] = there[u][j] ? weights[tk[u] + j0 + j] : 0.f;
        if (there[u][j]) raw[u][j] = *reinterpret_cast<const typename W::Raw*>(y + s * ys + at[u]);
      }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j)
        if (there[u][j]) {
          float f[V];
          W::widen(raw[u][j], f);
#pragma unroll
          for (int i = 0; i < V; ++i) sum[u][i] = fmaf(w[u][j], f[i], sum[u][i]);
        }
  }
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (in[u]) *reinterpret_cast<typename W::Raw*>(out + out_at[u]) = W::narrow(sum[u]);
}

template <typename T, int V, int U>
int combine_by(const void* y, int64_t rows, int64_t ys, int64_t n, const int32_t* slots, const float* weights, int64_t tokens,
               int64_t k, const void* add, int64_t as, void* out, int64_t os, cudaStream_t s) {
  const int64_t row_pieces = n / V, pieces = tokens * row_pieces;
  const int64_t ctas = (pieces + kSumThreads * U - 1) / (kSumThreads * U);
  if (ctas > 0x7fffffff) return UP_ERR_UNSUPPORTED;
  const T *from = static_cast<const T*>(y), *more = static_cast<const T*>(add);
  const cudaError_t e =
      pieces < ((int64_t)1 << 31) - kSumThreads * U
          ? launch_early(combine_kernel<T, V, U, Divide32>, (unsigned)ctas, kSumThreads, 0, s, from, rows, ys, slots, weights, (int)k,
                         more, as, static_cast<T*>(out), os, (uint32_t)pieces, (uint32_t)row_pieces, Divide32(row_pieces))
          : launch_early(combine_kernel<T, V, U, Divide64>, (unsigned)ctas, kSumThreads, 0, s, from, rows, ys, slots, weights, (int)k,
                         more, as, static_cast<T*>(out), os, (uint64_t)pieces, (uint64_t)row_pieces, Divide64(row_pieces));
  if (e != cudaSuccess) return cuda_status(e);
  note_launch();
  return check_launch();
}
template <typename T, int V>
int combine(const void* y, int64_t rows, int64_t ys, int64_t n, const int32_t* slots, const float* weights, int64_t tokens,
            int64_t k, const void* add, int64_t as, void* out, int64_t os, cudaStream_t s) {
  // several pieces a thread where one has few slots and the GPU is full all the same
  const bool full = tokens * (n / V) > (int64_t)sm_count() * 2048 * 4;
  if (full && k <= 2) return combine_by<T, V, 4>(y, rows, ys, n, slots, weights, tokens, k, add, as, out, os, s);
  if (full && k <= 4) return combine_by<T, V, 2>(y, rows, ys, n, slots, weights, tokens, k, add, as, out, os, s);
  return combine_by<T, V, 1>(y, rows, ys, n, slots, weights, tokens, k, add, as, out, os, s);
}

}  // namespace experts
}  // namespace up

using namespace up;
using namespace up::experts;

extern "C" size_t up_sm100_expert_route_workspace_bytes(int64_t tokens, int64_t experts) {
  if (tokens <= kOne || experts <= 0 || experts > kMaxExperts) return 256;
  int span, per;
  return (size_t)split(tokens, &span, &per) * experts * sizeof(uint32_t);
}

extern "C" int up_sm100_expert_route(const void* logits, int dtype, int64_t tokens, int64_t n_experts, int64_t stride,
                                     int64_t k, int score, int renormalise, float gain, int32_t* ids, float* weights,
                                     int32_t* rows, int32_t* slots, int32_t* offsets, void* workspace,
                                     size_t workspace_bytes, void* stream) {
  UP_CHECK_ARG(tokens >= 0 && n_experts >= 1 && k >= 1 && k <= n_experts && stride >= 0);
  UP_CHECK_ARG(score == UP_EXPERT_SOFTMAX || score == UP_EXPERT_SIGMOID);
  if (dtype != UP_EK_F32 && dtype != UP_EK_F16 && dtype != UP_EK_BF16) return UP_ERR_UNSUPPORTED;
  if (n_experts > kMaxExperts || k > kMaxK || tokens > (0x7fffffff - kTile) / k) return UP_ERR_UNSUPPORTED;
  UP_CHECK_ARG(offsets != nullptr);
  UP_CHECK_ARG(tokens == 0 || (logits && ids && weights && rows && slots && workspace));
  UP_CHECK_ARG(tokens <= 1 || stride >= n_experts);
  UP_CHECK_ARG(aligned(workspace, 256) && (tokens == 0 || workspace_bytes >= up_sm100_expert_route_workspace_bytes(tokens, n_experts)));
  Route a{};
  a.logits = logits, a.stride = stride, a.tokens = (int)tokens, a.experts = (int)n_experts, a.k = (int)k, a.score = score;
  a.renormalise = renormalise != 0, a.gain = gain, a.ids = ids, a.rows = rows, a.slots = slots, a.offsets = offsets;
  a.weights = weights, a.counts = static_cast<uint32_t*>(workspace), a.span = kTile, a.per = 1;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == UP_EK_F32) return route_sized<float>(a, s);
  if (dtype == UP_EK_F16) return route_sized<__half>(a, s);
  return route_sized<__nv_bfloat16>(a, s);
}

extern "C" int up_sm100_expert_combine(const void* y, int dtype, int64_t rows, int64_t y_stride, int64_t n,
                                       const int32_t* slots, const float* weights, int64_t tokens, int64_t k,
                                       const void* add, int64_t add_stride, void* out, int64_t out_stride, void* stream) {
  UP_CHECK_ARG(rows >= 0 && n >= 0 && tokens >= 0 && k >= 0 && y_stride >= 0 && add_stride >= 0 && out_stride >= 0);
  if (dtype != UP_EK_F32 && dtype != UP_EK_F16 && dtype != UP_EK_BF16) return UP_ERR_UNSUPPORTED;
  if (k > 0x7fffffff || n > ((int64_t)1 << 31) || tokens > ((int64_t)1 << 31)) return UP_ERR_UNSUPPORTED;
  if (tokens == 0 || n == 0) return UP_OK;
  UP_CHECK_ARG(out != nullptr && (y != nullptr || rows == 0) && (k == 0 || (slots && weights)));
  UP_CHECK_ARG((rows <= 1 || y_stride >= n) && (tokens <= 1 || (out_stride >= n && (!add || add_stride >= n))));
  if (rows <= 1) y_stride = 0;
  if (tokens == 1) add_stride = out_stride = 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int v = dtype == UP_EK_F32 ? 4 : 8;
  // 16 bytes a thread where every row starts on 16 bytes, single values else
  const bool wide = n % v == 0 && y_stride % v == 0 && out_stride % v == 0 && add_stride % v == 0 && aligned(y, 16) &&
                    aligned(out, 16) && aligned(add, 16);
#define UP_SUM(T, V) combine<T, V>(y, rows, y_stride, n, slots, weights, tokens, k, add, add_stride, out, out_stride, s)
  if (dtype == UP_EK_F32) return wide ? UP_SUM(float, 4) : UP_SUM(float, 1);
  if (dtype == UP_EK_F16) return wide ? UP_SUM(__half, 8) : UP_SUM(__half, 1);
  return wide ? UP_SUM(__nv_bfloat16, 8) : UP_SUM(__nv_bfloat16, 1);
#undef UP_SUM
}

UP_DEFINE_REVISION(experts)
