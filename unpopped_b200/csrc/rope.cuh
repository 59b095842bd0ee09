// rope.cuh — rotary positions: what rope.cu and kv4_append.cu share.
//
// A position p rotates the pairs of a head's first `rot` dimensions. With c = table[p][i] and s = table[p][rot/2 + i],
//   y0 = x0 c - x1 s,  y1 = x1 c + x0 s
// for the pairs (i, i + rot/2) (half layout) or (2i, 2i + 1) (interleaved), i < rot/2. The map's transpose, which is
// the gradient's, has -s in place of s. Every product and sum is rounded to f32 by itself (no fused multiply-add), so
// the result does not depend on how a compiler contracts the formula, and the quantised cache is reproducible bit for
// bit from it.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "divide.cuh"

namespace up {
namespace rp {

__device__ __forceinline__ int64_t load_id(const void* ids, int kind, int64_t i) {
  return kind == UP_EK_I64 ? (int64_t)__ldg(static_cast<const long long*>(ids) + i)
                           : (int64_t)__ldg(static_cast<const int*>(ids) + i);
}

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32(float v) { return __float2bfloat16_rn(v); }

// One pair: (a, b) becomes (a c - b s, b c + a s).
__device__ __forceinline__ void rotate(float& a, float& b, float c, float s) {
  const float y0 = __fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s));
  const float y1 = __fadd_rn(__fmul_rn(b, c), __fmul_rn(a, s));
  a = y0;
  b = y1;
}

// The 16 bytes of a chunk and their elements in f32.
template <typename T>
struct Chunk {
  static constexpr int N = 16 / sizeof(T);
  __device__ static __forceinline__ void unpack(uint4 u, float (&f)[N]) {
    const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = to_f32<T>(e[i]);
  }
  __device__ static __forceinline__ uint4 pack(const float (&f)[N]) {
    uint4 u;
    T* e = reinterpret_cast<T*>(&u);
#pragma unroll
    for (int i = 0; i < N; ++i) e[i] = from_f32<T>(f[i]);
    return u;
  }
};

// N consecutive f32 of a table row; N is 2 (8-byte aligned) or a multiple of 4 (16-byte aligned).
template <int N>
__device__ __forceinline__ void load_row(const float* p, float (&f)[N]) {
  if constexpr (N == 2) {
    const float2 v = __ldg(reinterpret_cast<const float2*>(p));
    f[0] = v.x, f[1] = v.y;
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const float4 v = __ldg(reinterpret_cast<const float4*>(p + i));
      f[i] = v.x, f[i + 1] = v.y, f[i + 2] = v.z, f[i + 3] = v.w;
    }
  }
}

struct Geometry {
  int64_t seq, heads, dim, rot;
  int64_t xb, xs, xh, ob, os, oh;  // strides in elements: batch, token, head
  const void* positions;           // NULL: a token's index in its sequence
  int index_dtype;
  int64_t pos_stride_b, n_pos;
};

__device__ __forceinline__ int64_t position(const Geometry& g, int64_t b, int64_t s) {
  return g.positions ? load_id(g.positions, g.index_dtype, b * g.pos_stride_b + s) : s;
}

// How items of the vector form are counted: unit fastest, then group of heads, token, sequence.
template <typename Div>
struct Items {
  Div units, groups, seq;
  typename Div::Int count;
};

// One item of the vector form: a unit of two 16-byte chunks of HEADS heads (head, head + groups, ...), whose loads are in
// flight together and which share the token's cosines and sines. The units of a head: half layout rot / 2N of chunk j of
// the first half and chunk j of the second, then neighbours of the dimensions that are only copied; interleaved
// neighbours throughout. The last unit may have one chunk.
template <typename T, bool HALF, int HEADS, typename Div>
__device__ __forceinline__ void rope_item(const T* x, T* out, const float* __restrict__ table, const Geometry& g,
                                          typename Div::Int item, const Items<Div>& n, int backward) {
  constexpr int N = Chunk<T>::N, C = HALF ? N : N / 2;  // cosines a chunk needs
  using I = typename Div::Int;
  const I row = n.units(item), u = item - row * n.units.d;
  const I tok = n.groups(row), hg = row - tok * n.groups.d;
  const I b = n.seq(tok), s = tok - b * n.seq.d;
  const int dim = (int)g.dim, rot = (int)g.rot, pairs = HALF ? rot / (2 * N) : 0;
  const bool paired = HALF && (int)u < pairs;
  const int e0 = paired ? (int)u * N : (HALF ? rot : 0) + 2 * ((int)u - pairs) * N;
  const int e1 = paired ? e0 + rot / 2 : e0 + N;
  const bool two = e1 < dim, turn0 = e0 < rot, turn1 = !HALF && e1 < rot;
  const T* xr = x + (int64_t)b * g.xb + (int64_t)s * g.xs + (int64_t)hg * g.xh;
  T* o = out + (int64_t)b * g.ob + (int64_t)s * g.os + (int64_t)hg * g.oh;
  const int64_t xstep = (int64_t)n.groups.d * g.xh, ostep = (int64_t)n.groups.d * g.oh;
  const int heads = (int)min((int64_t)HEADS, (g.heads - (int64_t)hg + n.groups.d - 1) / n.groups.d);
  uint4 lo[HEADS], hi[HEADS];
#pragma unroll
  for (int k = 0; k < HEADS; ++k) {
    if (k >= heads) continue;
    lo[k] = *reinterpret_cast<const uint4*>(xr + k * xstep + e0);
    if (two) hi[k] = *reinterpret_cast<const uint4*>(xr + k * xstep + e1);
  }
  float c[2 * C], sn[2 * C];  // of the first chunk, and (interleaved) of the second
  if (turn0) {
    const int64_t p = position(g, b, s);
    const bool in = p >= 0 && p < g.n_pos;
    const float* t = table + (in ? p : 0) * rot + (HALF ? e0 : e0 / 2);
#pragma unroll
    for (int i = 0; i < 2 * C; ++i) c[i] = sn[i] = __int_as_float(0x7fffffff);
    if (in) {
      float(&c0)[C] = *reinterpret_cast<float(*)[C]>(c), (&s0)[C] = *reinterpret_cast<float(*)[C]>(sn);
      load_row<C>(t, c0);
      load_row<C>(t + rot / 2, s0);
      if (turn1) {
        float(&c1)[C] = *reinterpret_cast<float(*)[C]>(c + C), (&s1)[C] = *reinterpret_cast<float(*)[C]>(sn + C);
        load_row<C>(t + C, c1);
        load_row<C>(t + rot / 2 + C, s1);
      }
    }
    if (backward)
#pragma unroll
      for (int i = 0; i < 2 * C; ++i) sn[i] = -sn[i];
  }
#pragma unroll
  for (int k = 0; k < HEADS; ++k) {
    if (k >= heads) continue;
    if (turn0) {
      float a[N], d[N];
      Chunk<T>::unpack(lo[k], a);
      if constexpr (HALF) {
        Chunk<T>::unpack(hi[k], d);
#pragma unroll
        for (int i = 0; i < N; ++i) rotate(a[i], d[i], c[i], sn[i]);
        hi[k] = Chunk<T>::pack(d);
      } else {
#pragma unroll
        for (int i = 0; i < N / 2; ++i) rotate(a[2 * i], a[2 * i + 1], c[i], sn[i]);
        if (turn1) {
          Chunk<T>::unpack(hi[k], d);
#pragma unroll
          for (int i = 0; i < N / 2; ++i) rotate(d[2 * i], d[2 * i + 1], c[C + i], sn[C + i]);
          hi[k] = Chunk<T>::pack(d);
        }
      }
      lo[k] = Chunk<T>::pack(a);
    }
    st_cs_v4(o + k * ostep + e0, lo[k]);
    if (two) st_cs_v4(o + k * ostep + e1, hi[k]);
  }
}

template <typename T>
inline int64_t rope_units(const Geometry& g, bool half) {
  constexpr int N = Chunk<T>::N;
  const int64_t pairs = half ? g.rot / (2 * N) : 0;
  return pairs + ((g.dim - 2 * pairs * N) / N + 1) / 2;
}

// Heads an item: four where that leaves a thousand threads an SM, two where that leaves half as many, else one. Forward and
// backward of 16384 x 64 x 128 bf16 take 171 us with four, 178 with two and 199 with one, of 1999 x 24 x 96 f32 (in L2) 16.8,
// 14.9 and 14.9, of one token of 64 x 128 2.6, 2.4 and 2.1; an append of 16001 tokens, read back, 132, 147 and 179.
template <typename T>
inline int rope_heads(const Geometry& g, int64_t tokens, bool half) {
  const int64_t units = rope_units<T>(g, half), sms = sm_count();
  if (tokens * ((g.heads + 3) / 4) * units >= sms * 1024) return 4;
  return tokens * ((g.heads + 1) / 2) * units >= sms * 512 ? 2 : 1;
}

// Whether the vector form serves: whole 16-byte chunks everywhere.
template <typename T>
inline bool rope_vector(const void* x, const void* out, const float* table, const Geometry& g, bool half) {
  constexpr int N = Chunk<T>::N;
  return (g.xb | g.xs | g.xh | g.ob | g.os | g.oh) % N == 0 && g.dim % N == 0 && g.rot % (half ? 2 * N : N) == 0 &&
         g.dim <= 0x3fffffff &&
         aligned(x, 16) && aligned(out, 16) && aligned(table, 16);
}

}  // namespace rp
}  // namespace up
