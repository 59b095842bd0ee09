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

}  // namespace rp
}  // namespace up
