// f8_quantise.cu — activations and weights as e4m3 values with an f32 scale for each block of 128.
//
// For a block with largest finite magnitude a: scale = a * f32(1/448), q = e4m3(y * (1/scale)). Every step is one IEEE
// operation in f32 (1/scale is a correctly rounded division), so values and scales are the plain formula's bit for bit, with a
// gate too: y = x / (1 + exp(-x)) * u by f32's exponential and rounded quotient. (By ex2.approx and rcp.approx y was up to
// 2^-19 off: of 32768 x 2048 values a third of the scales were other numbers, and 70 codes their neighbours.)
//
// Bound by HBM: 2 (4, 8) bytes read and 1.03 written a value; gated 16-bit values by instructions as well (82 % of the issue slots). Measured:
// 32768 x 2048 gated bf16 values 62.5 us (5.4 TB/s; 68 to 71 where many of the gates are far from 0), gated f32 87 (7.0), plain bf16 40
// (5.1); 64 x 4096 x 2048 bf16 weights 5.3 TB/s. Blocks that walk over the pieces with the next one's loads on their way took 61 to 120
// us where the same sums without took 59.
// The operator's other sources, which its revision hash covers through this line (build.py --sources):
// FNV-1a 64 of divide.cuh, launch.cuh: 2e2d27af524d7113
#include "common.cuh"
#include "divide.cuh"
#include "launch.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

namespace up {
namespace f8q {

constexpr int kThreads = 256;
constexpr int kBlock = 128;           // values a scale
constexpr float kMax = 448.f;         // e4m3's largest
constexpr float kSmallest = 1.17549435e-38f;  // 2^-126: a smaller scale has no finite 1/scale to rely on

// Sixteen values as they lie in memory (8 words of two, or 16), by loads of 32 bytes where they lie on such borders (ordinary ones: launch.cuh).
template <typename T>
struct Raw {
  uint32_t w[8];
};
template <>
struct Raw<float> {
  uint32_t w[16];
};
__device__ __forceinline__ void load32(const void* p, uint32_t* w, bool wide) {
  if (wide) {
    asm volatile("ld.global.L1::no_allocate.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                 : "l"(p));
  } else {
#pragma unroll
    for (int i = 0; i < 8; i += 4)
      asm volatile("ld.global.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(w[i]), "=r"(w[i + 1]), "=r"(w[i + 2]), "=r"(w[i + 3])
                   : "l"(static_cast<const char*>(p) + 4 * i));
  }
}
template <typename T>
__device__ __forceinline__ void load(const T* p, Raw<T>& r, bool wide) {
  load32(p, r.w, wide);
  if (sizeof(T) == 4) load32(reinterpret_cast<const char*>(p) + 32, r.w + (sizeof(T) == 4 ? 8 : 0), wide);
}
template <typename T>
__device__ __forceinline__ void clear(Raw<T>& r) {
#pragma unroll
  for (int i = 0; i < (int)(sizeof(r) / 4); ++i) r.w[i] = 0;
}
__device__ __forceinline__ void widen(const Raw<float>& r, float (&v)[16]) {
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r.w[i]);
}
__device__ __forceinline__ void widen(const Raw<__half>& r, float (&v)[16]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&r.w[i]));
    v[2 * i] = f.x, v[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ void widen(const Raw<__nv_bfloat16>& r, float (&v)[16]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) v[2 * i] = __uint_as_float(r.w[i] << 16), v[2 * i + 1] = __uint_as_float(r.w[i] & 0xffff0000u);
}

__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ float as_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float as_float(__nv_bfloat16 v) { return __bfloat162float(v); }

// Magnitudes compare as their bits do; those from kInfinity on are not finite.
constexpr uint32_t kInfinity = 0x7f800000u;
__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }
__device__ __forceinline__ float max_abs(float a, float b, float c) {  // a NaN if one of them is
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ uint32_t largest(const float (&v)[16]) {
  float a = v[0];
#pragma unroll
  for (int i = 1; i < 15; i += 2) a = max_abs(a, v[i], v[i + 1]);
  return magnitude(max_abs(a, v[15], 0.f));
}
__device__ __forceinline__ uint32_t largest_finite(const float (&v)[16]) {
  uint32_t a = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) a = max(a, magnitude(v[i]) < kInfinity ? magnitude(v[i]) : 0u);
  return a;
}

__device__ __forceinline__ float scale_of(uint32_t a) {
  const float s = __uint_as_float(a) * (1.f / kMax);
  return s >= kSmallest ? s : 0.f;
}

// Sixteen values as e4m3 bytes; |v * inv| is at most 448 (1 + 2^-22). CHECK: some may not be finite.
template <bool CHECK>
__device__ __forceinline__ uint4 codes(const float (&v)[16], float inv) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t two[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float a = v[4 * i + 2 * h], b = v[4 * i + 2 * h + 1];
      float2 f = make_float2(a * inv, b * inv);
      if (CHECK && magnitude(a) >= kInfinity) f.x = __int_as_float(0x7fc00000);
      if (CHECK && magnitude(b) >= kInfinity) f.y = __int_as_float(0x7fc00000);
      two[h] = __nv_cvt_float2_to_fp8x2(f, __NV_SATFINITE, __NV_E4M3);
    }
    w[i] = __byte_perm(two[0], two[1], 0x5410);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Two f32 operations in one instruction.
__device__ __forceinline__ uint64_t pair_of(float a, float b) { return (uint64_t)__float_as_uint(b) << 32 | __float_as_uint(a); }
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t c;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(c) : "l"(a), "l"(b));
  return c;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ float reciprocal_approx(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
// x / (1 + exp(-x)) * g with f32's exponential and quotient. The quotient is x times an approximate reciprocal with one correction by its
// remainder (Markstein, "Computation of elementary functions on the IBM RISC System/6000 processor", 1990), of both by 1/4 so that the
// reciprocal is a normal number: for each f32 x from -88.7 up, of 2^-100 at least, that is the rounded quotient (compared for all of them;
// 63 us where the compiler's quotient takes 89). Below, where exp(-x) leaves f32, and for values that are not finite it gives a NaN.
__device__ __forceinline__ void gated(float& x0, float& x1, float g0, float g1) {
  const float d0 = fmaf(expf(-x0), -0.25f, -0.25f), d1 = fmaf(expf(-x1), -0.25f, -0.25f);
  const uint64_t d = pair_of(d0, d1), r = pair_of(reciprocal_approx(-d0), reciprocal_approx(-d1));
  const uint64_t x = mul2(pair_of(x0, x1), pair_of(0.25f, 0.25f)), q = mul2(x, r);
  const uint64_t y = mul2(fma2(fma2(d, q, x), r, q), pair_of(g0, g1));
  x0 = __uint_as_float((uint32_t)y), x1 = __uint_as_float((uint32_t)(y >> 32));
}
// The same for all values: with exp(-x) out of range 1 + exp(-x) is exp(-x) to the last bit, which goes by halves.
__device__ __forceinline__ float gated_any(float x, float g) {
  const float d = 1.f + expf(-x);
  if (d < __uint_as_float(kInfinity)) return x / d * g;
  const float h = expf(0.5f * x);
  return x * h * g * h;
}

// Those of sixteen that are no finite numbers once more, from memory, so that the kernel need not hold its inputs for them.
template <typename T>
__device__ __forceinline__ void gate_again(const T* from, int k, float (&v)[16]) {
  uint32_t bad = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) bad |= magnitude(v[i]) >= kInfinity ? 1u << i : 0u;
#pragma unroll 1
  for (; bad != 0; bad &= bad - 1) {
    const int at = __ffs(bad) - 1;
    const float y = gated_any(as_float(from[at]), as_float(from[k + at]));
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = i == at ? y : v[i];
  }
}

// A piece is 16 values; 8 pieces (a quarter of a warp) are a block. The last block of a row may have fewer. A thread has U pieces, whose loads
// are all on their way before the first is looked at. Gated 16-bit values are held to 40 registers a thread, six blocks an SM: 62.5 us where five
// take 67. (With 8 values a piece the blocks' own instructions, 150 a piece, were the bound:
// 8192 x 8192 bf16 values took 52 us.)
template <typename T, bool GATE, int U, typename Div>
__global__ void __launch_bounds__(kThreads, GATE && sizeof(T) == 2 ? 6 : 0)
    quantise_kernel(const T* x, int64_t tokens, int64_t x_stride, const int32_t* rows,
                    typename Div::Int pieces, Div by_row, int k, bool wide, uint4* __restrict__ q, float* __restrict__ scale,
                    int64_t ss_r, int64_t ss_b) {
  using Int = typename Div::Int;
  const int row_pieces = (k + kBlock - 1) / kBlock * (kBlock / 16);
  const Int p0 = (Int)blockIdx.x * (kThreads * U) + threadIdx.x;
  const unsigned mask = 0xffu << (threadIdx.x & 24);
  Raw<T> raw[U][GATE ? 2 : 1];
  after_previous();
  let_next_begin();
  Int row[U];
  int at[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    // pieces is a multiple of 8, as kThreads is: the 8 lanes of a block are there together or not at all
    const Int p = p0 + u * kThreads;
    row[u] = p < pieces ? by_row(p) : 0;
    at[u] = p < pieces ? (int)(p - row[u] * (Int)row_pieces) * 16 : -1;
    const int64_t src = at[u] < 0 || at[u] >= k ? -1 : rows ? (int64_t)rows[row[u]] : (int64_t)row[u];
    if ((uint64_t)src < (uint64_t)tokens) {
      const T* from = x + src * x_stride + at[u];
      load(from, raw[u][0], wide);
      if (GATE) load(from + k, raw[u][GATE], wide);
    } else {
      clear(raw[u][0]);
      if (GATE) clear(raw[u][GATE]);
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (at[u] < 0) break;
    float v[16];
    widen(raw[u][0], v);
    if (GATE) {
      float g[16];
      widen(raw[u][GATE], g);
#pragma unroll
      for (int i = 0; i < 16; i += 2) gated(v[i], v[i + 1], g[i], g[i + 1]);
    }
    uint32_t a = largest(v);
    if (GATE && a >= kInfinity) {
      gate_again(x + (rows ? (int64_t)rows[row[u]] : (int64_t)row[u]) * x_stride + at[u], k, v);
      a = largest(v);
    }
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) a = max(a, __shfl_xor_sync(mask, a, o));
    const bool fine = a < kInfinity;  // alike in the block's lanes
    if (!fine) {
      a = largest_finite(v);
#pragma unroll
      for (int o = 4; o > 0; o >>= 1) a = max(a, __shfl_xor_sync(mask, a, o));
    }
    const float s = scale_of(a);
    const float inv = s > 0.f ? __frcp_rn(s) : 0.f;
    if (at[u] < k) q[((int64_t)row[u] * k + at[u]) >> 4] = fine ? codes<false>(v, inv) : codes<true>(v, inv);
    if ((threadIdx.x & 7) == 0) scale[(int64_t)row[u] * ss_r + (at[u] / kBlock) * ss_b] = s;
  }
}

// One CTA a block of 128 x 128 weights: its values stay in registers between the maximum and the codes.
template <typename T>
__global__ void __launch_bounds__(kThreads)
    weight_kernel(const T* w, int64_t n, int64_t k, int64_t stride_e, int64_t stride_n, uint32_t blocks_k,
                  uint32_t blocks_n, bool wide, uint4* __restrict__ q, float* __restrict__ scale) {
  const uint32_t rest = blockIdx.x / blocks_k, e = rest / blocks_n;
  const int64_t bk = blockIdx.x - rest * blocks_k, bn = rest - e * blocks_n;
  const int64_t col = bk * kBlock + (threadIdx.x & 7) * 16;
  constexpr int kApart = kThreads / 8, kEach = kBlock / kApart;  // rows from one to the next of a thread, and how many it has
  const int64_t row0 = bn * kBlock + (threadIdx.x >> 3);
  Raw<T> raw[kEach];
  uint32_t a = 0;
  after_previous();
  let_next_begin();
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    clear(raw[j]);
    if (row0 + j * kApart < n && col < k) load(w + e * stride_e + (row0 + j * kApart) * stride_n + col, raw[j], wide);
  }
  float v[16];
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    widen(raw[j], v);
    a = max(a, largest(v));
  }
  __shared__ uint32_t part[2][kThreads / 32];
  a = __reduce_max_sync(0xffffffffu, a);
  if ((threadIdx.x & 31) == 0) part[0][threadIdx.x >> 5] = a;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kThreads / 32; ++i) a = max(a, part[0][i]);
  const bool fine = a < kInfinity;
  if (!fine) {
    a = 0;
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      widen(raw[j], v);
      a = max(a, largest_finite(v));
    }
    a = __reduce_max_sync(0xffffffffu, a);
    if ((threadIdx.x & 31) == 0) part[1][threadIdx.x >> 5] = a;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kThreads / 32; ++i) a = max(a, part[1][i]);
  }
  const float s = scale_of(a);
  const float inv = s > 0.f ? __frcp_rn(s) : 0.f;
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    const int64_t row = row0 + j * kApart;
    if (row < n && col < k) {
      widen(raw[j], v);
      q[((e * n + row) * k + col) >> 4] = fine ? codes<false>(v, inv) : codes<true>(v, inv);
    }
  }
  if (threadIdx.x == 0) scale[blockIdx.x] = s;
}

template <typename T, bool GATE, int U>
int quantise_by(const T* x, int64_t tokens, int64_t x_stride, const int32_t* rows, int64_t pieces, int64_t row_pieces, int64_t k,
                uint4* q, float* scale, int64_t ss_r, int64_t ss_b, cudaStream_t s) {
  const int64_t ctas = (pieces + kThreads * U - 1) / (kThreads * U);
  if (ctas > 0x7fffffff) return UP_ERR_UNSUPPORTED;
  // gated values of 16 bits lie 2k bytes on, of 32 bits 4k: k is a multiple of 16, so on such borders as x is
  const bool wide = aligned(x, 32) && x_stride * sizeof(T) % 32 == 0;
  const cudaError_t e =
      pieces + kThreads * U < (int64_t)1 << 31
          ? launch_early(quantise_kernel<T, GATE, U, Divide32>, (unsigned)ctas, kThreads, 0, s, x, tokens, x_stride, rows,
                         (uint32_t)pieces, Divide32(row_pieces), (int)k, wide, q, scale, ss_r, ss_b)
          : launch_early(quantise_kernel<T, GATE, U, Divide64>, (unsigned)ctas, kThreads, 0, s, x, tokens, x_stride, rows,
                         (uint64_t)pieces, Divide64(row_pieces), (int)k, wide, q, scale, ss_r, ss_b);
  if (e != cudaSuccess) return cuda_status(e);
  note_launch();
  return check_launch();
}
template <typename T, bool GATE>
int quantise(const void* x, int64_t tokens, int64_t x_stride, const int32_t* rows, int64_t n_rows, int64_t k, uint8_t* q,
             float* scale, int64_t ss_r, int64_t ss_b, cudaStream_t s) {
  const int64_t row_pieces = (k + kBlock - 1) / kBlock * (kBlock / 16), pieces = n_rows * row_pieces;
  constexpr int kMany = sizeof(T) == 4 || GATE ? 1 : 2;  // 64 bytes a thread on their way
  const T* from = static_cast<const T*>(x);
  uint4* to = reinterpret_cast<uint4*>(q);
  // one piece a thread until the SMs are full
  if (pieces <= (int64_t)sm_count() * 2048)
    return quantise_by<T, GATE, 1>(from, tokens, x_stride, rows, pieces, row_pieces, k, to, scale, ss_r, ss_b, s);
  return quantise_by<T, GATE, kMany>(from, tokens, x_stride, rows, pieces, row_pieces, k, to, scale, ss_r, ss_b, s);
}

template <typename T>
int quantise_weight(const void* w, int64_t experts, int64_t n, int64_t k, int64_t se, int64_t sn, uint8_t* q, float* scale,
                    cudaStream_t s) {
  const int64_t bk = (k + kBlock - 1) / kBlock, bn = (n + kBlock - 1) / kBlock;
  const cudaError_t e = launch_early(weight_kernel<T>, (unsigned)(experts * bn * bk), kThreads, 0, s, static_cast<const T*>(w), n, k, se,
                                     sn, (uint32_t)bk, (uint32_t)bn,
                                     aligned(w, 32) && se * sizeof(T) % 32 == 0 && sn * sizeof(T) % 32 == 0,
                                     reinterpret_cast<uint4*>(q), scale);
  if (e != cudaSuccess) return cuda_status(e);
  note_launch();
  return check_launch();
}

int size_of(int dtype) { return dtype == UP_EK_F32 ? 4 : dtype == UP_EK_F16 || dtype == UP_EK_BF16 ? 2 : 0; }

}  // namespace f8q
}  // namespace up

using namespace up;
using namespace up::f8q;

extern "C" int up_sm100_f8_quantise(const void* x, int dtype, int64_t tokens, int64_t x_stride, const int32_t* rows,
                                    int64_t n_rows, int64_t k, int gate, uint8_t* q, float* scale, int64_t scale_stride_r,
                                    int64_t scale_stride_b, void* stream) {
  UP_CHECK_ARG(tokens >= 0 && n_rows >= 0 && k >= 0 && x_stride >= 0 && scale_stride_r >= 0 && scale_stride_b >= 0);
  UP_CHECK_ARG(rows != nullptr || n_rows == tokens);
  const int size = size_of(dtype);
  if (size == 0 || k % 16 != 0 || k > (1 << 30)) return UP_ERR_UNSUPPORTED;
  if (n_rows == 0 || k == 0) return UP_OK;
  UP_CHECK_ARG((x != nullptr || tokens == 0) && q != nullptr && scale != nullptr);
  UP_CHECK_ARG(tokens <= 1 || x_stride >= (gate ? 2 * k : k));
  if (tokens <= 1) x_stride = 0;
  if (!aligned(x, 16) || x_stride * size % 16 != 0 || !aligned(q, 16)) return UP_ERR_UNSUPPORTED;
  if (n_rows > ((int64_t)1 << 40) / k) return UP_ERR_UNSUPPORTED;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
#define UP_F8_CALL(T)                                                                                                     \
  (gate ? quantise<T, true>(x, tokens, x_stride, rows, n_rows, k, q, scale, scale_stride_r, scale_stride_b, s)            \
        : quantise<T, false>(x, tokens, x_stride, rows, n_rows, k, q, scale, scale_stride_r, scale_stride_b, s))
  if (dtype == UP_EK_F32) return UP_F8_CALL(float);
  if (dtype == UP_EK_F16) return UP_F8_CALL(__half);
  return UP_F8_CALL(__nv_bfloat16);
#undef UP_F8_CALL
}

extern "C" int up_sm100_f8_quantise_weight(const void* w, int dtype, int64_t experts, int64_t n, int64_t k,
                                           int64_t w_stride_e, int64_t w_stride_n, uint8_t* q, float* scale,
                                           void* stream) {
  UP_CHECK_ARG(experts >= 0 && n >= 0 && k >= 0 && w_stride_e >= 0 && w_stride_n >= 0);
  const int size = size_of(dtype);
  if (size == 0 || k % 16 != 0) return UP_ERR_UNSUPPORTED;
  if (experts == 0 || n == 0 || k == 0) return UP_OK;
  UP_CHECK_ARG(w != nullptr && q != nullptr && scale != nullptr);
  UP_CHECK_ARG(n <= 1 || w_stride_n >= k);
  if (n == 1) w_stride_n = 0;
  if (experts == 1) w_stride_e = 0;
  if (!aligned(w, 16) || w_stride_n * size % 16 != 0 || w_stride_e * size % 16 != 0 || !aligned(q, 16))
    return UP_ERR_UNSUPPORTED;
  const int64_t bk = (k + kBlock - 1) / kBlock, bn = (n + kBlock - 1) / kBlock;
  if (bk > 0x7fffffff / bn || experts > 0x7fffffff / (bn * bk)) return UP_ERR_UNSUPPORTED;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == UP_EK_F32) return quantise_weight<float>(w, experts, n, k, w_stride_e, w_stride_n, q, scale, s);
  if (dtype == UP_EK_F16) return quantise_weight<__half>(w, experts, n, k, w_stride_e, w_stride_n, q, scale, s);
  return quantise_weight<__nv_bfloat16>(w, experts, n, k, w_stride_e, w_stride_n, q, scale, s);
}

UP_DEFINE_REVISION(f8_quantise)
