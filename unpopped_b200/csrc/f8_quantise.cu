// f8_quantise.cu — activations and weights as e4m3 values with an f32 scale for each block of 128.
//
// For a block with largest finite magnitude a: scale = a * f32(1/448), q = e4m3(y * (1/scale)). Every step is one IEEE
// operation in f32 (1/scale is a correctly rounded division), so values and scales are the plain formula's bit for bit;
// with a gate, y itself goes by ex2.approx and rcp.approx (about 2^-21, an eighth of a thousandth of e4m3's half step).
//
// Bound by HBM: 2 (4, 8) bytes read and 1.03 written a value.
#include "common.cuh"
#include "divide.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

namespace up {
namespace f8q {

constexpr int kThreads = 256;
constexpr int kBlock = 128;           // values a scale
constexpr float kMax = 448.f;         // e4m3's largest
constexpr float kSmallest = 1.17549435e-38f;  // 2^-126: a smaller scale has no finite 1/scale to rely on

__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
  const float4 a = ld_nc_na_f4(p), b = ld_nc_na_f4(p + 4);
  v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}
__device__ __forceinline__ void load8(const __half* p, float (&v)[8]) {
  const uint4 u = ld_nc_na_v4(p);
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    v[2 * i] = f.x, v[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ void load8(const __nv_bfloat16* p, float (&v)[8]) {
  const uint4 u = ld_nc_na_v4(p);
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) v[2 * i] = __uint_as_float(w[i] << 16), v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
}

__device__ __forceinline__ bool finite(float v) { return fabsf(v) < __int_as_float(0x7f800000); }

__device__ __forceinline__ float largest(const float (&v)[8]) {
  float a = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) a = fmaxf(a, finite(v[i]) ? fabsf(v[i]) : 0.f);
  return a;
}

__device__ __forceinline__ float scale_of(float a) {
  const float s = a * (1.f / kMax);
  return s >= kSmallest ? s : 0.f;
}

// Eight values as e4m3 bytes. |y * inv| is at most 448 (1 + 2^-22), so only values that are not finite need a care.
__device__ __forceinline__ uint2 codes(const float (&v)[8], float inv) {
  uint32_t w[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float2 f;
    f.x = finite(v[2 * i]) ? v[2 * i] * inv : __int_as_float(0x7fc00000);
    f.y = finite(v[2 * i + 1]) ? v[2 * i + 1] * inv : __int_as_float(0x7fc00000);
    w[i >> 1] |= (uint32_t)__nv_cvt_float2_to_fp8x2(f, __NV_SATFINITE, __NV_E4M3) << (16 * (i & 1));
  }
  return make_uint2(w[0], w[1]);
}

// A piece is 8 values; 16 pieces (half a warp) are a block. The last block of a row may have fewer.
template <typename T, bool GATE, typename Div>
__global__ void __launch_bounds__(kThreads)
    quantise_kernel(const T* __restrict__ x, int64_t tokens, int64_t x_stride, const int32_t* __restrict__ rows,
                    typename Div::Int pieces, Div by_row, int k, uint2* __restrict__ q, float* __restrict__ scale, int64_t ss_r,
                    int64_t ss_b) {
  using Int = typename Div::Int;
  const int row_pieces = (k + kBlock - 1) / kBlock * (kBlock / 8);
  for (Int p = (Int)blockIdx.x * kThreads + threadIdx.x; p < pieces; p += (Int)gridDim.x * kThreads) {
    // pieces is a multiple of 16 and so is the step: the 16 lanes of a block come here together
    const Int r = by_row(p);
    const int at = (int)(p - r * (Int)row_pieces) * 8;
    const int64_t src = rows ? (int64_t)rows[r] : (int64_t)r;
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = 0.f;
    if (at < k && (uint64_t)src < (uint64_t)tokens) {
      const T* from = x + src * x_stride + at;
      load8(from, v);
      if (GATE) {
        float u[8];
        load8(from + k, u);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = __fdividef(v[i], 1.f + __expf(-v[i])) * u[i];
      }
    }
    float a = largest(v);
    const unsigned mask = 0xffffu << (threadIdx.x & 16);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) a = fmaxf(a, __shfl_xor_sync(mask, a, o));
    const float s = scale_of(a);
    const float inv = s > 0.f ? 1.f / s : 0.f;
    if (at < k) q[((int64_t)r * k + at) >> 3] = codes(v, inv);
    if ((threadIdx.x & 15) == 0) scale[(int64_t)r * ss_r + (at / kBlock) * ss_b] = s;
  }
}

// One CTA a block of 128 x 128 weights: its values stay in registers between the maximum and the codes.
template <typename T>
__global__ void __launch_bounds__(kThreads)
    weight_kernel(const T* __restrict__ w, int64_t n, int64_t k, int64_t stride_e, int64_t stride_n, int64_t blocks_k,
                  int64_t blocks_n, uint2* __restrict__ q, float* __restrict__ scale) {
  const int64_t bk = blockIdx.x % blocks_k, rest = blockIdx.x / blocks_k, bn = rest % blocks_n, e = rest / blocks_n;
  const int piece = threadIdx.x & 15;
  const int64_t col = bk * kBlock + piece * 8;
  constexpr int kEach = kBlock / (kThreads / 16);  // rows a thread
  float v[kEach][8];
  float a = 0.f;
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    const int64_t row = bn * kBlock + (threadIdx.x >> 4) + j * (kThreads / 16);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[j][i] = 0.f;
    if (row < n && col < k) load8(w + e * stride_e + row * stride_n + col, v[j]);
  }
#pragma unroll
  for (int j = 0; j < kEach; ++j) a = fmaxf(a, largest(v[j]));
  __shared__ float part[kThreads / 32];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, o));
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = a;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kThreads / 32; ++i) a = fmaxf(a, part[i]);
  const float s = scale_of(a);
  const float inv = s > 0.f ? 1.f / s : 0.f;
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    const int64_t row = bn * kBlock + (threadIdx.x >> 4) + j * (kThreads / 16);
    if (row < n && col < k) q[((e * n + row) * k + col) >> 3] = codes(v[j], inv);
  }
  if (threadIdx.x == 0) scale[blockIdx.x] = s;
}

template <typename T, bool GATE>
int quantise(const void* x, int64_t tokens, int64_t x_stride, const int32_t* rows, int64_t n_rows, int64_t k, uint8_t* q,
             float* scale, int64_t ss_r, int64_t ss_b, cudaStream_t s) {
  const int64_t row_pieces = (k + kBlock - 1) / kBlock * (kBlock / 8);
  const int64_t pieces = n_rows * row_pieces;
  const int64_t ctas = (pieces + kThreads - 1) / kThreads;
  const int64_t most = (int64_t)sm_count() * 64;
  const unsigned grid = (unsigned)(ctas < most ? ctas : most);
  const T* from = static_cast<const T*>(x);
  uint2* to = reinterpret_cast<uint2*>(q);
  if (pieces + most * kThreads < (int64_t)1 << 31)
    quantise_kernel<T, GATE, Divide32><<<grid, kThreads, 0, s>>>(from, tokens, x_stride, rows, (uint32_t)pieces,
                                                                 Divide32(row_pieces), (int)k, to, scale, ss_r, ss_b);
  else
    quantise_kernel<T, GATE, Divide64><<<grid, kThreads, 0, s>>>(from, tokens, x_stride, rows, (uint64_t)pieces,
                                                                 Divide64(row_pieces), (int)k, to, scale, ss_r, ss_b);
  note_launch();
  return check_launch();
}

template <typename T>
int quantise_weight(const void* w, int64_t experts, int64_t n, int64_t k, int64_t se, int64_t sn, uint8_t* q, float* scale,
                    cudaStream_t s) {
  const int64_t bk = (k + kBlock - 1) / kBlock, bn = (n + kBlock - 1) / kBlock;
  weight_kernel<T><<<(unsigned)(experts * bn * bk), kThreads, 0, s>>>(static_cast<const T*>(w), n, k, se, sn, bk, bn,
                                                                      reinterpret_cast<uint2*>(q), scale);
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
