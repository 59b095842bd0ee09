// rope.cu — rotary positions (rope.cuh has the formula): forward, the gradient, and the table of cosines and sines.
//
// What bounds it: HBM. Every element of x is read once and written once (2 * size bytes) for 3 flops; the table rows
// (4 * rot bytes a token, against heads * dim * size of x) are read again for each head, from L1. 16384 tokens of 64
// heads of 128, bf16, forward and backward: 171 us (1.09 GB: 6.4 TB/s).
//
// A thread owns two 16-byte chunks whose pairs are complete: in the half layout chunk j of the first half and chunk j of
// the second, in the interleaved one two neighbours. So a pair is rotated in one thread, nothing is exchanged, and a row
// may be rotated in place. Consecutive threads take consecutive chunks of a head, then heads, then tokens.
// The operator's other sources, which its revision hash covers through this line (build.py --sources):
// FNV-1a 64 of divide.cuh, rope.cuh: b29fc97861bc8e05
#include "rope.cuh"

#include <type_traits>

namespace up {
namespace rp {

constexpr int kThreads = 256;

template <typename T, bool HALF, int HEADS, typename Div>
__global__ void __launch_bounds__(kThreads) rope_vec_kernel(const T* x, T* out, const float* __restrict__ table,
                                                            const Geometry g, const Items<Div> n, int backward) {
  using I = typename Div::Int;
  const I item = (I)blockIdx.x * kThreads + threadIdx.x;
  if (item < n.count) rope_item<T, HALF, HEADS, Div>(x, out, table, g, item, n, backward);
}

// Any even rot, stride and alignment: a thread per pair, then per copied element.
template <typename T>
__global__ void __launch_bounds__(kThreads) rope_any_kernel(const T* x, T* out, const float* __restrict__ table,
                                                            const Geometry g, int64_t items, int half, int backward) {
  const int64_t units = g.rot / 2 + (g.dim - g.rot);
  for (int64_t item = (int64_t)blockIdx.x * kThreads + threadIdx.x; item < items;
       item += (int64_t)gridDim.x * kThreads) {
    const int64_t row = item / units, u = item - row * units;
    const int64_t tok = row / g.heads, h = row - tok * g.heads;
    const int64_t b = tok / g.seq, s = tok - b * g.seq;
    const T* xr = x + b * g.xb + s * g.xs + h * g.xh;
    T* o = out + b * g.ob + s * g.os + h * g.oh;
    if (u >= g.rot / 2) {
      o[u + g.rot / 2] = xr[u + g.rot / 2];
      continue;
    }
    const int64_t e0 = half ? u : 2 * u, e1 = half ? u + g.rot / 2 : 2 * u + 1;
    const int64_t p = position(g, b, s);
    const bool in = p >= 0 && p < g.n_pos;
    const float nan = __int_as_float(0x7fffffff);
    const float c = in ? __ldg(table + p * g.rot + u) : nan;
    float sn = in ? __ldg(table + p * g.rot + g.rot / 2 + u) : nan;
    if (backward) sn = -sn;
    float a = to_f32<T>(xr[e0]), d = to_f32<T>(xr[e1]);
    rotate(a, d, c, sn);
    o[e0] = from_f32<T>(a);
    o[e1] = from_f32<T>(d);
  }
}

template <typename T, bool HALF, int HEADS>
int launch_vec(const void* x, void* out, const float* table, const Geometry& g, int64_t tokens, int backward,
               cudaStream_t s) {
  const int64_t units = rope_units<T>(g, HALF), groups = (g.heads + HEADS - 1) / HEADS;
  const int64_t items = tokens * groups * units, blocks = (items + kThreads - 1) / kThreads;
  if (blocks > 0x7fffffff) return UP_ERR_UNSUPPORTED;
  const T* xt = static_cast<const T*>(x);
  T* ot = static_cast<T*>(out);
  if (items + kThreads <= 0x7fffffff && g.heads <= 0x7fffffff) {
    const Items<Divide32> n{Divide32(units), Divide32(groups), Divide32(g.seq), (uint32_t)items};
    rope_vec_kernel<T, HALF, HEADS, Divide32><<<(int)blocks, kThreads, 0, s>>>(xt, ot, table, g, n, backward);
  } else {
    const Items<Divide64> n{Divide64(units), Divide64(groups), Divide64(g.seq), (uint64_t)items};
    rope_vec_kernel<T, HALF, HEADS, Divide64><<<(int)blocks, kThreads, 0, s>>>(xt, ot, table, g, n, backward);
  }
  note_launch();
  return check_launch();
}

template <typename T>
int launch(const void* x, void* out, const float* table, const Geometry& g, int64_t tokens, int half, int backward,
           cudaStream_t s) {
  if (rope_vector<T>(x, out, table, g, half)) {
    const auto run = [&](auto heads) {
      constexpr int H = decltype(heads)::value;
      return half ? launch_vec<T, true, H>(x, out, table, g, tokens, backward, s)
                  : launch_vec<T, false, H>(x, out, table, g, tokens, backward, s);
    };
    const int heads = rope_heads<T>(g, tokens, half);
    if (heads == 4) return run(std::integral_constant<int, 4>{});
    return heads == 2 ? run(std::integral_constant<int, 2>{}) : run(std::integral_constant<int, 1>{});
  }
  const int64_t items = tokens * g.heads * (g.rot / 2 + (g.dim - g.rot));
  int64_t blocks = (items + kThreads - 1) / kThreads;
  const int64_t cap = (int64_t)sm_count() * 64;
  if (blocks > cap) blocks = cap;
  rope_any_kernel<T><<<(int)blocks, kThreads, 0, s>>>(static_cast<const T*>(x), static_cast<T*>(out), table, g, items,
                                                      half, backward);
  note_launch();
  return check_launch();
}

// A table is made once for a model, so nothing was done about its time: 32768 positions of 128 take 48 us, 53 scaled by
// WAVELENGTH and 69 by RAMP. Its bytes take 2.6; pow, log and sincos in f64, which a position times a frequency needs to keep
// f32's precision, bound it.
// One entry a thread, in f64 with one rounding: cos and sin of p * f_i. The frequencies f_i = base^(-2i / rot), and
// with `scaling` for contexts longer than a model was trained on (w = 2 pi / f_i is a frequency's wavelength):
//  LINEAR      f_i / factor
//  BASE        the base grown so that the last frequency is divided by factor: base * factor^(rot / (rot - 2))
//  WAVELENGTH  f_i where w < orig / high, f_i / factor where w > orig / low, between them the blend
//              (1 - t) f_i / factor + t f_i with t = (orig / w - low) / (high - low)
//  RAMP        the same blend with t = 1 - clamp((i - i_high) / (i_low - i_high), 0, 1), i_n the (rounded outwards)
//              index at which a wavelength fits `orig` n times
__global__ void __launch_bounds__(kThreads) rope_table_kernel(float* __restrict__ table, int64_t n_pos, int64_t rot,
                                                              double base, int scaling, double factor, double low,
                                                              double high, double orig, double gain) {
  const int64_t half = rot / 2;
  const double pi2 = 6.283185307179586476925;
  for (int64_t at = (int64_t)blockIdx.x * kThreads + threadIdx.x; at < n_pos * half;
       at += (int64_t)gridDim.x * kThreads) {
    const int64_t p = at / half, i = at - p * half;
    const double grown =
        scaling == UP_ROPE_BASE && rot > 2 ? base * pow(factor, (double)rot / (double)(rot - 2)) : base;
    double f = pow(grown, -2.0 * (double)i / (double)rot);
    if (scaling == UP_ROPE_LINEAR) f /= factor;
    if (scaling == UP_ROPE_WAVELENGTH) {
      const double turns = orig * f / pi2;  // orig / w
      const double t = turns >= high ? 1.0 : (turns <= low ? 0.0 : (turns - low) / (high - low));
      f = (1.0 - t) * f / factor + t * f;
    }
    if (scaling == UP_ROPE_RAMP) {
      const double per = (double)rot / (2.0 * log(base));
      const double a = fmax(floor(per * log(orig / (high * pi2))), 0.0);
      const double z = fmin(ceil(per * log(orig / (low * pi2))), (double)(rot - 1));
      const double t = 1.0 - fmin(fmax(((double)i - a) / (z > a ? z - a : 0.001), 0.0), 1.0);
      f = (1.0 - t) * f / factor + t * f;
    }
    double sn, c;
    sincos((double)p * f, &sn, &c);
    table[p * rot + i] = (float)(gain * c);
    table[p * rot + half + i] = (float)(gain * sn);
  }
}

}  // namespace rp
}  // namespace up

using namespace up;
using namespace up::rp;

extern "C" int up_sm100_rope(const void* x, int dtype, int64_t batch, int64_t seq, int64_t heads, int64_t dim,
                             int64_t x_stride_b, int64_t x_stride_s, int64_t x_stride_h, const void* positions,
                             int index_dtype, int64_t pos_stride_b, const float* table, int64_t n_pos, int64_t rot,
                             int layout, int backward, void* out, int64_t out_stride_b, int64_t out_stride_s,
                             int64_t out_stride_h, void* stream) {
  UP_CHECK_ARG(batch >= 0 && seq >= 0 && heads >= 0 && dim >= 0 && n_pos >= 0);
  UP_CHECK_ARG(rot >= 0 && rot <= dim && rot % 2 == 0);
  UP_CHECK_ARG(x_stride_b >= 0 && x_stride_s >= 0 && x_stride_h >= 0);
  // the output's rows must not overlap: each is written by threads of its own
  UP_CHECK_ARG((heads <= 1 || out_stride_h >= dim) && (seq <= 1 || out_stride_s >= dim) &&
               (batch <= 1 || out_stride_b >= dim));
  if (layout != UP_ROPE_HALF && layout != UP_ROPE_INTERLEAVED) return UP_ERR_UNSUPPORTED;
  if (positions != nullptr && index_dtype != UP_EK_I32 && index_dtype != UP_EK_I64) return UP_ERR_UNSUPPORTED;
  if (batch == 0 || seq == 0 || heads == 0 || dim == 0) return UP_OK;
  UP_CHECK_ARG(x != nullptr && out != nullptr && (table != nullptr || rot == 0) && pos_stride_b >= 0);
  // the stride of an extent of one is never used
  if (batch == 1) x_stride_b = out_stride_b = pos_stride_b = 0;
  if (seq == 1) x_stride_s = out_stride_s = 0;
  if (heads == 1) x_stride_h = out_stride_h = 0;
  const Geometry g{seq, heads, dim, rot, x_stride_b, x_stride_s, x_stride_h, out_stride_b, out_stride_s, out_stride_h,
                   positions, index_dtype, pos_stride_b, n_pos};
  const int half = layout == UP_ROPE_HALF;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case UP_EK_F32: return launch<float>(x, out, table, g, batch * seq, half, backward, s);
    case UP_EK_F16: return launch<__half>(x, out, table, g, batch * seq, half, backward, s);
    case UP_EK_BF16: return launch<__nv_bfloat16>(x, out, table, g, batch * seq, half, backward, s);
    default: return UP_ERR_UNSUPPORTED;
  }
}

extern "C" int up_sm100_rope_table(float* table, int64_t n_pos, int64_t rot, double base, int scaling, double factor,
                                   double low, double high, double orig, double gain, void* stream) {
  UP_CHECK_ARG(n_pos >= 0 && rot >= 0 && rot % 2 == 0 && base > 1.0);
  if (scaling < UP_ROPE_NONE || scaling > UP_ROPE_RAMP) return UP_ERR_UNSUPPORTED;
  UP_CHECK_ARG(scaling == UP_ROPE_NONE || factor > 0.0);
  UP_CHECK_ARG(scaling < UP_ROPE_WAVELENGTH || (low > 0.0 && high > low && orig > 0.0));
  if (n_pos == 0 || rot == 0) return UP_OK;
  UP_CHECK_ARG(table != nullptr);
  int64_t blocks = (n_pos * (rot / 2) + kThreads - 1) / kThreads;
  const int64_t cap = (int64_t)sm_count() * 32;
  if (blocks > cap) blocks = cap;
  rope_table_kernel<<<(int)blocks, kThreads, 0, static_cast<cudaStream_t>(stream)>>>(table, n_pos, rot, base, scaling,
                                                                                    factor, low, high, orig, gain);
  note_launch();
  return check_launch();
}

UP_DEFINE_REVISION(rope)
