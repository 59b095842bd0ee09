// kv4_append.cu — new tokens into the paged 4-bit cache: the position's rotation of queries and keys (rope.cuh), the
// quantisation of keys and values to int4 with an f16 scale a group, and the write to each token's slot, in one launch.
//
// A row is one head of one token; its dimensions fall into groups. With a the largest magnitude of a group (keys after
// their rotation, in f32),
//   scale = f16(min(a * f32(1/7), 65504)),   value = clamp(rint(x * (1 / scale)), -8, 7),   0 where scale is 0
// with every operation rounded to f32 by itself. A group that holds an infinity or a NaN gets a NaN scale and zero
// values: it reads back as NaN. The clamp is met only where f16 rounds a tiny scale down.
//
// What bounds it: HBM. q, k and v are read once, q is written once, and a cached row takes dim / 2 + 2 dim / group bytes.
// 16001 tokens of 64 and 8 heads of 128, f16: 112 us (612 MB: 5.5 TB/s, the slots' scattered rows in 64-byte pieces among
// them); one token 2.8 us, the launch's own time.
//
// Some blocks turn the queries as rope.cu does, the others take the rows of keys and values; they alternate over the grid,
// so that the queries' traffic fills the time in which the other rows wait for their slots, positions and scales. A row of
// keys or values is dim / 16 threads, and a block takes as many whole rows as fit into 256. A thread owns two 16-byte
// chunks (8 dimensions each) of its row, so that each rotated pair is in one thread: chunks j and rot / 16 + j of the half
// layout, two neighbours otherwise. A chunk's magnitude goes through shared memory: groups need not fall on a warp's lanes
// (dim 96 has 6 threads a row), and a group's maximum is then group / 32 16-byte reads.
// Four blocks an SM hide the rows' lookups best: 112 us for the 16001 tokens, with 64 registers a thread, against 128 for
// the three that 72 registers leave and 157 for five, which spill.
// Four rows a thread, loaded together, measured slower (231 us against 159 us for 16001 tokens of 64 and 8 heads, both with
// an earlier form of the queries' part): the registers that they take halve the queries' blocks on an SM.
// The operator's other sources, which its revision hash covers through this line (build.py --sources):
// FNV-1a 64 of divide.cuh, kv4.cuh, rope.cuh: 96ec8a3a8dd401a2
#include "kv4.cuh"
#include "rope.cuh"

namespace up {
namespace kv4 {

using namespace rp;

constexpr int kThreads = 256;

struct Append {
  int64_t tokens, q_heads, kv_heads, pages;
  int64_t qs, qh, ks, kh, vs, vh, qos, qoh;  // strides in elements: token, head
  const void* positions;
  int pos_dtype;
  const void* slots;
  int slot_dtype;
  const float* table;
  int64_t n_pos;
  int rot, half, page_log2, dim, group, groups;
  uint8_t *k4, *v4;
  __half *k_scale, *v_scale;
  Divide32 by_tpr, by_heads, by_per;  // threads a row, rows a token, chunks a group
};

// The 8 elements at dimension e of a row, in f32. VEC: 16-byte aligned.
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* row, int e, float (&f)[8]) {
  if constexpr (VEC) {
    Chunk<T>::unpack(*reinterpret_cast<const uint4*>(row + e), f);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = to_f32<T>(row[e + i]);
  }
}

// How the blocks that turn queries and those that take rows of keys and values alternate: `few` of the rarer kind, the
// last of each of the first `few` runs of `period` blocks.
struct Mix {
  uint32_t few, period;
  int few_are_queries;
};

// The rotated 8 elements at dimension e, whatever the pairs' other elements' place: each pair is computed from the row.
template <typename T>
__device__ __forceinline__ void rotate_any(const T* row, int e, const float* t, bool in, const Append& a,
                                           float (&f)[8]) {
  const float nan = __int_as_float(0x7fffffff);
  const int r2 = a.rot / 2;
  for (int i = 0; i < 8; ++i) {
    const int d = e + i;
    if (d >= a.rot) continue;
    const int pair = a.half ? (d < r2 ? d : d - r2) : d / 2;
    const bool second = a.half ? d >= r2 : (d & 1);
    const int other = a.half ? (second ? d - r2 : d + r2) : (d ^ 1);
    float x0 = second ? to_f32<T>(row[other]) : f[i], x1 = second ? f[i] : to_f32<T>(row[other]);
    rotate(x0, x1, in ? __ldg(t + pair) : nan, in ? __ldg(t + r2 + pair) : nan);
    f[i] = second ? x1 : x0;
  }
}

__device__ __forceinline__ uint32_t magnitude8(const float (&f)[8]) {  // as bits: a NaN is above every number
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(f[i]) & 0x7fffffffu);
  return m;
}

// VEC: blocks of queries (items of rope_item, HEADS heads each) and of rows. Else (rows or rotations that are not whole
// 16-byte chunks) every block takes rows, and the queries are rows like the others.
template <typename T, bool VEC, int HEADS>
__global__ void __launch_bounds__(kThreads, 4) kv4_append_kernel(const T* q, const T* __restrict__ k,
                                                              const T* __restrict__ v, T* q_out, const Append a,
                                                              const Geometry g, const Mix mix,
                                                              const Items<Divide32> n) {
  uint32_t block = blockIdx.x;
  if (VEC) {
    const uint32_t run = block / mix.period;  // runs before this block
    const bool rare = run < mix.few && block - run * mix.period == mix.period - 1;
    block = rare ? run : block - min(run, mix.few);
    if (rare == (mix.few_are_queries != 0)) {
      const uint32_t item = block * kThreads + threadIdx.x;
      if (item < n.count) {
        if (a.half) rope_item<T, true, HEADS, Divide32>(q, q_out, a.table, g, item, n, 0);
        else rope_item<T, false, HEADS, Divide32>(q, q_out, a.table, g, item, n, 0);
      }
      return;
    }
  }
  // the chunks' magnitudes of this block's rows: two chunks a thread
  __shared__ alignas(16) uint32_t mag[2 * kThreads];
  const int tpr = a.dim / 16, rows_per_block = kThreads / tpr;
  const int r = (int)a.by_tpr(threadIdx.x), u = (int)threadIdx.x - r * tpr;
  const uint32_t q_heads = VEC ? 0u : (uint32_t)a.q_heads, kv_heads = (uint32_t)a.kv_heads;
  const uint32_t heads = q_heads + 2 * kv_heads;  // the launch keeps tokens * heads below 2^31
  const uint32_t row = block * (uint32_t)rows_per_block + r;
  const uint32_t tok = a.by_heads(row), head = row - tok * heads;
  const bool live = r < rows_per_block && tok < a.tokens;
  const bool is_q = !VEC && head < q_heads, is_v = head >= q_heads + kv_heads;
  const int pairs = VEC && a.half ? a.rot / 16 : 0;  // half-layout pairs of chunks come first
  const int c0 = u < pairs ? u : 2 * u, c1 = u < pairs ? u + pairs : 2 * u + 1;
  float x[2][8];
  int64_t slot = -1;
  const int64_t h = is_q ? head : is_v ? head - q_heads - kv_heads : head - q_heads;
  if (live) {
    const T* src = is_q ? q + tok * a.qs + h * a.qh : is_v ? v + tok * a.vs + h * a.vh : k + tok * a.ks + h * a.kh;
    load8<T, VEC>(src, 8 * c0, x[0]);
    load8<T, VEC>(src, 8 * c1, x[1]);
    if (!is_q) {
      slot = load_id(a.slots, a.slot_dtype, tok);
      if (slot >= (a.pages << a.page_log2)) slot = -1;  // left out, like a negative one
    }
    if (!is_v && a.rot > 0) {
      const int64_t p = load_id(a.positions, a.pos_dtype, tok);
      const bool in = p >= 0 && p < a.n_pos;
      const float* t = a.table + (in ? p : 0) * a.rot;
      const float nan = __int_as_float(0x7fffffff);
      if constexpr (!VEC) {
        rotate_any(src, 8 * c0, t, in, a, x[0]);
        rotate_any(src, 8 * c1, t, in, a, x[1]);
      } else if (a.half) {
        if (u < pairs) {
          float c[8], s[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) c[i] = s[i] = nan;
          if (in) {
            load_row<8>(t + 8 * u, c);
            load_row<8>(t + a.rot / 2 + 8 * u, s);
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) rotate(x[0][i], x[1][i], c[i], s[i]);
        }
      } else {
#pragma unroll
        for (int z = 0; z < 2; ++z) {
          const int e = 8 * (z ? c1 : c0);
          if (e >= a.rot) continue;
          float c[4], s[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) c[i] = s[i] = nan;
          if (in) {
            load_row<4>(t + e / 2, c);
            load_row<4>(t + a.rot / 2 + e / 2, s);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) rotate(x[z][2 * i], x[z][2 * i + 1], c[i], s[i]);
        }
      }
    }
    if (!is_q) {
      mag[r * 2 * tpr + c0] = magnitude8(x[0]);
      mag[r * 2 * tpr + c1] = magnitude8(x[1]);
    }
  }
  __syncthreads();
  if (!live || (!is_q && slot < 0)) return;
  if (is_q) {
    T* o = q_out + tok * a.qos + h * a.qoh;
#pragma unroll
    for (int z = 0; z < 2; ++z)
#pragma unroll
      for (int i = 0; i < 8; ++i) o[8 * (z ? c1 : c0) + i] = from_f32<T>(x[z][i]);
    return;
  }
  // the row's place in the cache
  const int64_t page = slot >> a.page_log2, at = slot & (((int64_t)1 << a.page_log2) - 1);
  const int64_t line = (((page * a.kv_heads + h) << a.page_log2) + at);
  const int groups = a.groups, per = a.group / 8;  // chunks a group
  uint32_t* words = reinterpret_cast<uint32_t*>((is_v ? a.v4 : a.k4) + line * (a.dim / 2));
  __half* scales = (is_v ? a.v_scale : a.k_scale) + line * groups;
  __half sc = __half(0);
  float sf = 0.f, inv = 0.f;
  int last = -1;
#pragma unroll
  for (int z = 0; z < 2; ++z) {
    const int c = z ? c1 : c0, grp = (int)a.by_per((uint32_t)c);
    if (grp != last) {
      const uint4* m4 = reinterpret_cast<const uint4*>(mag + r * 2 * tpr + grp * per);
      uint32_t m = 0;
      for (int i = 0; i < per / 4; ++i) {
        const uint4 w = m4[i];
        m = max(max(m, max(w.x, w.y)), max(w.z, w.w));
      }
      sc = m >= 0x7f800000u ? __ushort_as_half(0x7fff)
                            : __float2half_rn(fminf(__fmul_rn(__uint_as_float(m), 1.0f / 7.0f), 65504.0f));
      sf = __half2float(sc);
      inv = sf > 0.0f ? __fdiv_rn(1.0f, sf) : 0.0f;
      last = grp;
    }
    uint32_t w = 0;
    if (sf > 0.0f)
#pragma unroll
      for (int i = 0; i < 8; ++i)
        w |= ((uint32_t)(int)fminf(fmaxf(rintf(__fmul_rn(x[z][i], inv)), -8.0f), 7.0f) & 15u) << (4 * i);
    words[c] = w;
    if (c == grp * per) scales[grp] = sc;
  }
}

template <typename T>
int launch_append(const void* q, const void* k, const void* v, void* q_out, Append a, const Geometry& g,
                  cudaStream_t s) {
  const bool strides = (a.ks | a.kh | a.vs | a.vh) % 8 == 0;
  const bool vec = strides && aligned(k, 16) && aligned(v, 16) && a.rot % (a.half ? 16 : 8) == 0 && aligned(a.table, 16) &&
                   (a.q_heads == 0 || rope_vector<T>(q, q_out, a.table, g, a.half));
  const int64_t limit = 0x7fffffff - kThreads;  // rows, items and blocks are counted in 32 bits
  const int64_t heads = (vec ? 0 : a.q_heads) + 2 * a.kv_heads;
  const int per = rope_heads<T>(g, a.tokens, a.half);
  const int64_t units = rope_units<T>(g, a.half), groups = (a.q_heads + per - 1) / per;
  if (heads > limit || a.tokens > limit / heads) return UP_ERR_UNSUPPORTED;
  if (a.q_heads > limit / units || a.tokens > limit / (a.q_heads > 0 ? a.q_heads * units : 1)) return UP_ERR_UNSUPPORTED;
  a.by_heads = Divide32(heads);
  const int rows_per_block = kThreads / (a.dim / 16);
  const int64_t rows = a.tokens * heads, row_blocks = (rows + rows_per_block - 1) / rows_per_block;
  const int64_t q_items = vec ? a.tokens * groups * units : 0, q_blocks = (q_items + kThreads - 1) / kThreads;
  if (row_blocks + q_blocks > limit) return UP_ERR_UNSUPPORTED;
  Mix mix;
  mix.few_are_queries = q_blocks < row_blocks;
  mix.few = (uint32_t)(mix.few_are_queries ? q_blocks : row_blocks);
  mix.period = (uint32_t)(mix.few > 0 ? (q_blocks + row_blocks) / mix.few : 1);
  const Items<Divide32> n{Divide32(units), Divide32(groups > 0 ? groups : 1), Divide32(a.tokens), (uint32_t)q_items};
  const auto kernel = !vec       ? kv4_append_kernel<T, false, 1>
                      : per == 4 ? kv4_append_kernel<T, true, 4>
                      : per == 2 ? kv4_append_kernel<T, true, 2>
                                 : kv4_append_kernel<T, true, 1>;
  kernel<<<(unsigned)(row_blocks + q_blocks), kThreads, 0, s>>>(
      static_cast<const T*>(q), static_cast<const T*>(k), static_cast<const T*>(v), static_cast<T*>(q_out), a, g, mix, n);
  note_launch();
  return check_launch();
}

}  // namespace kv4
}  // namespace up

using namespace up;
using namespace up::kv4;

extern "C" int up_sm100_kv4_append(const void* q, const void* k, const void* v, int dtype, int64_t tokens,
                                   int64_t q_heads, int64_t q_stride_t, int64_t q_stride_h, int64_t k_stride_t,
                                   int64_t k_stride_h, int64_t v_stride_t, int64_t v_stride_h, const void* positions,
                                   int pos_dtype, const float* table, int64_t n_pos, int64_t rot, int layout,
                                   const void* slots, int slot_dtype, const up_kv4_cache* cache, void* q_out,
                                   int64_t q_out_stride_t, int64_t q_out_stride_h, void* stream) {
  const int ok = check_cache(cache);
  if (ok != UP_OK) return ok;
  UP_CHECK_ARG(tokens >= 0 && q_heads >= 0 && n_pos >= 0);
  UP_CHECK_ARG(rot >= 0 && rot <= cache->dim && rot % 2 == 0);
  UP_CHECK_ARG(q_stride_t >= 0 && q_stride_h >= 0 && k_stride_t >= 0 && k_stride_h >= 0 && v_stride_t >= 0 &&
               v_stride_h >= 0);
  if (layout != UP_ROPE_HALF && layout != UP_ROPE_INTERLEAVED) return UP_ERR_UNSUPPORTED;
  if (dtype != UP_EK_BF16 && dtype != UP_EK_F16) return UP_ERR_UNSUPPORTED;
  if (slot_dtype != UP_EK_I32 && slot_dtype != UP_EK_I64) return UP_ERR_UNSUPPORTED;
  if (rot > 0 && pos_dtype != UP_EK_I32 && pos_dtype != UP_EK_I64) return UP_ERR_UNSUPPORTED;
  if (tokens == 0) return UP_OK;
  UP_CHECK_ARG(k != nullptr && v != nullptr && slots != nullptr);
  UP_CHECK_ARG(q_heads == 0 || (q != nullptr && q_out != nullptr));
  UP_CHECK_ARG(q_heads <= 1 || q_out_stride_h >= cache->dim);
  UP_CHECK_ARG(q_heads == 0 || tokens <= 1 || q_out_stride_t >= cache->dim);
  UP_CHECK_ARG(rot == 0 || (positions != nullptr && table != nullptr));
  // the stride of an extent of one is never used
  if (tokens == 1) q_stride_t = k_stride_t = v_stride_t = q_out_stride_t = 0;
  if (q_heads <= 1) q_stride_h = q_out_stride_h = 0;
  if (cache->kv_heads == 1) k_stride_h = v_stride_h = 0;
  Append a{};
  a.tokens = tokens, a.q_heads = q_heads, a.kv_heads = cache->kv_heads, a.pages = cache->pages;
  a.qs = q_stride_t, a.qh = q_stride_h, a.ks = k_stride_t, a.kh = k_stride_h, a.vs = v_stride_t, a.vh = v_stride_h;
  a.qos = q_out_stride_t, a.qoh = q_out_stride_h;
  a.positions = positions, a.pos_dtype = pos_dtype, a.slots = slots, a.slot_dtype = slot_dtype;
  a.table = table, a.n_pos = n_pos, a.rot = (int)rot, a.half = layout == UP_ROPE_HALF;
  a.page_log2 = log2_of(cache->page), a.dim = (int)cache->dim, a.group = (int)cache->group;
  a.groups = (int)(cache->dim / cache->group), a.by_tpr = Divide32(cache->dim / 16), a.by_per = Divide32(cache->group / 8);
  a.k4 = static_cast<uint8_t*>(cache->k), a.v4 = static_cast<uint8_t*>(cache->v);
  a.k_scale = static_cast<__half*>(cache->k_scale), a.v_scale = static_cast<__half*>(cache->v_scale);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const Geometry g{tokens, q_heads, cache->dim, rot, 0, q_stride_t, q_stride_h, 0, q_out_stride_t, q_out_stride_h,
                   positions, pos_dtype, 0, n_pos};
  return dtype == UP_EK_BF16 ? launch_append<__nv_bfloat16>(q, k, v, q_out, a, g, s)
                             : launch_append<__half>(q, k, v, q_out, a, g, s);
}

UP_DEFINE_REVISION(kv4_append)
