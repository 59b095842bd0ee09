// kv4_attention.cuh — what the attention kernels over the paged 4-bit cache share: the arguments, the visible range of a
// query tile, and the matrix instructions.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "divide.cuh"
#include "kv4.cuh"

namespace up {
namespace kv4 {

struct Args {
  const void* q;
  void* out;
  float* lse;
  int bf16;                            // q and out: bf16, else f16
  int64_t qs, qh, os, oh, ls;          // strides in elements: token, head (lse: token)
  int64_t tokens;
  const uint8_t *k4, *v4;
  const __half *k_scale, *v_scale;
  uint32_t pages;                      // below 2^31: a negative page number is not below it
  int kv_heads, ratio, page_log2;      // ratio: query heads a key/value head
  int cpg, groups;                     // 32-dimension chunks a group; groups a row
  const int32_t* table;
  int64_t table_stride, table_width;
  const int32_t *lens, *cu;
  int batch, causal, window;
  Divide32 by_ratio;
  float scale_log2;                    // scale * log2(e): logits are kept in powers of two
  uint32_t* header;                    // workspace: its error word is header[3]
  uint32_t* counters;
  float* partials;
};

constexpr float kLn2 = 0.69314718055994531f;
constexpr float kNoMax = -3.0e38f;     // a running maximum before anything was seen: below every logit, yet finite

constexpr int64_t kMaxTokens = (int64_t)1 << 30;  // cached tokens a sequence, query rows a head, window, sequences: sums fit an int

struct Seq {
  int len, nq;
  int64_t q0;
};

__device__ __forceinline__ Seq load_seq(const Args& a, int b) {
  Seq s;
  s.len = (int)min(max((int64_t)__ldg(a.lens + b), (int64_t)0), a.table_width << a.page_log2);  // at most 2^30
  if (a.cu) {
    s.q0 = min(max((int64_t)__ldg(a.cu + b), (int64_t)0), a.tokens);
    const int64_t q1 = min(max((int64_t)__ldg(a.cu + b + 1), s.q0), a.tokens);
    s.nq = (int)(q1 - s.q0);  // at most 2^30 / ratio
  } else {
    s.q0 = b;
    s.nq = 1;
  }
  return s;
}

// The cached tokens [lo, hi) that the query tokens i0 .. i1 of a sequence can see between them.
__device__ __forceinline__ void visible(const Args& a, const Seq& s, int i0, int i1, int& lo, int& hi) {
  hi = a.causal ? min(max(s.len - s.nq + i1 + 1, 0), s.len) : s.len;
  lo = a.window > 0 ? max(s.len - s.nq + i0 + 1 - a.window, 0) : 0;
}

__device__ __forceinline__ uint32_t smem_addr(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

// 16 bytes global -> shared; zeros where `bytes` is 0 (the source is then not read).
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void ldmatrix_x4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// d += a b: 16 x 8 x 16, f16 operands, f32 sums.
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, "
      "%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// d = a b + {c0, c1, c0, c1}: the same start for both of a thread's rows.
__device__ __forceinline__ void mma_f16_from(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1, float c0, float c1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %10, "
      "%11};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1));
}

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// (v & mask) ^ flip
__device__ __forceinline__ uint32_t pick(uint32_t v, uint32_t mask, uint32_t flip) {
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0x6a;" : "=r"(d) : "r"(v), "r"(mask), "r"(flip));
  return d;
}

// The nibbles of a word as f16 pairs without a conversion: a nibble with its sign bit flipped is n + 8, and as an f16's
// low bits the subnormal (n + 8) 2^-24; the odd nibbles, four bits higher, are 16 times that. e[i] holds nibbles i and
// i + 4. The product's other side takes the 2^24, the 16 and the sum of the eights.
__device__ __forceinline__ void expand_raw(uint32_t w, uint32_t (&e)[4]) {
  const uint32_t x = w >> 8;
  e[0] = pick(w, 0x000f000fu, 0x00080008u);
  e[1] = pick(w, 0x00f000f0u, 0x00800080u);
  e[2] = pick(x, 0x000f000fu, 0x00080008u);
  e[3] = pick(x, 0x00f000f0u, 0x00800080u);
}

// The nibbles of a word as f16 pairs, exactly: e[i] holds nibbles i and i + 4 (signed). A nibble's two's complement bits
// with the sign bit flipped are n + 8; OR-ed into the mantissa of 1024 they give 1024 + (n + 8), and 16 steps higher
// 1024 + 16 (n + 8), so that the odd nibbles need no shift of their own.
__device__ __forceinline__ void expand(uint32_t w, uint32_t (&e)[4]) {
  const uint32_t x = w >> 8;
  const __half2 off = __half2half2(__ushort_as_half(0x6408));  // 1032
  const __half2 sixteenth = __half2half2(__ushort_as_half(0x2c00)), off16 = __half2half2(__ushort_as_half(0xd480));  // -72
  auto low = [&](uint32_t v) {
    uint32_t u = pick(v, 0x000f000fu, 0x64086408u);
    const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&u), off);
    return *reinterpret_cast<const uint32_t*>(&h);
  };
  auto high = [&](uint32_t v) {
    uint32_t u = pick(v, 0x00f000f0u, 0x64806480u);
    const __half2 h = __hfma2(*reinterpret_cast<const __half2*>(&u), sixteenth, off16);
    return *reinterpret_cast<const uint32_t*>(&h);
  };
  e[0] = low(w);
  e[1] = high(w);
  e[2] = low(x);
  e[3] = high(x);
}

// The 8 elements of 16 bytes in f32.
__device__ __forceinline__ void unpack8(uint4 u, int bf16, float (&f)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (bf16) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    } else {
      const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      f[2 * i] = v.x;
      f[2 * i + 1] = v.y;
    }
  }
}

__device__ __forceinline__ uint32_t pack2_f16(float lo, float hi) {
  uint32_t d;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi, int bf16) {
  if (!bf16) return pack2_f16(lo, hi);
  uint32_t d;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}

// ---- host side ----
constexpr int kSplitWarps = 4;
constexpr int kSplitThreads = 32 * kSplitWarps;
constexpr int kUnitTokens = 32 * kSplitWarps;  // cached tokens of one unit: 32 a warp
constexpr int kMaxCtas = 1024;                 // counters in the workspace
constexpr int kMaxRows = 16;                   // query rows of a tile at most
constexpr int kGroup = 16;                     // parts of a split tile that are added at once
constexpr size_t kHeaderBytes = 256, kCounterBytes = kHeaderBytes + 3 * kMaxCtas * sizeof(uint32_t);

// Query rows a tile has in the split kernel: 8 a column group, a second one where the head size leaves registers (not
// above 128) and the rows of a sequence and key/value head need it on average: the host knows the batch's rows, not each
// sequence's, and a sequence of fewer rows then computes an empty group. Measured with 64 sequences of 2048 tokens, all of the
// same rows, 8 key/value heads of 128: 8 rows 41 us in tiles of 8 and 53 of 16, 12 rows 68 and 55, 32 rows 123 and 97; one
// sequence of 2048, where little but the start counts: 8 rows 10.1 and 11.7, 32 rows 12.5 and 15.4.
inline int split_rows(int64_t rows_a_sequence, int64_t dim) {
  return rows_a_sequence > 8 && (dim == 64 || dim == 96 || dim == 128) ? 16 : 8;
}

// Whether the kernel for many query rows (head sizes 64 and 128; 256 rows a CTA, one CTA an SM) takes less time than the
// split one, given `rows` query rows for each of `pairs` (sequence, key/value head): the first in as many turns as its
// CTAs fill the SMs, the second in 16-row tiles that are spread evenly. Against as many cached tokens a 256-row tile takes
// an SM as long as four 16-row ones at head size 128 and six at 64. `rows` is the batch's mean and the measurements are of
// equal sequences; a batch of unequal ones goes to one kernel whole (a prompt of 2048 and 63 single tokens, 4096 cached
// tokens each, 32 heads over 8: 617 us, as two calls 152 and 67). From one sequence of 4096 tokens to 32 of 2048, 8 key/value
// heads, 32 to 1024 rows each, the faster one is taken but within 4 %: 12 sequences of 4096 at size 128, 96 rows 102 us split
// and 118 not, 128 rows 129 and 116; 4 of them, 256 rows 90 and 102, 384 rows 127 and 114; at size 64, 12 of them, 128 rows
// 84 and 108, 192 rows 119 and 106.
inline bool many_rows(int64_t rows, int64_t pairs, int64_t dim, int64_t sms) {
  if (dim != 64 && dim != 128) return false;
  const int64_t turns = (pairs * ((rows + 255) / 256) + sms - 1) / sms;
  return turns * sms * (dim == 64 ? 6 : 4) < pairs * ((rows + 15) / 16);
}
int prompt_attention(const Args& a, int dim, cudaStream_t s);

int split_attention(const Args& a, int dim, int tile_rows, int ctas, cudaStream_t s);  // by head size
int split_attention_small(const Args& a, int dim, int tile_rows, int ctas, cudaStream_t s);
int split_attention_128(const Args& a, int tile_rows, int ctas, cudaStream_t s);
int split_attention_large(const Args& a, int dim, int ctas, cudaStream_t s);

}  // namespace kv4
}  // namespace up
