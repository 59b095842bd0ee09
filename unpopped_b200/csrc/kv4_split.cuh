// kv4_split.cuh — attention over the paged 4-bit cache for few query rows a key/value head (decode): the cache is read
// once, 4 bits a value, straight into matrix instructions.
//
//   s[j] = scale * sum_g k_scale[j][g] * sum_{d in g} q[d] n_k[j][d],   out[d] = sum_j p[j] v_scale[j][g(d)] n_v[j][d] / l
// with n the stored nibbles: a group's scale multiplies sums and probabilities, never single elements, so nibbles go into
// the products as exact f16 integers.
//
// Layout. A tile is 8 NT query rows (rows: query token x head of the group) of one sequence and key/value head. Both
// products run transposed, cached tokens or dimensions as the 16 rows and query rows as the 8 columns of mma m16n8k16,
// so one query head wastes no more than the 8 columns:
//  * K: ldmatrix gives lane (g, t) the word t (8 dimensions) of token g's 16-byte chunk. Its nibble pairs (0,4), (1,5),
//    (2,6), (3,7) are the A fragments of two k-steps; q's B fragments are laid out in the same order once a tile. The
//    fragments are the masked bits themselves, f16 subnormals (n + 8) 2^-24 and, for odd nibbles, 16 times that: q is
//    divided by 16 there, and the sums begin at -8 sum q.
//  * V: ldmatrix.trans moves 16-bit units, four nibbles: lane (g, t) gets dimensions 4g .. 4g + 3 of tokens 2t and 2t + 1
//    in the two halves of a word, which is the A fragment of V transposed after the same conversion.
//  * Probabilities: the score fragment times v_scale, rounded to f16, transposed by movmatrix, is the B fragment.
// q is scaled by a power of two a row to fit f16 (exactly, where it is within 2^-24 of the row's largest); the
// probabilities by a power of two a warp and row, the largest exponent of the v_scale that the row has seen, less 5, so that
// p * v_scale ends at 2^15 and f16 has 2^-30 of range below a weight of one, whatever the tokens hold that the row does not
// see. p * v_scale is rounded to f16; every sum is f32.
// The running maximum moves only when a lane's probabilities of a step sum to more than 2^9 (which the 2^15 above holds), so
// most steps need one vote, no reduction across lanes and no rescaling.
//
// Work. Units of 128 cached tokens, over sequences, tiles and heads in order, are split evenly over the launch's CTAs
// (each sequence's count comes from its length on the device: no host read, no launch bound by the longest sequence).
// CTAs do not run at one rate (of a launch that the memory bounds, the slowest take a fifth longer than the mean); drawing
// the last eighth of the units in items as CTAs finish cost more, by the items' starts, than it gained (attend over 32
// contexts of 8k to 16k tokens: 100.7 us with it, 95.7 us without).
// A warp takes 32 tokens of each unit through its own ring of cp.async stages, so no barrier stands in the loop. A tile
// that ends inside one CTA is written at once; parts of a split tile go to the workspace in f32 and the CTA that
// finishes last adds them in order. No CTA waits for another.
//
// What bounds it: HBM where contexts are long; while the loop runs it reads 6.0 to 6.4 TB/s, with about 560 instructions a
// warp and 32 tokens of size 128 (the schedulers issue in 60 % of their cycles). 64 query over 8 key/value heads of 128,
// bf16: 32 contexts of 8000 to 16384 tokens 89 us (412 MB: 4.6 TB/s), one of 131071 tokens 42 us (143 MB: 3.4 TB/s), one of
// 777 tokens 9.2 us. What is beside the loop, and all that short contexts cost: lengths, then pages, then the first data
// (3 to 5 us), the parts' merge (2 to 5 us), and CTAs that share an SM with slower ones.
#pragma once

#include "kv4_attention.cuh"

namespace up {
namespace kv4 {

template <int D, int NT>
struct SplitCfg {
  static constexpr int kChunks = D / 32;
  // Two stages: a third made the ring's share of the SM's memory leave 7 KB of L1 (94.3 against 91.7 us for 32 contexts of
  // 8k to 16k tokens), and a fifth CTA in place of it spilled registers (97.2 us).
  static constexpr int kStages = 2;
  static constexpr int kRows = 8 * NT;
  // a stage of one warp: 32 tokens of K and V (D / 2 bytes each) and of their scales (at most D / 32 f16 each)
  static constexpr int kKV = 16 * D, kSc = 2 * D, kStage = 2 * kKV + 2 * kSc;
  static constexpr int kPitch = D + 4;  // floats between the rows of the merge buffer: conflict-free 16-byte stores
  static constexpr int kRing = kSplitWarps * kStages * kStage;
  static constexpr int kMerge = kSplitWarps * kRows * kPitch * 4;
  static constexpr int kSmem = kRing > kMerge ? kRing : kMerge;
  static_assert(kStages == 2, "the tokens that exist are kept for the step at hand and the next");
  static constexpr int kOcc = D <= 128 ? (NT == 1 ? 4 : 3) : 2;
};

// Chunk c of token row r is stored at chunk c ^ swizzle(r): 8 rows of one chunk then fall on 8 different bank groups.
template <int D>
__device__ __forceinline__ int swizzle(int r) {
  constexpr int n = D / 32, z = n % 8 == 0 ? 8 : n % 4 == 0 ? 4 : n % 2 == 0 ? 2 : 1;
  return (r / (8 / z)) & (z - 1);
}

// A column's threshold and the exponent of v_scale that it stands for. p * v_scale is 2^kLift to 2^(kLift + 1) where a logit
// is at the running maximum and the v_scale the largest.
constexpr int kLift = 5;
__device__ __forceinline__ float exp_to_lim(int vexp) { return __uint_as_float((uint32_t)(136 + kLift - vexp) << 23); }
__device__ __forceinline__ int lim_to_exp(float lim) { return 136 + kLift - (int)(__float_as_uint(lim) >> 23); }

// a / b for a >= 0, b > 0, in 32 bits where both fit (a 64-bit division is a long sequence).
__device__ __forceinline__ int64_t divide(int64_t a, int64_t b) {
  return ((a | b) >> 32) == 0 ? (int64_t)((uint32_t)a / (uint32_t)b) : a / b;
}

// U units in order over P CTAs: the first `extra` take `each` + 1, the others `each`.
struct Shares {
  int64_t P, each, extra;
  __device__ __forceinline__ Shares(int64_t U, int64_t grid) {
    P = min(grid, U);
    each = P > 0 ? divide(U, P) : 0;
    extra = U - each * P;
  }
  __device__ __forceinline__ int64_t begin(int64_t cta) const { return cta * each + min(cta, extra); }
  __device__ __forceinline__ int64_t cta_of(int64_t u) const {
    const int64_t in_first = extra * (each + 1);
    return u < in_first ? divide(u, each + 1) : extra + divide(u - in_first, each);
  }
};

// What starting a tile costs, in units: its loads wait for one another (length, pages, cache) and its parts are added. The
// CTAs' shares count it, or CTAs that get many short sequences finish last: 64 sequences of 0 to 4096 tokens
// took 52.2 us without it and 45.8 with, 24 sequences of a few queries 42.2 and 28.4.
constexpr int kTileCost = 2;

// Units of one (tile, head) of a sequence: at least one, which writes the rows that see nothing.
template <int ROWS>
__device__ __forceinline__ int tile_units(const Args& a, const Seq& s, int tile, int& unit0) {
  const int rows = s.nq * a.ratio, i0 = (int)a.by_ratio(tile * ROWS), i1 = (int)a.by_ratio(min((tile + 1) * ROWS, rows) - 1);
  int lo, hi;
  visible(a, s, i0, i1, lo, hi);
  unit0 = lo / kUnitTokens;
  return max(1, (hi + kUnitTokens - 1) / kUnitTokens - unit0);
}

// The units of each lane's sequence b (0 where there is none), for a whole warp: a sequence of many tiles is counted by all
// lanes. Counted by one lane, and searched by each thread for itself, the 154 tiles of 818 queries took half of the time
// (head size 96, 911 cached tokens: 50 us where it is 33).
template <int ROWS>
__device__ __forceinline__ int64_t seq_units(const Args& a, int b, bool any) {
  Seq s{0, 0, 0};
  if (any) s = load_seq(a, b);
  const int lane = threadIdx.x & 31, tiles = (s.nq * a.ratio + ROWS - 1) / ROWS;
  int64_t n = 0;
  int unit0;
  if (tiles <= 4)
    for (int i = 0; i < tiles; ++i) n += kTileCost + tile_units<ROWS>(a, s, i, unit0);
  for (uint32_t many = __ballot_sync(0xffffffffu, tiles > 4); many; many &= many - 1) {
    const int src = __ffs(many) - 1, of = __shfl_sync(0xffffffffu, tiles, src);
    const Seq w{__shfl_sync(0xffffffffu, s.len, src), __shfl_sync(0xffffffffu, s.nq, src), 0};
    int64_t sum = 0;
    for (int i = lane; i < of; i += 32) sum += kTileCost + tile_units<ROWS>(a, w, i, unit0);
#pragma unroll 1
    for (int d = 1; d < 32; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    if (lane == src) n = sum;
  }
  return n * a.kv_heads;
}

// D: head size. CPG: 32-dimension chunks a group. EXACT: CPG is the cache's; else it is 1 and groups hold a.cpg chunks.
template <int D, int CPG, int NT, bool EXACT>
__global__ void __launch_bounds__(kSplitThreads, SplitCfg<D, NT>::kOcc) kv4_split_kernel(const Args a) {
  using C = SplitCfg<D, NT>;
  constexpr int ROWS = C::kRows, CH = C::kChunks, GT = CH / CPG;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ int64_t s_scan[kSplitWarps + 1], s_base;
  __shared__ int s_seq, s_last;
  __shared__ float s_ref[kSplitWarps][ROWS], s_sum[kSplitWarps][ROWS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;

  // ---- this CTA's share [u, u1) of the units, and the sequence it begins in ----
  const int per = (a.batch + kSplitThreads - 1) / kSplitThreads;
  const int my0 = min((int)threadIdx.x * per, a.batch), my1 = min(my0 + per, a.batch);
  int64_t mine = 0;
  for (int k = 0; k < per; ++k) mine += seq_units<ROWS>(a, my0 + k, my0 + k < my1);
  int64_t incl = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int64_t v = __shfl_up_sync(0xffffffffu, incl, d);
    if (lane >= d) incl += v;
  }
  if (lane == 31) s_scan[warp] = incl;
  __syncthreads();
  int64_t before = incl - mine, U = 0;
  for (int w = 0; w < kSplitWarps; ++w) {
    if (w < warp) before += s_scan[w];
    U += s_scan[w];
  }
  const Shares shares(U, gridDim.x);
  const int64_t cta = blockIdx.x;
  if (cta >= shares.P) return;
  // the sequence in which this CTA's share [u, u1) begins: the thread that counted it says so
  int64_t u = shares.begin(cta);
  const int64_t u1 = shares.begin(cta + 1);
  const bool here = u >= before && u < before + mine;
  if (__any_sync(0xffffffffu, here)) {
    int64_t base = before;
    int b = my0;
    for (int k = 0; k + 1 < per; ++k) {  // which of this thread's: the last one needs no count
      const int64_t n = seq_units<ROWS>(a, my0 + k, my0 + k < my1);
      if (b == my0 + k && u >= base + n) base += n, ++b;
    }
    if (here) s_seq = b, s_base = base;
  }
  __syncthreads();
  int b = s_seq, tile = 0;
  int64_t off = u - s_base;

  const uint32_t smem_base = smem_addr(smem), ring = smem_base + warp * (C::kStages * C::kStage);
  float* merge = reinterpret_cast<float*>(smem);
  // the scale runs of 8 tokens are 16 * groups bytes: `groups` 16-byte pieces
  const int groups = EXACT ? GT : a.groups;
  // a lane copies a piece of K's scales (the first 4 * groups lanes) or of V's; one of each where that is more than 32 lanes
  // or no power of two
  const bool sc_both = 8 * groups > 32 || (groups & (groups - 1)) != 0, sc_v = !sc_both && lane >= 4 * groups;
  const int sc_at = sc_both ? lane : lane & (4 * groups - 1);
  const bool sc_mine = sc_at < 4 * groups && (sc_both || lane < 8 * groups);
  const int sc_run = sc_mine ? sc_at / groups * 8 : 0, sc_part = sc_at % groups;
  // where piece lane + 32 i of a step's K (or V) lies in its stage
  auto copy_at = [&](int i) -> uint32_t {
    if constexpr (32 % CH == 0 && 32 / CH >= 8) {  // the swizzle repeats: one offset a lane, the rest are constants
      return ((lane / CH) * CH + ((lane % CH) ^ swizzle<D>(lane / CH))) * 16 + i * 512;
    } else {
      const int r = (lane + 32 * i) / CH, c = (lane + 32 * i) % CH;
      return (r * CH + (c ^ swizzle<D>(r))) * 16;
    }
  };
  // where row `lane` of chunk c lies
  auto chunk_at = [&](int c) -> uint32_t { return (lane * CH + (c ^ swizzle<D>(lane))) * 16; };

  while (u < u1) {
    const Seq seq = load_seq(a, b);
    const int rows = seq.nq * a.ratio, tiles = (rows + ROWS - 1) / ROWS;
    int unit0 = 0, n_units = 0;
    // off counts from this tile's first head: the tile that it falls into
    if (tile < tiles) {
      n_units = tile_units<ROWS>(a, seq, tile, unit0);
      const int64_t size = (int64_t)(n_units + kTileCost) * a.kv_heads;
      if (off >= size) {
        off -= size;
        ++tile;
        while (tile < tiles) {  // 32 tiles at a time
          int my_first = 0, my_units = -kTileCost;
          if (tile + lane < tiles) my_units = tile_units<ROWS>(a, seq, tile + lane, my_first);
          int end = my_units + kTileCost;  // of one head: 32 tiles of at most 2^23 units
#pragma unroll 1  // unrolled, the registers of the main loop suffer (91.2 against 89.1 us for the 32 long contexts)
          for (int d = 1; d < 32; d <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, end, d);
            if (lane >= d) end += v;
          }
          const uint32_t past = __ballot_sync(0xffffffffu, off < (int64_t)end * a.kv_heads);
          if (past) {
            const int at = __ffs(past) - 1;
            n_units = __shfl_sync(0xffffffffu, my_units, at);
            off -= (int64_t)(__shfl_sync(0xffffffffu, end, at) - n_units - kTileCost) * a.kv_heads;
            unit0 = __shfl_sync(0xffffffffu, my_first, at);
            tile += at;
            break;
          }
          off -= (int64_t)__shfl_sync(0xffffffffu, end, 31) * a.kv_heads;
          tile = min(tile + 32, tiles);
        }
      }
    }
    if (tile >= tiles) {  // past this sequence's last unit
      ++b;
      tile = 0;
      off = 0;
      continue;
    }
    // a tile's share is its cost and then its units: this CTA has [at, at + take) of it, the units [first, first + count)
    const int head = (int)divide(off, n_units + kTileCost), at = (int)(off - (int64_t)head * (n_units + kTileCost));
    const int take = (int)min((int64_t)(n_units + kTileCost - at), u1 - u);
    const int first = max(at - kTileCost, 0), count = max(at + take - kTileCost, 0) - first;
    const int64_t tile_u0 = u - at + kTileCost;  // the share of the first unit
    u += take;
    off += take;
    if (count == 0) continue;
    const int tok0 = (unit0 + first) * kUnitTokens + warp * 32;
    const int32_t* pages = a.table + (int64_t)b * a.table_stride;
    // the page of this lane's token of step k, -1 where it has none
    auto page_of = [&](int k) {
      const int j = tok0 + k * kUnitTokens + lane;
      if (k >= count || j >= seq.len) return -1;
      const int p = __ldg(pages + (j >> a.page_log2));
      return (uint32_t)p < a.pages ? p : -1;
    };
    int page0[C::kStages];
#pragma unroll
    for (int k = 0; k < C::kStages; ++k) page0[k] = page_of(k);
    // ---- the tile's queries (loads), and the first copies ----
    uint4 raw[NT][CH];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int row = tile * ROWS + nt * 8 + g, i = (int)a.by_ratio(row);
      const char* src = static_cast<const char*>(a.q) + 2 * ((seq.q0 + i) * a.qs + (int64_t)(head * a.ratio + row - i * a.ratio) * a.qh);
#pragma unroll
      for (int c = 0; c < CH; ++c)
        raw[nt][c] = row < rows ? __ldg(reinterpret_cast<const uint4*>(src + 2 * (32 * c + 8 * t))) : make_uint4(0, 0, 0, 0);
    }
    // A run is 8 tokens, which lie on one page. Rows past the sequence's end come with their run; they are masked. Offsets
    // count 16-byte pieces: a page of one head is page * CH of them (page * groups / 8 of scales).
    const uint32_t page_kv = (uint32_t)a.kv_heads << a.page_log2, head_kv = (uint32_t)head << a.page_log2;
    const uint32_t in_page = (1u << a.page_log2) - 1;
    const uint4* k_base = reinterpret_cast<const uint4*>(a.k4) + (uint64_t)head_kv * CH;
    const uint4* v_base = reinterpret_cast<const uint4*>(a.v4) + (uint64_t)head_kv * CH;
    const uint4* ks_base = reinterpret_cast<const uint4*>(sc_v ? a.v_scale : a.k_scale) + ((uint64_t)head_kv * groups >> 3);
    const uint4* vs_base = reinterpret_cast<const uint4*>(a.v_scale) + ((uint64_t)head_kv * groups >> 3);
    const uint32_t sc_dst = 2 * C::kKV + (sc_v ? C::kSc : 0) + sc_at * 16;
    uint32_t have = 0, have_next = 0;  // the tokens of the step at hand, and of the last one copied, that exist
    // Copies step k into the stage at `st`.
    auto issue = [&](int k, int page, uint32_t st) {
      if (k < count) {
        const uint32_t tok = (uint32_t)(tok0 + k * kUnitTokens) & in_page;
        have_next = __ballot_sync(0xffffffffu, page >= 0);
        if (a.page_log2 >= 5) {  // one page holds the step's 32 tokens
          const int pg = __shfl_sync(0xffffffffu, page, 0);
          const uint32_t bytes = pg >= 0 ? 16u : 0u;
          const uint64_t at = (uint64_t)(uint32_t)max(pg, 0) * (page_kv * CH) + (tok * CH + lane);
          const uint4 *k_at = k_base + at, *v_at = v_base + at;
#pragma unroll
          for (int i = 0; i < CH; ++i) {
            const uint32_t dst = st + copy_at(i);
            cp_async16(dst, k_at + 32 * i, bytes);
            cp_async16(dst + C::kKV, v_at + 32 * i, bytes);
          }
          if (sc_mine) {
            const uint64_t sc = (uint64_t)(uint32_t)max(pg, 0) * ((page_kv >> 3) * groups) + ((tok >> 3) * groups + sc_at);
            cp_async16(st + sc_dst, ks_base + sc, bytes);
            if (sc_both) cp_async16(st + sc_dst + C::kSc, vs_base + sc, bytes);
          }
        } else {
#pragma unroll
          for (int i = 0; i < CH; ++i) {
            const int r = (lane + 32 * i) / CH, run = r & ~7;
            const int pg = __shfl_sync(0xffffffffu, page, run);
            const uint32_t bytes = pg >= 0 ? 16u : 0u;
            const uint64_t at = (uint64_t)(uint32_t)max(pg, 0) * (page_kv * CH) +
                                (((tok + run) & in_page) * CH + (lane + 32 * i - run * CH));
            const uint32_t dst = st + copy_at(i);
            cp_async16(dst, k_base + at, bytes);
            cp_async16(dst + C::kKV, v_base + at, bytes);
          }
          const int pg = __shfl_sync(0xffffffffu, page, sc_run);
          if (sc_mine) {
            const uint32_t bytes = pg >= 0 ? 16u : 0u;
            const uint64_t at = (uint64_t)(uint32_t)max(pg, 0) * ((page_kv >> 3) * groups) +
                                ((((tok + sc_run) & in_page) >> 3) * groups + sc_part);
            cp_async16(st + sc_dst, ks_base + at, bytes);
            if (sc_both) cp_async16(st + sc_dst + C::kSc, vs_base + at, bytes);
          }
        }
      }
      cp_async_commit();
    };

#pragma unroll
    for (int k = 0; k < C::kStages - 1; ++k) issue(k, page0[k], ring + k * C::kStage);
    int page = page0[C::kStages - 1];

    // ---- B fragments of the queries, and per column (query row) its logit factor and visible range ----
    uint32_t qf[NT][CH][4];
    float qs[NT][2], zero[NT][GT][2];  // zero: where a group's sum begins, -8 sum q
    int last[NT][2], past[NT][2];      // a column sees the tokens past < j <= last
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float big = 0.f;
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        float f[8];
        unpack8(raw[nt][c], a.bf16, f);
#pragma unroll
        for (int k = 0; k < 8; ++k) big = fmaxf(big, fabsf(f[k]));
      }
      big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
      big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
      const int ex = (int)(__float_as_uint(big) >> 23) - 127;  // the row's largest magnitude becomes 2^14 .. 2^15
      const int sh = big == 0.f || ex == 128 ? 0 : min(14 - ex, 126);
      const float up = __uint_as_float((uint32_t)(sh + 127) << 23);
#pragma unroll
      for (int z = 0; z < GT; ++z) {
        float total = 0.f;
#pragma unroll
        for (int cc = 0; cc < CPG; ++cc) {
          const int c = z * CPG + cc;
          float f[8];
          unpack8(raw[nt][c], a.bf16, f);
#pragma unroll
          for (int k = 0; k < 8; ++k) total += f[k] *= up;
#pragma unroll
          for (int k = 0; k < 4; ++k)
            qf[nt][c][k] = (k & 1) ? pack2_f16(f[k] * 0.0625f, f[k + 4] * 0.0625f) : pack2_f16(f[k], f[k + 4]);
        }
        total += __shfl_xor_sync(0xffffffffu, total, 1);
        total += __shfl_xor_sync(0xffffffffu, total, 2);
#pragma unroll
        for (int j = 0; j < 2; ++j)
          zero[nt][z][j] = __shfl_sync(0xffffffffu, total, 4 * (2 * t + j)) * -0x1p-21f;  // -8 2^-24
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int s2 = __shfl_sync(0xffffffffu, sh, 4 * (2 * t + j));
        qs[nt][j] = a.scale_log2 * 0x1p24f * __uint_as_float((uint32_t)(127 - s2) << 23);
        const int r2 = tile * ROWS + nt * 8 + 2 * t + j;
        const int pos = seq.len - seq.nq + (int)a.by_ratio(r2);
        last[nt][j] = r2 >= rows ? -1 : a.causal ? min(pos, seq.len - 1) : seq.len - 1;
        past[nt][j] = a.window > 0 ? max(pos - a.window, -1) : -1;
      }
    }
    // every query of the tile sees the tokens (all_past, all_last]
    const int i0 = (int)a.by_ratio(tile * ROWS), i1 = (int)a.by_ratio(min((tile + 1) * ROWS, rows) - 1);
    const int all_last = a.causal ? seq.len - seq.nq + i0 : seq.len - 1;
    const int all_past = a.window > 0 ? seq.len - seq.nq + i1 - a.window : -1;

    float O[CH][2][NT][4];
    // p = 2^(logit - ref) with ref = mx + vexp - kLift: mx a recent maximum of the row's logits, vexp of the exponents of the
    // v_scale that it has seen, which its lim = 2^(9 + kLift - vexp) holds: a step's sum from there on raises mx. A column of
    // no row has the largest vexp, so that it asks for nothing.
    float ref[NT][2], sum[NT][2], lim[NT][2];
    uint32_t vbits = 0x0002u;  // the f16 2^(vexp + 1) of the least vexp: scales from here on may raise one
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        ref[nt][j] = kNoMax, sum[nt][j] = 0.f;  // (-3e38 + vexp - kLift is -3e38)
        lim[nt][j] = exp_to_lim(tile * ROWS + nt * 8 + 2 * t + j < rows ? -24 : 15);  // -24: the smallest exponent of an f16
      }
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int z = 0; z < 2; ++z)
#pragma unroll
          for (int i = 0; i < 4; ++i) O[c][z][nt][i] = 0.f;
    }

    // The scales of this lane's four tokens (g, g + 8, g + 16, g + 24): all groups where the count is known.
    auto scales = [&](const __half* sc, float (&f)[4][GT]) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const __half* row = sc + (g + 8 * i) * groups;
        if constexpr (EXACT && GT % 2 == 0) {
          uint32_t w[GT / 2];
          if constexpr (GT == 2) {
            w[0] = *reinterpret_cast<const uint32_t*>(row);
          } else if constexpr (GT == 4) {
            const uint2 v = *reinterpret_cast<const uint2*>(row);
            w[0] = v.x, w[1] = v.y;
          } else {
            const uint4 v = *reinterpret_cast<const uint4*>(row);
            w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
          }
#pragma unroll
          for (int z = 0; z < GT / 2; ++z) {
            const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w[z]));
            f[i][2 * z] = v.x, f[i][2 * z + 1] = v.y;
          }
        } else {
#pragma unroll
          for (int z = 0; z < GT; ++z) f[i][z] = __half2float(row[EXACT ? z : z / a.cpg]);
        }
      }
    };

    auto consume = [&](int tok, uint32_t have, uint32_t st, auto masked) {
      constexpr bool MASKED = decltype(masked)::value;
      const uint8_t* sp = smem + (st - smem_base);
      const __half* vs = reinterpret_cast<const __half*>(sp + 2 * C::kKV + C::kSc);
      // ---- scores ----
      float S[2][NT][4];
      {
        float f[4][GT];
        scales(reinterpret_cast<const __half*>(sp + 2 * C::kKV), f);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int z = 0; z < GT; ++z) f[i][z] = fmaf(f[i][z], 0.f, f[i][z]);  // infinity * a nibble of 0 is NaN: so is the logit
#pragma unroll
        for (int z = 0; z < GT; ++z) {
          float acc[2][NT][4];
#pragma unroll
          for (int cc = 0; cc < CPG; ++cc) {
            const int c = z * CPG + cc;
            uint32_t w[4], e[4][4];
            ldmatrix_x4(st + chunk_at(c), w);
#pragma unroll
            for (int i = 0; i < 4; ++i) expand_raw(w[i], e[i]);
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                if (cc == 0)
                  mma_f16_from(acc[h][nt], e[2 * h][0], e[2 * h + 1][0], e[2 * h][1], e[2 * h + 1][1], qf[nt][c][0],
                               qf[nt][c][1], zero[nt][z][0], zero[nt][z][1]);
                else
                  mma_f16(acc[h][nt], e[2 * h][0], e[2 * h + 1][0], e[2 * h][1], e[2 * h + 1][1], qf[nt][c][0], qf[nt][c][1]);
                mma_f16(acc[h][nt], e[2 * h][2], e[2 * h + 1][2], e[2 * h][3], e[2 * h + 1][3], qf[nt][c][2], qf[nt][c][3]);
              }
          }
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int i = 0; i < 4; ++i)
                S[h][nt][i] = z == 0 ? acc[h][nt][i] * f[2 * h + i / 2][0]
                                     : fmaf(acc[h][nt][i], f[2 * h + i / 2][z], S[h][nt][i]);
        }
      }
      if (MASKED) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int r = h * 16 + (i / 2) * 8 + g, j = tok + r;
              const bool see = ((have >> r) & 1u) && j <= last[nt][i & 1] && j > past[nt][i & 1];
              S[h][nt][i] = see ? S[h][nt][i] * qs[nt][i & 1] : -INFINITY;
            }
      }
      // ---- probabilities, against the running reference ----
      // this lane's token: the largest of its v_scale, as bits, where it exists
      uint32_t vb = 0;
      if constexpr (!MASKED && EXACT && GT % 2 == 0) {
#pragma unroll
        for (int z = 0; z < GT / 2; ++z) {
          const uint32_t w = reinterpret_cast<const uint32_t*>(vs + lane * GT)[z] & 0x7fff7fffu;
          vb = max(vb, max(w >> 16, w & 0xffffu));
        }
        vb = min(vb, 0x7bffu);
      } else {
        for (int z = 0; z < groups; ++z) {
          const uint32_t w = __half_as_ushort(vs[lane * groups + z]) & 0x7fffu;
          vb = max(vb, MASKED ? (((have >> lane) & 1u) && w < 0x7c00u ? w : 0u) : min(w, 0x7bffu));
        }
      }
      float p[2][NT][4], part[NT][2];
      auto weigh = [&]() {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            part[nt][j] = 0.f;
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int i = j; i < 4; i += 2) {
                p[h][nt][i] = exp2_approx(MASKED ? S[h][nt][i] - ref[nt][j] : fmaf(S[h][nt][i], qs[nt][j], -ref[nt][j]));
                part[nt][j] += p[h][nt][i];
              }
          }
      };
      weigh();
      bool over = vb >= vbits;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) over |= part[nt][0] > lim[nt][0] || part[nt][1] > lim[nt][1];
      if (__any_sync(0xffffffffu, over)) {
        // each column's largest logit and, where scales have grown, the largest finite v_scale of the tokens that it sees
        auto finite_scale = [&](int tok) {  // of a token, as bits
          uint32_t most = 0;
          for (int z = 0; z < groups; ++z) {
            const uint32_t w = __half_as_ushort(vs[tok * groups + z]) & 0x7fffu;
            most = max(most, w < 0x7c00u ? w : 0u);
          }
          return most;
        };
        const bool grown = __any_sync(0xffffffffu, vb >= vbits);
        uint32_t all = 0, own[4] = {0, 0, 0, 0};  // own: of this lane's tokens g, g + 8, g + 16, g + 24
        if (!MASKED) {
          all = __reduce_max_sync(0xffffffffu, finite_scale(lane));
        } else if (grown) {
#pragma unroll
          for (int i = 0; i < 4; ++i) own[i] = finite_scale(g + 8 * i);
        }
        vbits = 0x8000u;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            int vexp = lim_to_exp(lim[nt][j]);
            float m = ref[nt][j] - (float)(vexp - kLift);
            uint32_t most = all;
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int i = j; i < 4; i += 2) {
                m = fmaxf(m, MASKED ? S[h][nt][i] : S[h][nt][i] * qs[nt][j]);
                if (MASKED && S[h][nt][i] != -INFINITY) most = max(most, own[2 * h + i / 2]);
              }
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
            if (MASKED && grown) {
#pragma unroll
              for (int d = 4; d < 32; d <<= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, d));
            }
            if (most) vexp = max(vexp, (int)(__float_as_uint(__half2float(__ushort_as_half((unsigned short)most))) >> 23) - 127);
            lim[nt][j] = exp_to_lim(vexp);
            if (vexp < 15) vbits = min(vbits, (uint32_t)__half_as_ushort(__float2half_rn(__uint_as_float((uint32_t)(vexp + 128) << 23))));
            const float now = m + (float)(vexp - kLift), f = exp2_approx(ref[nt][j] - now);
            ref[nt][j] = now;
            sum[nt][j] *= f;
#pragma unroll
            for (int c = 0; c < CH; ++c)
#pragma unroll
              for (int z = 0; z < 2; ++z) O[c][z][nt][j] *= f, O[c][z][nt][2 + j] *= f;
          }
        vbits = min(vbits, __shfl_xor_sync(0xffffffffu, vbits, 1));
        vbits = min(vbits, __shfl_xor_sync(0xffffffffu, vbits, 2));
        weigh();
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) sum[nt][0] += part[nt][0], sum[nt][1] += part[nt][1];
      // ---- output ----
      float f[4][GT];
      scales(vs, f);
#pragma unroll
      for (int z = 0; z < GT; ++z) {
        uint32_t pf[2][NT][2];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 2; ++i) {  // a masked token's scale may be anything, a NaN too: 0 stays 0
              const float p0 = p[h][nt][2 * i], p1 = p[h][nt][2 * i + 1], v = f[2 * h + i][z];
              pf[h][nt][i] = movmatrix_trans(pack2_f16(MASKED && p0 == 0.f ? 0.f : p0 * v, MASKED && p1 == 0.f ? 0.f : p1 * v));
            }
#pragma unroll
        for (int cc = 0; cc < CPG; ++cc) {
          const int c = z * CPG + cc;
          uint32_t w[4], e[4][4];
          ldmatrix_x4_trans(st + C::kKV + chunk_at(c), w);
#pragma unroll
          for (int i = 0; i < 4; ++i) expand(w[i], e[i]);
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              mma_f16(O[c][0][nt], e[2 * h][0], e[2 * h][1], e[2 * h + 1][0], e[2 * h + 1][1], pf[h][nt][0], pf[h][nt][1]);
              mma_f16(O[c][1][nt], e[2 * h][2], e[2 * h][3], e[2 * h + 1][2], e[2 * h + 1][3], pf[h][nt][0], pf[h][nt][1]);
            }
        }
      }
    };

    // ---- this warp's 32 tokens of each unit ----
    int slot = 0, slot_in = C::kStages - 1;
    for (int k = 0; k < count; ++k) {
      have = have_next;
      issue(k + C::kStages - 1, page, ring + slot_in * C::kStage);
      page = page_of(k + C::kStages);
      cp_async_wait<C::kStages - 1>();
      __syncwarp();
      const int tok = tok0 + k * kUnitTokens;
      if (have == 0xffffffffu && tok > all_past && tok + 31 <= all_last)
        consume(tok, have, ring + slot * C::kStage, std::false_type{});
      else
        consume(tok, have, ring + slot * C::kStage, std::true_type{});
      __syncwarp();
      slot_in = slot;
      slot = slot + 1 == C::kStages ? 0 : slot + 1;
    }
    cp_async_wait<0>();

    // ---- the warps' parts of the tile, through shared memory ----
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float l = sum[nt][j];
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
        if (g == 0) {
          s_ref[warp][nt * 8 + 2 * t + j] = ref[nt][j];
          s_sum[warp][nt * 8 + 2 * t + j] = l;
        }
      }
    __syncthreads();  // every warp is done with its ring
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int j = 0; j < 2; ++j)
          *reinterpret_cast<float4*>(merge + (warp * ROWS + nt * 8 + 2 * t + j) * C::kPitch + 32 * c + 4 * g) =
              make_float4(O[c][0][nt][j], O[c][0][nt][2 + j], O[c][1][nt][j], O[c][1][nt][2 + j]);
    __syncthreads();
    const bool whole = first == 0 && count == n_units;
    const int live = min(ROWS, rows - tile * ROWS);
    // a row's output from its sums (in f32) and its place
    auto store = [&](int r, int d, float4 o, float m, float l) {
      const int row = tile * ROWS + r, i = (int)a.by_ratio(row);
      const int64_t tk = seq.q0 + i;
      const int h = head * a.ratio + row - i * a.ratio;
      const float inv = l == 0.f ? 0.f : 1.f / l;
      uint2 w;
      w.x = pack2(l == 0.f ? 0.f : o.x * inv, l == 0.f ? 0.f : o.y * inv, a.bf16);
      w.y = pack2(l == 0.f ? 0.f : o.z * inv, l == 0.f ? 0.f : o.w * inv, a.bf16);
      *reinterpret_cast<uint2*>(static_cast<char*>(a.out) + 2 * (tk * a.os + h * a.oh + d)) = w;
      if (a.lse && d == 0) a.lse[tk * a.ls + h] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
    };
    // parts: [CTA][whether the tile begins in it]: [ROWS][D] sums, [ROWS] references, [ROWS] sums of p, and the latter
    // two again once the part holds its group
    constexpr int PART = ROWS * (D + 4);
    float* part = a.partials + (cta * 2 + (first > 0 ? 0 : 1)) * PART;
    for (int at = threadIdx.x; at < live * (D / 4); at += kSplitThreads) {
      const int r = at / (D / 4), d = 4 * (at - r * (D / 4));
      float m = s_ref[0][r];
#pragma unroll
      for (int w = 1; w < kSplitWarps; ++w) m = fmaxf(m, s_ref[w][r]);
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
      float l = 0.f;
#pragma unroll
      for (int w = 0; w < kSplitWarps; ++w) {
        const float f = exp2_approx(s_ref[w][r] - m);
        const float4 v = *reinterpret_cast<const float4*>(merge + (w * ROWS + r) * C::kPitch + d);
        o.x = fmaf(v.x, f, o.x), o.y = fmaf(v.y, f, o.y), o.z = fmaf(v.z, f, o.z), o.w = fmaf(v.w, f, o.w);
        l = fmaf(s_sum[w][r], f, l);
      }
      if (whole) {
        store(r, d, o, m, l);
      } else {
        __stcg(reinterpret_cast<float4*>(part + r * D + d), o);
        if (d == 0) {
          __stcg(part + ROWS * D + r, m);
          __stcg(part + ROWS * D + ROWS + r, l);
        }
      }
    }
    if (!whole) {
      // The tile's parts are added in order, kGroup at a time: the CTA that completes a group adds its parts into the
      // group's first, and the one that completes the last group adds the groups. The counters belong to CTAs that a tile
      // begins in (the first group's, the groups') or that it reaches from before (the other groups').
      const int64_t c0 = shares.cta_of(tile_u0), c1 = shares.cta_of(tile_u0 + n_units - 1);
      const int n = (int)(c1 - c0) + 1, n_groups = (n + kGroup - 1) / kGroup;
      const int mine_in = (int)(cta - c0) / kGroup, from = mine_in * kGroup;
      auto part_of = [&](int i) { return a.partials + ((c0 + i) * 2 + (i == 0 ? 1 : 0)) * PART; };
      // counts this CTA in; true in the one that completes the count
      auto arrive = [&](uint32_t* counter, int of) {
        __syncthreads();  // orders the block's stores before thread 0's release
        if (threadIdx.x == 0) {
          uint32_t before;
          asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(before) : "l"(counter) : "memory");
          const bool done = before == (uint32_t)(of - 1);
          if (done) *counter = 0;  // ready for the next launch
          s_last = done;
        }
        __syncthreads();
        return s_last != 0;
      };
      // Adds the parts base, base + step, ...: into part base, or as the tile's output. kGroup parts' loads are on the way
      // together.
      auto add = [&](int base, int step, int of, int level, bool out) {
        const int refs = ROWS * D + level * 2 * ROWS;
        const float* begin = part_of(base);
        const int64_t skip = part_of(base + step) - begin;  // part 0 of the tile lies apart from the others'
        const int64_t next = part_of(base + 2 * step) - part_of(base + step);
#pragma unroll 1
        for (int at = threadIdx.x; at < live * (D / 4); at += kSplitThreads) {
          const int r = at / (D / 4), d = 4 * (at - r * (D / 4));
          float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
          float l = 0.f, m = kNoMax;
#pragma unroll 1
          for (int i0 = 0; i0 < of; i0 += kGroup) {
            float4 v[kGroup];
            float vm[kGroup], vl[kGroup];
#pragma unroll
            for (int i = 0; i < kGroup; ++i) {
              const bool is = i0 + i < of;
              const float* q = begin + (i0 + i == 0 ? 0 : skip + (i0 + i - 1) * next);
              v[i] = is ? __ldcg(reinterpret_cast<const float4*>(q + r * D + d)) : make_float4(0.f, 0.f, 0.f, 0.f);
              vm[i] = is ? __ldcg(q + refs + r) : kNoMax;
              vl[i] = is ? __ldcg(q + refs + ROWS + r) : 0.f;
            }
            float now = m;
#pragma unroll
            for (int i = 0; i < kGroup; ++i) now = fmaxf(now, vm[i]);
            const float f = exp2_approx(m - now);
            o.x *= f, o.y *= f, o.z *= f, o.w *= f, l *= f;
            m = now;
#pragma unroll
            for (int i = 0; i < kGroup; ++i) {
              const float w = exp2_approx(vm[i] - m);
              o.x = fmaf(v[i].x, w, o.x), o.y = fmaf(v[i].y, w, o.y), o.z = fmaf(v[i].z, w, o.z), o.w = fmaf(v[i].w, w, o.w);
              l = fmaf(vl[i], w, l);
            }
          }
          if (out) {
            store(r, d, o, m, l);
          } else {
            float* q = part_of(base);
            __stcg(reinterpret_cast<float4*>(q + r * D + d), o);
            if (d == 0) __stcg(q + refs + 2 * ROWS + r, m), __stcg(q + refs + 3 * ROWS + r, l);
          }
        }
      };
      if (arrive(a.counters + (mine_in == 0 ? 0 : kMaxCtas) + c0 + from, min(kGroup, n - from))) {
#pragma unroll 1
        for (int level = 0;; ++level) {
          const bool top = level > 0 || n_groups == 1;
          add(level ? 0 : from, level ? kGroup : 1, level ? n_groups : min(kGroup, n - from), level, top);
          if (top || !arrive(a.counters + 2 * kMaxCtas + c0, n_groups)) break;
        }
      }
    }
    __syncthreads();  // the ring and the small arrays are free again
  }
}

template <int D, int CPG, int NT, bool EXACT>
int launch_split(const Args& a, int ctas, cudaStream_t s) {
  constexpr int smem = SplitCfg<D, NT>::kSmem;
  const auto kernel = kv4_split_kernel<D, CPG, NT, EXACT>;
  if (smem > 48 * 1024) {
    const cudaError_t e = ensure_smem_attr(reinterpret_cast<const void*>(kernel), smem);
    if (e != cudaSuccess) return cuda_status(e);
  }
  kernel<<<min(ctas, sm_count() * SplitCfg<D, NT>::kOcc), kSplitThreads, smem, s>>>(a);
  note_launch();
  return check_launch();
}

}  // namespace kv4
}  // namespace up
