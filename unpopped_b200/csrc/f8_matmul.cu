// f8_matmul.cu — products of e4m3 activations and weights with an f32 scale for each block of 128, dense or by expert.
//
//   out[m][j] = sum_b xs[m][b] ws[j / 128][b] (sum_{k in b} x[m][k] w[j][k])
//
// The scales change every 128 k and are not powers of two, so no accumulator can run over a row: each block's product is a
// tcgen05.mma of its own into tensor memory (four steps of 32 k, f32), and the epilogue warps add it, times its two scales,
// to f32 sums in registers while the next blocks are multiplied.
//
// Two forms, by which operand takes the MMA's rows:
//  * Narrow, for few tokens: 128 weight rows, up to 32 tokens as columns. Bound by HBM: every weight once. Columns are dealt in steps of 16,
//    so a group of one token costs little, and four blocks share an accumulator slot, so that handing it to the epilogue costs once
//    for all four. A thread of the epilogue has one weight row; the tokens' scales come to it through shared memory.
//  * Wide: 128 tokens as rows (256 of two CTAs, tcgen05's cta_group::2), 256 weight rows as columns. A thread of the epilogue has one
//    token, so a block's scales are one factor for all of its columns. (With tokens as columns every thread needs every token's
//    factor: at 128 bytes a cycle shared memory gives those of 128 x 128 values in 512 cycles, in which the MMA takes 256.)
#include "common.cuh"
#include "divide.cuh"
#include "launch.cuh"
#include "tc.cuh"

#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <mutex>

namespace up {
namespace f8 {

constexpr int kBlock = 128;               // k a scale, and weight rows a scale
constexpr int kTile = 128 * kBlock;       // bytes of 128 rows of a block
constexpr int kBox = 16;                  // tokens of a small TMA box
constexpr int kMaxExperts = 1024;
constexpr int kRuns = 4;                  // runs of blocks that the roles may be apart
constexpr int kMaxCtas = (UP_F8_COUNTER_BYTES - 64) / 4;  // a counter each

template <int TOKENS>
struct Narrow {
  static constexpr bool kWide = false;
  static constexpr int kCtas = 1, kTokens = TOKENS, kStep = 16, kWeights = 128;  // of a tile; tokens go in steps
  static constexpr int kGroup = 4;                                  // blocks of an accumulator slot
  static constexpr int kDBlock = TOKENS;                            // columns of tensor memory a block
  static constexpr int kBBytes = TOKENS * kBlock, kStages = TOKENS == 64 ? 8 : 10;
  static constexpr int kRunsWarp = 4, kEpi0 = 5;                    // the warp that deals the runs, the first of the epilogue's
  static constexpr int kEpiWarps = TOKENS == 32 ? 4 : 8, kSums = TOKENS * 4 / kEpiWarps;  // sums a thread
  static constexpr int kMinBlocks = 8;                              // of an owner: fewer do not pay for joining the parts
  static constexpr int kScRing = 4, kScSlot = kGroup * TOKENS;  // tokens' scales in shared memory, a group a slot
};
template <int CTAS>
struct Wide {
  static constexpr bool kWide = true;
  static constexpr int kCtas = CTAS, kTokens = 128 * CTAS, kStep = kTokens, kWeights = 256;
  static constexpr int kGroup = 1;
  static constexpr int kDBlock = 256;
  static constexpr int kBBytes = 256 / CTAS * kBlock, kStages = CTAS == 2 ? 6 : 4;
  static constexpr int kRunsWarp = 2, kEpi0 = 4;
  static constexpr int kEpiWarps = 8, kSums = 128;
  static constexpr int kMinBlocks = 16;
  static constexpr int kScRing = 0, kScSlot = 0;
};
// What follows from them.
template <typename C>
struct Of {
  static constexpr int kStage = kTile + C::kBBytes;
  static constexpr int kDSlot = C::kDBlock * C::kGroup, kDRing = 512 / kDSlot;  // accumulators in tensor memory
  static constexpr int kEpiThreads = 32 * C::kEpiWarps, kThreads = 32 * C::kEpi0 + kEpiThreads;
  static constexpr size_t kPart = (size_t)C::kSums * kEpiThreads;  // values of a CTA's part of a tile
  // One thread issues the MMAs and commits of a block in some 450 cycles, so two take the blocks in turn; the ring's even
  // depth then gives each stage to one of them, which sees all of its phases.
  static constexpr int kIssuers = 2;
  static constexpr int kBars = 2 * C::kStages + 2 * kDRing + 2 * C::kScRing + 3 * kRuns + 3;
  static constexpr int kSmem = 1024 + C::kStages * kStage + C::kScRing * C::kScSlot * 4 + kRuns * 48 + kBars * 8 + 16 + (kMaxExperts + 1) * 2 * 4;
  static_assert(C::kStages % 2 == 0 && (C::kGroup > 1 || kDRing % 2 == 0) && kSmem <= 232448, "rings, shared memory");
};

struct Header {
  uint32_t ticket, done, epoch, error;    // `error` at byte 12, as in every workspace
  uint32_t pad[12];
};
static_assert(sizeof(Header) == 64, "header");

struct Args {
  const float *xs, *ws;
  int64_t xs_m, xs_b;
  int64_t m;
  int experts, n, kb, nb, tb, groups;     // kb: blocks of k, in `groups` groups; nb: of weight rows, in tb tiles
  Divide32 by_owners = Divide32(1), by_groups = Divide32(1);
  const int32_t* offsets;
  void* out;
  int64_t out_stride;
  int out_dtype, wide_out;                // wide_out: its rows begin on 32 bytes
  Header* header;
  uint32_t* counters;                     // one a CTA: the parts of the tile that it begins
  float* partials;                        // [CTA][2][Of<C>::kPart]
  uint64_t wait_ns;
};

// Waits for the barrier's phase, at most a.wait_ns; false when that ran out or another role gave up. The clock is read only after
// many attempts.
__device__ __forceinline__ bool try_wait(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(tc::smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, const Args& a, volatile int* abort) {
  for (int it = 0; it < 64; ++it)
    if (try_wait(bar, parity)) return true;
  const uint64_t t0 = globaltimer_ns();
  for (uint32_t it = 1;; ++it) {
    if (try_wait(bar, parity)) return true;
    if ((it & 255u) == 0) {
      if (abort && *abort) return false;
      if (globaltimer_ns() - t0 > a.wait_ns) return false;
    }
  }
}

// A role's place in the ring of runs.
struct Runs {
  int at = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void next() {
    if (++at == kRuns) at = 0, phase ^= 1u;
  }
};

// A unit is one group of k of one tile; tiles are numbered by expert, then weight rows, then tokens, so the tiles that
// share weights are neighbours. An owner is a CTA, or a pair. Of the tiles, as many as fill whole rounds of the owners are dealt out one
// by one; the units of the `rest` others, the first ones, are shared evenly, so that all owners end together. An owner's units are
// runs of groups of a tile, one after the other: first its share of the rest, whose parts are then joined while others still
// work. One thread of a CTA goes over them and leaves each run in shared memory, where the other roles read it.
struct Run {
  int t, g0, g1;                          // the tile, its groups from g0 to before g1; no groups: the end
  int e, tb, m0, n;                       // the tile's expert, place among the weight rows, first row and number of tokens
  int c0, c1;                             // the first and last of the owners that share the tile (by a barrier of their own)
  int pad[3];
};
static_assert(sizeof(Run) == 48, "Run");
template <typename C>
struct Walk {
  const int *start, *begin;               // first tile, first row of each expert
  int groups;                             // a tile's
  int base, more;                         // shares of the rest: base + 1 units for the first `more` owners, base for the others
  int left;                               // units of this owner's share, from r.g0 of tile r.t on
  int whole_t, whole_left, owners;        // the next of the tiles dealt out, and how many are left
  Run r;

  __device__ __forceinline__ int first_unit(int owner) const { return owner * base + min(owner, more); }
  __device__ __forceinline__ int owner_of(int unit) const {
    return unit < more * (base + 1) ? unit / (base + 1) : more + (unit - more * (base + 1)) / base;
  }
  __device__ __forceinline__ Walk(const Args& a, const int* start_, const int* begin_, int owner, int owners_)
      : start(start_), begin(begin_), groups(a.groups), left(0), owners(owners_) {
    const int tiles = start[a.experts];
    const int rounds = (int)a.by_owners(tiles);
    int rest = tiles - rounds * owners;
    if (10 * rest > 9 * owners) rest = 0;  // a last round that is nearly full: parts would cost more than they save
    const int units = rest * groups, most = units * C::kGroup / C::kMinBlocks, sharers = most < 1 ? 1 : most < owners ? most : owners;
    base = sharers == owners ? (int)a.by_owners(units) : units / sharers, more = units - base * sharers;
    r.e = 0, r.t = 0, r.g0 = 0;
    if (owner < sharers) {
      left = base + (owner < more ? 1 : 0);
      r.t = (int)a.by_groups(first_unit(owner));
      r.g0 = first_unit(owner) - r.t * groups;
    }
    whole_t = rest + owner;
    whole_left = rounds + (rest == 0 && owner < tiles - rounds * owners ? 1 : 0);
    const int first = left > 0 ? r.t : whole_t;
    int hi = a.experts - 1;               // the last expert that starts at or before the first tile
    while (r.e < hi) {
      const int mid = (r.e + hi + 1) >> 1;
      if (start[mid] <= first) r.e = mid;
      else hi = mid - 1;
    }
  }
  // the next run; the one without groups at the end
  __device__ __forceinline__ bool next() {
    if (left > 0) {
      r.g1 = min(groups, r.g0 + left);
      left -= r.g1 - r.g0;
    } else if (whole_left > 0) {
      --whole_left;
      r.t = whole_t, r.g0 = 0, r.g1 = groups;
      whole_t += owners;
    } else {
      r.g1 = r.g0;
      return false;
    }
    while (r.t >= start[r.e + 1]) ++r.e;
    const int rows = begin[r.e + 1] - begin[r.e], wide = (rows + C::kTokens - 1) / C::kTokens, at = r.t - start[r.e];
    r.tb = at, r.m0 = begin[r.e], r.n = rows;
    if (wide > 1) {
      // the group's tokens in tiles of equal width; the last may have fewer, and has some: (wide - 1) * kTokens < rows
      r.tb = at / wide;
      const int each = ((rows + wide - 1) / wide + C::kStep - 1) / C::kStep * C::kStep, first = (at - r.tb * wide) * each;
      r.m0 += first;
      r.n = min(each, rows - first);
    }
    return true;
  }
  __device__ __forceinline__ void passed() {  // the run was taken over
    if (left > 0) ++r.t, r.g0 = 0;
  }
};

__device__ __forceinline__ uint32_t cta_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// The address of the first CTA's copy of a barrier in the cluster's shared memory.
__device__ __forceinline__ uint32_t in_leader(const uint64_t* bar) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(tc::smem_u32(bar)));
  return r;
}
__device__ __forceinline__ void arrive_in_leader(uint32_t bar) {  // of in_leader
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

template <bool PAIR>
__device__ __forceinline__ void load_w(void* dst, const CUtensorMap* m, uint32_t bar, int32_t x, int32_t y, int32_t z) {
  if (PAIR)
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], "
        "[%2];" ::"r"(tc::smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(m)), "r"(bar), "r"(x), "r"(y), "r"(z)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
            tc::smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(m)), "r"(bar), "r"(x), "r"(y), "r"(z)
        : "memory");
}
template <bool PAIR>
__device__ __forceinline__ void load_x(void* dst, const CUtensorMap* m, uint32_t bar, int32_t x, int32_t y) {
  if (PAIR)
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(
            tc::smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(m)), "r"(bar), "r"(x), "r"(y)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(
            tc::smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(m)), "r"(bar), "r"(x), "r"(y)
        : "memory");
}

// D[tmem] (+)= A[smem] * B[smem], e4m3 inputs, f32 sums.
template <bool PAIR>
__device__ __forceinline__ void mma_f8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  if (PAIR)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, {%5, %5, %5, %5, %5, %5, %5, %5}, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(0u)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, {%5, %5, %5, %5}, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(0u)
        : "memory");
}
// Arrives on `bar`, in both CTAs of a pair, when every tcgen05 op that this thread issued before has completed.
template <bool PAIR>
__device__ __forceinline__ void commit(uint64_t* bar) {
  if (PAIR)
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
            tc::smem_u32(bar)),
        "h"((uint16_t)3)
        : "memory");
  else
    tc::commit(bar);
}
template <bool PAIR>
__device__ __forceinline__ void tmem_alloc(uint32_t* slot) {
  if (PAIR) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(tc::smem_u32(slot)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  } else {
    tc::tmem_alloc(slot, 512);
    tc::tmem_relinquish();
  }
}
template <bool PAIR>
__device__ __forceinline__ void tmem_free(uint32_t at) {
  if (PAIR)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(at) : "memory");
  else
    tc::tmem_dealloc(at, 512);
}

// Instruction descriptor, kind::f8f6f4: e4m3 A and B (K-major), f32 D.
__device__ __forceinline__ constexpr uint32_t idesc_f8(int m, int n) {
  return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

// 16 or 32 consecutive columns of this thread's lane of tensor memory. The registers hold them after wait_loads; what uses them is
// volatile too, so nothing moves it before the wait.
__device__ __forceinline__ void load16(uint32_t from, uint32_t (&v)[16]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
               : "r"(from)
               : "memory");
}
__device__ __forceinline__ void load32(uint32_t from, uint32_t (&v)[32]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
               : "r"(from)
               : "memory");
}
__device__ __forceinline__ void wait_loads() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fma_after(float& sum, uint32_t v, float f) {
  asm volatile("fma.rn.f32 %0, %1, %2, %0;" : "+f"(sum) : "f"(__uint_as_float(v)), "f"(f));
}
__device__ __forceinline__ float4 shared4(uint32_t at) {
  float4 f;
  asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(f.x), "=f"(f.y), "=f"(f.z), "=f"(f.w) : "r"(at));
  return f;
}

// The schedule: begin[e] (rows) and start[e] (tiles) of every expert, from the offsets on the device; each entry is held to
// [0, m] and to its predecessors. One warp.
template <typename C>
__device__ __forceinline__ void schedule(const Args& a, int* start, int* begin, int lane) {
  constexpr int kTokens = C::kTokens;
  int run_tiles = 0, run_row = 0;
  for (int e0 = 0; e0 <= a.experts; e0 += 32) {
    const int e = e0 + lane;
    int row = 0;
    if (e <= a.experts) {
      const int64_t o = a.offsets ? (int64_t)a.offsets[e] : (e == 0 ? 0 : a.m);
      row = (int)(o < 0 ? 0 : o > a.m ? a.m : o);
    }
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, row, o);
      if (lane >= o) row = max(row, v);
    }
    row = max(row, run_row);
    int before = __shfl_up_sync(0xffffffffu, row, 1);  // begin[e - 1]
    if (lane == 0) before = run_row;
    // tiles of expert e - 1, which ends where e begins
    int tiles = e >= 1 && e <= a.experts ? (row - before + kTokens - 1) / kTokens * a.tb : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, tiles, o);
      if (lane >= o) tiles += v;
    }
    if (e <= a.experts) begin[e] = row, start[e] = run_tiles + tiles;
    run_row = __shfl_sync(0xffffffffu, row, 31);
    run_tiles += __shfl_sync(0xffffffffu, tiles, 31);
  }
}

__device__ __forceinline__ uint16_t half_bits(float v, bool bf16) {
  return bf16 ? __bfloat16_as_ushort(__float2bfloat16_rn(v)) : __half_as_ushort(__float2half_rn(v));
}
__device__ __forceinline__ uint32_t half_pair(float a, float b, bool bf16) {
  const __nv_bfloat162 x = __floats2bfloat162_rn(a, b);
  const __half2 y = __floats2half2_rn(a, b);
  return bf16 ? *reinterpret_cast<const uint32_t*>(&x) : *reinterpret_cast<const uint32_t*>(&y);
}
__device__ __forceinline__ void store32(void* to, const uint32_t (&v)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]),
               "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}

template <typename C>
__device__ __forceinline__ void matmul(const CUtensorMap& wmap, const CUtensorMap& xmap, const CUtensorMap& xmap_full, const Args& a) {
  using O = Of<C>;
  constexpr bool PAIR = C::kCtas == 2;
  constexpr int kGroup = C::kGroup, kStages = C::kStages, kDRing = O::kDRing, kScRing = C::kScRing, kSums = C::kSums;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* stages = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* sc = reinterpret_cast<float*>(stages + kStages * O::kStage);  // [kScRing][4 blocks][32]
  uint64_t* full = reinterpret_cast<uint64_t*>(sc + kScRing * C::kScSlot);
  uint64_t* empty = full + kStages;
  uint64_t* d_full = empty + kStages;
  uint64_t* d_empty = d_full + kDRing;
  uint64_t* sc_full = d_empty + kDRing;
  uint64_t* sc_empty = sc_full + kScRing;
  uint64_t* seg_in = sc_empty + kScRing;
  uint64_t* seg_out = seg_in + 1;
  uint64_t* drain = seg_out + 1;
  uint64_t* run_full = drain + 1;
  uint64_t* run_empty = run_full + kRuns;
  uint64_t* run_owners = run_empty + kRuns;
  static_assert((kStages * O::kStage + kScRing * C::kScSlot * 4 + O::kBars * 8) % 8 == 0, "alignment");
  Run* runs = reinterpret_cast<Run*>(run_owners + kRuns);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(runs + kRuns);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile uint32_t* verdict = tmem_slot + 2;
  int* start = reinterpret_cast<int*>(tmem_slot + 4);
  int* begin = start + kMaxExperts + 1;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = PAIR ? cta_rank() : 0;
  if (warp == 0) {
    if (lane == 0) {
      for (int s = 0; s < kStages; ++s) tc::mbar_init(&full[s], 1), tc::mbar_init(&empty[s], 1);
      for (int d = 0; d < kDRing; ++d) tc::mbar_init(&d_full[d], kGroup > 1 ? O::kIssuers : 1), tc::mbar_init(&d_empty[d], C::kEpiWarps * C::kCtas);
      for (int q = 0; q < kScRing; ++q) tc::mbar_init(&sc_full[q], 1), tc::mbar_init(&sc_empty[q], C::kEpiWarps);
      // readers of the runs: the loads, the issuers (a pair's are the first CTA's), the scales, the epilogue's warps
      for (int i = 0; i < kRuns; ++i)
        tc::mbar_init(&run_full[i], 1), tc::mbar_init(&run_owners[i], 1), tc::mbar_init(&run_empty[i], 1 + (rank == 0 ? O::kIssuers : 0) + (C::kWide ? 0 : 1) + C::kEpiWarps);
      tc::mbar_init(seg_in, C::kEpiWarps), tc::mbar_init(seg_out, 1), tc::mbar_init(drain, O::kIssuers);
      *abort_flag = 0;
      tc::mbar_fence_init();
      tc::tma_prefetch_desc(&wmap), tc::tma_prefetch_desc(&xmap), tc::tma_prefetch_desc(&xmap_full);
    }
  } else if (warp == 1) {
    tmem_alloc<PAIR>(tmem_slot);
  } else if (warp == 2) {
    after_previous();
    schedule<C>(a, start, begin, lane);
  }
  after_previous();
  let_next_begin();
  tc::fence_before_sync();
  __syncthreads();
  if (PAIR) cluster_sync();
  tc::fence_after_sync();
  const uint32_t tmem = *tmem_slot;

  auto give_up = [&]() {
    *abort_flag = 1;
    atomicOr(&a.header->error, 1u);
  };
  // waits for the next run; false at the end or when a wait ran out (good is false then)
  auto take = [&](const Runs& at, bool& good) {
    good = good && wait(&run_full[at.at], at.phase, a, abort_flag);
    return good && runs[at.at].g1 > runs[at.at].g0;
  };

  if (warp < C::kEpi0) {
    if (C::kWide) asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    if (warp == 0) {
      // ---------------- loads ----------------
      if (lane == 0) {
        int64_t issued = 0;
        int s = 0;
        uint32_t ph = 1;
        const uint32_t full0 = PAIR ? in_leader(full) : tc::smem_u32(full);  // a pair's loads all count on the leader's barriers
        bool good = true;
        for (Runs at; take(at, good); at.next()) {
          const Run w = runs[at.at];
          tc::mbar_arrive(&run_empty[at.at]);
          const int boxes = (w.n + kBox - 1) / kBox;
          const uint32_t bytes = C::kWide ? C::kCtas * O::kStage : kTile + boxes * (kBox * kBlock);
          const int row = w.tb * C::kWeights + (int)rank * kBlock, m0 = w.m0 + (int)rank * 128;
          for (int kb = w.g0 * kGroup, end = min(a.kb, w.g1 * kGroup); kb < end; ++kb) {
            good = wait(&empty[s], ph, a, abort_flag);
            if (!good) break;
            uint8_t* to = stages + (size_t)s * O::kStage;
            const uint32_t bar = full0 + 8 * s;
            const int k = kb * kBlock;
            if (rank == 0) tc::mbar_arrive_expect_tx(&full[s], bytes);
            if (C::kWide) {
              load_w<PAIR>(to + kTile, &wmap, bar, k, row, w.e);
              if (!PAIR) load_w<PAIR>(to + 2 * kTile, &wmap, bar, k, row + kBlock, w.e);
              load_x<PAIR>(to, &xmap_full, bar, k, m0);
            } else {
              load_w<PAIR>(to, &wmap, bar, k, row, w.e);
              if (boxes * kBox == C::kTokens)
                load_x<PAIR>(to + kTile, &xmap_full, bar, k, m0);
              else
                for (int b = 0; b < boxes; ++b) load_x<PAIR>(to + kTile + b * (kBox * kBlock), &xmap, bar, k, m0 + b * kBox);
            }
            ++issued;
            if (++s == kStages) s = 0, ph ^= 1u;
          }
        }
        if (!good) give_up();
        // every load lands before shared memory is released
        if (rank == 0)
          for (int64_t j = issued > kStages ? issued - kStages : 0; j < issued; ++j)
            wait(&full[j % kStages], (uint32_t)((j / kStages) & 1), a, nullptr);
      }
    } else if (warp == 1 || warp == 3) {
      // ---------------- MMA: the issuers take the blocks in turn; a group's accumulators are done when both have committed ----------------
      if (lane == 0 && rank == 0) {
        int s = 0, d = 0;
        bool mine = warp == 1;
        uint32_t ph = 0, dph = 1;
        bool good = true;
        for (Runs at; take(at, good); at.next()) {
          const Run w = runs[at.at];
          tc::mbar_arrive(&run_empty[at.at]);
          const uint32_t id = C::kWide ? idesc_f8(128 * C::kCtas, 256) : idesc_f8(128, (w.n + 15) / 16 * 16);
          const int end = min(a.kb, w.g1 * kGroup);
          for (int kb = w.g0 * kGroup; kb < end && good; kb += kGroup) {
            if (kGroup > 1 || mine) good = wait(&d_empty[d], dph, a, abort_flag);
#pragma unroll 1
            for (int j = 0; j < kGroup && kb + j < end && good; ++j, mine = !mine) {
              if (mine) {
                good = wait(&full[s], ph, a, abort_flag);
                if (!good) break;
                tc::fence_after_sync();
                const uint32_t stage = tc::smem_u32(stages) + s * O::kStage;
                const uint64_t ad = tc::sdesc_kmajor_sw128(stage), bd = tc::sdesc_kmajor_sw128(stage + kTile);
#pragma unroll
                for (int i = 0; i < kBlock / 32; ++i) mma_f8<PAIR>(tmem + d * O::kDSlot + j * C::kDBlock, ad + 2 * i, bd + 2 * i, id, i > 0);
                commit<PAIR>(&empty[s]);
                if (kGroup == 1) commit<PAIR>(&d_full[d]);
              }
              if (++s == kStages) s = 0, ph ^= 1u;
            }
            if (kGroup > 1) commit<PAIR>(&d_full[d]);
            if (++d == kDRing) d = 0, dph ^= 1u;
          }
        }
        if (!good) give_up();
        commit<PAIR>(drain);
        wait(drain, 0, a, nullptr);
      }
    } else if (warp == 2 && !C::kWide) {
      // ---------------- scales: x's times the weight's, four blocks of a run at a time, the next four's loads on their way ----------------
      constexpr int kEach = C::kTokens / 32;
      float xs[2][4][kEach], ws[2];
      int cnt[2], n[2], kb = 0, end = 0;
      Run w;
      Runs at;
      bool good = true, more = true;
      auto load = [&](int h) {
        cnt[h] = 0;
        if (kb >= end && more) {
          more = __all_sync(0xffffffffu, take(at, good));
          if (more) {
            w = runs[at.at];
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(&run_empty[at.at]);
            at.next();
            kb = w.g0 * kGroup, end = min(a.kb, w.g1 * kGroup);
          }
        }
        if (more) {
          cnt[h] = min(4, end - kb), n[h] = w.n;
          ws[h] = lane < cnt[h] ? a.ws[((int64_t)w.e * a.nb + w.tb) * a.kb + kb + lane] : 0.f;
          const float* from = a.xs + (w.m0 + lane) * a.xs_m + kb * a.xs_b;
#pragma unroll
          for (int c = 0; c < kEach; ++c)
#pragma unroll
            for (int j = 0; j < 4; ++j) xs[h][j][c] = c * 32 + lane < w.n && j < cnt[h] ? from[c * 32 * a.xs_m + j * a.xs_b] : 0.f;
          kb += 4;
        }
      };
      int q = 0;
      uint32_t ph = 1;
      auto store = [&](int h) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (j >= cnt[h]) break;
          if (j % kGroup == 0) good = __all_sync(0xffffffffu, wait(&sc_empty[q], ph, a, abort_flag));
          if (!good) break;
          const float f = __shfl_sync(0xffffffffu, ws[h], j);
#pragma unroll
          for (int c = 0; c < kEach; ++c)
            if (c * 32 < n[h]) sc[q * C::kScSlot + j % kGroup * C::kTokens + c * 32 + lane] = xs[h][j][c] * f;
          if (j % kGroup == kGroup - 1 || j + 1 == cnt[h]) {
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(&sc_full[q]);
            if (++q == kScRing) q = 0, ph ^= 1u;
          }
        }
      };
      load(0);
      while (cnt[0] > 0 && good) {
        load(1);
        store(0);
        if (cnt[1] == 0 || !good) break;
        load(0);
        store(1);
      }
      if (!good) give_up();
    } else if (warp == C::kRunsWarp) {
      // ---------------- runs ----------------
      if (lane == 0) {
        Walk<C> w(a, start, begin, blockIdx.x / C::kCtas, gridDim.x / C::kCtas);
        Runs at;
        bool good = true;
        for (bool more = true; more; at.next()) {
          more = w.next();  // the run without groups is handed over too
          good = wait(&run_empty[at.at], at.phase ^ 1u, a, abort_flag);
          if (!good) break;
          runs[at.at] = w.r;
          tc::mbar_arrive(&run_full[at.at]);
          if (w.r.g0 > 0 || w.r.g1 < a.groups) {  // who shares the tile is needed last
            runs[at.at].c0 = w.owner_of(w.r.t * a.groups);
            runs[at.at].c1 = w.owner_of(w.r.t * a.groups + a.groups - 1);
          }
          tc::mbar_arrive(&run_owners[at.at]);
          w.passed();
        }
        if (!good) give_up();
      }
    }
  } else {
    // ---------------- sums: lanes 32 (warp % 4) .. of tensor memory ----------------
    if (C::kWide) asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    const int quarter = warp & 3, part = (warp - C::kEpi0) >> 2, thread = threadIdx.x - 32 * C::kEpi0, row = quarter * 32 + lane;
    const uint32_t d_empty0 = PAIR ? in_leader(d_empty) : 0;
    const uint32_t from = tmem + ((uint32_t)(quarter * 32) << 16) + kSums * part;
    float sum[kSums];
    uint32_t v[2][C::kWide ? 16 : 32];
    int d = 0, q = 0;
    uint32_t dph = 0, qph = 0, joined = 0;
    bool good = true;
    auto accumulators = [&]() {  // waits for the next slot's
      good = __all_sync(0xffffffffu, wait(&d_full[d], dph, a, abort_flag));
      tc::fence_after_sync();
    };
    auto free_accumulators = [&]() {
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) {
        if (PAIR)
          arrive_in_leader(d_empty0 + 8 * d);
        else
          tc::mbar_arrive(&d_empty[d]);
      }
      if (++d == kDRing) d = 0, dph ^= 1u;
    };
    for (Runs at; __all_sync(0xffffffffu, take(at, good)); at.next()) {
#pragma unroll
      for (int j = 0; j < kSums; ++j) sum[j] = 0.f;
      const volatile Run& w = runs[at.at];  // kept until the tile is written: read where it is needed, not held in registers
      const int first = w.g0 * kGroup, end = min(a.kb, w.g1 * kGroup);
      if constexpr (C::kWide) {
        // The thread's row is a token, its columns 128 weight rows with one scale. A token behind the group's last one goes by the last one's
        // scale, a block of weights behind the last by the last's; neither is written.
        const int nb = min(w.tb * 2 + part, a.nb - 1), m = w.m0 + min((int)rank * 128 + row, w.n - 1);
        const float* xs = a.xs + m * a.xs_m + first * a.xs_b;
        const float* ws = a.ws + ((int64_t)w.e * a.nb + nb) * a.kb + first;
        constexpr int kAhead = 4;  // blocks whose scales are on their way
        float xs_next[kAhead], ws_next[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
          xs_next[j] = first + j < end ? xs[j * a.xs_b] : 0.f;
          ws_next[j] = first + j < end ? ws[j] : 0.f;
        }
        accumulators();
        if (!good) break;
        // Two sets of 16 columns at a time; the next ones' loads run beside the sums, the next block's too. (Sets of 32 left too few
        // registers for the 128 sums: 574 against 562 us for 8192 rows by 8192 x 8192 weights; packed fma.rn.f32x2 needs its operands moved: 565.)
        load16(from + d * O::kDSlot, v[0]);
        load16(from + d * O::kDSlot + 16, v[1]);
        for (int kb = first; kb < end; ++kb) {
          const float f = xs_next[0] * ws_next[0];
#pragma unroll
          for (int j = 0; j + 1 < kAhead; ++j) xs_next[j] = xs_next[j + 1], ws_next[j] = ws_next[j + 1];
          if (kb + kAhead < end) xs_next[kAhead - 1] = xs[kAhead * a.xs_b], ws_next[kAhead - 1] = ws[kAhead];
          xs += a.xs_b, ++ws;
          const uint32_t in = from + d * O::kDSlot;
#pragma unroll
          for (int c = 0; c < kSums; c += 32) {
            const bool last = c + 32 == kSums;
            wait_loads();
            if (last) free_accumulators();
#pragma unroll
            for (int j = 0; j < 16; ++j) fma_after(sum[c + j], v[0][j], f);
            if (!last) {
              load16(in + c + 32, v[0]);
            } else if (kb + 1 < end) {
              accumulators();
              if (!good) break;
              load16(from + d * O::kDSlot, v[0]);
            }
#pragma unroll
            for (int j = 0; j < 16; ++j) fma_after(sum[c + 16 + j], v[1][j], f);
            if (!last)
              load16(in + c + 48, v[1]);
            else if (kb + 1 < end)
              load16(from + d * O::kDSlot + 16, v[1]);
          }
          if (!good) break;
        }
      } else {
        // The thread's row is a weight row, its columns the tokens, each with a factor of its own.
        for (int kb = first; kb < end; kb += kGroup) {
          accumulators();
          if (!good) break;
          good = __all_sync(0xffffffffu, wait(&sc_full[q], qph, a, abort_flag));
          if (!good) break;
          const uint32_t f = tc::smem_u32(sc + q * C::kScSlot + kSums * part);
          auto add = [&](int j, int c, const uint32_t(&x)[32]) {  // block j's columns c to c + 31
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
              const float4 f4 = shared4(f + (j * C::kTokens + c + i) * 4);
              fma_after(sum[c + i], x[i], f4.x), fma_after(sum[c + i + 1], x[i + 1], f4.y);
              fma_after(sum[c + i + 2], x[i + 2], f4.z), fma_after(sum[c + i + 3], x[i + 3], f4.w);
            }
          };
          const uint32_t in = from + d * O::kDSlot;
#pragma unroll
          for (int j = 0; j < kGroup; j += kSums > 32 ? 1 : 2) {
            if (kb + j >= end) break;
            if constexpr (kSums > 32) {
              load32(in + j * C::kDBlock, v[0]);
              load32(in + j * C::kDBlock + 32, v[1]);
              wait_loads();
              add(j, 0, v[0]);
              add(j, 32, v[1]);
            } else {
              load32(in + j * C::kDBlock, v[0]);
              if (kb + j + 1 < end) load32(in + (j + 1) * C::kDBlock, v[1]);
              wait_loads();
              add(j, 0, v[0]);
              if (kb + j + 1 < end) add(j + 1, 0, v[1]);
            }
          }
          free_accumulators();
          if (lane == 0) tc::mbar_arrive(&sc_empty[q]);  // free_accumulators synchronised the warp
          if (++q == kScRing) q = 0, qph ^= 1u;
        }
      }
      if (!good) break;

      bool write = true;
      if (w.g0 > 0 || w.g1 < a.groups) {
        // A part of a tile: published, and whichever owner comes last adds the parts in the order of the owners.
        good = __all_sync(0xffffffffu, wait(&run_owners[at.at], at.phase, a, abort_flag));
        if (!good) break;
        const int c0 = w.c0, c1 = w.c1, owner = blockIdx.x / C::kCtas;
        float* parts = a.partials + thread;
        float* to = parts + ((size_t)blockIdx.x * 2 + (c0 == owner ? 1 : 0)) * O::kPart;
#pragma unroll
        for (int j = 0; j < kSums; ++j) __stcg(to + j * O::kEpiThreads, sum[j]);
        __syncwarp();
        const uint32_t jp = joined & 1u;
        ++joined;
        if (lane == 0) tc::mbar_arrive(seg_in);
        if (warp == C::kEpi0 && lane == 0) {
          // one release for all warps' stores, which the barrier put before it
          good = wait(seg_in, jp, a, abort_flag);
          if (good) {
            uint32_t* counter = a.counters + c0 * C::kCtas + rank;
            uint32_t before;
            asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(before) : "l"(counter) : "memory");
            const bool done = before == (uint32_t)(c1 - c0);
            if (done) *counter = 0u;  // ready for the next launch
            *verdict = done ? 1u : 0u;
            tc::mbar_arrive(seg_out);
          }
        }
        good = __all_sync(0xffffffffu, good && wait(seg_out, jp, a, abort_flag));
        if (!good) break;
        write = *verdict != 0u;
        if (write) {
          constexpr int kAt = kSums < 64 ? kSums : 64;  // values in flight
          const float* in = parts + (size_t)rank * 2 * O::kPart;
          auto fetch = [&](int p, int j, float(&x)[kAt]) {
            const float* of = in + ((size_t)p * C::kCtas * 2 + (p == c0 ? 1 : 0)) * O::kPart + j * O::kEpiThreads;
#pragma unroll
            for (int i = 0; i < kAt; ++i) x[i] = __ldcg(of + i * O::kEpiThreads);
          };
#pragma unroll
          for (int j = 0; j < kSums; j += kAt) {
            float x[kAt];
            fetch(c0, j, x);
#pragma unroll
            for (int i = 0; i < kAt; ++i) sum[j + i] = x[i];
            for (int p = c0 + 1; p <= c1; ++p) {
              fetch(p, j, x);
#pragma unroll
              for (int i = 0; i < kAt; ++i) sum[j + i] += x[i];
            }
          }
        }
      }
      const bool bf16 = a.out_dtype == UP_EK_BF16;
      if (!write) {
      } else if constexpr (C::kWide) {
        const int token = (int)rank * 128 + row, col0 = w.tb * C::kWeights + kSums * part;
        if (token < w.n) {
          const int64_t at = (int64_t)(w.m0 + token) * a.out_stride + col0;
          if (a.out_dtype == UP_EK_F32) {
            float* to = static_cast<float*>(a.out) + at;
#pragma unroll
            for (int j = 0; j < kSums; j += 8) {
              if (a.wide_out && col0 + j + 8 <= a.n) {
                uint32_t r[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) r[i] = __float_as_uint(sum[j + i]);
                store32(to + j, r);
              } else {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                  if (col0 + j + i < a.n) to[j + i] = sum[j + i];
              }
            }
          } else {
            uint16_t* to = static_cast<uint16_t*>(a.out) + at;
#pragma unroll
            for (int j = 0; j < kSums; j += 16) {
              uint32_t r[8];
#pragma unroll
              for (int i = 0; i < 8; ++i) r[i] = half_pair(sum[j + 2 * i], sum[j + 2 * i + 1], bf16);
              if (a.wide_out && col0 + j + 16 <= a.n) {
                store32(to + j, r);
              } else {
#pragma unroll
                for (int i = 0; i < 16; ++i)
                  if (col0 + j + i < a.n) to[j + i] = (uint16_t)(r[i >> 1] >> (16 * (i & 1)));
              }
            }
          }
        }
      } else {
        const int col = w.tb * C::kWeights + row, n = w.n - kSums * part;
        if (col < a.n) {
          const int64_t at = (int64_t)(w.m0 + kSums * part) * a.out_stride + col;
          if (a.out_dtype == UP_EK_F32) {
            float* to = static_cast<float*>(a.out) + at;
#pragma unroll
            for (int j = 0; j < kSums; ++j, to += a.out_stride)
              if (j < n) *to = sum[j];
          } else {
            uint16_t* to = static_cast<uint16_t*>(a.out) + at;
#pragma unroll
            for (int j = 0; j < kSums; ++j, to += a.out_stride)
              if (j < n) *to = half_bits(sum[j], bf16);
          }
        }
      }
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&run_empty[at.at]);
    }
    if (!good) give_up();
  }

  tc::fence_before_sync();
  __syncthreads();
  if (PAIR) cluster_sync();  // neither leaves while the other's MMAs or arrivals may still reach it
  tc::fence_after_sync();
  if (warp == 1) tmem_free<PAIR>(tmem);
}

template <typename C>
__global__ void __launch_bounds__(Of<C>::kThreads, 1)
    matmul_kernel(const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap xmap,
                  const __grid_constant__ CUtensorMap xmap_full, const __grid_constant__ Args a) {
  matmul<C>(wmap, xmap, xmap_full, a);
}
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(Of<Wide<2>>::kThreads, 1)
    matmul_pair_kernel(const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap xmap,
                       const __grid_constant__ CUtensorMap xmap_full, const __grid_constant__ Args a) {
  matmul<Wide<2>>(wmap, xmap, xmap_full, a);
}

// ---- host side ----
// One CTA an SM.
static int cta_count() { return sm_count() < kMaxCtas ? sm_count() : kMaxCtas; }

enum Form { kNarrow32, kNarrow64, kWide, kPair };

// The form that takes the least time by a model of what was measured: a fixed part (launch, first loads, joining of parts) and so many
// microseconds a block of an owner's tile, fitted to calls of 1 to 2048 rows by 1024 x 8192 to 28672 x 8192 weights. Measured, us,
// Narrow<32>, Narrow<64>, Wide<1>, Wide<2>: by 8192 x 8192 weights 1 row 21, 23, 28, 37; 64 rows 27, 24, 29, 37; 128 rows 40, 31, 29, 37; 256
// rows 72, 47, 40, 39; 2048 rows 501, 281, 151, 143. 128 experts of 4096 x 2048: 512 rows 162, 181, 171, 266; 8192 rows 439, 316, 213, 333;
// 65536 rows 2327, 1685, 749, 784.
static Form form_of(int64_t m, int64_t experts, int64_t n, int64_t kb) {
  struct Cost {
    int tokens, weights, ctas;  // of a tile
    double fixed, block;
  };
  static const Cost cost[4] = {{32, 128, 1, 10.5, 0.275}, {64, 128, 1, 13, 0.30}, {128, 256, 1, 20, 0.59}, {256, 256, 2, 20, 0.56}};
  const double used = (double)(m < experts ? m : experts), per = m / used;  // experts that have rows, at most; rows of each
  int best = 0;
  double least = 0;
  for (int i = 0; i < 4; ++i) {
    const Cost& c = cost[i];
    // a ragged group's last tile is half full in the mean
    const double tiles = experts == 1 ? (double)((m + c.tokens - 1) / c.tokens) : per / c.tokens + 0.5 > 1 ? per / c.tokens + 0.5 : 1;
    const double us = c.fixed + c.block * tiles * used * (double)((n + c.weights - 1) / c.weights) * (double)kb * c.ctas / cta_count();
    if (i == 0 || us < least) best = i, least = us;
  }
  return (Form)best;
}

static PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, []() {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  });
  return fn;
}


// A tensor map of e4m3 rows in boxes of 128 bytes of k by `rows`; what lies outside reads 0.
static bool encode(CUtensorMap* map, const void* at, int dims, int64_t k, int64_t n, int64_t experts, int64_t stride, int rows) {
  const cuuint64_t size[3] = {(cuuint64_t)k, (cuuint64_t)n, (cuuint64_t)experts};
  const cuuint64_t strides[2] = {(cuuint64_t)stride, (cuuint64_t)(n * stride)};
  const cuuint32_t box[3] = {kBlock, (cuuint32_t)rows, 1}, one[3] = {1, 1, 1};
  return encode_fn()(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, dims, const_cast<void*>(at), size, strides, box, one,
                     CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

struct Operands {
  const uint8_t *x, *w;
  int64_t m, x_stride, experts, n, k;
};

template <typename C, typename K>
static int launch(K kernel, unsigned grid, Args& a, const Operands& o, cudaStream_t s) {
  a.groups = (a.kb + C::kGroup - 1) / C::kGroup;
  a.by_groups = Divide32(a.groups), a.by_owners = Divide32(grid / C::kCtas);
  a.tb = (a.nb + C::kWeights / kBlock - 1) / (C::kWeights / kBlock);
  CUtensorMap wmap, xmap, xmap_full;
  if (!encode(&wmap, o.w, 3, o.k, o.n, o.experts, o.k, kBlock) || !encode(&xmap, o.x, 2, o.k, o.m, 1, o.x_stride, kBox) ||
      !encode(&xmap_full, o.x, 2, o.k, o.m, 1, o.x_stride, C::kTokens / C::kCtas))
    return fail_with(UP_ERR_CUDA, "cuTensorMapEncodeTiled refused an operand's tensor map");
  const cudaError_t e = ensure_smem_attr((const void*)kernel, Of<C>::kSmem);
  if (e != cudaSuccess) return cuda_status(e);
  const cudaError_t l = launch_early(kernel, grid, Of<C>::kThreads, Of<C>::kSmem, s, wmap, xmap, xmap_full, a);
  if (l != cudaSuccess) return cuda_status(l);
  note_launch();
  return check_launch();
}

}  // namespace f8
}  // namespace up

using namespace up;
using namespace up::f8;

extern "C" size_t up_sm100_f8_matmul_workspace_bytes(int64_t m, int64_t experts, int64_t n, int64_t k) {
  if (m <= 0 || experts <= 0 || n <= 0 || k <= 0) return UP_F8_COUNTER_BYTES;
  return UP_F8_COUNTER_BYTES + (size_t)cta_count() * 2 * Of<Wide<1>>::kPart * sizeof(float);
}

extern "C" int up_sm100_f8_matmul(const uint8_t* x, int64_t m, int64_t x_stride, const float* x_scale, int64_t xs_stride_m,
                                  int64_t xs_stride_b, const uint8_t* w, const float* w_scale, int64_t experts, int64_t n,
                                  int64_t k, const int32_t* offsets, void* out, int out_dtype, int64_t out_stride,
                                  void* workspace, size_t workspace_bytes, void* stream) {
  UP_CHECK_ARG(m >= 0 && x_stride >= 0 && xs_stride_m >= 0 && xs_stride_b >= 0 && experts >= 1 && n >= 0 && k >= 0);
  UP_CHECK_ARG(out_stride >= 0 && (offsets != nullptr || experts == 1));
  if (out_dtype != UP_EK_F32 && out_dtype != UP_EK_F16 && out_dtype != UP_EK_BF16) return UP_ERR_UNSUPPORTED;
  if (k == 0 || k % 16 != 0 || experts > kMaxExperts) return UP_ERR_UNSUPPORTED;
  if (m == 0 || n == 0) return UP_OK;
  UP_CHECK_ARG(x && x_scale && w && w_scale && out && workspace);
  UP_CHECK_ARG(m <= 1 || (x_stride >= k && out_stride >= n));
  if (m == 1) x_stride = (k + 15) / 16 * 16, out_stride = 0;
  if (!aligned(x, 16) || !aligned(w, 16) || x_stride % 16 != 0) return UP_ERR_UNSUPPORTED;
  const int64_t nb = (n + kBlock - 1) / kBlock, kb = (k + kBlock - 1) / kBlock;
  if (m > 0x3fffffff || n > 0x3fffffff || k > 0x3fffffff || x_stride >= ((int64_t)1 << 40) || n * k >= ((int64_t)1 << 40) ||
      nb > 0x7fffffff / (m / 32 + experts + 1))
    return UP_ERR_UNSUPPORTED;
  UP_CHECK_ARG(aligned(workspace, 256) && workspace_bytes >= up_sm100_f8_matmul_workspace_bytes(m, experts, n, k));
  if (encode_fn() == nullptr) return fail_with(UP_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
  const Operands o{x, w, m, x_stride, experts, n, k};
  Args a{};
  a.xs = x_scale, a.ws = w_scale, a.xs_m = xs_stride_m, a.xs_b = xs_stride_b, a.m = m, a.experts = (int)experts, a.n = (int)n;
  a.kb = (int)kb, a.nb = (int)nb, a.offsets = offsets, a.out = out, a.out_stride = out_stride;
  a.out_dtype = out_dtype, a.wide_out = out_stride % (out_dtype == UP_EK_F32 ? 8 : 16) == 0 && aligned(out, 32), a.header = static_cast<Header*>(workspace);
  a.counters = reinterpret_cast<uint32_t*>(static_cast<char*>(workspace) + sizeof(Header));
  a.partials = reinterpret_cast<float*>(static_cast<char*>(workspace) + UP_F8_COUNTER_BYTES);
  a.wait_ns = wait_limit_ns();
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (form_of(m, experts, n, kb)) {
    case kPair: return launch<Wide<2>>(matmul_pair_kernel, (unsigned)(cta_count() & ~1), a, o, s);
    case kWide: return launch<Wide<1>>(matmul_kernel<Wide<1>>, (unsigned)cta_count(), a, o, s);
    case kNarrow64: return launch<Narrow<64>>(matmul_kernel<Narrow<64>>, (unsigned)cta_count(), a, o, s);
    default: return launch<Narrow<32>>(matmul_kernel<Narrow<32>>, (unsigned)cta_count(), a, o, s);
  }
}

namespace up {
size_t f8_matmul_smem_bytes() {  // for the kernel interface: the largest form's
  size_t most = 0;
  for (const size_t n : {(size_t)Of<Narrow<32>>::kSmem, (size_t)Of<Narrow<64>>::kSmem, (size_t)Of<Wide<1>>::kSmem, (size_t)Of<Wide<2>>::kSmem})
    most = n > most ? n : most;
  return most;
}
}  // namespace up

UP_DEFINE_REVISION(f8_matmul)
