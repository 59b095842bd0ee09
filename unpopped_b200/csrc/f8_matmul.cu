// f8_matmul.cu — products of e4m3 activations and weights with an f32 scale for each block of 128, dense or by expert.
//
//   out[m][j] = sum_b xs[m][b] ws[j / 128][b] (sum_{k in b} x[m][k] w[j][k])
//
// The scales change every 128 k and are not powers of two, so no accumulator can run over a row: each block's product is a
// tcgen05.mma of its own into tensor memory (four steps of 32 k, f32), and the epilogue warps add it, times its two scales,
// to f32 sums in registers while the next blocks are multiplied.
//
// Two kinds, by which operand takes the MMA's rows:
//  * Narrow, for few tokens: 128 weight rows, up to 32 tokens as columns. Bound by HBM: every weight once. Columns are dealt in steps of 16,
//    so a group of one token costs little, and four blocks share an accumulator slot, so that handing it to the epilogue costs once
//    for all four. A thread of the epilogue has one weight row; the tokens' scales come to it through shared memory.
//  * Wide: 128 tokens as rows (256 of two CTAs, tcgen05's cta_group::2), 256 or 128 weight rows as columns. A thread of the epilogue has one
//    token, so a block's scales are one factor for all of its columns. (With tokens as columns every thread needs every token's
//    factor: at 128 bytes a cycle shared memory gives those of 128 x 128 values in 512 cycles, in which the MMA takes 256.) Bound by
//    the two accumulators' round: an MMA of 512 cycles, its commit, the epilogue's loads and 128 sums a thread, the arrival that frees it.
// Measured: 1 row by 8192 x 8192 weights 16.3 us (4.1 TB/s of weights), by 28672 x 8192 42 (5.6 TB/s); 512 rows of 128 experts by 4096 x 2048
// 150 (958 MB of weights: 6.4 TB/s). Where calls follow one another for seconds and the clock falls to the power limit, 8192 rows by
// 8192 x 8192 take 583 us (1.89 PFLOP/s; 513 alone), 65536 rows of 128 experts by 4096 x 2048 853 (1.29 PFLOP/s; 729 alone).
// The operator's other sources, which its revision hash covers through this line (build.py --sources):
// FNV-1a 64 of divide.cuh, f8_walk.cuh, launch.cuh: 45adde3f9cc64f52
#include "common.cuh"
#include "f8_walk.cuh"
#include "launch.cuh"
#include "tc.cuh"

#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <mutex>
#include <type_traits>

namespace up {
namespace f8 {

constexpr int kBox = 16;                  // tokens of a small TMA box
constexpr int kMaxExperts = 1024;
constexpr int kRuns = 4;                  // runs of blocks that the roles may be apart
constexpr uint64_t kSettleNs = 10000000;  // loads land in some microseconds
constexpr int kMaxCtas = (UP_F8_COUNTER_BYTES - 64) / 4;  // a counter each

// What follows from a form (f8_walk.cuh).
template <typename C>
struct Of {
  static constexpr int kStage = kTile + C::kBBytes;
  static constexpr int kDSlot = C::kDBlock * C::kGroup, kDRing = 512 / kDSlot;  // accumulators in tensor memory
  static constexpr int kEpiThreads = 32 * C::kEpiWarps, kThreads = 32 * C::kEpi0 + kEpiThreads;
  // factors in shared memory, four blocks a slot, twice (Scales), and whether the second are there
  static constexpr int kScRing = C::kFactors > 0 ? 4 : 0, kScSlot = 8 * C::kFactors + 4;
  static constexpr int kStaged = C::kWide ? 32 * 17 : 0;             // values a warp, for rows of `out` that do not begin on 32 bytes
  static constexpr size_t kPart = (size_t)C::kSums * kEpiThreads;  // values of a CTA's part of a tile
  // One thread issues the MMAs and commits of a block in some 450 cycles, so two take the blocks in turn; the ring's even
  // depth then gives each stage to one of them, which sees all of its phases.
  static constexpr int kIssuers = 2;
  static constexpr int kBars = 2 * C::kStages + 2 * kDRing + 2 * kScRing + 3 * kRuns + 3;
  static constexpr int kSmem = 1024 + C::kStages * kStage + kScRing * kScSlot * 4 + kRuns * 48 + kBars * 8 + 16 + (kMaxExperts + 1) * 2 * 4 +
                               C::kEpiWarps * kStaged * 4;
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
  int panel_rows;                         // of an expert: more go by panels
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
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, const Args& a, volatile int* abort) {
  for (int it = 0; it < 64; ++it)
    if (tc::mbar_try_wait(bar, parity)) return true;
  const uint64_t t0 = globaltimer_ns();
  for (uint32_t it = 1;; ++it) {
    if (tc::mbar_try_wait(bar, parity)) return true;
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

// 32 consecutive columns of this thread's lane of tensor memory. The registers hold them after wait_loads; what uses them is
// volatile too, so nothing moves it before the wait.
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
__device__ __forceinline__ void mul_after(uint32_t& v, float f) {
  float r;
  asm volatile("mul.rn.f32 %0, %1, %2;" : "=f"(r) : "f"(__uint_as_float(v)), "f"(f));
  v = __float_as_uint(r);
}
// Whether the product of two scales is no normal number (0 included). Then v * x * w goes by both, the larger first, as it may be an ordinary number
// all the same: where x * w is too small, v * (the larger) is not too large, and where it is and x * w is as well, the result is.
__device__ __forceinline__ bool out_of_range(float product) { return (__float_as_uint(product) << 1) - 0x01000000u >= 0xfe000000u; }
struct Scales {
  float first, then;
  __device__ __forceinline__ Scales(float x, float w) : first(1.f), then(x * w) {
    if (out_of_range(then) && x != 0.f && w != 0.f) {
      const bool larger = fabsf(x) > fabsf(w);
      first = larger ? x : w, then = larger ? w : x;
    }
  }
};
__device__ __forceinline__ float shared1(uint32_t at) {
  float f;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(f) : "r"(at));
  return f;
}
__device__ __forceinline__ float4 shared4(uint32_t at) {
  float4 f;
  asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(f.x), "=f"(f.y), "=f"(f.z), "=f"(f.w) : "r"(at));
  return f;
}

// The schedule: begin[e] (rows) and start[e] (tiles) of every expert, from the offsets on the device, which all threads have put into
// `begin` held to [0, m]; each entry is held to its predecessors. One warp, a lane with some experts that follow one another: one scan
// of the lanes for the rows and one for the tiles.
template <typename C>
__device__ __forceinline__ void schedule(const Args& a, int* start, int* begin, int lane) {
  constexpr int kTokens = C::kTokens;
  const int each = (a.experts + 32) / 32, e0 = min(lane * each, a.experts + 1), e1 = min(e0 + each, a.experts + 1);
  int most = 0;
  for (int e = e0; e < e1; ++e) most = max(most, begin[e]);
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, most, o);
    if (lane >= o) most = max(most, v);
  }
  int row = __shfl_up_sync(0xffffffffu, most, 1);  // where the expert before this lane's first entry begins
  if (lane == 0) row = 0;
  int tiles = 0;
  for (int e = e0; e < e1; ++e) {
    const int before = row;
    row = max(row, begin[e]);
    // tiles of expert e - 1, which ends where e begins
    if (e > 0) tiles += (row - before + kTokens - 1) / kTokens * a.tb;
    begin[e] = row, start[e] = tiles;
  }
  int all = tiles;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, all, o);
    if (lane >= o) all += v;
  }
  for (int e = e0; e < e1; ++e) start[e] += all - tiles;
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
  constexpr int kGroup = C::kGroup, kStages = C::kStages, kDRing = O::kDRing, kScRing = O::kScRing, kSums = C::kSums;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* stages = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* sc = reinterpret_cast<float*>(stages + kStages * O::kStage);  // [kScRing][4 blocks][kFactors]
  uint64_t* full = reinterpret_cast<uint64_t*>(sc + kScRing * O::kScSlot);
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
  static_assert((kStages * O::kStage + kScRing * O::kScSlot * 4 + O::kBars * 8) % 8 == 0, "alignment");
  Run* runs = reinterpret_cast<Run*>(run_owners + kRuns);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(runs + kRuns);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile uint32_t* verdict = tmem_slot + 2;
  int* start = reinterpret_cast<int*>(tmem_slot + 4);
  int* begin = start + kMaxExperts + 1;
  float* staged = reinterpret_cast<float*>(begin + kMaxExperts + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = PAIR ? cta_rank() : 0;
  if (warp == 0) {
    if (lane == 0) {
      for (int s = 0; s < kStages; ++s) tc::mbar_init(&full[s], 1), tc::mbar_init(&empty[s], 1);
      for (int d = 0; d < kDRing; ++d) tc::mbar_init(&d_full[d], kGroup > 1 ? O::kIssuers : 1), tc::mbar_init(&d_empty[d], C::kEpiWarps * C::kCtas);
      for (int q = 0; q < kScRing; ++q) tc::mbar_init(&sc_full[q], 1), tc::mbar_init(&sc_empty[q], C::kEpiWarps);
      // readers of the runs: the factors, the issuers (a pair's are the first CTA's), the tokens' loads, the epilogue's warps
      for (int i = 0; i < kRuns; ++i)
        tc::mbar_init(&run_full[i], 1), tc::mbar_init(&run_owners[i], 1),
            tc::mbar_init(&run_empty[i], (C::kFactors > 0 ? 1 : 0) + (rank == 0 ? O::kIssuers : 0) + (C::kWide ? 0 : 1) + C::kEpiWarps);
      tc::mbar_init(seg_in, C::kEpiWarps), tc::mbar_init(seg_out, 1), tc::mbar_init(drain, O::kIssuers);
      *abort_flag = 0;
      tc::mbar_fence_init();
      tc::tma_prefetch_desc(&wmap), tc::tma_prefetch_desc(&xmap), tc::tma_prefetch_desc(&xmap_full);
    }
  } else if (warp == 1) {
    tmem_alloc<PAIR>(tmem_slot);
  }
  // Without offsets nothing of the launch before is read until after the first runs are dealt out. No wait with a limit begins before its end.
  if (a.offsets) {
    after_previous();
    for (int e = threadIdx.x; e <= a.experts; e += O::kThreads) begin[e] = (int)min((int64_t)max(a.offsets[e], 0), a.m);
    __syncthreads();
    if (warp == 2) schedule<C>(a, start, begin, lane);
  } else if (threadIdx.x == 64) {  // one matrix and all rows
    start[0] = begin[0] = 0, begin[1] = (int)a.m;
    start[1] = (int)((a.m + C::kTokens - 1) / C::kTokens) * a.tb;
  }
  let_next_begin();
  tc::fence_before_sync();
  __syncthreads();
  if (PAIR) cluster_sync();
  tc::fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  if (a.offsets == nullptr && warp > 0) after_previous();

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
    if (C::kSums > 64) asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");  // 56 x 128 + 224 x 256 threads: what 168 each are
    if (warp == 0) {
      // ---------------- runs, and the loads of weights (Wide: of tokens too) ----------------
      if (lane == 0) {
        Walk<C> walk(a, start, begin, blockIdx.x / C::kCtas, gridDim.x / C::kCtas);
        int64_t issued = 0;
        int s = 0;
        uint32_t ph = 1;
        const uint32_t full0 = PAIR ? in_leader(full) : tc::smem_u32(full);  // a pair's loads all count on the leader's barriers
        bool good = true;
        Runs at;
        for (bool more = true; more && good; at.next()) {
          more = walk.next();  // the run without groups is handed over too
          good = wait(&run_empty[at.at], at.phase ^ 1u, a, abort_flag);
          if (!good) break;
          const Run w = walk.r;
          runs[at.at] = w;
          tc::mbar_arrive(&run_full[at.at]);
          walk.passed();
          if (issued == 0 && a.offsets == nullptr) after_previous();
          const int boxes = (w.n + kBox - 1) / kBox;
          const uint32_t bytes = C::kWide ? C::kCtas * O::kStage : kTile + boxes * (kBox * kBlock);
          const int row = w.tb * C::kWeights + (int)rank * (C::kWeights / C::kCtas);
          for (int kb = w.g0 * kGroup, end = min(a.kb, w.g1 * kGroup); kb < end; ++kb) {
            good = wait(&empty[s], ph, a, abort_flag);
            if (!good) break;
            uint8_t* to = stages + (size_t)s * O::kStage + (C::kWide ? kTile : 0);
            const uint32_t bar = full0 + 8 * s;
            if (rank == 0) tc::mbar_arrive_expect_tx(&full[s], bytes);
            load_w<PAIR>(to, &wmap, bar, kb * kBlock, row, w.e);
            if (C::kWeights / C::kCtas > 128) load_w<PAIR>(to + kTile, &wmap, bar, kb * kBlock, row + 128, w.e);
            if (C::kWide) load_x<PAIR>(to - kTile, &xmap_full, bar, kb * kBlock, w.m0 + (int)rank * 128);
            ++issued;
            if (++s == kStages) s = 0, ph ^= 1u;
          }
          // who shares the tile is needed last
          if (w.g0 > 0 || w.g1 < a.groups) {
            runs[at.at].c0 = walk.owner_of(w.t * a.groups);
            runs[at.at].c1 = walk.owner_of(w.t * a.groups + a.groups - 1);
          }
          tc::mbar_arrive(&run_owners[at.at]);
        }
        // every load lands before shared memory is released; where a role gave up, its loads' barriers may never complete (see the end)
        if (rank == 0 && good)
          for (int64_t j = issued > kStages ? issued - kStages : 0; j < issued && good; ++j)
            good = wait(&full[j % kStages], (uint32_t)((j / kStages) & 1), a, abort_flag);
        if (!good) give_up();
      }
    } else if (!C::kWide && warp == C::kXWarp) {
      // ---------------- the loads of tokens: on the same barriers, which the weights' loads give the bytes of both ----------------
      if (lane == 0) {
        int s = 0;
        uint32_t ph = 1;
        const uint32_t full0 = tc::smem_u32(full);
        bool good = true;
        for (Runs at; take(at, good); at.next()) {
          const Run w = runs[at.at];
          tc::mbar_arrive(&run_empty[at.at]);
          const int boxes = (w.n + kBox - 1) / kBox;
          for (int kb = w.g0 * kGroup, end = min(a.kb, w.g1 * kGroup); kb < end; ++kb) {
            good = wait(&empty[s], ph, a, abort_flag);
            if (!good) break;
            uint8_t* to = stages + (size_t)s * O::kStage + kTile;
            const uint32_t bar = full0 + 8 * s;
            if (boxes * kBox == C::kTokens)
              load_x<PAIR>(to, &xmap_full, bar, kb * kBlock, w.m0);
            else
              for (int b = 0; b < boxes; ++b) load_x<PAIR>(to + b * (kBox * kBlock), &xmap, bar, kb * kBlock, w.m0 + b * kBox);
            if (++s == kStages) s = 0, ph ^= 1u;
          }
        }
        if (!good) give_up();
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
          const uint32_t id = C::kWide ? idesc_f8(128 * C::kCtas, C::kWeights) : idesc_f8(128, (w.n + 15) / 16 * 16);
          const int end = min(a.kb, w.g1 * kGroup);
          for (int kb = w.g0 * kGroup; kb < end && good; kb += kGroup) {
            if (kGroup > 1) good = wait(&d_empty[d], dph, a, abort_flag);
#pragma unroll 1
            for (int j = 0; j < kGroup && kb + j < end && good; ++j, mine = !mine) {
              if (mine) {
                // the operands first: they are there before the slot is free, which the next block's time hangs on
                good = wait(&full[s], ph, a, abort_flag);
                if (!good) break;
                const uint32_t stage = tc::smem_u32(stages) + s * O::kStage;
                const uint64_t ad = tc::sdesc_kmajor_sw128(stage), bd = tc::sdesc_kmajor_sw128(stage + kTile);
                if (kGroup == 1) good = wait(&d_empty[d], dph, a, abort_flag);
                if (!good) break;
                tc::fence_after_sync();
#pragma unroll
                for (int i = 0; i < kBlock / 32; ++i) mma_f8<PAIR>(tmem + d * O::kDSlot + j * C::kDBlock, ad + 2 * i, bd + 2 * i, id, i > 0);
                if (kGroup == 1) commit<PAIR>(&d_full[d]);
                commit<PAIR>(&empty[s]);
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
    } else if (warp == 2) {
      if constexpr (C::kFactors > 0) {
        // ---------------- factors: x's scales times the weights', four blocks of a run at a time, the next four's loads on their way ----------------
        constexpr int kEach = C::kFactors / 32;
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
          good = __all_sync(0xffffffffu, wait(&sc_empty[q], ph, a, abort_flag));
          if (!good) return;
          float* slot = sc + q * O::kScSlot + lane;
          bool odd = false;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float f = __shfl_sync(0xffffffffu, ws[h], j);
#pragma unroll
            for (int c = 0; c < kEach; ++c)
              if (c * 32 < n[h]) {
                const float by = xs[h][j][c] * f;
                slot[j * C::kFactors + c * 32] = by;
                odd = odd || (out_of_range(by) && xs[h][j][c] != 0.f);
              }
          }
          odd = __any_sync(0xffffffffu, odd);
          if (odd) {
#pragma unroll 1
            for (int j = 0; j < 4; ++j) {
              const float f = __shfl_sync(0xffffffffu, ws[h], j);
#pragma unroll
              for (int c = 0; c < kEach; ++c) {
                const Scales two(j == 0 ? xs[h][0][c] : j == 1 ? xs[h][1][c] : j == 2 ? xs[h][2][c] : xs[h][3][c], f);
                slot[j * C::kFactors + c * 32] = two.then, slot[(4 + j) * C::kFactors + c * 32] = two.first;
              }
            }
          }
          if (lane == 0) slot[8 * C::kFactors] = odd ? 1.f : 0.f;
          __syncwarp();
          if (lane == 0) tc::mbar_arrive(&sc_full[q]);
          if (++q == kScRing) q = 0, ph ^= 1u;
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
      }
    }
  } else {
    // ---------------- sums: lanes 32 (warp % 4) .. of tensor memory ----------------
    if (C::kSums > 64) asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
    const int quarter = warp & 3, part = (warp - C::kEpi0) >> 2, thread = threadIdx.x - 32 * C::kEpi0, row = quarter * 32 + lane;
    const uint32_t d_empty0 = PAIR ? in_leader(d_empty) : 0;
    const uint32_t from = tmem + ((uint32_t)(quarter * 32) << 16) + kSums * part;
    float sum[kSums];
    uint32_t v[2][32];
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
        // The thread's row is a token, its columns weight rows with one scale, so a block has one factor for it. A token behind the group's last one
        // goes by the last one's scale, a block of weights behind the last by the last's; neither is written.
        const int nb = min(w.tb * (C::kWeights / kBlock) + part * kSums / kBlock, a.nb - 1), m = w.m0 + min((int)rank * 128 + row, w.n - 1);
        const float* xs = a.xs + m * a.xs_m + first * a.xs_b;
        const float* ws = a.ws + ((int64_t)w.e * a.nb + nb) * a.kb + first;
        float xs_next[2], ws_next[2];  // two blocks' scales on their way
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          xs_next[j] = first + j < end ? xs[j * a.xs_b] : 0.f;
          ws_next[j] = first + j < end ? ws[j] : 0.f;
        }
        accumulators();
        if (!good) break;
        // Two sets of 32 columns at a time, whose successors' loads run beside the sums. A slot is free as soon as its last loads are
        // done: a later block's MMA waits for that. `odd`: the accumulators times g first (Scales).
        load32(from + d * O::kDSlot, v[0]);
        load32(from + d * O::kDSlot + 32, v[1]);
        auto block = [&](int kb, auto odd, float f, float g) {
          const uint32_t in = from + d * O::kDSlot;
#pragma unroll
          for (int c = 0; c < kSums; c += 64) {
            const bool last = c + 64 == kSums;
            wait_loads();
            if (last) free_accumulators();
            if constexpr (odd.value) {
#pragma unroll
              for (int j = 0; j < 32; ++j) mul_after(v[0][j], g), mul_after(v[1][j], g);
            }
#pragma unroll
            for (int j = 0; j < 32; ++j) fma_after(sum[c + j], v[0][j], f);
            if (!last) {
              load32(in + c + 64, v[0]);
            } else if (kb + 1 < end) {
              accumulators();
              if (!good) return;
              load32(from + d * O::kDSlot, v[0]);
            }
#pragma unroll
            for (int j = 0; j < 32; ++j) fma_after(sum[c + 32 + j], v[1][j], f);
            if (!last)
              load32(in + c + 96, v[1]);
            else if (kb + 1 < end)
              load32(from + d * O::kDSlot + 32, v[1]);
          }
        };
        float x_new, w_new;
        auto fetch = [&](int kb) {
          x_new = 0.f, w_new = 0.f;
          if (kb + 2 < end) x_new = xs[2 * a.xs_b], w_new = ws[2];
          xs += a.xs_b, ++ws;
        };
        auto move_up = [&]() { xs_next[0] = xs_next[1], ws_next[0] = ws_next[1], xs_next[1] = x_new, ws_next[1] = w_new; };
        auto any_odd = [&](int j, float f) { return __any_sync(0xffffffffu, out_of_range(f) && xs_next[j] != 0.f && ws_next[j] != 0.f) != 0; };
        // From the first block on where a row's scales leave f32's range, the run goes on in a loop of its own. The vote is on the block after, beside
        // the wait for tensor memory: 8192 rows by 8192 x 8192 weights 503 us without any, 511 so, 514 to 542 with the vote or a branch in
        // each block's own way.
        int kb = first;
        float f = xs_next[0] * ws_next[0];
        for (bool odd = any_odd(0, f); kb < end && !odd; ++kb) {
          fetch(kb);
          const float f_next = xs_next[1] * ws_next[1];
          odd = any_odd(1, f_next);
          block(kb, std::false_type(), f, 1.f);
          if (!good) break;
          move_up();
          f = f_next;
        }
        if (good)
#pragma unroll 1
          for (; kb < end; ++kb) {
            const Scales two(xs_next[0], ws_next[0]);
            fetch(kb);
            block(kb, std::true_type(), two.then, two.first);
            if (!good) break;
            move_up();
          }
      } else {
        // The thread's row is a weight row, its columns the tokens, each with a factor of its own.
        for (int kb = first; kb < end; kb += kGroup) {
          accumulators();
          if (!good) break;
          good = __all_sync(0xffffffffu, wait(&sc_full[q], qph, a, abort_flag));
          if (!good) break;
          const uint32_t f = tc::smem_u32(sc + q * O::kScSlot + kSums * part);
          const float flag = shared1(f + 8 * C::kFactors * 4);
          const uint32_t in = from + d * O::kDSlot;
          auto blocks = [&](auto odd) {
            auto add = [&](int j, uint32_t(&x)[32]) {  // block j's
#pragma unroll
              for (int i = 0; i < 32; i += 4) {
                if constexpr (odd.value) {
                  const float4 g4 = shared4(f + ((4 + j) * C::kFactors + i) * 4);
                  mul_after(x[i], g4.x), mul_after(x[i + 1], g4.y), mul_after(x[i + 2], g4.z), mul_after(x[i + 3], g4.w);
                }
                const float4 f4 = shared4(f + (j * C::kFactors + i) * 4);
                fma_after(sum[i], x[i], f4.x), fma_after(sum[i + 1], x[i + 1], f4.y);
                fma_after(sum[i + 2], x[i + 2], f4.z), fma_after(sum[i + 3], x[i + 3], f4.w);
              }
            };
#pragma unroll
            for (int j = 0; j < kGroup; j += 2) {
              if (kb + j >= end) break;
              load32(in + j * C::kDBlock, v[0]);
              if (kb + j + 1 < end) load32(in + (j + 1) * C::kDBlock, v[1]);
              wait_loads();
              add(j, v[0]);
              if (kb + j + 1 < end) add(j + 1, v[1]);
            }
          };
          if (__builtin_expect(flag != 0.f, 0))
            blocks(std::true_type());
          else
            blocks(std::false_type());
          free_accumulators();
          if (lane == 0) tc::mbar_arrive(&sc_empty[q]);  // free_accumulators synchronised the warp
          if (++q == kScRing) q = 0, qph ^= 1u;
        }
      }
      if (!good) break;

      bool write = true;
      if (w.g0 > 0 || w.g1 < a.groups) {
        // A part of a tile: published, and whichever owner comes last adds the parts in the order of the owners, its own among them, so that
        // the sums do not depend on who that is.
        good = __all_sync(0xffffffffu, wait(&run_owners[at.at], at.phase, a, abort_flag));
        if (!good) break;
        const int c0 = w.c0, c1 = w.c1, owner = blockIdx.x / C::kCtas;
        float* parts = a.partials + thread;
        float* to = parts + ((size_t)blockIdx.x * 2 + (c0 == owner ? 1 : 0)) * O::kPart;
#pragma unroll
        for (int j = 0; j < kSums; ++j) {
          if (!C::kWide && j % C::kStep == 0 && j >= w.n) break;  // columns of no token
          __stcg(to + j * O::kEpiThreads, sum[j]);
        }
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
          constexpr int kAt = C::kWide ? 64 : C::kStep;  // values of a part in flight
          const float* in = parts + (size_t)rank * 2 * O::kPart;
          auto fetch = [&](int p, int j, float(&x)[kAt]) {
            const float* of = in + ((size_t)p * C::kCtas * 2 + (p == c0 ? 1 : 0)) * O::kPart + j * O::kEpiThreads;
#pragma unroll
            for (int i = 0; i < kAt; ++i) x[i] = __ldcg(of + i * O::kEpiThreads);
          };
#pragma unroll
          for (int j = 0; j < kSums; j += kAt) {
#pragma unroll
            for (int i = 0; i < kAt; ++i) sum[j + i] = 0.f;
            if constexpr (C::kWide) {
              for (int p = c0; p <= c1; ++p) {
                float x[kAt];
                fetch(p, j, x);
#pragma unroll
                for (int i = 0; i < kAt; ++i) sum[j + i] += x[i];
              }
            } else {
              if (j >= w.n) break;
              float x[2][kAt];  // the next part's are on their way beside a part's sums
              fetch(c0, j, x[0]);
              for (int p = c0; p <= c1; p += 2) {
                if (p + 1 <= c1) fetch(p + 1, j, x[1]);
#pragma unroll
                for (int i = 0; i < kAt; ++i) sum[j + i] += x[0][i];
                if (p + 1 > c1) break;
                if (p + 2 <= c1) fetch(p + 2, j, x[0]);
#pragma unroll
                for (int i = 0; i < kAt; ++i) sum[j + i] += x[1][i];
              }
            }
          }
        }
      }
      const bool bf16 = a.out_dtype == UP_EK_BF16;
      if (!write) {
      } else if constexpr (C::kWide) {
        const int token = (int)rank * 128 + row, col0 = w.tb * C::kWeights + kSums * part;
        if (!a.wide_out || col0 + kSums > a.n) {
          // Stores of single values would each touch 32 rows, so 16 columns at a time go through shared memory and a store is 16
          // neighbours of each of two rows.
          float* own = staged + (warp - C::kEpi0) * O::kStaged;
          const int n = w.n - (token - lane) < 32 ? w.n - (token - lane) : 32;  // the warp's rows
          const int64_t at = (int64_t)(w.m0 + token - lane) * a.out_stride;
#pragma unroll
          for (int c = 0; c < kSums; c += 16) {
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 16; ++i) own[lane * 17 + i] = sum[c + i];
            __syncwarp();
            const int col = col0 + c + (lane & 15);
#pragma unroll 4
            for (int r = lane >> 4; r < n; r += 2) {
              if (col >= a.n) break;
              const float v = own[r * 17 + (lane & 15)];
              const int64_t to = at + r * a.out_stride + col;
              if (a.out_dtype == UP_EK_F32)
                static_cast<float*>(a.out)[to] = v;
              else
                static_cast<uint16_t*>(a.out)[to] = (uint16_t)half_pair(v, 0.f, bf16);
            }
          }
        } else if (token < w.n) {
          const int64_t at = (int64_t)(w.m0 + token) * a.out_stride + col0;
          if (a.out_dtype == UP_EK_F32) {
            float* to = static_cast<float*>(a.out) + at;
#pragma unroll
            for (int j = 0; j < kSums; j += 8) {
              uint32_t r[8];
#pragma unroll
              for (int i = 0; i < 8; ++i) r[i] = __float_as_uint(sum[j + i]);
              store32(to + j, r);
            }
          } else {
            uint16_t* to = static_cast<uint16_t*>(a.out) + at;
#pragma unroll
            for (int j = 0; j < kSums; j += 16) {
              uint32_t r[8];
#pragma unroll
              for (int i = 0; i < 8; ++i) r[i] = half_pair(sum[j + 2 * i], sum[j + 2 * i + 1], bf16);
              store32(to + j, r);
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
            for (int j = 0; j < kSums; ++j, to += a.out_stride) {
              if (j >= n) break;
              *to = sum[j];
            }
          } else {
            uint16_t* to = static_cast<uint16_t*>(a.out) + at;
#pragma unroll
            for (int j = 0; j < kSums; ++j, to += a.out_stride) {
              if (j >= n) break;
              *to = half_bits(sum[j], bf16);
            }
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
  if (*abort_flag) {
    // Some loads were issued whose others were not, so no barrier tells when they have landed: shared memory is kept for a time in which every
    // load of this GPU's memory has.
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < kSettleNs) __nanosleep(1000);
  }
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
template <typename C>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(Of<C>::kThreads, 1)
    matmul_pair_kernel(const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap xmap,
                       const __grid_constant__ CUtensorMap xmap_full, const __grid_constant__ Args a) {
  matmul<C>(wmap, xmap, xmap_full, a);
}

// ---- host side ----
// One CTA an SM.
static int cta_count() { return sm_count() < kMaxCtas ? sm_count() : kMaxCtas; }

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
  if (!encode(&wmap, o.w, 3, o.k, o.n, o.experts, o.k, 128) || !encode(&xmap, o.x, 2, o.k, o.m, 1, o.x_stride, kBox) ||
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
  return UP_F8_COUNTER_BYTES + (size_t)cta_count() * 2 * Of<Wide<1, 256>>::kPart * sizeof(float);
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
  a.panel_rows = (int)(kPanelBytes / (kb * kBlock));
  a.kb = (int)kb, a.nb = (int)nb, a.offsets = offsets, a.out = out, a.out_stride = out_stride;
  a.out_dtype = out_dtype, a.wide_out = out_stride % (out_dtype == UP_EK_F32 ? 8 : 16) == 0 && aligned(out, 32);
  a.header = static_cast<Header*>(workspace);
  a.counters = reinterpret_cast<uint32_t*>(static_cast<char*>(workspace) + sizeof(Header));
  a.partials = reinterpret_cast<float*>(static_cast<char*>(workspace) + UP_F8_COUNTER_BYTES);
  a.wait_ns = wait_limit_ns();
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (form_of(m, experts, n, kb, cta_count())) {
    case kWide256: return launch<Wide<1, 256>>(matmul_kernel<Wide<1, 256>>, (unsigned)cta_count(), a, o, s);
    case kPair256: return launch<Wide<2, 256>>(matmul_pair_kernel<Wide<2, 256>>, (unsigned)(cta_count() & ~1), a, o, s);
    case kWide128: return launch<Wide<1, 128>>(matmul_kernel<Wide<1, 128>>, (unsigned)cta_count(), a, o, s);
    default: return launch<Narrow>(matmul_kernel<Narrow>, (unsigned)cta_count(), a, o, s);
  }
}

namespace up {
size_t f8_matmul_smem_bytes() {  // for the kernel interface: the largest form's
  size_t most = 0;
  for (const size_t n : {(size_t)Of<Narrow>::kSmem, (size_t)Of<Wide<1, 256>>::kSmem, (size_t)Of<Wide<2, 256>>::kSmem, (size_t)Of<Wide<1, 128>>::kSmem})
    most = n > most ? n : most;
  return most;
}
}  // namespace up

UP_DEFINE_REVISION(f8_matmul)
