// f8_matmul.cu — products of e4m3 activations and weights with an f32 scale for each block of 128, dense or by expert.
//
//   out[m][j] = sum_b xs[m][b] ws[j / 128][b] (sum_{k in b} x[m][k] w[j][k])
//
// The scales change every 128 k and are not powers of two, so no accumulator can run over a row: each block's product is a
// tcgen05.mma of its own into tensor memory (four steps of 32 k, f32), and the epilogue warps add it, times its two scales,
// to f32 sums in registers while the next blocks are multiplied.
//
// The weights are the MMA's 128 rows and the tokens its columns: a group of any number of tokens costs columns in steps of 16
// and no padding to 128, and one weight scale serves a whole tile's block.
#include "common.cuh"
#include "tc.cuh"

#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <mutex>

namespace up {
namespace f8 {

constexpr int kBlock = 128;               // k a scale
constexpr int kRows = 128;                // weight rows a tile: the MMA's M
constexpr int kCols = 128;                // tokens a tile: at most, the MMA's N is the tokens there are, in steps of 16
constexpr int kBox = 16;                  // tokens a TMA box
constexpr int kMaxExperts = 1024;
constexpr int kStages = 6;
constexpr int kWBytes = kRows * kBlock, kXBytes = kCols * kBlock, kStage = kWBytes + kXBytes;
constexpr int kDRing = 512 / kCols;       // accumulators in tensor memory
constexpr int kScRing = 8;                // blocks of scales in shared memory
constexpr int kEpiWarps = 8, kEpi0 = 4;   // warps 0 to 3: loads, MMA, scales, tensor memory
constexpr int kThreads = 32 * (kEpi0 + kEpiWarps);
constexpr int kChunks = kCols / 16 / 2;   // 16-column chunks an epilogue warp holds (the two halves take them in turn)
constexpr int kMinUnits = 4;              // blocks of a CTA at least: fewer do not pay for joining the parts
constexpr int kMaxCtas = (UP_F8_COUNTER_BYTES - 64) / 4;  // a counter each

struct Header {
  uint32_t ticket, done, epoch, error;    // `error` at byte 12, as in every workspace
  uint32_t pad[12];
};
static_assert(sizeof(Header) == 64, "header");

struct Args {
  const float *xs, *ws;
  int64_t xs_m, xs_b;
  int64_t m;
  int experts, n, k, kb, nb;
  const int32_t* offsets;
  void* out;
  int64_t out_stride;
  int out_dtype;
  Header* header;
  uint32_t* counters;                     // one a CTA: the parts of the tile that it begins
  float* partials;                        // [CTA][2][kCols][kRows]
  uint64_t wait_ns;
};

constexpr int kSmemSched = (kMaxExperts + 1) * 2 * 4;
constexpr int kSmemBars = 512;
constexpr int kSmem = 1024 + kStages * kStage + kScRing * kCols * 4 + kSmemSched + kSmemBars;
static_assert(kSmem <= 232448, "shared memory");

// A unit is one block of k of one tile; tiles are numbered by expert, then weight rows, then tokens, so the tiles that
// share weights are neighbours. A walk goes from unit to unit.
struct Walk {
  const int *start, *begin;               // first tile, first row of each expert
  int experts, kbs, t, kb;
  int e, nb, m0, n;                       // the tile's expert, block of weight rows, first row and number of tokens
  __device__ __forceinline__ void set() {
    while (t >= start[e + 1]) ++e;
    const int rows = begin[e + 1] - begin[e], wide = (rows + kCols - 1) / kCols, at = t - start[e];
    nb = at / wide;
    const int mt = at - nb * wide;
    m0 = begin[e] + mt * kCols;
    n = min(kCols, rows - mt * kCols);
  }
  __device__ __forceinline__ void init(const int* start_, const int* begin_, int experts_, int kbs_, int64_t u) {
    start = start_, begin = begin_, experts = experts_, kbs = kbs_;
    t = (int)(u / kbs);
    kb = (int)(u - (int64_t)t * kbs);
    int lo = 0, hi = experts - 1;         // the last expert that starts at or before t
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (start[mid] <= t) lo = mid;
      else hi = mid - 1;
    }
    e = lo;
    set();
  }
  // to the next unit; `more`: there is one
  __device__ __forceinline__ void next(bool more) {
    if (++kb == kbs) {
      kb = 0;
      ++t;
      if (more) set();
    }
  }
};

__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* m, uint64_t* bar, int32_t x, int32_t y, int32_t z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
          tc::smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(m)), "r"(tc::smem_u32(bar)), "r"(x), "r"(y), "r"(z)
      : "memory");
}

// D[tmem] (+)= A[smem] * B[smem], e4m3 (or e5m2) inputs, f32 sums.
__device__ __forceinline__ void mma_f8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, {%5, %5, %5, %5}, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(0u)
      : "memory");
}

// Instruction descriptor, kind::f8f6f4: e4m3 A and B (K-major), f32 D.
__device__ __forceinline__ constexpr uint32_t idesc_f8(int m, int n) {
  return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

__device__ __forceinline__ void store_out(const Args& a, int64_t at, float v) {
  if (a.out_dtype == UP_EK_BF16)
    static_cast<__nv_bfloat16*>(a.out)[at] = __float2bfloat16_rn(v);
  else if (a.out_dtype == UP_EK_F16)
    static_cast<__half*>(a.out)[at] = __float2half_rn(v);
  else
    static_cast<float*>(a.out)[at] = v;
}

__device__ __forceinline__ int64_t cta_of_unit(int64_t u, int64_t units, int64_t ctas) {
  int64_t c = (u * ctas) / units;
  while (c + 1 < ctas && ((c + 1) * units) / ctas <= u) ++c;
  while (c > 0 && (c * units) / ctas > u) --c;
  return c;
}

// The schedule: begin[e] (rows) and start[e] (tiles) of every expert, from the offsets on the device; each entry is held to
// [0, m] and to its predecessors. One warp.
__device__ __forceinline__ void schedule(const Args& a, int* start, int* begin, int lane) {
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
    int tiles = e >= 1 && e <= a.experts ? (row - before + kCols - 1) / kCols * a.nb : 0;
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

__global__ void __launch_bounds__(kThreads, 1)
    matmul_kernel(const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap xmap, const Args a) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* stages = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* sc = reinterpret_cast<float*>(stages + kStages * kStage);  // [kScRing][kCols]
  int* start = reinterpret_cast<int*>(sc + kScRing * kCols);
  int* begin = start + kMaxExperts + 1;
  uint64_t* full = reinterpret_cast<uint64_t*>(begin + kMaxExperts + 1);
  uint64_t* empty = full + kStages;
  uint64_t* d_full = empty + kStages;
  uint64_t* d_empty = d_full + kDRing;
  uint64_t* sc_full = d_empty + kDRing;
  uint64_t* sc_empty = sc_full + kScRing;
  uint64_t* seg_in = sc_empty + kScRing;
  uint64_t* seg_out = seg_in + 1;
  uint64_t* drain = seg_out + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile uint32_t* verdict = tmem_slot + 2;
  static_assert((2 * kStages + 2 * kDRing + 2 * kScRing + 3) * 8 + 12 <= kSmemBars && kSmemSched % 8 == 0, "barriers");

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (warp == 0) {
    if (lane == 0) {
      for (int s = 0; s < kStages; ++s) tc::mbar_init(&full[s], 1), tc::mbar_init(&empty[s], 1);
      for (int d = 0; d < kDRing; ++d) tc::mbar_init(&d_full[d], 1), tc::mbar_init(&d_empty[d], kEpiWarps);
      for (int q = 0; q < kScRing; ++q) tc::mbar_init(&sc_full[q], 1), tc::mbar_init(&sc_empty[q], kEpiWarps);
      tc::mbar_init(seg_in, kEpiWarps), tc::mbar_init(seg_out, 1), tc::mbar_init(drain, 1);
      *abort_flag = 0;
      tc::mbar_fence_init();
      tc::tma_prefetch_desc(&wmap), tc::tma_prefetch_desc(&xmap);
    }
  } else if (warp == 1) {
    tc::tmem_alloc(tmem_slot, 512);
    tc::tmem_relinquish();
  } else if (warp == 2) {
    schedule(a, start, begin, lane);
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = *tmem_slot;

  const int64_t units = (int64_t)start[a.experts] * a.kb;
  const int64_t by_units = units / kMinUnits;
  const int64_t ctas = by_units < 1 ? 1 : by_units < (int64_t)gridDim.x ? by_units : (int64_t)gridDim.x;
  const int64_t lo = blockIdx.x < ctas ? (int64_t)blockIdx.x * units / ctas : units;
  const int64_t hi = blockIdx.x < ctas ? ((int64_t)blockIdx.x + 1) * units / ctas : units;
  const int64_t mine = hi - lo;
  auto give_up = [&]() {
    *abort_flag = 1;
    atomicOr(&a.header->error, 1u);
  };

  if (mine > 0) {
    Walk w;
    if (warp == 0) {
      // ---------------- loads: one box of 128 weight rows, boxes of 16 tokens ----------------
      if (lane == 0) {
        w.init(start, begin, a.experts, a.kb, lo);
        int64_t issued = 0;
        int s = 0;
        uint32_t ph = 1;
        for (int64_t i = 0; i < mine; ++i) {
          if (!tc::mbar_wait(&empty[s], ph, a.wait_ns, abort_flag)) {
            give_up();
            break;
          }
          const int boxes = (w.n + kBox - 1) / kBox;
          uint8_t* to = stages + (size_t)s * kStage;
          tc::mbar_arrive_expect_tx(&full[s], kWBytes + boxes * (kBox * kBlock));
          tma_load_3d(to, &wmap, &full[s], w.kb * kBlock, w.nb * kRows, w.e);
          for (int b = 0; b < boxes; ++b)
            tc::tma_load_2d(to + kWBytes + b * (kBox * kBlock), &xmap, &full[s], w.kb * kBlock, w.m0 + b * kBox);
          issued = i + 1;
          w.next(issued < mine);
          if (++s == kStages) s = 0, ph ^= 1u;
        }
        // every load lands before this CTA's shared memory is released
        for (int64_t j = issued > kStages ? issued - kStages : 0; j < issued; ++j)
          tc::mbar_wait(&full[j % kStages], (uint32_t)((j / kStages) & 1), a.wait_ns, nullptr);
      }
    } else if (warp == 1) {
      // ---------------- MMA ----------------
      if (lane == 0) {
        w.init(start, begin, a.experts, a.kb, lo);
        int s = 0, d = 0;
        uint32_t ph = 0, dph = 1;
        bool good = true;
        for (int64_t i = 0; i < mine && good; ++i) {
          good = tc::mbar_wait(&d_empty[d], dph, a.wait_ns, abort_flag) && tc::mbar_wait(&full[s], ph, a.wait_ns, abort_flag);
          if (!good) {
            give_up();
            break;
          }
          tc::fence_after_sync();
          const uint32_t at = tc::smem_u32(stages + (size_t)s * kStage);
          const uint64_t ad = tc::sdesc_kmajor_sw128(at), bd = tc::sdesc_kmajor_sw128(at + kWBytes);
          const uint32_t id = idesc_f8(kRows, (w.n + 15) & ~15);
#pragma unroll
          for (int j = 0; j < kBlock / 32; ++j) mma_f8(tmem + d * kCols, ad + 2 * j, bd + 2 * j, id, j > 0);
          tc::commit(&empty[s]);
          tc::commit(&d_full[d]);
          w.next(i + 1 < mine);
          if (++s == kStages) s = 0, ph ^= 1u;
          if (++d == kDRing) d = 0, dph ^= 1u;
        }
        tc::commit(drain);
        tc::mbar_wait(drain, 0, a.wait_ns, nullptr);
      }
    } else if (warp == 2) {
      // ---------------- scales: xs * ws of the unit's tokens, four units' loads in flight ----------------
      w.init(start, begin, a.experts, a.kb, lo);
      constexpr int kAhead = 4, kEach = kCols / 32;
      float next[kAhead][kEach];
      int n_next[kAhead];
      auto load = [&](int64_t i) {
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
          n_next[j] = 0;
          if (i + j < mine) {
            n_next[j] = w.n;
            const float ws = a.ws[((int64_t)w.e * a.nb + w.nb) * a.kb + w.kb];
#pragma unroll
            for (int c = 0; c < kEach; ++c)
              next[j][c] = c * 32 + lane < w.n ? ws * a.xs[(w.m0 + c * 32 + lane) * a.xs_m + w.kb * a.xs_b] : 0.f;
            w.next(i + j + 1 < mine);
          }
        }
      };
      load(0);
      int q = 0;
      uint32_t ph = 1;
      bool good = true;
      for (int64_t i = 0; i < mine && good; i += kAhead) {
        float f[kAhead][kEach];
        int n[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
          n[j] = n_next[j];
#pragma unroll
          for (int c = 0; c < kEach; ++c) f[j][c] = next[j][c];
        }
        load(i + kAhead);
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
          if (!good || i + j >= mine) break;
          good = __all_sync(0xffffffffu, tc::mbar_wait(&sc_empty[q], ph, a.wait_ns, abort_flag));
          if (!good) {
            give_up();
            break;
          }
#pragma unroll
          for (int c = 0; c < kEach; ++c)
            if (c * 32 < n[j]) sc[q * kCols + c * 32 + lane] = f[j][c];
          __syncwarp();
          if (lane == 0) tc::mbar_arrive(&sc_full[q]);
          if (++q == kScRing) q = 0, ph ^= 1u;
        }
      }
    } else if (warp >= kEpi0) {
      // ---------------- sums: lanes 32 (warp % 4) .. of tensor memory, every second chunk of 16 columns ----------------
      w.init(start, begin, a.experts, a.kb, lo);
      const int quarter = warp & 3, half = (warp - kEpi0) >> 2, row = quarter * 32 + lane;
      const uint32_t from = tmem + ((uint32_t)(quarter * 32) << 16);
      float sum[kChunks][16];
      int d = 0, q = 0;
      uint32_t dph = 0, qph = 0, joined = 0;
      bool fresh = true, whole = false;
      for (int64_t i = 0; i < mine; ++i) {
        if (fresh) {
          whole = w.kb == 0;
          fresh = false;
#pragma unroll
          for (int c = 0; c < kChunks; ++c)
#pragma unroll
            for (int j = 0; j < 16; ++j) sum[c][j] = 0.f;
        }
        bool good = tc::mbar_wait(&sc_full[q], qph, a.wait_ns, abort_flag) && tc::mbar_wait(&d_full[d], dph, a.wait_ns, abort_flag);
        if (!__all_sync(0xffffffffu, good)) {
          give_up();
          break;
        }
        tc::fence_after_sync();
        const int chunks = (w.n + 15) >> 4;
        uint32_t v[kChunks][16];
#pragma unroll
        for (int c = 0; c < kChunks; ++c)
          if (2 * c + half < chunks) tc::ld_32x32b_x16(from + d * kCols + (2 * c + half) * 16, v[c]);
        tc::wait_ld();
        tc::fence_before_sync();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(&d_empty[d]);
#pragma unroll
        for (int c = 0; c < kChunks; ++c)
          if (2 * c + half < chunks) {
            const float4* f = reinterpret_cast<const float4*>(sc + q * kCols + (2 * c + half) * 16);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float4 s4 = f[j];
              sum[c][4 * j] = fmaf(__uint_as_float(v[c][4 * j]), s4.x, sum[c][4 * j]);
              sum[c][4 * j + 1] = fmaf(__uint_as_float(v[c][4 * j + 1]), s4.y, sum[c][4 * j + 1]);
              sum[c][4 * j + 2] = fmaf(__uint_as_float(v[c][4 * j + 2]), s4.z, sum[c][4 * j + 2]);
              sum[c][4 * j + 3] = fmaf(__uint_as_float(v[c][4 * j + 3]), s4.w, sum[c][4 * j + 3]);
            }
          }
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(&sc_empty[q]);
        if (++d == kDRing) d = 0, dph ^= 1u;
        if (++q == kScRing) q = 0, qph ^= 1u;

        const bool last = w.kb + 1 == a.kb;
        if (last || i + 1 == mine) {
          whole = whole && last;
          bool write = whole;
          if (!whole) {
            // A part of a tile: published, and whichever CTA comes last adds the parts in the order of the CTAs.
            const int64_t first = (int64_t)w.t * a.kb;
            const int64_t c0 = cta_of_unit(first, units, ctas), c1 = cta_of_unit(first + a.kb - 1, units, ctas);
            const size_t part = (size_t)kCols * kRows;
            float* to = a.partials + ((size_t)blockIdx.x * 2 + (c0 == (int64_t)blockIdx.x ? 1 : 0)) * part;
#pragma unroll
            for (int c = 0; c < kChunks; ++c)
              if (2 * c + half < chunks)
#pragma unroll
                for (int j = 0; j < 16; ++j) __stcg(to + ((2 * c + half) * 16 + j) * kRows + row, sum[c][j]);
            __threadfence();
            __syncwarp();
            const uint32_t jp = joined & 1u;
            ++joined;
            if (lane == 0) tc::mbar_arrive(seg_in);
            if (!__all_sync(0xffffffffu, tc::mbar_wait(seg_in, jp, a.wait_ns, abort_flag))) {
              give_up();
              break;
            }
            if (warp == kEpi0 && lane == 0) {
              __threadfence();
              const uint32_t parts = (uint32_t)(c1 - c0 + 1);
              const bool done = atomicAdd(&a.counters[c0], 1u) == parts - 1;
              if (done) a.counters[c0] = 0u;  // ready for the next launch
              __threadfence();
              *verdict = done ? 1u : 0u;
              tc::mbar_arrive(seg_out);
            }
            if (!__all_sync(0xffffffffu, tc::mbar_wait(seg_out, jp, a.wait_ns, abort_flag))) {
              give_up();
              break;
            }
            write = *verdict != 0u;
            if (write) {
              __threadfence();
#pragma unroll
              for (int c = 0; c < kChunks; ++c)
                if (2 * c + half < chunks) {
                  for (int64_t p = c0; p <= c1; ++p) {
                    const float* in = a.partials + ((size_t)p * 2 + (p == c0 ? 1 : 0)) * part;
                    float v2[16];
#pragma unroll
                    for (int j = 0; j < 16; ++j) v2[j] = __ldcg(in + ((2 * c + half) * 16 + j) * kRows + row);
#pragma unroll
                    for (int j = 0; j < 16; ++j) sum[c][j] = p == c0 ? v2[j] : sum[c][j] + v2[j];
                  }
                }
            }
          }
          const int col = w.nb * kRows + row;
          if (write && col < a.n) {
#pragma unroll
            for (int c = 0; c < kChunks; ++c)
#pragma unroll
              for (int j = 0; j < 16; ++j) {
                const int t = (2 * c + half) * 16 + j;
                if (t < w.n) store_out(a, (int64_t)(w.m0 + t) * a.out_stride + col, sum[c][j]);
              }
          }
          fresh = true;
        }
        w.next(i + 1 < mine);
      }
    }
  }

  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  if (warp == 1) tc::tmem_dealloc(tmem, 512);
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

}  // namespace f8
}  // namespace up

using namespace up;
using namespace up::f8;

extern "C" size_t up_sm100_f8_matmul_workspace_bytes(int64_t m, int64_t experts, int64_t n, int64_t k) {
  if (m <= 0 || experts <= 0 || n <= 0 || k <= 0) return UP_F8_COUNTER_BYTES;
  return UP_F8_COUNTER_BYTES + (size_t)cta_count() * 2 * kCols * kRows * sizeof(float);
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
  const int64_t nb = (n + kRows - 1) / kRows, kb = (k + kBlock - 1) / kBlock;
  if (m > 0x3fffffff || n > 0x3fffffff || k > 0x3fffffff || x_stride >= ((int64_t)1 << 40) || n * k >= ((int64_t)1 << 40) ||
      nb > 0x7fffffff / (m / kCols + experts + 1))
    return UP_ERR_UNSUPPORTED;
  UP_CHECK_ARG(aligned(workspace, 256) && workspace_bytes >= up_sm100_f8_matmul_workspace_bytes(m, experts, n, k));
  auto enc = encode_fn();
  if (enc == nullptr) return fail_with(UP_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
  // weights as [experts, n, k] bytes in boxes of 128 rows, activations as [m, k] in boxes of 16; what lies outside reads 0
  CUtensorMap wmap, xmap;
  const cuuint32_t one[3] = {1, 1, 1};
  const cuuint64_t wdims[3] = {(cuuint64_t)k, (cuuint64_t)n, (cuuint64_t)experts};
  const cuuint64_t wstrides[2] = {(cuuint64_t)k, (cuuint64_t)(n * k)};
  const cuuint32_t wbox[3] = {kBlock, kRows, 1};
  if (enc(&wmap, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<uint8_t*>(w), wdims, wstrides, wbox, one,
          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
    return fail_with(UP_ERR_CUDA, "cuTensorMapEncodeTiled refused the weights' tensor map");
  const cuuint64_t xdims[2] = {(cuuint64_t)k, (cuuint64_t)m};
  const cuuint64_t xstrides[1] = {(cuuint64_t)x_stride};
  const cuuint32_t xbox[2] = {kBlock, kBox};
  if (enc(&xmap, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t*>(x), xdims, xstrides, xbox, one,
          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
    return fail_with(UP_ERR_CUDA, "cuTensorMapEncodeTiled refused the activations' tensor map");
  const cudaError_t e = ensure_smem_attr((const void*)matmul_kernel, kSmem);
  if (e != cudaSuccess) return cuda_status(e);
  Args a{};
  a.xs = x_scale, a.ws = w_scale, a.xs_m = xs_stride_m, a.xs_b = xs_stride_b, a.m = m, a.experts = (int)experts, a.n = (int)n;
  a.k = (int)k, a.kb = (int)kb, a.nb = (int)nb, a.offsets = offsets, a.out = out, a.out_stride = out_stride;
  a.out_dtype = out_dtype, a.header = static_cast<Header*>(workspace);
  a.counters = reinterpret_cast<uint32_t*>(static_cast<char*>(workspace) + sizeof(Header));
  a.partials = reinterpret_cast<float*>(static_cast<char*>(workspace) + UP_F8_COUNTER_BYTES);
  a.wait_ns = wait_limit_ns();
  matmul_kernel<<<(unsigned)cta_count(), kThreads, kSmem, static_cast<cudaStream_t>(stream)>>>(wmap, xmap, a);
  note_launch();
  return check_launch();
}

UP_DEFINE_REVISION(f8_matmul)
