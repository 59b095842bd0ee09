// kv4_prompt.cu — attention over the paged 4-bit cache for many query rows a key/value head (prompts), on the tcgen05
// tensor cores: the cache's tiles are turned into f16 once a CTA and serve 256 query rows.
//
// What bounds it: no one unit. At dim 128 a tile of 256 query rows and 128 cached tokens takes about 5300 cycles, of which
// the tensor cores are busy 4200 (an M128 N64 K16 product takes 49 cycles, not 32: it reads its A operand from shared
// memory again), the exponentials 2050 (16 a clock and SM), and the schedulers issue in half. Leaving out half of the
// products, the exponentials or the conversion of the cache gains 6, 1 and 5 % each: the chain from S to P to the next S
// is what takes the time. Starting and ending a CTA takes 14000 cycles more. Three sequences of 1500 to 2048 query
// tokens, 32 heads over 8, dim 128: bf16 311 us (198 GFLOP, 636 TFLOP/s; the second products of the parts not counted).
//
// A CTA takes 256 query rows (query token x head of the group) of one sequence and key/value head as two tiles of 128,
// and walks the cached tokens that any of them sees, 128 at a time. Per tile of tokens, S = Q K^T (128 x 128) and
// O += P V (128 x dim) run per query tile with f32 accumulators in tensor memory. A tile of tokens is two halves of 64,
// each with an S of its own, so that a query tile's probabilities of one half are computed while the tensor cores work
// on the other.
//  * warp groups 0 and 1 (probabilities): group w holds query tile w, a thread a row. A thread reads its row of S twice,
//    for the largest logit and for p = 2^(logit - ref + 7), and writes P as f16 over it: the A operand of the second product.
//    ref moves only when a logit is more than 8 above it; then the thread scales its row of O. So p ends at 2^15, and f16
//    takes weights down to 2^-30 of the largest (without the 7, 65536 weights of 2^-26, a thousandth together, were lost).
//  * warp groups 2 and 3 (cache, K and V): read 128 tokens' nibbles and scales, a tile ahead in registers, and write
//    them as f16 into 128-byte swizzled shared memory, a place a half, free again when the half's products are done. Both
//    have a row a token: K is the B operand with its contraction (the dimensions) contiguous, V
//    the one with its output (the dimensions) contiguous. The nibble conversion pairs dimensions k and k + 4 of each 8;
//    q is stored in the same order and the output's columns are read in it.
//  * warps 16 and 17 (products): each issues the tcgen05.mma of one query tile, so neither tile's products wait for the
//    other's probabilities.
// Scales. A tile's scales are multiplied by a power of two (separately for K and V) that takes the largest to 2^12 .. 2^13,
// so nibble * scale ends just inside f16's range; the logits take K's power, the probabilities V's, relative to the one that
// O has (O is scaled when a tile's is above it, or below a quarter of it). That leaves 2^26 below the largest scale in which
// a scale keeps all of its bits, so a row's precision does not hang on tokens that it does not see: an f16 scale loses bits
// only below 2^-11 and only beside one of 8192 or more in its 128 tokens (then it is off by at most 2^-22).
// The logits are exact up to their f32 sums, as a row's logsumexp is in f32:
// each of K's scales is split into its first 8 bits and the rest, a nibble times either is exact in f16, and both
// products are added in one S (with one scale a token, multiplying the columns of S by it in the softmax instead took 381
// us where this took 320). So is V for f16 outputs. For bf16 ones, which round to 8 bits, nibble * scale is rounded to f16:
// that is one product, and the second part's memory is a second stage (311 us against 367). p is rounded to f16. All sums
// are f32.
// A token with an infinite or NaN v_scale is left out of the products (its rows would reach queries that do not see it)
// and the outputs of the queries that do see it become NaN; their logsumexp, which no value is part of, stays.
// Every wait is bounded; one that runs out sets the workspace's error word and the CTA unwinds.
//
// The tile of 2 x 128 rows is what 512 columns of tensor memory hold (S and O of both tiles at dim 128) and 227 KB of
// shared memory (q 64 KB, K and V in two parts 64 KB each).
#include "kv4_attention.cuh"
#include "tc.cuh"

namespace up {
namespace kv4 {

namespace {

constexpr int kRowsCta = 256, kTok = 128, kHalf = kTok / 2;
constexpr int kThreads = 32 * 18, kCacheWarp = 8, kMmaWarp = 16;
constexpr int kTop = 12, kLeastExp = -24 - kTop;  // the largest scale of a tile becomes 2^kTop .. 2^(kTop + 1): times -8, -65504
constexpr int kLift = 7;  // p = 2^kLift where a logit is at the reference
constexpr int kBlockBytes = kTok * 128;       // 128 query rows of 64 dimensions (128 bytes), swizzled
constexpr int kHalfBlockBytes = kHalf * 128;  // 64 tokens of 64 dimensions

template <int D>
struct Cfg {
  static constexpr int kBlocks = D / 64;
  static constexpr int kTile = kBlocks * kBlockBytes;       // 128 rows of D f16
  static constexpr int kPart = kTile / 2;                   // K or V of a half: 64 rows, with the scales' first bits or the rest
  static constexpr int kQ = 0, kK = 2 * kTile, kV = kK + 4 * kPart;
  static constexpr int kScale = kV + 4 * kPart;             // f16 pairs [2 (K, V)][128][up to D / 32]
  static constexpr int kSmem = kScale + 2 * kTok * (D / 32) * 4 + 1024 /* alignment */;
  static constexpr int kS = 0, kO = 2 * kTok;               // tensor memory columns: S (and P) of both tiles, then O
  static constexpr int kCols = 512;
};

struct Meta {          // what the cache warps say of a tile of tokens
  int k_exp, v_exp;    // its scales were multiplied by 2^-these
  uint32_t valid[4];   // tokens that exist
  uint32_t bad[4];     // of these, the ones with an infinite or NaN v_scale
};

struct Shared {
  uint64_t k_full[2], k_empty[2], v_full[2][2], v_empty[2][2];  // K: [half], V: [stage][half]
  // V's part of a tile's meta is there; of tile t in t mod 4, as up to three tiles' come before the first one's is waited
  // for, and a wait must not find its barrier two phases on.
  uint64_t v_meta[4];
  uint64_t s_full[2][2], p_full[2][2], pv_done[2], all_done[2], q_full, drain;  // [query tile][half]
  uint32_t tmem;
  int abort;
  Meta meta[4];
  uint32_t big[2][4];          // [K, V][warp]
};

__device__ __forceinline__ uint64_t desc_v(uint32_t addr) {  // dimensions contiguous: 64-dimension blocks kHalfBlockBytes apart
  uint64_t d = 0;
  d |= (uint64_t)((addr >> 4) & 0x3fffu);
  d |= (uint64_t)(kHalfBlockBytes >> 4) << 16;  // leading offset: the next 64 dimensions
  d |= (uint64_t)(1024u >> 4) << 32;        // stride offset: the next 8 tokens
  d |= (uint64_t)1u << 46;
  d |= (uint64_t)2u << 61;                  // 128-byte swizzle
  return d;
}

// kind::f16 with f16 operands and f32 sums; `mn`: B's output dimension is the contiguous one.
__host__ __device__ constexpr uint32_t idesc_f16(int M, int N, bool mn) {
  return (1u << 4) | (mn ? 1u << 16 : 0u) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}

__device__ __forceinline__ void ld_x32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}

// D[tmem] (+)= A B, kind::f16: A from shared memory (a descriptor) or tensor memory. The thread that issues shares its
// scheduler with warps that compute, so what an issue costs is its instructions: no lane mask, constant tensor memory
// addresses (the CTA holds all of it, from address 0).
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)add)
      : "memory");
}
__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
  return one != 0;
}

__device__ __forceinline__ float pow2f(int e) { return __uint_as_float((uint32_t)(min(max(e, -126), 127) + 127) << 23); }
template <int ID, int THREADS>
__device__ __forceinline__ void named_sync() { asm volatile("bar.sync %0, %1;" ::"n"(ID), "n"(THREADS) : "memory"); }
__device__ __forceinline__ void cache_sync(int z) { z ? named_sync<2, 128>() : named_sync<1, 128>(); }  // K's, V's group

template <int D, bool BF16>  // BF16: q and out, else f16
__global__ void __launch_bounds__(kThreads, 1) kv4_prompt_kernel(const Args a, const uint64_t wait_ns) {
  using C = Cfg<D>;
  constexpr int CH = D / 32;
  extern __shared__ uint8_t raw_smem[];
  __shared__ Shared sh;
  uint8_t* smem = raw_smem + ((1024 - (smem_addr(raw_smem) & 1023)) & 1023);
  const uint32_t sbase = smem_addr(smem);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      tc::mbar_init(&sh.k_full[i], 2);   // the warps that fill it
      tc::mbar_init(&sh.k_empty[i], 2);  // a commit of each issuer
      for (int h = 0; h < 2; ++h) {
        tc::mbar_init(&sh.v_full[i][h], 2);
        tc::mbar_init(&sh.v_empty[i][h], 2);
        tc::mbar_init(&sh.s_full[i][h], 2);  // the issuer (it has seen the tile's meta) and a commit
        tc::mbar_init(&sh.p_full[i][h], 4);  // the tile's warps
      }
      tc::mbar_init(&sh.pv_done[i], 1);
      tc::mbar_init(&sh.all_done[i], 1);
    }
    for (int i = 0; i < 4; ++i) tc::mbar_init(&sh.v_meta[i], 1);
    tc::mbar_init(&sh.q_full, kCacheWarp);
    tc::mbar_init(&sh.drain, 2);
    tc::mbar_fence_init();
    sh.abort = 0;
  }
  if (warp == kMmaWarp) {
    tc::tmem_alloc(&sh.tmem, C::kCols);
    tc::tmem_relinquish();
  }
  // ---- which sequence, tile and head: sequences in order, a sequence's last (longest) tiles first ----
  // Each warp finds it for itself, 32 sequences at a time: no exchange between them.
  const int64_t work = blockIdx.x;
  int64_t base = 0;  // CTAs of the sequences before
  int b = 0;
  Seq seq;
  for (;; b += 32) {
    seq = Seq{0, 0, 0};
    if (b + lane < a.batch) seq = load_seq(a, b + lane);
    const int64_t mine = (int64_t)((seq.nq * a.ratio + kRowsCta - 1) / kRowsCta) * a.kv_heads;
    int64_t incl = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t v = __shfl_up_sync(0xffffffffu, incl, d);
      if (lane >= d) incl += v;
    }
    const uint32_t past = __ballot_sync(0xffffffffu, work < base + incl);
    if (past) {
      const int at = __ffs(past) - 1;
      base = __shfl_sync(0xffffffffu, base + incl - mine, at);
      seq.len = __shfl_sync(0xffffffffu, seq.len, at);
      seq.nq = __shfl_sync(0xffffffffu, seq.nq, at);
      seq.q0 = __shfl_sync(0xffffffffu, seq.q0, at);
      b += at;
      break;
    }
    base += __shfl_sync(0xffffffffu, incl, 31);
    if (b + 32 >= a.batch) {  // more CTAs were launched than there are tiles; all warps see this
      b = -1;
      break;
    }
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  if (b < 0) {
    if (warp == kMmaWarp) tc::tmem_dealloc(0, C::kCols);
    return;
  }
  const int rows = seq.nq * a.ratio, tiles = (rows + kRowsCta - 1) / kRowsCta;
  const int in_seq = (int)(work - base), tile = tiles - 1 - in_seq / a.kv_heads, head = in_seq % a.kv_heads;
  const int row0 = tile * kRowsCta, live = min(kRowsCta, rows - row0);
  int lo, hi;
  visible(a, seq, (int)a.by_ratio(row0), (int)a.by_ratio(row0 + live - 1), lo, hi);
  const int tok0 = lo / kTok * kTok, n = hi > tok0 ? (hi - tok0 + kTok - 1) / kTok : 0;

  constexpr int LPR = D / 8;  // lanes a row of queries
  constexpr uint32_t tmem = 0;  // all 512 columns were allocated: they begin at 0
  volatile int* abort_flag = &sh.abort;
  auto give_up = [&]() {
    *abort_flag = 1;
    a.header[3] = 1u;
  };

  if (warp < kCacheWarp) {
    // ---------------- probabilities ----------------
    const int w = warp >> 2, r = threadIdx.x;  // r: the CTA's row
    const int row = row0 + r, in_q = (int)a.by_ratio(row), head_q = head * a.ratio + row - in_q * a.ratio;
    const int64_t token = seq.q0 + in_q;
    // ---- queries: f16 with a power of two a row and the logits' sign, swizzled ----
    // A warp copies its 32 rows to their places as they are; then each thread turns its row into f16 there.
    const uint32_t q_rows = sbase + C::kQ + w * C::kTile + (r & 96) * 128;
    auto place = [&](uint32_t rows, int rr, int o) {  // 8 dimensions of one of the warp's rows
      return rows + (o / 8) * kBlockBytes + rr * 128 + ((o % 8) ^ (rr & 7)) * 16;
    };
    {
      const int64_t q_off = 2 * (token * a.qs + (int64_t)head_q * a.qh);
      const int o = lane % LPR;
#pragma unroll 8
      for (int k = 0; k < LPR; ++k) {  // 32 / LPR rows at a time
        const int rr = k * (32 / LPR) + lane / LPR;
        const int64_t off = __shfl_sync(0xffffffffu, q_off, rr);
        const bool in = (r & ~31) + rr < live;
        cp_async16(place(q_rows, rr, o), static_cast<const char*>(a.q) + (in ? off + 16 * o : 0), in ? 16 : 0);
      }
      cp_async_commit();
      cp_async_wait<0>();
      __syncwarp();
    }
    auto piece = [&](int o) {
      uint4 x;
      asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w)
                   : "r"(place(q_rows, lane, o))
                   : "memory");
      return x;
    };
    uint32_t big = 0;  // the row's largest magnitude, by its 16 bits
#pragma unroll
    for (int o = 0; o < LPR; ++o) {
      const uint4 x = piece(o);
      big = __vmaxu2(big, __vmaxu2(__vmaxu2(x.x & 0x7fff7fffu, x.y & 0x7fff7fffu), __vmaxu2(x.z & 0x7fff7fffu, x.w & 0x7fff7fffu)));
    }
    big = max(big & 0xffffu, big >> 16);
    const float most = BF16 ? __uint_as_float(big << 16) : __half2float(__ushort_as_half((unsigned short)big));
    const int ex = (int)(__float_as_uint(most) >> 23) - 127;  // it becomes 2^7 .. 2^8
    const int up = big == 0 || ex == 128 ? 0 : min(7 - ex, 126);
    const float q_mul = a.scale_log2 < 0.f ? -pow2f(up) : pow2f(up), row_scale = fabsf(a.scale_log2) * pow2f(-up);
#pragma unroll 4
    for (int o = 0; o < LPR; ++o) {
      float f[8];
      unpack8(piece(o), BF16, f);
#pragma unroll
      for (int x = 0; x < 8; ++x) f[x] *= q_mul;
      asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(place(q_rows, lane, o)), "r"(pack2_f16(f[0], f[4])),
                   "r"(pack2_f16(f[1], f[5])), "r"(pack2_f16(f[2], f[6])), "r"(pack2_f16(f[3], f[7]))
                   : "memory");
    }
    tc::fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) tc::mbar_arrive(&sh.q_full);
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;
    const uint32_t ts = tmem + C::kS + w * kTok + lanes, to = tmem + C::kO + w * D + lanes;
    const int pos = seq.len - seq.nq + in_q;
    const int last = r >= live ? -1 : a.causal ? min(pos, seq.len - 1) : seq.len - 1;
    const int past = a.window > 0 ? max(pos - a.window, -1) : -1;
    float mx = kNoMax, sum = 0.f;
    int vexp = kLeastExp;  // O is in units of 2^vexp
    bool ok = true, not_finite = false;  // whether a value that the row sees is not
    const bool wide = ((reinterpret_cast<uintptr_t>(a.out) | (uint64_t)(2 * (a.os | a.oh))) & 15) == 0;  // 16-byte stores
    auto wait = [&](uint64_t* bar, int parity) {
      return __all_sync(0xffffffffu, tc::mbar_wait(bar, parity & 1, wait_ns, abort_flag)) != 0;
    };
#pragma unroll 1
    for (int u = 0; u < 2 * n; ++u) {  // half h of tile t
      const int t = u >> 1, h = u & 1;
      ok = wait(&sh.s_full[w][h], t);
      if (!ok) break;
      tc::fence_after_sync();
      const Meta& meta = sh.meta[t & 3];
      const int j0 = tok0 + u * kHalf;
      const uint32_t th = ts + h * kHalf;
      const float c = row_scale * pow2f(meta.k_exp);
      const int ve = meta.v_exp;
      const uint32_t valid0 = meta.valid[2 * h], valid1 = meta.valid[2 * h + 1];
      const bool masked = !__all_sync(0xffffffffu, (valid0 & valid1) == 0xffffffffu && j0 > past && j0 + kHalf - 1 <= last);
      // the visible tokens of chunk g (32 of them)
      auto seen = [&](int g) -> uint32_t {
        const int from = past + 1 - (j0 + 32 * g), to_ = last + 1 - (j0 + 32 * g);  // in [from, to_)
        uint32_t m = g ? valid1 : valid0;
        m &= from >= 32 ? 0u : from <= 0 ? 0xffffffffu : 0xffffffffu << from;
        m &= to_ <= 0 ? 0u : to_ >= 32 ? 0xffffffffu : (1u << to_) - 1u;
        return m;
      };
      // the largest logit, against the reference
      float m = -INFINITY;
#pragma unroll 1
      for (int g = 0; g < 2; ++g) {
        uint32_t v[32];
        ld_x32(th + 32 * g, v);
        tc::wait_ld();
        if (masked) {
          const uint32_t see = seen(g);
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = (see >> i) & 1u ? v[i] : 0x7fffffffu;  // a NaN is no maximum
        }
        float m1 = m;
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
          m = fmaxf(m, __uint_as_float(v[i]));
          m1 = fmaxf(m1, __uint_as_float(v[i + 1]));
        }
        m = fmaxf(m, m1);
      }
      m = fmaxf(mx, m * c);  // c is not negative; where nothing is seen, -infinity or (c = 0) NaN
      const bool rise = __any_sync(0xffffffffu, m > mx + 8.f), move = ve > vexp || ve < vexp - 2;
      if (rise || move) {
        float fo = 1.f;
        if (rise) {
          fo = exp2_approx(mx - m);
          sum *= fo;
          mx = m;
        }
        if (move) {
          fo *= pow2f(vexp - ve);
          vexp = ve;
        }
        if (u > 0) {
          // Phases are told apart by parity. PV of half u - 2 is done (S of half u was issued after it) and PV of half u
          // waits for this warp, so the barrier is in the phase asked for or just past it.
          ok = wait(&sh.pv_done[w], u - 1);
          if (!ok) break;
          tc::fence_after_sync();
#pragma unroll 1
          for (int g = 0; g < D / 32; ++g) {
            uint32_t v[32];
            ld_x32(to + 32 * g, v);
            tc::wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * fo);
            tc::st_32x32b_x32(to + 32 * g, v);
          }
        }
      }
      // p = 2^(c S - ref + kLift), in units of O, as f16 over columns that were read, and their sum
      const float add = (float)(ve - vexp + kLift) - mx;
      float s0 = 0.f, s1 = 0.f;
#pragma unroll 1
      for (int g = 0; g < 2; ++g) {
        uint32_t v[32], p[16];
        ld_x32(th + 32 * g, v);
        tc::wait_ld();
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(exp2_approx(fmaf(__uint_as_float(v[i]), c, add)));
        if (masked) {
          const uint32_t see = seen(g);
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = (see >> i) & 1u ? v[i] : 0u;
        }
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
          s0 += __uint_as_float(v[i]);
          s1 += __uint_as_float(v[i + 1]);
          p[i / 2] = pack2_f16(__uint_as_float(v[i]), __uint_as_float(v[i + 1]));
        }
        tc::st_32x32b_x16(th + 16 * g, p);
      }
      sum = fmaf(s0 + s1, pow2f(vexp - ve - kLift), sum);
      const uint32_t bad0 = meta.bad[2 * h], bad1 = meta.bad[2 * h + 1];
      if (bad0 | bad1) not_finite |= ((seen(0) & bad0) | (seen(1) & bad1)) != 0;
      tc::wait_st();
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&sh.p_full[w][h]);
    }
    if (ok && n > 0) ok = wait(&sh.all_done[w], 0);
    if (!ok) {
      give_up();
    } else {
      tc::fence_after_sync();
      // the row, rounded, into the warp's part of the query tile (its products are done), then out in whole rows
      const float scale = not_finite ? __int_as_float(0x7fffffff) : sum == 0.f ? 0.f : pow2f(vexp - kLift) / sum;  // O is 0 where the sum is
#pragma unroll 1
      for (int g = 0; g < D / 32; ++g) {
        uint32_t v[32] = {};
        if (n > 0) {
          ld_x32(to + 32 * g, v);
          tc::wait_ld();
        }
#pragma unroll
        for (int k = 0; k < 32; ++k) v[k] = __float_as_uint(__uint_as_float(v[k]) * scale);
#pragma unroll
        for (int k = 0; k < 4; ++k) {  // columns 0 .. 7 hold dimensions 0, 4, 1, 5, 2, 6, 3, 7
          auto two = [&](int x, int y) { return pack2(__uint_as_float(v[8 * k + x]), __uint_as_float(v[8 * k + y]), BF16); };
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(place(q_rows, lane, 4 * g + k)), "r"(two(0, 2)),
                       "r"(two(4, 6)), "r"(two(1, 3)), "r"(two(5, 7))
                       : "memory");
        }
      }
      __syncwarp();
      const int64_t out_off = 2 * (token * a.os + (int64_t)head_q * a.oh);
      const int o = lane % LPR;
#pragma unroll 4
      for (int k = 0; k < LPR; ++k) {  // 32 / LPR rows at a time
        const int rr = k * (32 / LPR) + lane / LPR;
        char* dst = static_cast<char*>(a.out) + __shfl_sync(0xffffffffu, out_off, rr) + 16 * o;
        if ((r & ~31) + rr >= live) continue;
        uint4 v;
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                     : "r"(place(q_rows, rr, o))
                     : "memory");
        if (wide) {
          *reinterpret_cast<uint4*>(dst) = v;
        } else {
          *reinterpret_cast<uint2*>(dst) = make_uint2(v.x, v.y);
          *reinterpret_cast<uint2*>(dst + 8) = make_uint2(v.z, v.w);
        }
      }
      if (a.lse && r < live) a.lse[token * a.ls + head_q] = sum == 0.f ? -INFINITY : (mx + log2f(sum)) * kLn2;
    }
  } else if (warp < kMmaWarp) {
    // ---------------- cache: nibbles and scales to f16; group z: 0 K, 1 V ----------------
    const int z = (warp - kCacheWarp) >> 2, w = warp & 3, tid = threadIdx.x & 127, groups = a.groups;
    const uint8_t* nibbles = z ? a.v4 : a.k4;
    const __half* scales = z ? a.v_scale : a.k_scale;
    uint32_t* sc = reinterpret_cast<uint32_t*>(smem + C::kScale) + z * kTok * CH;  // a scale's first 8 bits, the rest
    const bool two = !BF16 || z == 0;
    const int32_t* pages = a.table + (int64_t)b * a.table_stride;
    const int in_page = (1 << a.page_log2) - 1, cpg_log2 = 31 - __clz(a.cpg);  // 1, 2 or 4 chunks a group
    auto page_of = [&](int t) {
      const int j = tok0 + t * kTok + tid;
      if (t >= n || j >= seq.len) return -1;
      const int p = __ldg(pages + (j >> a.page_log2));
      return (uint32_t)p < a.pages ? p : -1;
    };
    // a tile's nibbles: unit u = lane / 8 + 4 i of this warp's 32 tokens is run u / CH (8 tokens, lane % 8), chunk u % CH
    uint4 raw[CH];
    uint16_t sk[CH];  // this thread's token's scales (one a group)
    const uint32_t page_lines = (uint32_t)a.kv_heads << a.page_log2, head_line = (uint32_t)head << a.page_log2;
    // a run of 8 is on one page; one whose first token has no page is not read, as there may be no page at all
    auto fetch = [&](int t, int page) {
      const int at = (tok0 + t * kTok + 32 * w) & in_page;
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        const int u = (lane >> 3) + 4 * i, run = u / CH, c = u - run * CH;
        const int pg = __shfl_sync(0xffffffffu, page, 8 * run);
        const int64_t ln = (int64_t)(uint32_t)pg * page_lines + (head_line + ((at + 8 * run) & in_page) + (lane & 7));
        raw[i] = pg >= 0 ? ld_nc_na_v4(nibbles + ln * (D / 2) + 16 * c) : make_uint4(0, 0, 0, 0);
      }
    };
    auto fetch_scales = [&](int t, int page) {
      const int64_t line = (int64_t)(uint32_t)max(page, 0) * page_lines + (head_line + ((tok0 + t * kTok + tid) & in_page));
#pragma unroll
      for (int g = 0; g < CH; ++g) {
        sk[g] = 0;
        if (g < groups && page >= 0) sk[g] = __half_as_ushort(__ldg(scales + line * groups + g));
      }
    };
    auto put = [](uint32_t at, const uint32_t (&e)[4]) {
      asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(e[0]), "r"(e[1]), "r"(e[2]), "r"(e[3]) : "memory");
    };
    auto times = [](const uint32_t (&e)[4], __half2 s, uint32_t (&o)[4]) {
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const __half2 v = __hmul2(*reinterpret_cast<const __half2*>(&e[x]), s);
        o[x] = *reinterpret_cast<const uint32_t*>(&v);
      }
    };
    auto convert = [&](int stage) {
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        const int u = (lane >> 3) + 4 * i, run = u / CH, c = u - run * CH, tok = 32 * w + 8 * run + (lane & 7);
        const uint32_t words[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
        const int in_row = tok * groups + (c >> cpg_log2);
        const __half2 s = *reinterpret_cast<const __half2*>(&sc[in_row]);
        const uint32_t at = sbase + (z ? C::kV : C::kK) + ((tok / kHalf) * 2 + stage) * C::kPart + (c / 2) * kHalfBlockBytes + (tok % kHalf) * 128;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t to = at + ((((c & 1) * 4 + k) ^ (tok & 7)) << 4);
          uint32_t e[4], o[4];
          expand(words[k], e);
          times(e, __low2half2(s), o);
          put(to, o);
          if (two) {
            times(e, __high2half2(s), o);
            put(to + C::kPart, o);
          }
        }
      }
    };
    int page = page_of(0);
    if (n > 0) {
      fetch_scales(0, page);
      fetch(0, page);
    }
    for (int t = 0; t < n; ++t) {
      const int next = page_of(t + 1);
      Meta& meta = sh.meta[t & 3];
      // the tile's power of two, and its scales divided by it
      uint32_t big = 0;
      bool bad = false;
#pragma unroll
      for (int g = 0; g < CH; ++g) {
        const uint32_t m = sk[g] & 0x7fffu;
        if (m < 0x7c00u) big = max(big, m);
        bad |= m >= 0x7c00u;
      }
      big = __reduce_max_sync(0xffffffffu, big);
      const uint32_t marks = __ballot_sync(0xffffffffu, z ? bad : page >= 0);
      if (lane == 0) {
        sh.big[z][w] = big;
        (z ? meta.bad : meta.valid)[w] = marks;
      }
      cache_sync(z);  // also: every warp is done with the last tile's scales
      big = max(max(sh.big[z][0], sh.big[z][1]), max(sh.big[z][2], sh.big[z][3]));
      const int e = big ? (int)(__float_as_uint(__half2float(__ushort_as_half((unsigned short)big))) >> 23) - 127 - kTop : kLeastExp;
#pragma unroll
      for (int g = 0; g < CH; ++g) {
        if (g >= groups) continue;
        const bool finite = (sk[g] & 0x7fffu) < 0x7c00u;
        const uint32_t s = __half_as_ushort(__float2half_rn(__half2float(__ushort_as_half(sk[g])) * pow2f(-e)));
        const uint32_t first = two ? s & 0xfff8u : s;
        const __half rest = __hsub(__ushort_as_half((unsigned short)s), __ushort_as_half((unsigned short)first));
        // where it is not finite, a key makes its logit NaN, a value is left out: its token is marked
        sc[tid * groups + g] = finite ? first | (uint32_t)__half_as_ushort(rest) << 16 : z ? 0u : 0x7fff7fffu;
      }
      if (tid == 0) {
        (z ? meta.v_exp : meta.k_exp) = e;
        if (z) tc::mbar_arrive(&sh.v_meta[t & 3]);
      }
      cache_sync(z);
      page = next;
      if (t + 1 < n) fetch_scales(t + 1, page);
      // this warp's half, of the stage
      const int h = w >> 1, stage = two ? 0 : t & 1, turn = two ? t : t >> 1;
      if (__all_sync(0xffffffffu, tc::mbar_wait(z ? &sh.v_empty[stage][h] : &sh.k_empty[h], (turn & 1) ^ 1, wait_ns, abort_flag))) {
        convert(stage);
        tc::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(z ? &sh.v_full[stage][h] : &sh.k_full[h]);
        if (t + 1 < n) fetch(t + 1, page);
      } else {
        give_up();  // a named barrier still counts this warp: it keeps step with the others, without the work
      }
    }
  } else {
    // ---------------- products of query tile w ----------------
    if (n > 0) {
      constexpr uint32_t id_qk = idesc_f16(128, kHalf, false), id_pv = idesc_f16(128, D, true);
      const int w = warp - kMmaWarp;
      // descriptors of the first step; a step further adds its bytes / 16 to the address field
      const uint64_t q0 = tc::sdesc_kmajor_sw128(sbase + C::kQ + w * C::kTile);
      const uint64_t k0 = tc::sdesc_kmajor_sw128(sbase + C::kK), v0 = desc_v(sbase + C::kV);
      const uint32_t ts = tmem + C::kS + w * kTok, to = tmem + C::kO + w * D;
      auto wait = [&](uint64_t* bar, int parity) {
        return __all_sync(0xffffffffu, tc::mbar_wait(bar, parity & 1, wait_ns, abort_flag)) != 0;
      };
      auto qk = [&](int h) {
        const uint64_t k = k0 + (uint64_t)(h * (2 * C::kPart >> 4));
        if (elect_one()) {
#pragma unroll
          for (int x = 0; x < 2 * (D / 16); ++x) {  // 16 dimensions: 32 bytes; the scales' first bits, the rest
            const int i = x % (D / 16), part = x / (D / 16);
            mma_ss(ts + h * kHalf, q0 + (uint64_t)((i / 4) * (kBlockBytes >> 4) + (i % 4) * 2),
                   k + (uint64_t)(part * (C::kPart >> 4) + (i / 4) * (kHalfBlockBytes >> 4) + (i % 4) * 2), id_qk, x > 0);
          }
          tc::mbar_arrive(&sh.s_full[w][h]);
          tc::commit(&sh.s_full[w][h]);
          tc::commit(&sh.k_empty[h]);
        }
        __syncwarp();
      };
      // K of a half, and with the first one V's part of the tile's meta, which the probabilities take
      auto cached = [&](int t, int h) { return wait(&sh.k_full[h], t) && (h == 1 || wait(&sh.v_meta[t & 3], t >> 2)); };
      constexpr bool two = !BF16;
      bool ok = wait(&sh.q_full, 0);
      for (int h = 0; ok && h < 2; ++h) {
        ok = cached(0, h);
        if (!ok) break;
        tc::fence_after_sync();
        qk(h);
      }
#pragma unroll 1
      for (int u = 0; ok && u < 2 * n; ++u) {
        const int t = u >> 1, h = u & 1;
        const int stage = two ? 0 : t & 1;
        ok = wait(&sh.v_full[stage][h], two ? t : t >> 1) && wait(&sh.p_full[w][h], t);
        if (!ok) break;
        tc::fence_after_sync();
        const uint64_t v = v0 + (uint64_t)((2 * h + stage) * (C::kPart >> 4));
        if (elect_one()) {
#pragma unroll
          for (int i = 0; i < kHalf / 16; ++i)  // 16 tokens: 2048 bytes
            mma_ts(to, ts + h * kHalf + 8 * i, v + (uint64_t)(i * 128), id_pv, u + i > 0);
          if (two) {
#pragma unroll
            for (int i = 0; i < kHalf / 16; ++i)
              mma_ts(to, ts + h * kHalf + 8 * i, v + (uint64_t)((C::kPart >> 4) + i * 128), id_pv, true);
          }
          tc::commit(&sh.pv_done[w]);
          if (u + 1 == 2 * n) tc::commit(&sh.all_done[w]);
          tc::commit(&sh.v_empty[stage][h]);
        }
        __syncwarp();
        if (t + 1 == n) continue;
        ok = cached(t + 1, h);
        if (!ok) break;
        tc::fence_after_sync();
        qk(h);  // over S and P of tile t's half: issued after the products that read them
      }
      if (!ok) give_up();
      if (elect_one()) tc::commit(&sh.drain);  // nothing may be in flight when the tensor memory goes
      if (!tc::mbar_wait(&sh.drain, 0, wait_ns, nullptr)) give_up();
    }
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  if (warp == kMmaWarp) tc::tmem_dealloc(tmem, C::kCols);
}

template <int D, bool BF16>
int launch_prompt(const Args& a, int64_t ctas, cudaStream_t s) {
  const auto kernel = kv4_prompt_kernel<D, BF16>;
  const cudaError_t e = ensure_smem_attr(reinterpret_cast<const void*>(kernel), Cfg<D>::kSmem);
  if (e != cudaSuccess) return cuda_status(e);
  kernel<<<(unsigned)ctas, kThreads, Cfg<D>::kSmem, s>>>(a, wait_limit_ns());
  note_launch();
  return check_launch();
}

}  // namespace

int prompt_attention(const Args& a, int dim, cudaStream_t s) {
  const int64_t ctas = (a.tokens * a.ratio / kRowsCta + a.batch) * a.kv_heads;
  if (ctas > 0x7fffffff) return UP_ERR_UNSUPPORTED;
  if (dim == 64) return a.bf16 ? launch_prompt<64, true>(a, ctas, s) : launch_prompt<64, false>(a, ctas, s);
  return a.bf16 ? launch_prompt<128, true>(a, ctas, s) : launch_prompt<128, false>(a, ctas, s);
}

}  // namespace kv4
}  // namespace up
