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
//    (2,6), (3,7) are the A fragments of two k-steps; q's B fragments are laid out in the same order once a tile.
//  * V: ldmatrix.trans moves 16-bit units, four nibbles: lane (g, t) gets dimensions 4g .. 4g + 3 of tokens 2t and 2t + 1
//    in the two halves of a word, which is the A fragment of V transposed after the same conversion.
//  * Probabilities: the score fragment times v_scale, rounded to f16, transposed by movmatrix, is the B fragment.
// q is scaled by a power of two a row to fit f16 (exactly, where it is within 2^-22 of the row's largest); the
// probabilities by a power of two a warp, the largest exponent of the v_scale seen, so that p * v_scale fits f16 with
// 2^-23 of range below its largest value. p is rounded to f16 (2^-12); every sum is f32.
// The running maximum moves only when a logit exceeds it by more than 2^8 (f32 sums and the f16 range above hold that),
// so most steps need no reduction across lanes and no rescaling.
//
// Work. Units of 128 cached tokens, over sequences, tiles and heads in order, are split evenly over the launch's CTAs
// (each sequence's count comes from its length on the device: no host read, no launch bound by the longest sequence).
// A warp takes 32 tokens of each unit through its own ring of cp.async stages, so no barrier stands in the loop. A tile
// that ends inside one CTA is written at once; parts of a split tile go to the workspace in f32 and the CTA that
// finishes last adds them in order. No CTA waits for another.
#pragma once

#include "kv4_attention.cuh"

namespace up {
namespace kv4 {

template <int D, int NT>
struct SplitCfg {
  static constexpr int kChunks = D / 32;
  static constexpr int kStages = 3;
  static constexpr int kRows = 8 * NT;
  // a stage of one warp: 32 tokens of K and V (D / 2 bytes each) and of their scales (at most D / 32 f16 each)
  static constexpr int kKV = 16 * D, kSc = 2 * D, kStage = 2 * kKV + 2 * kSc;
  static constexpr int kPitch = D + 4;  // floats between the rows of the merge buffer: conflict-free 16-byte stores
  static constexpr int kRing = kSplitWarps * kStages * kStage;
  static constexpr int kMerge = kSplitWarps * kRows * kPitch * 4;
  static constexpr int kSmem = kRing > kMerge ? kRing : kMerge;
  static constexpr int kOcc = D <= 128 ? (NT == 1 ? 4 : 3) : 2;
};

// Chunk c of token row r is stored at chunk c ^ swizzle(r): 8 rows of one chunk then fall on 8 different bank groups.
template <int D>
__device__ __forceinline__ int swizzle(int r) {
  constexpr int n = D / 32, z = n % 8 == 0 ? 8 : n % 4 == 0 ? 4 : n % 2 == 0 ? 2 : 1;
  return (r / (8 / z)) & (z - 1);
}

__device__ __forceinline__ int64_t cta_of(int64_t u, int64_t U, int64_t P) {
  int64_t c = (u * P) / U;
  while (c + 1 < P && ((c + 1) * U) / P <= u) ++c;
  while (c > 0 && (c * U) / P > u) --c;
  return c;
}

// Units of one (tile, head) of a sequence: at least one, which writes the rows that see nothing.
template <int ROWS>
__device__ __forceinline__ int tile_units(const Args& a, const Seq& s, int tile, int& unit0) {
  const int rows = s.nq * a.ratio, i0 = tile * ROWS / a.ratio, i1 = (min((tile + 1) * ROWS, rows) - 1) / a.ratio;
  int lo, hi;
  visible(a, s, i0, i1, lo, hi);
  unit0 = lo / kUnitTokens;
  return max(1, (hi + kUnitTokens - 1) / kUnitTokens - unit0);
}

template <int ROWS>
__device__ __forceinline__ int64_t seq_units(const Args& a, int b) {
  const Seq s = load_seq(a, b);
  const int tiles = (s.nq * a.ratio + ROWS - 1) / ROWS;
  int64_t n = 0;
  int unit0;
  for (int i = 0; i < tiles; ++i) n += tile_units<ROWS>(a, s, i, unit0);
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
  __shared__ uint32_t s_mask[kSplitWarps][C::kStages];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;

  // ---- this CTA's share [u, u1) of the units, and the sequence it begins in ----
  const int per = (a.batch + kSplitThreads - 1) / kSplitThreads;
  const int my0 = min((int)threadIdx.x * per, a.batch), my1 = min(my0 + per, a.batch);
  int64_t mine = 0;
  for (int b = my0; b < my1; ++b) mine += seq_units<ROWS>(a, b);
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
  const int64_t P = min((int64_t)gridDim.x, U), cta = blockIdx.x;
  if (cta >= P) return;
  int64_t u = cta * U / P;
  const int64_t u1 = (cta + 1) * U / P;
  if (u >= before && u < before + mine) {
    int64_t base = before;
    int b = my0;
    for (;; ++b) {
      const int64_t n = seq_units<ROWS>(a, b);
      if (u < base + n) break;
      base += n;
    }
    s_seq = b;
    s_base = base;
  }
  __syncthreads();
  int b = s_seq;
  int64_t off = u - s_base;

  const uint32_t ring = smem_addr(smem) + warp * (C::kStages * C::kStage);
  float* merge = reinterpret_cast<float*>(smem);
  // the scale runs of 8 tokens are 16 * groups bytes: `groups` 16-byte pieces
  const int groups = EXACT ? GT : a.groups;
  const int sc_run = lane / groups, sc_part = lane - sc_run * groups;
  const bool sc_mine = lane < 4 * groups;

  while (u < u1) {
    const Seq seq = load_seq(a, b);
    const int rows = seq.nq * a.ratio, tiles = (rows + ROWS - 1) / ROWS;
    int tile = 0, unit0 = 0, n_units = 0;
    int64_t in_tile = off;  // off counts from the sequence's first unit
    for (; tile < tiles; ++tile) {
      n_units = tile_units<ROWS>(a, seq, tile, unit0);
      if (in_tile < (int64_t)n_units * a.kv_heads) break;
      in_tile -= (int64_t)n_units * a.kv_heads;
    }
    if (tile == tiles) {  // past this sequence's last unit
      ++b;
      off = 0;
      continue;
    }
    const int head = (int)(in_tile / n_units), first = (int)(in_tile - (int64_t)head * n_units);
    const int count = (int)min((int64_t)(n_units - first), u1 - u);
    const int64_t tile_u0 = u - first;

    // ---- the tile's queries: B fragments, and per column (query row) its logit factor and visible range ----
    uint32_t qf[NT][CH][4];
    float qs[NT][2];
    int last[NT][2], past[NT][2];  // a column sees the tokens past < j <= last
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int row = tile * ROWS + nt * 8 + g;
      const bool in = row < rows;
      const int i = in ? row / a.ratio : 0;
      const char* src = static_cast<const char*>(a.q) +
                        2 * ((seq.q0 + i) * a.qs + (int64_t)(head * a.ratio + (in ? row - i * a.ratio : 0)) * a.qh);
      uint4 raw[CH];
#pragma unroll
      for (int c = 0; c < CH; ++c)
        raw[c] = in ? __ldg(reinterpret_cast<const uint4*>(src + 2 * (32 * c + 8 * t))) : make_uint4(0, 0, 0, 0);
      float mx = 0.f;
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        float f[8];
        unpack8(raw[c], a.bf16, f);
#pragma unroll
        for (int k = 0; k < 8; ++k) mx = fmaxf(mx, fabsf(f[k]));
      }
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      const int ex = (int)(__float_as_uint(mx) >> 23) - 127;  // the row's largest magnitude becomes 2^7 .. 2^8
      const int sh = mx == 0.f || ex == 128 ? 0 : min(7 - ex, 126);
      const float up = __uint_as_float((uint32_t)(sh + 127) << 23);
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        float f[8];
        unpack8(raw[c], a.bf16, f);
#pragma unroll
        for (int k = 0; k < 4; ++k) qf[nt][c][k] = pack2_f16(f[k] * up, f[k + 4] * up);
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int s2 = __shfl_sync(0xffffffffu, sh, 4 * (2 * t + j));
        qs[nt][j] = a.scale_log2 * __uint_as_float((uint32_t)(127 - s2) << 23);
        const int r2 = tile * ROWS + nt * 8 + 2 * t + j;
        const int pos = seq.len - seq.nq + r2 / a.ratio;
        last[nt][j] = r2 >= rows ? -1 : a.causal ? min(pos, seq.len - 1) : seq.len - 1;
        past[nt][j] = a.window > 0 ? max(pos - a.window, -1) : -1;
      }
    }
    // every query of the tile sees the tokens (all_past, all_last]
    const int i0 = tile * ROWS / a.ratio, i1 = (min((tile + 1) * ROWS, rows) - 1) / a.ratio;
    const int all_last = a.causal ? seq.len - seq.nq + i0 : seq.len - 1;
    const int all_past = a.window > 0 ? seq.len - seq.nq + i1 - a.window : -1;

    float O[CH][2][NT][4];
    float ref[NT][2], sum[NT][2], mx[NT][2];
    int vexp = -24;  // the smallest exponent of an f16
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int j = 0; j < 2; ++j) ref[nt][j] = mx[nt][j] = kNoMax, sum[nt][j] = 0.f;
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int z = 0; z < 2; ++z)
#pragma unroll
          for (int i = 0; i < 4; ++i) O[c][z][nt][i] = 0.f;
    }

    const int tok0 = (unit0 + first) * kUnitTokens + warp * 32;
    const int32_t* pages = a.table + (int64_t)b * a.table_stride;
    // the page of this lane's token of step k, -1 where it has none
    auto page_of = [&](int k) {
      const int j = tok0 + k * kUnitTokens + lane;
      if (k >= count || j >= seq.len) return -1;
      const int p = __ldg(pages + (j >> a.page_log2));
      return p >= 0 && (int64_t)p < a.pages ? p : -1;
    };
    auto issue = [&](int k, int page) {
      if (k < count) {
        const uint32_t st = ring + (k % C::kStages) * C::kStage;
        const int tok = tok0 + k * kUnitTokens;
        const int in_page = (1 << a.page_log2) - 1;
        const uint32_t have = __ballot_sync(0xffffffffu, page >= 0);
        if (lane == 0) s_mask[warp][k % C::kStages] = have;
        // this lane's token as a row of the cache
        const int64_t line = ((((int64_t)page * a.kv_heads + head)) << a.page_log2) + ((tok + lane) & in_page);
#pragma unroll
        for (int i = 0; i < CH; ++i) {
          const int p = lane + 32 * i, r = p / CH, c = p - r * CH;
          const int64_t ln = __shfl_sync(0xffffffffu, line, r);
          const bool ok = (have >> r) & 1u;
          const int64_t src = ok ? ln * (D / 2) + c * 16 : 0;
          const uint32_t dst = st + (r * CH + (c ^ swizzle<D>(r))) * 16;
          cp_async16(dst, a.k4 + src, ok ? 16 : 0);
          cp_async16(dst + C::kKV, a.v4 + src, ok ? 16 : 0);
        }
        const int r8 = (8 * sc_run) & 31;
        const int64_t ln = __shfl_sync(0xffffffffu, line, r8);
        if (sc_mine) {
          const bool ok = (have >> r8) & 1u;
          const int64_t src = ok ? ln * groups + sc_part * 8 : 0;
          const uint32_t dst = st + 2 * C::kKV + lane * 16;
          cp_async16(dst, a.k_scale + src, ok ? 16 : 0);
          cp_async16(dst + C::kSc, a.v_scale + src, ok ? 16 : 0);
        }
      }
      cp_async_commit();
    };

    // The scales of group z of this lane's four tokens (g, g + 8, g + 16, g + 24).
    auto scales = [&](const __half* sc, int z, float (&f)[4]) {
      const int at = EXACT ? z : z / a.cpg;
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] = __half2float(sc[(g + 8 * i) * groups + at]);
    };

    auto consume = [&](int k, auto masked) {
      constexpr bool MASKED = decltype(masked)::value;
      const int slot = k % C::kStages, tok = tok0 + k * kUnitTokens;
      const uint32_t st = ring + slot * C::kStage;
      const uint8_t* sp = smem + warp * (C::kStages * C::kStage) + slot * C::kStage;
      const __half* ks = reinterpret_cast<const __half*>(sp + 2 * C::kKV);
      const __half* vs = reinterpret_cast<const __half*>(sp + 2 * C::kKV + C::kSc);
      const uint32_t have = MASKED ? s_mask[warp][slot] : 0xffffffffu;
      float S[2][NT][4];
#pragma unroll
      for (int z = 0; z < GT; ++z) {
        float acc[2][NT][4] = {};
#pragma unroll
        for (int cc = 0; cc < CPG; ++cc) {
          const int c = z * CPG + cc;
          uint32_t w[4], e[4][4];
          ldmatrix_x4(st + (lane * CH + (c ^ swizzle<D>(lane))) * 16, w);
#pragma unroll
          for (int i = 0; i < 4; ++i) expand(w[i], e[i]);
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              mma_f16(acc[h][nt], e[2 * h][0], e[2 * h + 1][0], e[2 * h][1], e[2 * h + 1][1], qf[nt][c][0], qf[nt][c][1]);
              mma_f16(acc[h][nt], e[2 * h][2], e[2 * h + 1][2], e[2 * h][3], e[2 * h + 1][3], qf[nt][c][2], qf[nt][c][3]);
            }
        }
        float f[4];
        scales(ks, z, f);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              S[h][nt][i] = z == 0 ? acc[h][nt][i] * f[2 * h + i / 2] : fmaf(acc[h][nt][i], f[2 * h + i / 2], S[h][nt][i]);
      }
      // the largest exponent of this step's v_scale; what is not finite or not visible to any row does not count
      uint32_t big = 0;
      {
        const bool mine_in = !MASKED || ((have >> lane) & 1u);
        for (int z = 0; z < groups; ++z) {
          const uint32_t bits = __half_as_ushort(vs[lane * groups + z]) & 0x7fffu;
          if (mine_in && bits < 0x7c00u) big = max(big, bits);
        }
        big = __reduce_max_sync(0xffffffffu, big);
      }
      const int ve = big ? (int)(__float_as_uint(__half2float(__ushort_as_half((unsigned short)big))) >> 23) - 127 : -24;
      bool over = false;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            S[h][nt][i] *= qs[nt][i & 1];
            if (MASKED) {
              const int r = h * 16 + (i / 2) * 8 + g, j = tok + r;
              if (!((have >> r) & 1u) || j > last[nt][i & 1] || j <= past[nt][i & 1]) S[h][nt][i] = -INFINITY;
            }
            over |= S[h][nt][i] > mx[nt][i & 1] + 8.f;
          }
      if (__any_sync(0xffffffffu, over) || ve > vexp) {
        vexp = max(vexp, ve);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            float m = mx[nt][j];
#pragma unroll
            for (int h = 0; h < 2; ++h) m = fmaxf(m, fmaxf(S[h][nt][j], S[h][nt][2 + j]));
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
            const float now = m + (float)vexp, f = exp2_approx(ref[nt][j] - now);
            mx[nt][j] = m;
            ref[nt][j] = now;
            sum[nt][j] *= f;
#pragma unroll
            for (int c = 0; c < CH; ++c)
#pragma unroll
              for (int z = 0; z < 2; ++z) O[c][z][nt][j] *= f, O[c][z][nt][2 + j] *= f;
          }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            S[h][nt][i] = exp2_approx(S[h][nt][i] - ref[nt][i & 1]);
            sum[nt][i & 1] += S[h][nt][i];
          }
#pragma unroll
      for (int z = 0; z < GT; ++z) {
        float f[4];
        scales(vs, z, f);
        uint32_t p[2][NT][2];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 2; ++i) {  // a masked token's scale may be anything, a NaN too: 0 stays 0
              const float p0 = S[h][nt][2 * i], p1 = S[h][nt][2 * i + 1], v = f[2 * h + i];
              p[h][nt][i] = movmatrix_trans(pack2_f16(MASKED && p0 == 0.f ? 0.f : p0 * v, MASKED && p1 == 0.f ? 0.f : p1 * v));
            }
#pragma unroll
        for (int cc = 0; cc < CPG; ++cc) {
          const int c = z * CPG + cc;
          uint32_t w[4], e[4][4];
          ldmatrix_x4_trans(st + C::kKV + (lane * CH + (c ^ swizzle<D>(lane))) * 16, w);
#pragma unroll
          for (int i = 0; i < 4; ++i) expand(w[i], e[i]);
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              mma_f16(O[c][0][nt], e[2 * h][0], e[2 * h][1], e[2 * h + 1][0], e[2 * h + 1][1], p[h][nt][0], p[h][nt][1]);
              mma_f16(O[c][1][nt], e[2 * h][2], e[2 * h][3], e[2 * h + 1][2], e[2 * h + 1][3], p[h][nt][0], p[h][nt][1]);
            }
        }
      }
    };

    // ---- this warp's 32 tokens of each unit ----
#pragma unroll
    for (int k = 0; k < C::kStages - 1; ++k) issue(k, page_of(k));
    int page = page_of(C::kStages - 1);
    for (int k = 0; k < count; ++k) {
      issue(k + C::kStages - 1, page);
      page = page_of(k + C::kStages);
      cp_async_wait<C::kStages - 1>();
      __syncwarp();
      const int tok = tok0 + k * kUnitTokens;
      const bool full = s_mask[warp][k % C::kStages] == 0xffffffffu && tok > all_past && tok + 31 <= all_last;
      if (full)
        consume(k, std::false_type{});
      else
        consume(k, std::true_type{});
      __syncwarp();
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
      const int row = tile * ROWS + r, i = row / a.ratio;
      const int64_t tk = seq.q0 + i;
      const int h = head * a.ratio + row - i * a.ratio;
      const float inv = l == 0.f ? 0.f : 1.f / l;
      uint2 w;
      w.x = pack2(l == 0.f ? 0.f : o.x * inv, l == 0.f ? 0.f : o.y * inv, a.bf16);
      w.y = pack2(l == 0.f ? 0.f : o.z * inv, l == 0.f ? 0.f : o.w * inv, a.bf16);
      *reinterpret_cast<uint2*>(static_cast<char*>(a.out) + 2 * (tk * a.os + h * a.oh + d)) = w;
      if (a.lse && d == 0) a.lse[tk * a.ls + h] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
    };
    // parts: [cta][whether the tile began in an earlier CTA][ROWS][D sums, then the reference and the sum]
    constexpr int PART = ROWS * (D + 2);
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
      // the tile's counter belongs to the CTA that it begins in; whoever arrives last adds the parts in order
      const int64_t c0 = cta_of(tile_u0, U, P), c1 = cta_of(tile_u0 + n_units - 1, U, P);
      __threadfence();
      __syncthreads();
      if (threadIdx.x == 0) {
        const bool done = atomicAdd(a.counters + c0, 1u) == (uint32_t)(c1 - c0);
        if (done) a.counters[c0] = 0;  // ready for the next launch
        s_last = done;
        __threadfence();
      }
      __syncthreads();
      if (s_last) {
        for (int at = threadIdx.x; at < live * (D / 4); at += kSplitThreads) {
          const int r = at / (D / 4), d = 4 * (at - r * (D / 4));
          float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
          float l = 0.f, m = kNoMax;
          for (int64_t c = c0; c <= c1; ++c) {
            const float* q = a.partials + (c * 2 + (c == c0 ? 1 : 0)) * PART;
            const float m1 = __ldcg(q + ROWS * D + r), l1 = __ldcg(q + ROWS * D + ROWS + r);
            const float4 v = __ldcg(reinterpret_cast<const float4*>(q + r * D + d));
            const float now = fmaxf(m, m1), f = exp2_approx(m - now), f1 = exp2_approx(m1 - now);
            o.x = fmaf(v.x, f1, o.x * f), o.y = fmaf(v.y, f1, o.y * f);
            o.z = fmaf(v.z, f1, o.z * f), o.w = fmaf(v.w, f1, o.w * f);
            l = fmaf(l1, f1, l * f);
            m = now;
          }
          store(r, d, o, m, l);
        }
      }
    }
    __syncthreads();  // the ring and the small arrays are free again
    u += count;
    off += count;
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
