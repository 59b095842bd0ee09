// f8_walk.cuh — the forms of the 8-bit products' kernel, the choice among them, and how a form's tiles are dealt out.
//
// Nothing here needs a GPU: with __device__, __forceinline__, __umulhi, __fdividef, min and max given, a C++ compiler takes it, and
// tests/f8_walk_host.cpp looks at the schedule itself.
#pragma once

#include <stdint.h>

#include <cmath>

#include "divide.cuh"

namespace up {
namespace f8 {

constexpr int kBlock = 128;               // k a scale, and weight rows a scale
constexpr int kTile = 128 * kBlock;       // bytes of 128 rows of a block
// The tiles of an expert with more rows than some 42 MB hold (a third of L2) go by panels of 16 tiles' weights, token by token; else those of one
// tile's weights follow one another and the rows stay in L2. 8192 rows by 8192 x 8192 weights 544 us without panels, 502 with; 16384 rows
// 1177, 991; but 4096 rows 247, 255. Panels of 8 tiles 510 and 1011, of 32 524 and 1044.
constexpr int kPanel = 16;
constexpr int64_t kPanelBytes = 42 << 20;

struct Narrow {
  static constexpr bool kWide = false;
  static constexpr int kCtas = 1, kTokens = 32, kStep = 16, kWeights = 128;  // of a tile; tokens go in steps
  static constexpr int kGroup = 4;                                  // blocks of an accumulator slot
  static constexpr int kDBlock = 32;                                // columns of tensor memory a block
  static constexpr int kBBytes = 32 * kBlock, kStages = 10;
  static constexpr int kXWarp = 4, kEpi0 = 5;                       // the warp that loads the tokens, the first of the epilogue's
  static constexpr int kEpiWarps = 4, kSums = 32;                   // sums a thread
  static constexpr int kMinBlocks = 8, kJoinBlocks = 12;            // of an owner's share of a tile, at least; blocks that joining parts takes
  static constexpr int kFactors = 32;                               // of a block, through shared memory: the tokens'
};
template <int CTAS, int WEIGHTS>
struct Wide {
  static constexpr bool kWide = true;
  static constexpr int kCtas = CTAS, kTokens = 128 * CTAS, kStep = kTokens, kWeights = WEIGHTS;
  static constexpr int kGroup = 1;
  static constexpr int kDBlock = WEIGHTS;
  static constexpr int kBBytes = WEIGHTS / CTAS * kBlock, kStages = 204800 / (kTile + kBBytes) / 2 * 2;
  static constexpr int kXWarp = 0, kEpi0 = 4;
  static constexpr int kEpiWarps = 8, kSums = WEIGHTS / 2;
  static constexpr int kMinBlocks = 16, kJoinBlocks = WEIGHTS == 256 ? 24 : 12;
  // none through shared memory: a thread's row is one token, so it loads its own, some blocks ahead. Measured against a warp that hands them
  // over as for the narrow forms: 8192 rows by 8192 x 8192 weights 543 against 580 us, 2048 by 4096 x 4096 (128 columns) 50 against 59
  static constexpr int kFactors = 0;
};

// A unit is one group of k of one tile; tiles are numbered by expert, then weight rows, then tokens (or by panels), so the tiles that
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
  int groups, tb, panel_rows;             // a tile's; tiles over the weight rows; Args'
  int base, more;                         // shares of the rest: base + 1 units for the first `more` owners, base for the others
  int left;                               // units of this owner's share, from r.g0 of tile r.t on
  int whole_t, whole_left, owners;        // the next of the tiles dealt out, and how many are left
  Run r;

  __device__ __forceinline__ int first_unit(int owner) const { return owner * base + min(owner, more); }
  __device__ __forceinline__ int owner_of(int unit) const {
    return unit < more * (base + 1) ? unit / (base + 1) : more + (unit - more * (base + 1)) / base;
  }
  template <typename A>
  __device__ __forceinline__ Walk(const A& a, const int* start_, const int* begin_, int owner, int owners_)
      : start(start_), begin(begin_), groups(a.groups), tb(a.tb), panel_rows(a.panel_rows), left(0), owners(owners_) {
    const int tiles = start[a.experts];
    const int rounds = (int)a.by_owners(tiles);
    int rest = tiles - rounds * owners;
    // Shared only where that saves an owner more blocks than the joining of parts takes: else whole as well. With 256 columns a part is 128 KB
    // a CTA, written and read again by all at one time: 512 rows by 8192 x 8192 weights 53 us shared, 41 whole; 8 blocks: 53, 12 to 32: 41.
    const int blocks = groups * C::kGroup;
    int most = min(owners, rest * blocks / C::kMinBlocks);
    // As many owners for each tile, where its groups divide by them, few owners are left idle and few blocks more come to one: nobody then joins two
    // tiles (1 row by 8192 x 8192 weights, 64 tiles: 18.0 us on 148 owners, 16.1 on 128; but 40 tiles of 5120 x 5120: 11.0 on 148, 11.6 on 120.
    // 48 tiles of 16 groups, 6144 x 8192, on 144: 15.6, on 148: 15.4).
    const int parts = (int)__fdividef(most + 0.5f, (float)max(rest, 1));  // most / rest: both are below 2^12
    if (parts >= 2 && groups % parts == 0 && 6 * parts * rest >= 5 * most && blocks * (most - parts * rest) <= 8 * parts * most)
      most = parts * rest;
    if (blocks * (most - rest) <= C::kJoinBlocks * most) rest = 0;
    const int units = rest * groups, sharers = rest > 0 ? most : 1;
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
      int place;
      if (C::kWide && rows > panel_rows) {
        const int panel = at / (kPanel * wide), in = at - panel * (kPanel * wide), across = min(kPanel, tb - panel * kPanel);
        place = in / across;
        r.tb = panel * kPanel + in - place * across;
      } else {
        r.tb = at / wide;
        place = at - r.tb * wide;
      }
      const int each = ((rows + wide - 1) / wide + C::kStep - 1) / C::kStep * C::kStep, first = place * each;
      r.m0 += first;
      r.n = min(each, rows - first);
    }
    return true;
  }
  __device__ __forceinline__ void passed() {  // the run was taken over
    if (left > 0) ++r.t, r.g0 = 0;
  }
};

enum Form { kNarrow, kWide256, kPair256, kWide128 };

// The form that takes the least time by a model: a fixed part (launch, first loads, output), then so many microseconds for each block of k of
// the tiles of one owner. It was fitted before the tiles of many rows went by panels and those of few by equal numbers of owners, and knows of
// neither: a tile's parts are counted here as if every owner had one share of them. Measured since, on 86 calls of 1 to 65536 rows, dense and by
// expert, by 512 x 1024 to 28672 x 8192 weights, the choice takes 0.4 % longer than the fastest form in the mean, 9 % at most (2048 rows by
// 1024 x 8192 weights: 32.4 us, where a pair takes 29.8). Without one of the forms the best of the others takes 1.0 to 5.4 % longer in the mean,
// 12 to 47 % at most. (A form of 64 tokens as columns was the fastest by 4 to 12 % for some calls of 64 to 256 rows, by 0.2 % in the mean; one of
// 256 tokens by 128 weights never was.) Measured, us, in the order of the table:
//   rows by 2048 x 1024 weights:   512: 9.3, 9.4, 9.8, 6.6;     8192: 76, 30.5, 31.0, 31.6
//   rows by 8192 x 8192 weights:   1: 16.5, 26.4, 30.2, 24.2;   128: 34.4, 28.6, 30.4, 24.3;  512: 102, 40.5, 39.3, 50.8;  8192: 1604, 539, 512, 853
//   128 experts' 4096 x 2048:      512: 147, 165, 248, 188;     8192: 303, 210, 319, 269;     65536: 1732, 723, 758, 893
inline Form form_of(int64_t m, int64_t experts, int64_t n, int64_t kb, int ctas) {
  struct Cost {
    int tokens, weights, ctas, least, join;  // of a tile; Walk's
    double fixed, block;
  };
  static const Cost cost[4] = {{Narrow::kTokens, Narrow::kWeights, 1, Narrow::kMinBlocks, Narrow::kJoinBlocks, 3.8, 0.214},
                               {128, 256, 1, Wide<1, 256>::kMinBlocks, Wide<1, 256>::kJoinBlocks, 3.4, 0.653},
                               {256, 256, 2, Wide<2, 256>::kMinBlocks, Wide<2, 256>::kJoinBlocks, 4.2, 0.600},
                               {128, 128, 1, Wide<1, 128>::kMinBlocks, Wide<1, 128>::kJoinBlocks, 3.5, 0.415}};
  const double used = (double)(m < experts ? m : experts), per = m / used;  // experts that have rows, at most; rows of each
  int best = 0;
  double least = 0;
  for (int i = 0; i < 4; ++i) {
    const Cost& c = cost[i];
    const int owners = ctas / c.ctas;
    // a ragged group's last tile is half full in the mean
    const double wide = experts == 1 ? (double)((m + c.tokens - 1) / c.tokens) : per / c.tokens + 0.5 > 1 ? per / c.tokens + 0.5 : 1;
    const double tiles = wide * used * (double)((n + c.weights - 1) / c.weights), rounds = floor(tiles / owners), rest = tiles - rounds * owners;
    const double shares = rest * kb / c.least < owners ? rest * kb / c.least : owners;
    const double blocks = rest == 0                                ? 0
                          : kb * (shares - rest) <= c.join * shares ? (double)kb
                                                                    : kb * rest / shares + c.join;
    const double us = c.fixed + c.block * (rounds * kb + blocks);
    if (i == 0 || us < least) best = i, least = us;
  }
  return (Form)best;
}

}  // namespace f8
}  // namespace up
