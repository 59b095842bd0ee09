// The 8-bit products' schedule and choice of form (unpopped_b200/csrc/f8_walk.cuh) as host code, for the tests.
#include <stdint.h>

#include <algorithm>
#include <cmath>

#define __device__
#define __host__
#define __forceinline__ inline
static inline uint32_t __umulhi(uint32_t a, uint32_t b) { return (uint32_t)(((uint64_t)a * b) >> 32); }
static inline float __fdividef(float a, float b) { return a / b; }
using std::max;
using std::min;

#include "f8_walk.cuh"

using namespace up;
using namespace up::f8;

struct Args {
  int experts, groups, tb, panel_rows;
  Divide32 by_owners, by_groups;
};

// An owner's runs, 9 numbers each (t, g0, g1, e, tb, m0, n, c0, c1; the last two -1 for a whole tile). Returns how many there are.
template <typename C>
int runs_of(int experts, const int* begin, int n, int kb, int owner, int owners, int panel_rows, int* out, int most) {
  const int nb = (n + 127) / 128, weights = C::kWeights / 128;
  int start[1025];
  Args a{experts, (kb + C::kGroup - 1) / C::kGroup, (nb + weights - 1) / weights, panel_rows, Divide32(owners),
         Divide32((kb + C::kGroup - 1) / C::kGroup)};
  start[0] = 0;
  for (int e = 0; e < experts; ++e) start[e + 1] = start[e] + (begin[e + 1] - begin[e] + C::kTokens - 1) / C::kTokens * a.tb;
  Walk<C> walk(a, start, begin, owner, owners);
  int count = 0;
  while (walk.next()) {
    const Run w = walk.r;
    walk.passed();
    if (count < most) {
      int* o = out + 9 * count;
      o[0] = w.t, o[1] = w.g0, o[2] = w.g1, o[3] = w.e, o[4] = w.tb, o[5] = w.m0, o[6] = w.n, o[7] = o[8] = -1;
      if (w.g0 > 0 || w.g1 < a.groups) o[7] = walk.owner_of(w.t * a.groups), o[8] = walk.owner_of(w.t * a.groups + a.groups - 1);
    }
    ++count;
  }
  return count;
}

extern "C" int f8_runs(int form, int experts, const int* begin, int n, int kb, int owner, int owners, int panel_rows, int* out, int most) {
  switch (form) {
    case kNarrow: return runs_of<Narrow>(experts, begin, n, kb, owner, owners, panel_rows, out, most);
    case kWide256: return runs_of<Wide<1, 256>>(experts, begin, n, kb, owner, owners, panel_rows, out, most);
    case kPair256: return runs_of<Wide<2, 256>>(experts, begin, n, kb, owner, owners, panel_rows, out, most);
    default: return runs_of<Wide<1, 128>>(experts, begin, n, kb, owner, owners, panel_rows, out, most);
  }
}
extern "C" int f8_form(int64_t m, int64_t experts, int64_t n, int64_t k, int ctas) {
  return (int)form_of(m, experts, n, (k + kBlock - 1) / kBlock, ctas);
}
extern "C" int f8_panel_rows(int64_t k) { return (int)(kPanelBytes / ((k + kBlock - 1) / kBlock * kBlock)); }
