// kv4_split_small.cu — the split kernel (kv4_split.cuh) for head sizes 32, 64 and 96.
#include "kv4_split.cuh"

namespace up {
namespace kv4 {

int split_attention_small(const Args& a, int dim, int rows, int ctas, cudaStream_t s) {
  if (dim == 32) return launch_split<32, 1, 1, true>(a, ctas, s);
  if (dim == 64) {
    if (a.cpg == 1) return rows == 8 ? launch_split<64, 1, 1, true>(a, ctas, s) : launch_split<64, 1, 2, true>(a, ctas, s);
    return rows == 8 ? launch_split<64, 2, 1, true>(a, ctas, s) : launch_split<64, 2, 2, true>(a, ctas, s);
  }
  if (a.cpg == 1) return rows == 8 ? launch_split<96, 1, 1, true>(a, ctas, s) : launch_split<96, 1, 2, true>(a, ctas, s);
  return rows == 8 ? launch_split<96, 3, 1, true>(a, ctas, s) : launch_split<96, 3, 2, true>(a, ctas, s);
}

}  // namespace kv4
}  // namespace up
