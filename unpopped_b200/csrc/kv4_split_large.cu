// kv4_split_large.cu — the split kernel (kv4_split.cuh) for head sizes from 160 to 256. 256 has a variant a group size;
// the others take every group as groups of 32 that share scales.
#include "kv4_split.cuh"

namespace up {
namespace kv4 {

int split_attention_large(const Args& a, int dim, int ctas, cudaStream_t s) {
  if (dim == 160) return launch_split<160, 1, 1, false>(a, ctas, s);
  if (dim == 192) return launch_split<192, 1, 1, false>(a, ctas, s);
  if (dim == 224) return launch_split<224, 1, 1, false>(a, ctas, s);
  if (a.cpg == 1) return launch_split<256, 1, 1, true>(a, ctas, s);
  if (a.cpg == 2) return launch_split<256, 2, 1, true>(a, ctas, s);
  if (a.cpg == 4) return launch_split<256, 4, 1, true>(a, ctas, s);
  return launch_split<256, 8, 1, true>(a, ctas, s);
}

}  // namespace kv4
}  // namespace up
