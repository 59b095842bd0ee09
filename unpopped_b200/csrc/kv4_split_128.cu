// kv4_split_128.cu — the split kernel (kv4_split.cuh) for heads of 128.
#include "kv4_split.cuh"

namespace up {
namespace kv4 {

int split_attention_128(const Args& a, int rows, int ctas, cudaStream_t s) {
  if (rows == 8) {
    if (a.cpg == 1) return launch_split<128, 1, 1, true>(a, ctas, s);
    if (a.cpg == 2) return launch_split<128, 2, 1, true>(a, ctas, s);
    return launch_split<128, 4, 1, true>(a, ctas, s);
  }
  if (a.cpg == 1) return launch_split<128, 1, 2, true>(a, ctas, s);
  if (a.cpg == 2) return launch_split<128, 2, 2, true>(a, ctas, s);
  return launch_split<128, 4, 2, true>(a, ctas, s);
}

}  // namespace kv4
}  // namespace up
