// kv4_attention.cu — attention over the paged 4-bit cache: argument checks, workspace and the choice of kernel.
// The operator's other sources, which its revision hash covers through this line (build.py --sources):
// FNV-1a 64 of divide.cuh, kv4.cuh, kv4_attention.cuh, kv4_prompt.cu, kv4_split.cuh, kv4_split_128.cu, kv4_split_large.cu, kv4_split_small.cu: 68c4624a8b9ca682
#include "kv4_attention.cuh"

namespace up {
namespace kv4 {

int split_attention(const Args& a, int dim, int rows, int ctas, cudaStream_t s) {
  if (dim <= 96) return split_attention_small(a, dim, rows, ctas, s);
  if (dim == 128) return split_attention_128(a, rows, ctas, s);
  return split_attention_large(a, dim, ctas, s);
}

// f32 parts of the split tiles: two a CTA (one tile begins earlier, one ends later), each rows x (dim + 4).
static size_t partial_bytes(int64_t ctas, int64_t rows, int64_t dim) {
  return (size_t)ctas * 2 * rows * (dim + 4) * sizeof(float);
}

static int split_ctas() { return sm_count() * 4 < kMaxCtas ? sm_count() * 4 : kMaxCtas; }

}  // namespace kv4
}  // namespace up

using namespace up;
using namespace up::kv4;

extern "C" size_t up_sm100_kv4_attention_workspace_bytes(int64_t tokens, int64_t q_heads, int64_t batch,
                                                         int64_t kv_heads, int64_t dim) {
  if (tokens <= 0 || batch <= 0 || kv_heads <= 0 || q_heads <= 0 || dim <= 0 || dim > kMaxDim) return kCounterBytes;
  const int64_t rows = (tokens + batch - 1) / batch * (q_heads / kv_heads);
  return kCounterBytes + partial_bytes(split_ctas(), split_rows(rows, dim), dim);
}

extern "C" int up_sm100_kv4_attention(const void* q, int dtype, int64_t tokens, int64_t q_heads, int64_t q_stride_t,
                                      int64_t q_stride_h, const up_kv4_cache* cache, const int32_t* block_table,
                                      int64_t table_stride, int64_t table_width, const int32_t* seq_lens,
                                      const int32_t* cu_q, int64_t batch, int causal, int64_t window, float scale,
                                      void* out, int64_t out_stride_t, int64_t out_stride_h, float* lse,
                                      int64_t lse_stride_t, void* workspace, size_t workspace_bytes, void* stream) {
  const int ok = check_cache(cache);
  if (ok != UP_OK) return ok;
  UP_CHECK_ARG(tokens >= 0 && q_heads >= 0 && batch >= 0 && window >= 0 && table_width >= 0 && table_stride >= 0);
  UP_CHECK_ARG(q_stride_t >= 0 && q_stride_h >= 0);
  if (dtype != UP_EK_BF16 && dtype != UP_EK_F16) return UP_ERR_UNSUPPORTED;
  if (q_heads % cache->kv_heads != 0 || batch > kMaxTokens) return UP_ERR_UNSUPPORTED;
  UP_CHECK_ARG(cu_q != nullptr || tokens == batch);
  if (tokens == 0 || q_heads == 0 || batch == 0) return UP_OK;
  const int64_t ratio = q_heads / cache->kv_heads;
  if (tokens > kMaxTokens / ratio || table_width > kMaxTokens / cache->page) return UP_ERR_UNSUPPORTED;
  UP_CHECK_ARG(q != nullptr && out != nullptr && seq_lens != nullptr && workspace != nullptr);
  UP_CHECK_ARG(block_table != nullptr || table_width == 0);
  UP_CHECK_ARG(batch <= 1 || table_stride >= table_width);
  UP_CHECK_ARG((q_heads <= 1 || out_stride_h >= cache->dim) && (tokens <= 1 || out_stride_t >= cache->dim));
  UP_CHECK_ARG(lse == nullptr || tokens <= 1 || lse_stride_t >= q_heads);
  // the stride of an extent of one is never used
  if (tokens == 1) q_stride_t = out_stride_t = lse_stride_t = 0;
  if (q_heads == 1) q_stride_h = out_stride_h = 0;
  // 16-byte loads of q, 8-byte stores of out
  if (!aligned(q, 16) || q_stride_t % 8 != 0 || q_stride_h % 8 != 0) return UP_ERR_UNSUPPORTED;
  if (!aligned(out, 8) || out_stride_t % 4 != 0 || out_stride_h % 4 != 0) return UP_ERR_UNSUPPORTED;
  UP_CHECK_ARG(aligned(workspace, 256));
  UP_CHECK_ARG(workspace_bytes >= up_sm100_kv4_attention_workspace_bytes(tokens, q_heads, batch, cache->kv_heads, cache->dim));
  Args a{};
  a.q = q, a.out = out, a.lse = lse, a.bf16 = dtype == UP_EK_BF16;
  a.qs = q_stride_t, a.qh = q_stride_h, a.os = out_stride_t, a.oh = out_stride_h, a.ls = lse_stride_t;
  a.tokens = tokens;
  a.k4 = static_cast<const uint8_t*>(cache->k), a.v4 = static_cast<const uint8_t*>(cache->v);
  a.k_scale = static_cast<const __half*>(cache->k_scale), a.v_scale = static_cast<const __half*>(cache->v_scale);
  if (cache->pages == 0) {  // every token is left out and nothing is read; copies of no bytes still name an address
    a.k4 = a.v4 = static_cast<const uint8_t*>(q);
    a.k_scale = a.v_scale = static_cast<const __half*>(q);
  }
  a.pages = (uint32_t)cache->pages, a.kv_heads = (int)cache->kv_heads, a.ratio = (int)ratio, a.page_log2 = log2_of(cache->page);
  a.cpg = (int)(cache->group / 32), a.groups = (int)(cache->dim / cache->group);
  a.table = block_table, a.table_stride = table_stride, a.table_width = table_width;
  a.lens = seq_lens, a.cu = cu_q, a.batch = (int)batch, a.causal = causal != 0, a.by_ratio = Divide32(ratio);
  a.window = (int)(window > kMaxTokens ? kMaxTokens : window);
  a.scale_log2 = scale * 1.44269504088896341f;
  a.header = static_cast<uint32_t*>(workspace);
  a.counters = reinterpret_cast<uint32_t*>(static_cast<char*>(workspace) + kHeaderBytes);
  a.partials = reinterpret_cast<float*>(static_cast<char*>(workspace) + kCounterBytes);
  const int64_t per = (tokens + batch - 1) / batch * ratio;  // query rows a sequence and key/value head
  if (many_rows(per, batch * cache->kv_heads, cache->dim, sm_count()))
    return prompt_attention(a, (int)cache->dim, static_cast<cudaStream_t>(stream));
  const int rows = split_rows(per, cache->dim);
  return split_attention(a, (int)cache->dim, rows, split_ctas(), static_cast<cudaStream_t>(stream));
}

UP_DEFINE_REVISION(kv4_attention)
