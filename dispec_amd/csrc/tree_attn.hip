// Attention of a drafted tree over the paged cache.
#include "dsp_common.h"
#include "dsp_internal.h"

namespace {

constexpr int kMaskThreads = 256;

// One thread a node: its mask row is its own bit and its ancestors'.  Parents come before their
// children, so the chain up ends; a node whose parent is not an earlier one is a root.
__global__ __launch_bounds__(kMaskThreads) void tree_mask_kernel(
    const int32_t* __restrict__ parents, const int32_t* __restrict__ cu_q, int64_t rows,
    int32_t max_q_len, int32_t words, uint32_t* __restrict__ mask) {
  const int b = blockIdx.y, i = blockIdx.x * kMaskThreads + threadIdx.x;
  const int at = cu_q[b], n = min(cu_q[b + 1] - at, max_q_len);
  if (at < 0 || i >= n || int64_t(at) + i >= rows) return;
  uint32_t* row = mask + (int64_t(at) + i) * words;
  int a = i, w = i >> 5;
  uint32_t bits = 0;
  for (int x = words - 1; x > w; --x) row[x] = 0u;
  while (a >= 0) {
    for (; (a >> 5) < w; --w) {
      row[w] = bits;
      bits = 0;
    }
    bits |= 1u << (a & 31);
    const int p = parents ? parents[at + a] : a - 1;
    a = p < a ? p : -1;
  }
  for (; w >= 0; --w) {
    row[w] = bits;
    bits = 0;
  }
}

}  // namespace

extern "C" int dsp_tree_mask(const int32_t* parents, const int32_t* cu_q, int64_t num_rows,
                             int32_t B, int32_t max_q_len, int32_t mask_words, int32_t* mask,
                             dsp_stream_t stream) {
  DSP_HOST_CHECK(cu_q && mask, DSP_EINVAL);
  DSP_HOST_CHECK(B >= 0 && B <= 65535 && max_q_len >= 0 && num_rows >= 0 &&
                     int64_t(mask_words) * 32 >= max_q_len,
                 DSP_EINVAL);
  if (B == 0 || max_q_len == 0) return DSP_OK;
  const dim3 grid(unsigned((max_q_len + kMaskThreads - 1) / kMaskThreads), unsigned(B));
  tree_mask_kernel<<<grid, kMaskThreads, 0, static_cast<hipStream_t>(stream)>>>(
      parents, cu_q, num_rows, max_q_len, mask_words, reinterpret_cast<uint32_t*>(mask));
  return dsp_launch_status();
}

extern "C" size_t dsp_paged_tree_workspace_bytes(int32_t B, int32_t Hq, int32_t KVH, int32_t D,
                                                 int32_t max_q_len, int32_t max_ctx) {
  if (B <= 0 || KVH <= 0 || Hq <= 0 || Hq % KVH != 0 || max_q_len <= 0 || max_ctx <= 0) return 0;
  return dsp_detail::generic_workspace_bytes(
      B, Hq, D, max_q_len, max_ctx,
      dsp_paged_mq_partition_tokens(B, Hq, KVH, D, max_q_len, max_ctx));
}

extern "C" int dsp_paged_tree_attention(
    const void* q, int64_t q_stride_t, int64_t q_stride_h, const void* k_cache,
    const void* v_cache, int64_t num_slots, int64_t kv_stride_slot, int64_t kv_stride_head,
    const int32_t* block_table, int64_t bt_stride, int32_t block_size, const int32_t* cu_q,
    const int32_t* ctx_lens, const int32_t* tree_mask, int32_t mask_words, int32_t B, int32_t Hq,
    int32_t KVH, int32_t D, float scale, int32_t max_q_len, int32_t max_ctx, void* workspace,
    size_t workspace_bytes, void* out, int64_t o_stride_t, int64_t o_stride_h, int32_t dtype,
    int32_t* err_count, dsp_stream_t stream) {
  DSP_HOST_CHECK(q && k_cache && v_cache && block_table && cu_q && ctx_lens && tree_mask && out,
                 DSP_EINVAL);
  DSP_HOST_CHECK(B >= 0 && B <= 65535 && Hq > 0 && KVH > 0 && KVH <= 65535 && Hq % KVH == 0 &&
                     max_q_len >= 0 && max_ctx >= 0 && num_slots >= 0 &&
                     int64_t(mask_words) * 32 >= max_q_len,
                 DSP_EINVAL);
  DSP_HOST_CHECK(dtype == DSP_BF16 || dtype == DSP_F16 || dtype == DSP_F32, DSP_EUNSUPPORTED);
  DSP_HOST_CHECK(dsp_detail::generic_head_dim(D), DSP_EUNSUPPORTED);
  DSP_HOST_CHECK(dsp_is_pow2(block_size) && bt_stride * block_size >= max_ctx, DSP_EINVAL);
  if (B == 0 || max_q_len == 0) return DSP_OK;
  const int64_t es = dtype == DSP_F32 ? 4 : 2;
  DSP_HOST_CHECK(dsp_aligned(q, es) && dsp_aligned(k_cache, es) && dsp_aligned(v_cache, es) &&
                     dsp_aligned(out, es),
                 DSP_EALIGN);
  const size_t need = dsp_paged_tree_workspace_bytes(B, Hq, KVH, D, max_q_len, max_ctx);
  DSP_HOST_CHECK(workspace_bytes >= need && (need == 0 || workspace != nullptr), DSP_EWORKSPACE);
  DSP_HOST_CHECK(need == 0 || dsp_aligned(workspace, 16), DSP_EALIGN);
  return dsp_detail::generic_attention(
      q, q_stride_t, q_stride_h, k_cache, v_cache, num_slots, kv_stride_slot, kv_stride_head,
      block_table, bt_stride, dsp_log2i(block_size), cu_q, ctx_lens, B, Hq, KVH, D, scale,
      max_q_len, max_ctx, dsp_paged_mq_partition_tokens(B, Hq, KVH, D, max_q_len, max_ctx),
      workspace, out, o_stride_t, o_stride_h, dtype, err_count, static_cast<hipStream_t>(stream),
      reinterpret_cast<const uint32_t*>(tree_mask), mask_words);
}
