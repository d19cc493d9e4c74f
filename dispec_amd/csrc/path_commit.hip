// Commit of the kept path of a drafted tree: the K and V rows of its nodes, every layer, move to
// the places right behind the context, in place.  The reference keeps a prefix of a chain, whose
// rows need no move (dispec/spec/speculative.py:135, BlockManager.truncate); the nodes of a
// tree's path are not neighbours.
//
// Node a of a tree whose first token is the context's token `base` lies at position base + a; the
// j-th node of the path, path[j], goes to base + j.  A path goes down the tree, so path[j] >
// path[j - 1] and path[j] >= j: a row that is read is never one that was written before it, if the
// rows move in order.  One thread takes one 16-byte column of a (sequence, layer, K or V) through
// all of its rows, so nothing but its own program order is needed: kBatch rows are read before the
// first of them is written.  Rows in their place already are not touched.
// What it reads and writes, and a chain of four loads before it (the path, the table's ids, the
// rows): 32 trees that keep up to 8 nodes, 36 layers of 8 heads of 128 in bf16, 8.8 us; one tree in
// 24 layers of 2 heads of 64 3.5 us.
#include "dsp_common.h"

namespace {

constexpr int kThreads = 256;
constexpr int kBatch = 8;
constexpr int kMaxPath = 1024;

template <int VEC>
__global__ __launch_bounds__(kThreads) void commit_path_kernel(
    char* k_pool, char* v_pool, int64_t layer_stride, int64_t slot_stride, int64_t num_slots,
    int32_t num_layers, int32_t cols, int32_t log2_bs, const int32_t* __restrict__ bt,
    int64_t bt_stride, int32_t bt_cols, const int32_t* __restrict__ cu_q,
    const int32_t* __restrict__ ctx_lens, const int32_t* __restrict__ path, int64_t path_stride,
    int32_t path_cols, const int32_t* __restrict__ num, int32_t* __restrict__ err_count) {
  using V = typename dsp_vec<VEC>::type;
  __shared__ int64_t s_src[kMaxPath], s_dst[kMaxPath];  // byte offsets of the rows; < 0: no move
  __shared__ int32_t s_bad;
  const int b = blockIdx.y, tid = threadIdx.x;
  const int n = cu_q[b + 1] - cu_q[b], base = ctx_lens[b] - n;
  const int m = min(num[b], path_cols - 1);
  if (m <= 0) return;
  if (tid == 0) s_bad = m + 1;
  __syncthreads();
  const bool reports = blockIdx.x == 0 && err_count;
  // (a path that does not go down its tree: nothing from there on is moved)
  for (int j = 1 + tid; j <= m; j += kThreads) {
    const int a = path[b * path_stride + j], prev = path[b * path_stride + j - 1];
    if (base < 0 || a <= prev || a < j || a >= n || prev < j - 1) atomicMin(&s_bad, j);
  }
  __syncthreads();
  const int end = min(m, s_bad - 1);
  if (s_bad <= m && tid == 0 && reports) atomicAdd(err_count, 1);
  auto slot_of = [&](int pos) -> int64_t {
    const int blk = pos >> log2_bs;
    if (blk >= bt_cols) return -1;
    const int64_t s = (int64_t(bt[b * bt_stride + blk]) << log2_bs) + (pos & ((1 << log2_bs) - 1));
    return s >= 0 && s < num_slots ? s : -1;
  };
  for (int j = 1 + tid; j <= end; j += kThreads) {
    const int a = path[b * path_stride + j];
    int64_t src = -1, dst = -1;
    if (a != j) {
      src = slot_of(base + a);
      dst = slot_of(base + j);
      if ((src < 0 || dst < 0) && reports) atomicAdd(err_count, 1);
    }
    const bool moves = src >= 0 && dst >= 0;
    s_src[j - 1] = moves ? src * slot_stride : -1;
    s_dst[j - 1] = moves ? dst * slot_stride : -1;
  }
  __syncthreads();
  const int64_t item = int64_t(blockIdx.x) * kThreads + tid;
  const int64_t plane = item / cols;
  if (plane >= 2 * int64_t(num_layers)) return;
  char* const at = (plane & 1 ? v_pool : k_pool) + (plane >> 1) * layer_stride +
                   (item - plane * cols) * VEC;
  for (int j0 = 0; j0 < end; j0 += kBatch) {
    V row[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i)
      if (j0 + i < end && s_src[j0 + i] >= 0) row[i] = *reinterpret_cast<const V*>(at + s_src[j0 + i]);
#pragma unroll
    for (int i = 0; i < kBatch; ++i)
      if (j0 + i < end && s_src[j0 + i] >= 0) *reinterpret_cast<V*>(at + s_dst[j0 + i]) = row[i];
  }
}

}  // namespace

extern "C" int dsp_kv_commit_path(void* k_pool, void* v_pool, int64_t num_layers,
                                  int64_t pool_layer_stride_bytes, int64_t pool_slot_stride_bytes,
                                  int64_t num_slots, int64_t row_bytes, int32_t block_size,
                                  const int32_t* block_table, int64_t bt_stride, int32_t bt_cols,
                                  const int32_t* cu_q, const int32_t* ctx_lens,
                                  const int32_t* path, int64_t path_stride, int32_t path_cols,
                                  const int32_t* num_accepted, int32_t B, int32_t* err_count,
                                  dsp_stream_t stream) {
  DSP_HOST_CHECK(k_pool && v_pool && block_table && cu_q && ctx_lens && path && num_accepted,
                 DSP_EINVAL);
  DSP_HOST_CHECK(num_layers >= 0 && num_layers < (int64_t(1) << 24) && num_slots >= 0 &&
                     row_bytes >= 0 && B >= 0 && bt_cols >= 0 && path_cols >= 0 &&
                     dsp_is_pow2(block_size),
                 DSP_EINVAL);
  DSP_HOST_CHECK(B <= 65535 && path_cols <= kMaxPath, DSP_EUNSUPPORTED);
  if (B == 0 || num_layers == 0 || row_bytes == 0 || path_cols <= 1 || num_slots == 0)
    return DSP_OK;
  const int vec = dsp_vec_width({row_bytes, pool_layer_stride_bytes, pool_slot_stride_bytes,
                                 int64_t(reinterpret_cast<uintptr_t>(k_pool)),
                                 int64_t(reinterpret_cast<uintptr_t>(v_pool))});
  const int64_t cols = row_bytes / vec, grid = (2 * num_layers * cols + kThreads - 1) / kThreads;
  DSP_HOST_CHECK(cols < (int64_t(1) << 31) && grid < (int64_t(1) << 31), DSP_EUNSUPPORTED);
  hipStream_t s = static_cast<hipStream_t>(stream);
  auto launch = [&](auto kernel) {
    kernel<<<dim3(unsigned(grid), unsigned(B)), kThreads, 0, s>>>(
        static_cast<char*>(k_pool), static_cast<char*>(v_pool), pool_layer_stride_bytes,
        pool_slot_stride_bytes, num_slots, int32_t(num_layers), int32_t(cols),
        dsp_log2i(block_size), block_table, bt_stride, bt_cols, cu_q, ctx_lens, path, path_stride,
        path_cols, num_accepted, err_count);
    return dsp_launch_status();
  };
  switch (vec) {
    case 16: return launch(commit_path_kernel<16>);
    case 8: return launch(commit_path_kernel<8>);
    case 4: return launch(commit_path_kernel<4>);
    case 2: return launch(commit_path_kernel<2>);
    default: return launch(commit_path_kernel<1>);
  }
}
