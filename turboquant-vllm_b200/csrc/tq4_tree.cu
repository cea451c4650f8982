// Trees of drafted tokens: the mask of a tree, and the entry point of attention with such masks over the packed cache.
#include "tq4_attention.cuh"

namespace tq4 {
namespace {

constexpr int kMaskThreads = 256;
constexpr int kMaskNodes = 2048;  // drafts of a sequence whose parents a block keeps in shared memory

struct MaskArgs {
  const int32_t* parents;
  const int32_t* starts;  // [seqs + 1]
  int64_t rows;
  int seqs, words;
  int32_t* mask;   // [rows][words]
  int32_t* depth;  // [rows]
  int* err_flag;
};

// Row j of a sequence: bits of j, its parent, the parent's parent, ...  A thread makes one word of a row: it walks up the whole
// branch (parents in shared memory) and keeps the bits of its word, so a row's words are made side by side and stored once.
// Bound by the walk's latency, about 30 cycles a step.
// blockIdx.x: sequence (the one behind the last stands for rows of no sequence), blockIdx.y: share of its words
__global__ void __launch_bounds__(kMaskThreads) tree_mask_kernel(const MaskArgs a) {
  __shared__ int s_parent[kMaskNodes];
  const int seq = blockIdx.x;
  const int64_t rows = a.rows;
  int64_t r0, r1;
  if (seq < a.seqs) {
    r0 = min(max((int64_t)a.starts[seq], (int64_t)0), rows);
    r1 = min(max((int64_t)a.starts[seq + 1], r0), rows);
  } else {
    r0 = min(max((int64_t)a.starts[a.seqs], (int64_t)0), rows);
    r1 = rows;
  }
  const int64_t n = r1 - r0, items = n * a.words;
  const bool held = n <= kMaskNodes;
  if (seq < a.seqs && held) {
    for (int i = threadIdx.x; i < (int)n; i += kMaskThreads) s_parent[i] = a.parents[r0 + i];
    __syncthreads();
  }
  const int32_t* parents = a.parents + r0;
  for (int64_t i = (int64_t)blockIdx.y * kMaskThreads + threadIdx.x; i < items; i += (int64_t)gridDim.y * kMaskThreads) {
    const int64_t j = i / a.words;
    const int w = (int)(i - j * a.words);
    unsigned bits = 0;
    int depth = -1;
    if (seq < a.seqs) {
      // (a parent is an earlier draft: the walk goes down in j and ends)
      int64_t k = j;
      while (true) {
        if ((k >> 5) == w) bits |= 1u << (k & 31);
        ++depth;
        const int p = held ? s_parent[k] : parents[k];
        if (p < 0 || p >= k) {  // the first of its branch; what is no earlier draft is reported and ends the walk
          if ((p < -1 || p >= k) && a.err_flag) atomicOr(a.err_flag, TQ4_DEV_BAD_TREE);
          break;
        }
        k = p;
      }
      if (j >= 32ll * a.words && w == 0 && a.err_flag) atomicOr(a.err_flag, TQ4_DEV_BAD_TREE);  // (its own bit has no room)
    }
    a.mask[r0 * a.words + i] = (int32_t)bits;
    if (w == 0) a.depth[r0 + j] = depth;
  }
}

}  // namespace
}  // namespace tq4

extern "C" int tq4_tree_mask(const int32_t* parents, const int32_t* query_start_loc, int64_t num_rows, int num_seqs, int words,
                             int32_t* mask, int32_t* depth, int* err_flag, void* stream) {
  using namespace tq4;
  if (num_rows < 0 || num_rows > 0x7fffffff || num_seqs < 0 || words <= 0) return TQ4_ERR_INVALID_ARG;
  if (num_rows == 0) return TQ4_OK;
  if (!parents || !query_start_loc || !mask || !depth) return TQ4_ERR_INVALID_ARG;
  const MaskArgs a{parents, query_start_loc, num_rows, num_seqs, words, mask, depth, err_flag};
  // (an even share of the words for every block, as if the sequences were alike)
  const int64_t items = (num_rows * words + num_seqs) / (num_seqs > 0 ? num_seqs : 1);
  int64_t shares = (items + kMaskThreads - 1) / kMaskThreads;
  if (shares > 64) shares = 64;
  if (launch_kernel(tree_mask_kernel, dim3((unsigned)num_seqs + 1, (unsigned)shares), dim3(kMaskThreads), 0, (cudaStream_t)stream, false,
                    a) != cudaSuccess)
    return TQ4_ERR_CUDA;
  TQ4_CHECK_LAUNCH();
  return TQ4_OK;
}

extern "C" size_t tq4_tree_attention_workspace_bytes(int64_t max_query_rows, int num_q_heads, int num_kv_heads, int head_dim) {
  using namespace tq4;
  AttnShape sh{};
  if (max_query_rows <= 0 || !supported_head_dim(head_dim) || !make_shape(sh, num_q_heads, num_kv_heads, head_dim) || sh.G > 128) return 0;
  int64_t vectors = 32 * max_query_rows * num_q_heads;
  if (vectors > kPrefillSplitVectors) vectors = kPrefillSplitVectors;
  // (a vector set of Hq and the alignment of the image on top: tree_tc_splits counts whole sets)
  return 128 + prefill_tc_image_bytes(head_dim) + (size_t)(vectors + num_q_heads) * (head_dim + 1) * 4;
}

extern "C" int tq4_tree_attention(
    const void* q, int q_dtype, int64_t num_rows, int num_seqs, int num_q_heads, int num_kv_heads, int head_dim, int64_t q_token_stride,
    int64_t q_head_stride, const uint8_t* cache, int64_t cache_block_stride, int64_t cache_token_stride, int64_t num_blocks,
    int block_size, const int32_t* block_table, int64_t bt_stride, int64_t bt_width, const int32_t* seq_lens, const int32_t* query_start_loc,
    int64_t max_seq_len, const int32_t* tree_mask, int64_t tree_mask_stride, int tree_mask_words, const float* k_centroids,
    int n_k_centroids, const float* v_centroids, int n_v_centroids, const float* rotation, float sm_scale, int sliding_window, void* out,
    int out_dtype, int64_t out_token_stride, int64_t out_head_stride, float* lse_out, int out_rotated, void* workspace,
    size_t workspace_bytes, int* err_flag, void* stream) {
  using namespace tq4;
  if (num_rows < 0 || num_rows > 0x7fffffff || num_seqs < 0 || block_size <= 0 || num_blocks < 0 || bt_width < 0 || tree_mask_words < 0)
    return TQ4_ERR_INVALID_ARG;
  if (!supported_head_dim(head_dim) || q_dtype < 0 || q_dtype > 2 || out_dtype < 0 || out_dtype > 2) return TQ4_ERR_UNSUPPORTED;
  if (n_k_centroids <= 0 || n_k_centroids > TQ4_MAX_CENTROIDS || n_v_centroids <= 0 || n_v_centroids > TQ4_MAX_CENTROIDS)
    return TQ4_ERR_UNSUPPORTED;
  AttnArgs a{};
  if (!make_shape(a.sh, num_q_heads, num_kv_heads, head_dim)) return TQ4_ERR_UNSUPPORTED;
  if (num_rows == 0) return TQ4_OK;
  if (!q || !cache || !block_table || !seq_lens || !query_start_loc || (!tree_mask && tree_mask_words) || !k_centroids || !v_centroids ||
      !rotation || !out || !workspace)
    return TQ4_ERR_INVALID_ARG;
  if (((uintptr_t)cache & 3) || (cache_token_stride & 3) || (cache_block_stride & 3) || ((uintptr_t)workspace & 15) ||
      cache_token_stride < row_data_bytes(num_kv_heads, head_dim))
    return TQ4_ERR_INVALID_ARG;
  if (workspace_bytes < tq4_tree_attention_workspace_bytes(num_rows, num_q_heads, num_kv_heads, head_dim)) return TQ4_ERR_WORKSPACE;
  a.sh.rows = (int)num_rows;
  a.sh.num_seqs = num_seqs;
  a.q = q;
  a.q_dtype = q_dtype;
  a.q_token_stride = q_token_stride;
  a.q_head_stride = q_head_stride;
  a.cache = cache;
  a.cache_block_stride = cache_block_stride;
  a.cache_token_stride = cache_token_stride;
  a.num_blocks = num_blocks;
  a.block_size = block_size;
  a.block_table = block_table;
  a.bt_stride = bt_stride;
  a.seq_lens = seq_lens;
  a.query_start_loc = query_start_loc;
  a.table_width = bt_width;
  a.max_keys = bt_width * block_size;
  if (max_seq_len > 0 && max_seq_len < a.max_keys) a.max_keys = max_seq_len;
  a.tree_mask = tree_mask;
  a.tree_stride = tree_mask_stride;
  a.tree_words = tree_mask_words;
  a.k_centroids = k_centroids;
  a.v_centroids = v_centroids;
  a.n_k_centroids = n_k_centroids;
  a.n_v_centroids = n_v_centroids;
  a.rotation = rotation;
  a.scale_log2e = sm_scale * 1.4426950408889634f;
  a.lut_scale_k = lut_scale(head_dim, n_k_centroids);
  a.lut_scale_v = lut_scale(head_dim, n_v_centroids);
  a.causal = 1;
  a.sliding_window = sliding_window > 0 ? sliding_window : 0;
  a.out = out;
  a.out_dtype = out_dtype;
  a.out_token_stride = out_token_stride;
  a.out_head_stride = out_head_stride;
  a.lse_out = lse_out;
  a.out_rotated = out_rotated;
  a.err_flag = err_flag;
  if (!prefill_tc_supported(a)) return TQ4_ERR_UNSUPPORTED;
  cudaStream_t st = (cudaStream_t)stream;
  // scratch: Pi's image, then the partials of a call cut along the keys
  uint8_t* image = reinterpret_cast<uint8_t*>(((uintptr_t)workspace + 127) & ~(uintptr_t)127);
  float* part_o = reinterpret_cast<float*>(image + prefill_tc_image_bytes(head_dim));
  const int64_t room = (int64_t)((uintptr_t)workspace + workspace_bytes) - (int64_t)(uintptr_t)part_o;
  const int splits = tree_tc_splits(a, room / ((int64_t)num_q_heads * (head_dim + 1) * 4) - 1);
  const bool to_parts = splits > 1;
  float* part_m = part_o + (size_t)splits * num_rows * num_q_heads * head_dim;
  prof_begin(TQ4_PROF_ATTENTION, st);
  const int rc = launch_tree_tc(a, st, splits, to_parts, image, part_o, part_m);
  prof_end(TQ4_PROF_ATTENTION, st);
  if (rc != TQ4_OK || !to_parts) return rc;
  CombineArgs c{};
  c.world = splits;
  c.part_o = part_o;
  c.part_m = part_m;
  c.rows = (int)num_rows;
  c.Hq = num_q_heads;
  c.rotation = rotation;
  c.out = out;
  c.out_dtype = out_dtype;
  c.out_token_stride = out_token_stride;
  c.out_head_stride = out_head_stride;
  c.lse_out = lse_out;
  c.out_rotated = out_rotated;
  prof_begin(TQ4_PROF_COMBINE, st);
  const int rc2 = launch_combine(c, head_dim, st, true);
  prof_end(TQ4_PROF_COMBINE, st);
  return rc2;
}
