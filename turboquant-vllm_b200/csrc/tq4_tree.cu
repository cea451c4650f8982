// Trees of drafted tokens: the mask of a tree, and the entry point of attention with such masks over the packed cache.
#include "tq4_attention.cuh"

namespace tq4 {
namespace {

constexpr int kMaskThreads = 128;
constexpr int kMaskBytes = 96 * 1024;  // words of a block's rows
constexpr int kMaskNodes = 2048;  // drafts of a sequence whose parents a block keeps in shared memory

struct MaskArgs {
  const int32_t* parents;
  const int32_t* starts;  // [seqs + 1]
  int64_t rows;
  int seqs, words;
  int block_rows;         // rows of a block
  int32_t* mask;   // [rows][words]
  int32_t* depth;  // [rows]
  int* err_flag;
};

// Row j of a sequence: bits of j, its parent, the parent's parent, ...  A thread walks up from one row, with the parents and the rows'
// words in shared memory; a block then stores its rows' words side by side.  Bound by the walk, 0.1 us a step (the parents from shared memory,
// behind the bit that went into it before): 64 trees of 200 to 512 drafts and chains of up to 37 7.0 us, 2.6 of them the launch and its
// round trips, 1.1 zeroing and storing 16 words a row; 3.7 without a parent, 53 with chains of 509.  (A thread for each word of a row
// walked every branch once a word: 10.3 us.)
// blockIdx.x: sequence (the one behind the last stands for rows of no sequence), blockIdx.y: share of its rows
__global__ void __launch_bounds__(kMaskThreads) tree_mask_kernel(const MaskArgs a) {
  extern __shared__ unsigned s_bits[];  // [rows of a block][pitch]
  __shared__ int s_parent[kMaskNodes];
  const int seq = blockIdx.x, tid = threadIdx.x;
  int64_t r0 = min(max((int64_t)a.starts[seq], (int64_t)0), a.rows), r1 = a.rows;
  if (seq < a.seqs) r1 = min(max((int64_t)a.starts[seq + 1], r0), a.rows);
  const int n = (int)(r1 - r0), words = a.words, pitch = words | 1;  // (odd: rows lie in different banks)
  const bool held = n <= kMaskNodes;
  const int32_t* parents = a.parents + r0;
  if (seq < a.seqs && held && (int)blockIdx.y * a.block_rows < n)
    for (int i = tid; i < n; i += kMaskThreads) s_parent[i] = parents[i];
  for (int b0 = (int)blockIdx.y * a.block_rows; b0 < n; b0 += (int)gridDim.y * a.block_rows) {
    const int rows = min(a.block_rows, n - b0);
    for (int i = tid; i < rows * pitch; i += kMaskThreads) s_bits[i] = 0u;
    __syncthreads();
    for (int i = tid; i < rows; i += kMaskThreads) {
      const int j = b0 + i;
      int depth = -1;
      if (seq < a.seqs) {
        unsigned* mine = s_bits + i * pitch;
        int k = j;
        while (true) {  // (a parent is an earlier draft: the walk goes down in k and ends)
          if ((k >> 5) < words) mine[k >> 5] |= 1u << (k & 31);
          ++depth;
          const int p = held ? s_parent[k] : parents[k];
          if (p < 0 || p >= k) {  // the first of its branch; what is no earlier draft is reported and ends the walk
            if ((p < -1 || p >= k) && a.err_flag) atomicOr(a.err_flag, TQ4_DEV_BAD_TREE);
            break;
          }
          k = p;
        }
        if ((j >> 5) >= words && a.err_flag) atomicOr(a.err_flag, TQ4_DEV_BAD_TREE);  // (its own bit has no room)
      }
      a.depth[r0 + j] = depth;
    }
    __syncthreads();
    int32_t* out = a.mask + (r0 + b0) * words;
    for (int i = tid; i < rows * words; i += kMaskThreads) {
      const int row = i / words;
      out[i] = (int32_t)s_bits[row * pitch + (i - row * words)];
    }
    __syncthreads();
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
  MaskArgs a{parents, query_start_loc, num_rows, num_seqs, words, 0, mask, depth, err_flag};
  // as many rows as there are threads, where their words fit
  const int row_bytes = (words | 1) * 4;
  a.block_rows = kMaskBytes / row_bytes < kMaskThreads ? kMaskBytes / row_bytes : kMaskThreads;
  if (a.block_rows < 1) return TQ4_ERR_UNSUPPORTED;
  if ((int64_t)a.block_rows > num_rows) a.block_rows = (int)num_rows;
  const int smem = a.block_rows * row_bytes;
  if (!ensure_dynamic_smem<tree_mask_kernel>(kMaskBytes)) return TQ4_ERR_CUDA;
  // (blocks for sequences of as many drafts as there are bits)
  int64_t shares = (32 * (int64_t)words + a.block_rows - 1) / a.block_rows;
  if (shares > 64) shares = 64;
  if (launch_kernel(tree_mask_kernel, dim3((unsigned)num_seqs + 1, (unsigned)shares), dim3(kMaskThreads), (size_t)smem, (cudaStream_t)stream, false,
                    a) != cudaSuccess)
    return TQ4_ERR_CUDA;
  TQ4_CHECK_LAUNCH();
  return TQ4_OK;
}

extern "C" size_t tq4_tree_attention_workspace_bytes(int64_t max_query_rows, int num_q_heads, int num_kv_heads, int head_dim) {
  using namespace tq4;
  AttnShape sh{};
  if (max_query_rows <= 0 || !supported_head_dim(head_dim) || !make_shape(sh, num_q_heads, num_kv_heads, head_dim) || sh.G > 128) return 0;
  // (parts only where the rows leave SMs idle: two CTAs of 128 rows each an SM)
  int64_t vectors = 64 * max_query_rows * num_q_heads;
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
    size_t workspace_bytes, int mode, int* err_flag, void* stream) {
  using namespace tq4;
  if (mode != 0 && mode != 3 && mode != 4) return TQ4_ERR_INVALID_ARG;
  if (mode == 4 && q_dtype != TQ4_BF16) return TQ4_ERR_UNSUPPORTED;
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
  // (a window that every position of a row of the table lies within is none: positions minus it stay in 32 bits)
  a.sliding_window = sliding_window > 0 && sliding_window < bt_width * block_size + 32 * (int64_t)tree_mask_words ? sliding_window : 0;
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
  // The kernel for few drafts takes 128 / G rows of a sequence a CTA, the other twice that: the first, unless sequences fill more than one of
  // its CTAs on average, which would dequantise every tile again.  64 sequences of 4096 tokens, 32 / 8 heads of 128, few / other:
  // 32 drafts (128 rows) 339 / 451 us, 64 drafts 662 / 616, 128 drafts 1261 / 1079 (single terms: 265 / 421, 518 / 509, 984 / 912).
  // (Offsets are on the device: the average is over sequences with and without drafts.  One tree of many drafts among empty ones
  // goes to the first.)
  const bool few = tree_few_supported(a) && num_rows * a.sh.G <= 128 * (int64_t)(num_seqs > 0 ? num_seqs : 1);
  // queries, weights and (few drafts) Pi as single fp16 terms: the caller's choice only, as in tq4_paged_attention.  What that adds to the output's error
  // grows with the scores and passes the rounding of a bf16 output (1.7e-3 of relative 2-norm): 5e-4, 9e-4, 1.9e-3 and 2.8e-3 at
  // scores with a standard deviation of 1.7, 7, 28 and 55 (4096 keys, head_dim 128), where two terms have 1e-4, 1.4e-4, 2.7e-4 and 4e-4.
  const bool fast = mode == 4;
  const int64_t slots = room / ((int64_t)num_q_heads * (head_dim + 1) * 4) - 1;
  const int splits = few ? tree_few_splits(a, slots) : tree_tc_splits(a, slots);
  const bool to_parts = splits > 1;
  float* part_m = part_o + (size_t)splits * num_rows * num_q_heads * head_dim;
  prof_begin(TQ4_PROF_ATTENTION, st);
  const int rc = few ? launch_tree_few(a, st, fast, splits, to_parts, image, part_o, part_m)
                     : launch_tree_tc(a, st, fast, splits, to_parts, image, part_o, part_m);
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
  c.out_rotated = few || out_rotated;  // (that kernel's parts are un-rotated already)
  prof_begin(TQ4_PROF_COMBINE, st);
  const int rc2 = launch_combine(c, head_dim, st, true);
  prof_end(TQ4_PROF_COMBINE, st);
  return rc2;
}
