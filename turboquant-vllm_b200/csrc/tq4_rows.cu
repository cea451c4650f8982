// Moving what the packed cache holds: pages copied, and token rows that stay moved together, in the caches of all layers at once.
//
// Both move the H (D + 8) bytes of a token row that carry data, never its padding.  They are bound by HBM where there is much to
// move (rows of 1088 bytes, 8 layers: 2048 pages copied 103 to 107 us, 5.4 TB/s; half of four contexts of 16384 moved together 112 to 116
// us, 5.0 TB/s) and by two or three dependent round trips to memory (list, block table, rows) where there is little (8 pages in 32 layers
// 3.6 us, 64 accepted branches in 32 layers 5.0 us), so a launch covers every layer.  Rows that start on 16 bytes and are a multiple of them go through shared memory by bulk copies, a row each, which
// cost a lane two instructions a row and keep whole pages in flight; others (an odd number of heads) by 8- or 4-byte loads, several a
// thread before the first is stored.
#include "tq4_common.cuh"

namespace tq4 {
namespace {

constexpr int kMaxLayers = 128;   // caches a launch takes (their addresses travel with it)
constexpr int kThreads = 256;
constexpr int kBatch = 8;         // pieces a thread has in flight
// Copies that every block compares its own with; above, a map of the pages is made first, by two more launches.  Pages of 16 rows of
// 1088 bytes, one layer: 384 copies 6.4 us compared, 8.3 by map; 512 13.2 and 8.5; 1024 29.9 and 11.2.
constexpr int kScanPairs = 384;
constexpr int kStages = 4;        // sets of rows that a block of copies has under way
constexpr uint32_t kStageBytes = 17408;  // ... of at most so many bytes, and a row a lane
constexpr int kShortKeep = 64;    // kept rows of a sequence that one block sees to

struct Caches {
  uint8_t* at[kMaxLayers];
};
struct Geometry {
  int64_t num_blocks, block_stride, token_stride;
  int block_size, row_units;  // pieces of a row
};

template <int U>
struct Piece;
template <>
struct Piece<16> { using T = uint4; };
template <>
struct Piece<8> { using T = uint2; };
template <>
struct Piece<4> { using T = uint32_t; };

__device__ __forceinline__ int64_t index_at(const void* p, int is64, int64_t i) {
  return is64 ? reinterpret_cast<const int64_t*>(p)[i] : (int64_t)reinterpret_cast<const int32_t*>(p)[i];
}
__device__ __forceinline__ void report(int* flag, int bits) {
  if (flag) atomicOr(flag, bits);
}

__device__ __forceinline__ uint32_t smem_of(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void bulk_in(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
__device__ __forceinline__ void bulk_out(void* dst, uint32_t src, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst), "r"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
// the lane's copies out of shared memory: all but the last `N` sets have been read from it / all have been written
template <int N>
__device__ __forceinline__ void bulk_wait_read() { asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void bulk_wait_all() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }
__device__ __forceinline__ void bar_init(uint32_t bar) { asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// Bounded wait for copies of this warp's own.
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity) {
  for (int it = 0; it < (1 << 22); ++it) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done) : "r"(bar), "r"(parity) : "memory");
    if (done) return true;
  }
  return false;
}
__device__ __forceinline__ void bar_fence() { asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory"); }
// The mark of a segment of rows says that they have been loaded; a bounded wait for one.
__device__ __forceinline__ void mark_set(int* mark) { asm volatile("st.release.gpu.global.s32 [%0], 1;" ::"l"(mark) : "memory"); }
__device__ __forceinline__ bool mark_wait(const int* mark) {
  for (int it = 0; it < (1 << 20); ++it) {
    int there;
    asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(there) : "l"(mark) : "memory");
    if (there) return true;
  }
  return false;
}
// marks are read like any memory, what bulk copies write is not
__device__ __forceinline__ void mark_fence() { asm volatile("fence.proxy.async.global;" ::: "memory"); }

// ======================================================================================
// Pages copied
// ======================================================================================
struct CopyArgs {
  Geometry g;
  const void* pairs;  // [n][2]: source and destination page
  int pairs_64;
  int64_t n;
  int layers, per_block;  // caches; ... of a block
  int rows;               // (bulk copies) of a stage
  const unsigned* claim;  // (many pairs) first pair with this destination, by page; ~0: none
  int* err_flag;
};

// A page may be the destination of one pair only, and no destination may be a source: with neither, the pages can be copied in any order.
// Of several pairs with one destination the first is carried out, and a pair whose source another pair writes to is not;
// both are reported.  (Decided from the list alone, so the result does not depend on the order in which blocks run.)
__global__ void __launch_bounds__(kThreads) claim_kernel(const CopyArgs a, unsigned* claim) {
  pdl_trigger();
  const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (i >= a.n) return;
  const int64_t src = index_at(a.pairs, a.pairs_64, 2 * i), dst = index_at(a.pairs, a.pairs_64, 2 * i + 1);
  if (src != dst && src >= 0 && src < a.g.num_blocks && dst >= 0 && dst < a.g.num_blocks) atomicMin(claim + dst, (unsigned)i);
}

// Whether pair (src, dst) is to be carried out; what is wrong with it is reported.  (All threads of the block.)
__device__ __forceinline__ bool pair_counts(const CopyArgs& a, int64_t pair, int64_t src, int64_t dst) {
  if (a.claim) pdl_wait();
  const bool in_range = src >= 0 && src < a.g.num_blocks && dst >= 0 && dst < a.g.num_blocks;
  if (!in_range) {
    if (threadIdx.x == 0) report(a.err_flag, TQ4_DEV_BAD_BLOCK);
    return false;
  }
  if (src == dst) return false;
  int skip = 0, clash = 0;
  if (a.claim) {
    const unsigned first = a.claim[dst];
    skip = first != (unsigned)pair;
    clash = (skip && index_at(a.pairs, a.pairs_64, 2 * (int64_t)first) != src) || a.claim[src] != ~0u;
  } else {
    for (int i = threadIdx.x; i < (int)a.n; i += blockDim.x) {
      const int64_t s = index_at(a.pairs, a.pairs_64, 2 * i), d = index_at(a.pairs, a.pairs_64, 2 * i + 1);
      if (s == d || s < 0 || s >= a.g.num_blocks) continue;
      if (d == dst && i < (int)pair) {
        skip = 1;
        clash |= s != src;
      }
      clash |= d == src;
    }
    skip = __syncthreads_or(skip);
    clash = __syncthreads_or(clash);
  }
  if (clash && threadIdx.x == 0) report(a.err_flag, TQ4_DEV_PAGE_CONFLICT);
  return !skip && !clash;
}

template <int U>
__global__ void __launch_bounds__(kThreads) copy_blocks_kernel(const __grid_constant__ Caches caches, const CopyArgs a) {
  using T = typename Piece<U>::T;
  const int groups = (a.layers + a.per_block - 1) / a.per_block;
  const int64_t pair = blockIdx.x / groups;
  const int layer0 = ((int)blockIdx.x % groups) * a.per_block, layer1 = min(a.layers, layer0 + a.per_block);
  const int64_t src = index_at(a.pairs, a.pairs_64, 2 * pair), dst = index_at(a.pairs, a.pairs_64, 2 * pair + 1);
  if (!pair_counts(a, pair, src, dst)) return;
  // ---- the page, layer by layer ---------------------------------------------------------------------------
  const int page = a.g.block_size * a.g.row_units, all = page * (layer1 - layer0);
  for (int i0 = threadIdx.x; i0 < all; i0 += kBatch * kThreads) {
    T x[kBatch];
    int64_t at[kBatch];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int i = i0 + b * kThreads;
      if (i >= all) continue;
      const int layer = i / page, r = i - layer * page, row = r / a.g.row_units;
      at[b] = (int64_t)row * a.g.token_stride + (r - row * a.g.row_units) * U;
      x[b] = *reinterpret_cast<const T*>(caches.at[layer0 + layer] + src * a.g.block_stride + at[b]);
    }
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int i = i0 + b * kThreads;
      if (i < all) *reinterpret_cast<T*>(caches.at[layer0 + i / page] + dst * a.g.block_stride + at[b]) = x[b];
    }
  }
}

// The same by bulk copies: one warp, a lane a row of the set of rows that a stage holds.  A lane stores what it loaded itself, so it
// may ask for its next row as soon as its own copy out of that place has read it.
__global__ void __launch_bounds__(32) copy_blocks_bulk_kernel(const __grid_constant__ Caches caches, const CopyArgs a) {
  extern __shared__ __align__(128) unsigned char s_rows[];
  __shared__ __align__(8) uint64_t s_bar[kStages];
  const int lane = threadIdx.x;
  const int groups = (a.layers + a.per_block - 1) / a.per_block;
  const int64_t pair = blockIdx.x / groups;
  const int layer0 = ((int)blockIdx.x % groups) * a.per_block, layers = min(a.layers - layer0, a.per_block);
  const int64_t src = index_at(a.pairs, a.pairs_64, 2 * pair), dst = index_at(a.pairs, a.pairs_64, 2 * pair + 1);
  const uint32_t bytes = (uint32_t)a.g.row_units * 16, slot = smem_of(s_rows) + lane * bytes;
  if (lane < kStages) bar_init(smem_of(&s_bar[lane]));
  bar_fence();
  __syncwarp();
  if (!pair_counts(a, pair, src, dst)) return;
  const int sets = (a.g.block_size + a.rows - 1) / a.rows, all = sets * layers;  // of a page; of the block
  const uint32_t stage = a.rows * bytes;
  auto rows_of = [&](int i) { return min(a.rows, a.g.block_size - (i % sets) * a.rows); };
  auto at = [&](int i, int64_t page) {
    return caches.at[layer0 + i / sets] + page * a.g.block_stride + (int64_t)((i % sets) * a.rows + lane) * a.g.token_stride;
  };
  auto ask = [&](int i) {
    const int n = rows_of(i);
    const uint32_t bar = smem_of(&s_bar[i % kStages]);
    if (lane == 0) bar_expect(bar, n * bytes);
    __syncwarp();
    if (lane < n) bulk_in(slot + (i % kStages) * stage, at(i, src), bytes, bar);
  };
  auto landed = [&](int i) { return bar_wait(smem_of(&s_bar[i % kStages]), (i / kStages) & 1); };
  int asked = 0;
  while (asked < min(kStages, all)) ask(asked++);
  for (int i = 0; i < all; ++i) {
    if (!__all_sync(0xffffffffu, landed(i))) {
      if (lane == 0) report(a.err_flag, TQ4_DEV_TIMEOUT);
      for (int k = i; k < asked; ++k) landed(k);  // (copies under way: the shared memory is another CTA's after this one)
      break;
    }
    if (lane < rows_of(i)) bulk_out(at(i, dst), slot + (i % kStages) * stage, bytes);
    bulk_commit();
    if (i > 0 && asked < all) {
      bulk_wait_read<1>();
      ask(asked++);
    }
  }
  bulk_wait_all();
}

// ======================================================================================
// Rows that stay, moved together
// ======================================================================================
struct CompactArgs {
  Geometry g;
  const int32_t* table;
  int64_t table_stride, table_width;
  const int32_t* first;      // [seqs] position of the first row that the list is about
  const int32_t* keep;       // [seqs][>= kept] strictly increasing, from `first`
  int64_t keep_stride;
  int keep_width;
  const int32_t* kept;       // [seqs]
  int32_t* lens_out;         // (optional) [seqs] first + kept
  int seqs, layers, per_block;
  int rows;                  // (short lists, bulk copies) of a set
  // long lists
  int segments, seg_rows;    // segments of a sequence, rows of a segment
  int* ticket;
  int* valid;                // [seqs] rows to move (0: the list is not in order)
  int* loaded;               // [layers][seqs][segments]
  int* err_flag;
};

// rows of a sequence's list; -1: more than the list has places, or fewer than none
__device__ __forceinline__ int kept_of(const CompactArgs& a, int seq) {
  const int n = a.kept[seq];
  return n < 0 || n > a.keep_width ? -1 : n;
}

// Byte offset of position `pos` of a sequence in a cache, or -1 (reported): past its row of the table, or a page out of range.
__device__ __forceinline__ int64_t row_at(const CompactArgs& a, const int32_t* table, int64_t pos) {
  const int64_t col = pos >= 0 ? pos / a.g.block_size : -1;
  if (col < 0 || col >= a.table_width) {
    report(a.err_flag, TQ4_DEV_BAD_BLOCK);
    return -1;
  }
  const int32_t page = table[col];
  if (page < 0 || page >= a.g.num_blocks) {
    report(a.err_flag, TQ4_DEV_BAD_BLOCK);
    return -1;
  }
  return page * a.g.block_stride + (pos - col * a.g.block_size) * a.g.token_stride;
}

// A block has a sequence in some layers.  Row j goes from first + keep[j] to first + j <= that: no destination is the source
// of a later row, so batches of rows in ascending order are safe as long as each is loaded before it is stored.
template <int U>
__global__ void __launch_bounds__(kThreads) compact_short_kernel(const __grid_constant__ Caches caches, const CompactArgs a) {
  using T = typename Piece<U>::T;
  __shared__ int64_t s_src[kShortKeep], s_dst[kShortKeep];
  const int groups = (a.layers + a.per_block - 1) / a.per_block;
  const int seq = (int)blockIdx.x / groups, layer0 = ((int)blockIdx.x % groups) * a.per_block;
  const int layers = min(a.layers - layer0, a.per_block), tid = threadIdx.x;
  const int n = kept_of(a, seq);
  const int32_t* keep = a.keep + seq * a.keep_stride;
  const int64_t first = a.first[seq];
  if (layer0 == 0 && tid == 0 && a.lens_out) a.lens_out[seq] = a.first[seq] + a.kept[seq];
  int bad = n < 0;
  if (tid < n) {
    const int k = keep[tid];
    bad = k < 0 || (tid > 0 && keep[tid - 1] >= k);
    s_src[tid] = s_dst[tid] = -1;
    if (!bad && k != tid) {  // (rows that stay where they are are not touched)
      const int32_t* table = a.table + seq * a.table_stride;
      s_src[tid] = row_at(a, table, first + k);
      s_dst[tid] = row_at(a, table, first + tid);
    }
  }
  if (__syncthreads_or(bad)) {  // a list out of order: reported, the sequence is left as it is
    if (tid == 0) report(a.err_flag, TQ4_DEV_KEEP_ORDER);
    return;
  }
  const int per_layer = n * a.g.row_units, all = per_layer * layers;
  for (int i0 = 0; i0 < all; i0 += kBatch * kThreads) {
    T x[kBatch];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int i = i0 + b * kThreads + tid;
      if (i >= all) continue;
      const int layer = i / per_layer, r = i - layer * per_layer, row = r / a.g.row_units;
      if (s_src[row] >= 0 && s_dst[row] >= 0)
        x[b] = *reinterpret_cast<const T*>(caches.at[layer0 + layer] + s_src[row] + (r - row * a.g.row_units) * U);
    }
    __syncthreads();
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int i = i0 + b * kThreads + tid;
      if (i >= all) continue;
      const int layer = i / per_layer, r = i - layer * per_layer, row = r / a.g.row_units;
      if (s_src[row] >= 0 && s_dst[row] >= 0)
        *reinterpret_cast<T*>(caches.at[layer0 + layer] + s_dst[row] + (r - row * a.g.row_units) * U) = x[b];
    }
    __syncthreads();
  }
}

// The same by bulk copies: one warp, a lane a row of a layer, layer by layer and in ascending order; a set of them is loaded before the
// first of it is stored.  (Accepted drafts of 64 trees of 16 in 32 layers: 9.5 us by loads of 16 bytes, most of it for dividing
// them among the threads, 5.0 us so.)
__global__ void __launch_bounds__(32) compact_short_bulk_kernel(const __grid_constant__ Caches caches, const CompactArgs a) {
  extern __shared__ __align__(128) unsigned char s_rows[];
  __shared__ __align__(8) uint64_t s_bar;
  const int lane = threadIdx.x;
  const uint32_t bar = smem_of(&s_bar), bytes = (uint32_t)a.g.row_units * 16, slot = smem_of(s_rows) + lane * bytes;
  const int groups = (a.layers + a.per_block - 1) / a.per_block;
  const int seq = (int)blockIdx.x / groups, layer0 = ((int)blockIdx.x % groups) * a.per_block;
  const int layers = min(a.layers - layer0, a.per_block);
  const int n = kept_of(a, seq);
  const int32_t* keep = a.keep + seq * a.keep_stride;
  const int32_t* table = a.table + seq * a.table_stride;
  const int64_t first = a.first[seq];
  if (lane == 0) {
    bar_init(bar);
    if (layer0 == 0 && a.lens_out) a.lens_out[seq] = a.first[seq] + a.kept[seq];
  }
  bar_fence();
  int bad = n < 0;
  for (int j = lane; j < n; j += 32) bad |= keep[j] < 0 || (j > 0 && keep[j - 1] >= keep[j]);
  if (__any_sync(0xffffffffu, bad)) {  // a list out of order: reported, the sequence is left as it is
    if (lane == 0) report(a.err_flag, TQ4_DEV_KEEP_ORDER);
    return;
  }
  const int all = n * layers;
  for (int i0 = 0, phase = 0; i0 < all; i0 += a.rows, phase ^= 1) {
    const int i = i0 + lane, layer = i / n, row = i - layer * n;
    int64_t src = -1, dst = -1;
    if (lane < a.rows && i < all && keep[row] != row) {  // (rows that stay where they are are not touched)
      src = row_at(a, table, first + keep[row]);
      dst = row_at(a, table, first + row);
    }
    const bool moves = src >= 0 && dst >= 0;
    const unsigned movers = __ballot_sync(0xffffffffu, moves);
    if (lane == 0) bar_expect(bar, __popc(movers) * bytes);
    __syncwarp();
    if (moves) {
      bulk_wait_read<0>();  // (the lane's row before is out of its place)
      bulk_in(slot, caches.at[layer0 + layer] + src, bytes, bar);
    }
    if (!__all_sync(0xffffffffu, bar_wait(bar, phase))) {
      if (lane == 0) report(a.err_flag, TQ4_DEV_TIMEOUT);
      bar_wait(bar, phase);  // (copies under way: the shared memory is another CTA's after this one)
      break;
    }
    if (moves) bulk_out(caches.at[layer0 + layer] + dst, slot, bytes);
    bulk_commit();
  }
  bulk_wait_all();
}

// Long lists, first kernel: is each in order, and the marks of the second one to zero.
__global__ void __launch_bounds__(1024) compact_check_kernel(const CompactArgs a) {
  pdl_trigger();
  const int64_t marks = (int64_t)a.layers * a.seqs * a.segments;
  for (int64_t i = (int64_t)blockIdx.x * 1024 + threadIdx.x; i < marks; i += (int64_t)gridDim.x * 1024) a.loaded[i] = 0;
  if (blockIdx.x == 0 && threadIdx.x == 0) *a.ticket = 0;
  for (int seq = blockIdx.x; seq < a.seqs; seq += gridDim.x) {
    const int n = kept_of(a, seq);
    const int32_t* keep = a.keep + seq * a.keep_stride;
    int bad = n < 0;
#pragma unroll 4
    for (int j = threadIdx.x; j < n; j += 1024) bad |= keep[j] < 0 || (j > 0 && keep[j - 1] >= keep[j]);
    bad = __syncthreads_or(bad);
    if (threadIdx.x == 0) {
      if (bad) report(a.err_flag, TQ4_DEV_KEEP_ORDER);
      a.valid[seq] = bad ? 0 : n;
      if (a.lens_out) a.lens_out[seq] = a.first[seq] + a.kept[seq];
    }
  }
}

// First place in keep[0 .. n) that holds `value` or more: a warp looks at 32 places a step.
__device__ __forceinline__ int lower_bound_warp(const int32_t* keep, int n, int value, int lane) {
  int lo = 0, hi = n;
  while (lo < hi) {
    const int step = (hi - lo + 31) / 32, at = lo + lane * step;
    const unsigned below = __ballot_sync(0xffffffffu, at < hi && keep[at] < value);
    if (below == 0) return lo;
    const int last = 31 - __clz(below);  // (in ascending order: lanes 0 .. last)
    hi = min(hi, lo + (last + 1) * step);
    lo += last * step + 1;
  }
  return lo;
}

// ... second kernel: a block has a segment of consecutive rows of a sequence in one layer.  It loads them into shared memory, says
// so, waits until every block that reads rows it is about to overwrite has said so too, and stores.  Those are blocks of
// earlier rows (keep[j] >= j) with earlier tickets: they run or have run, and none of them waits before it has loaded.  So a
// row is read once and written once, in place.
template <int U>
__global__ void __launch_bounds__(kThreads) compact_long_kernel(const __grid_constant__ Caches caches, const CompactArgs a) {
  using T = typename Piece<U>::T;
  extern __shared__ __align__(128) unsigned char s_rows[];
  __shared__ int64_t s_src[32], s_dst[32];
  __shared__ int s_ticket, s_range[2], s_stuck;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  pdl_wait();
  if (tid == 0) {
    s_ticket = atomicAdd(a.ticket, 1);
    s_stuck = 0;
  }
  __syncthreads();
  // ticket -> (segment, sequence, layer), layers fastest: the blocks to wait for have a long start
  const int per_seg = a.layers * a.seqs, seg = s_ticket / per_seg, rest = s_ticket - seg * per_seg;
  const int seq = rest / a.layers, layer = rest - seq * a.layers;
  const int j0 = seg * a.seg_rows, rows = min(a.seg_rows, a.valid[seq] - j0);
  if (rows <= 0) return;
  const int32_t* keep = a.keep + seq * a.keep_stride;
  const int64_t first = a.first[seq];
  if (tid < rows) {
    const int k = keep[j0 + tid];
    const int32_t* table = a.table + seq * a.table_stride;
    s_src[tid] = s_dst[tid] = -1;
    if (k != j0 + tid) {
      const int64_t src = row_at(a, table, first + k), dst = row_at(a, table, first + j0 + tid);
      if (src >= 0 && dst >= 0) {
        s_src[tid] = src;
        s_dst[tid] = dst;
      }
    }
  }
  __syncthreads();
  uint8_t* cache = caches.at[layer];
  const int all = rows * a.g.row_units;
  const uint32_t base = (uint32_t)__cvta_generic_to_shared(s_rows);
  for (int i = tid; i < all; i += kThreads) {
    const int row = i / a.g.row_units;
    if (s_src[row] < 0) continue;
    const uint8_t* from = cache + s_src[row] + (i - row * a.g.row_units) * U;
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(base + i * U), "l"(from), "n"(U) : "memory");
  }
  // rows k < j0 that come from the places of this block's rows
  if (warp < 2) {
    const int k = lower_bound_warp(keep, j0, warp == 0 ? j0 : j0 + rows, lane);
    if (lane == 0) s_range[warp] = k;
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncthreads();
  int* loaded = a.loaded + ((int64_t)layer * a.seqs + seq) * a.segments;
  if (tid == 0) {
    __threadfence();
    mark_set(loaded + seg);
  }
  if (s_range[0] < s_range[1]) {
    for (int s = s_range[0] / a.seg_rows + tid; s <= (s_range[1] - 1) / a.seg_rows; s += kThreads)
      if (!mark_wait(loaded + s)) s_stuck = 1;
    __threadfence();
    __syncthreads();
    if (s_stuck) {
      if (tid == 0) report(a.err_flag, TQ4_DEV_TIMEOUT);
      return;
    }
  }
  for (int i = tid; i < all; i += kThreads) {
    const int row = i / a.g.row_units;
    if (s_src[row] >= 0) *reinterpret_cast<T*>(cache + s_dst[row] + (i - row * a.g.row_units) * U) = *reinterpret_cast<const T*>(s_rows + i * U);
  }
}

// The same by bulk copies: one warp, a row a lane.  One segment in one layer a block, with a dozen blocks an SM: with several layers
// behind one another the mark's release waits for the copies out of the layer before (half of four contexts of 16384 in 8 layers:
// 129 us with up to four layers a block, 112 so).
__global__ void __launch_bounds__(32) compact_long_bulk_kernel(const __grid_constant__ Caches caches, const CompactArgs a) {
  extern __shared__ __align__(128) unsigned char s_rows[];
  __shared__ __align__(8) uint64_t s_bar;
  const int lane = threadIdx.x;
  const uint32_t bar = smem_of(&s_bar), bytes = (uint32_t)a.g.row_units * 16, slot = smem_of(s_rows) + lane * bytes;
  if (lane == 0) bar_init(bar);
  bar_fence();
  __syncwarp();
  pdl_wait();
  int ticket = 0;
  if (lane == 0) ticket = atomicAdd(a.ticket, 1);
  ticket = __shfl_sync(0xffffffffu, ticket, 0);
  const int per_seg = a.layers * a.seqs, seg = ticket / per_seg, rest = ticket - seg * per_seg;
  const int seq = rest / a.layers, layer = rest - seq * a.layers;
  const int j0 = seg * a.seg_rows, rows = min(a.seg_rows, a.valid[seq] - j0);
  if (rows <= 0) return;
  const int32_t* keep = a.keep + seq * a.keep_stride;
  const int64_t first = a.first[seq];
  int64_t src = -1, dst = -1;
  if (lane < rows) {
    const int k = keep[j0 + lane];
    const int32_t* table = a.table + seq * a.table_stride;
    if (k != j0 + lane) {
      src = row_at(a, table, first + k);
      dst = row_at(a, table, first + j0 + lane);
    }
  }
  const bool moves = src >= 0 && dst >= 0;
  const unsigned movers = __ballot_sync(0xffffffffu, moves);
  uint8_t* cache = caches.at[layer];
  if (lane == 0) bar_expect(bar, __popc(movers) * bytes);
  __syncwarp();
  if (moves) bulk_in(slot, cache + src, bytes, bar);
  // rows k < j0 that come from the places of this block's rows, and the segments that have them
  const int k0 = lower_bound_warp(keep, j0, j0, lane), k1 = lower_bound_warp(keep, j0, j0 + rows, lane);
  if (!__all_sync(0xffffffffu, bar_wait(bar, 0))) {  // no mark: nobody overwrites what has not been read
    if (lane == 0) report(a.err_flag, TQ4_DEV_TIMEOUT);
    bar_wait(bar, 0);  // (copies under way: the shared memory is another CTA's after this one)
    return;
  }
  int* loaded = a.loaded + ((int64_t)layer * a.seqs + seq) * a.segments;
  bool ok = true;
  if (lane == 0) mark_set(loaded + seg);
  if (k0 < k1)
    for (int s = k0 / a.seg_rows + lane; s <= (k1 - 1) / a.seg_rows; s += 32) ok = mark_wait(loaded + s) && ok;
  if (!__all_sync(0xffffffffu, ok)) {
    if (lane == 0) report(a.err_flag, TQ4_DEV_TIMEOUT);
    return;
  }
  mark_fence();
  if (moves) bulk_out(cache + dst, slot, bytes);
  bulk_commit();
  bulk_wait_all();
}

// Largest piece that the caches' addresses and strides, and the bytes of a row, are multiples of.
int piece_of(const Caches& c, int layers, int64_t block_stride, int64_t token_stride, int row_bytes) {
  uintptr_t all = (uintptr_t)block_stride | (uintptr_t)token_stride | (uintptr_t)row_bytes | 16;
  for (int i = 0; i < layers; ++i) all |= (uintptr_t)c.at[i];
  return all % 16 == 0 ? 16 : all % 8 == 0 ? 8 : 4;
}

// rows of a bulk copy's stage, or of a segment of a long list
int stage_rows(int row_bytes, uint32_t stage = kStageBytes) {
  const int n = (int)stage / row_bytes;
  return n < 1 ? 1 : n > 32 ? 32 : n;
}

struct CompactSpace {
  size_t ticket, valid, loaded, bytes;
  int segments;
};
CompactSpace compact_space(int layers, int seqs, int keep_width, int row_bytes) {
  CompactSpace s{};
  s.segments = (keep_width + stage_rows(row_bytes) - 1) / stage_rows(row_bytes);
  s.valid = 16;
  s.loaded = s.valid + ((size_t)seqs * 4 + 15) / 16 * 16;
  s.bytes = s.loaded + (size_t)(layers < kMaxLayers ? layers : kMaxLayers) * seqs * s.segments * 4;
  return s;
}

// caches and geometry of a call, checked
int check_caches(uint8_t* const* caches, int layers, int64_t num_blocks, int block_size, int64_t block_stride, int64_t token_stride,
                 int num_kv_heads, int head_dim) {
  if (layers < 0 || num_blocks < 0 || block_size <= 0 || num_kv_heads <= 0 || head_dim <= 0) return TQ4_ERR_INVALID_ARG;
  if (!supported_head_dim(head_dim)) return TQ4_ERR_UNSUPPORTED;
  if (layers > 0 && !caches) return TQ4_ERR_INVALID_ARG;
  if ((block_stride & 3) || (token_stride & 3) || token_stride < row_data_bytes(num_kv_heads, head_dim)) return TQ4_ERR_INVALID_ARG;
  for (int i = 0; i < layers; ++i)
    if (!caches[i] || ((uintptr_t)caches[i] & 3)) return TQ4_ERR_INVALID_ARG;
  return TQ4_OK;
}

int launch_copy_bulk(const Caches& c, CopyArgs a, cudaStream_t st) {
  const int row_bytes = a.g.row_units * 16;
  a.rows = stage_rows(row_bytes);
  if (a.rows > a.g.block_size) a.rows = a.g.block_size;
  const size_t smem = (size_t)kStages * a.rows * row_bytes;
  if (!ensure_dynamic_smem<copy_blocks_bulk_kernel>((int)smem, true)) return TQ4_ERR_CUDA;
  // Layers of a block: enough blocks to fill the GPU at few pages, and as few looks at the list as there can be at many
  const int64_t fill = 3 * (int64_t)sm_count();
  const int64_t groups = fill / a.n < 1 ? 1 : fill / a.n < a.layers ? fill / a.n : a.layers;
  a.per_block = (int)((a.layers + groups - 1) / groups);
  const int64_t blocks = a.n * ((a.layers + a.per_block - 1) / a.per_block);
  if (blocks > 0x7fffffff || (int64_t)a.per_block * a.g.block_size > 0x3fffffff) return TQ4_ERR_UNSUPPORTED;
  if (launch_kernel(copy_blocks_bulk_kernel, dim3((unsigned)blocks), dim3(32), smem, st, a.claim != nullptr, c, a) != cudaSuccess) return TQ4_ERR_CUDA;
  TQ4_CHECK_LAUNCH();
  return TQ4_OK;
}

template <int U>
int launch_copy(const Caches& c, CopyArgs a, cudaStream_t st) {
  if constexpr (U == 16)
    if (kStages * a.g.row_units * 16 <= 200 * 1024) return launch_copy_bulk(c, a, st);
  // A block moves about 32 KB: enough blocks to fill the GPU at few pages, and no more than one look at the list for each
  const int page = a.g.block_size * a.g.row_units;
  a.per_block = (kBatch * kThreads + page - 1) / page;
  if (a.per_block > a.layers) a.per_block = a.layers;
  const int64_t groups = (a.layers + a.per_block - 1) / a.per_block;
  if ((int64_t)page * a.per_block > 0x3fffffff || a.n * groups > 0x7fffffff) return TQ4_ERR_UNSUPPORTED;
  if (launch_kernel(copy_blocks_kernel<U>, dim3((unsigned)(a.n * groups)), dim3(kThreads), 0, st, a.claim != nullptr, c, a) != cudaSuccess)
    return TQ4_ERR_CUDA;
  TQ4_CHECK_LAUNCH();
  return TQ4_OK;
}

template <int U>
int launch_compact(const Caches& c, CompactArgs a, int row_bytes, cudaStream_t st) {
  if (a.keep_width <= kShortKeep) {
    if constexpr (U == 16) {
      a.rows = stage_rows(row_bytes, 2 * kStageBytes);
      const size_t smem = (size_t)a.rows * row_bytes;
      a.per_block = a.keep_width < a.rows ? a.rows / (a.keep_width > 0 ? a.keep_width : 1) : 1;  // as many layers as make a set
      if (a.per_block > a.layers) a.per_block = a.layers;
      const int64_t grid = (int64_t)a.seqs * ((a.layers + a.per_block - 1) / a.per_block);
      if (grid <= 0x7fffffff && smem <= 200 * 1024) {
        if (!ensure_dynamic_smem<compact_short_bulk_kernel>((int)smem, true)) return TQ4_ERR_CUDA;
        if (launch_kernel(compact_short_bulk_kernel, dim3((unsigned)grid), dim3(32), smem, st, false, c, a) != cudaSuccess) return TQ4_ERR_CUDA;
        TQ4_CHECK_LAUNCH();
        return TQ4_OK;
      }
    }
    // (a few rows a sequence: as many layers a block as make a batch of every thread's)
    a.per_block = kBatch * kThreads / (4 * a.g.row_units);
    if (a.per_block < 1) a.per_block = 1;
    if (a.per_block > a.layers) a.per_block = a.layers;
    const int64_t grid = (int64_t)a.seqs * ((a.layers + a.per_block - 1) / a.per_block);
    if (grid > 0x7fffffff || (int64_t)kShortKeep * a.g.row_units * a.per_block > 0x3fffffff) return TQ4_ERR_UNSUPPORTED;
    if (launch_kernel(compact_short_kernel<U>, dim3((unsigned)grid), dim3(kThreads), 0, st, false, c, a) != cudaSuccess) return TQ4_ERR_CUDA;
    TQ4_CHECK_LAUNCH();
    return TQ4_OK;
  }
  const int64_t marks = (int64_t)a.seqs * a.layers * a.segments;
  constexpr bool bulk = U == 16;
  const size_t smem = (size_t)a.seg_rows * row_bytes;
  if (marks > 0x7fffffff || smem > 200 * 1024) return TQ4_ERR_UNSUPPORTED;
  if constexpr (bulk) {
    if (!ensure_dynamic_smem<compact_long_bulk_kernel>((int)smem, true)) return TQ4_ERR_CUDA;
  } else {
    if (!ensure_dynamic_smem<compact_long_kernel<U>>((int)smem, true)) return TQ4_ERR_CUDA;
  }
  const int64_t want = (marks + 1023) / 1024 > a.seqs ? (marks + 1023) / 1024 : a.seqs, most = sm_count();
  if (launch_kernel(compact_check_kernel, dim3((unsigned)(want < most ? want : most)), dim3(1024), 0, st, false, a) != cudaSuccess)
    return TQ4_ERR_CUDA;
  TQ4_CHECK_LAUNCH();
  cudaError_t e;
  if constexpr (bulk) e = launch_kernel(compact_long_bulk_kernel, dim3((unsigned)marks), dim3(32), smem, st, true, c, a);
  else e = launch_kernel(compact_long_kernel<U>, dim3((unsigned)marks), dim3(kThreads), smem, st, true, c, a);
  if (e != cudaSuccess) return TQ4_ERR_CUDA;
  TQ4_CHECK_LAUNCH();
  return TQ4_OK;
}

}  // namespace
}  // namespace tq4

extern "C" size_t tq4_copy_blocks_workspace_bytes(int64_t n_pairs, int64_t num_blocks) {
  return n_pairs > tq4::kScanPairs && num_blocks > 0 ? (size_t)num_blocks * sizeof(unsigned) : 0;
}

extern "C" int tq4_copy_blocks(uint8_t* const* caches, int num_caches, int64_t num_blocks, int block_size, int64_t cache_block_stride,
                               int64_t cache_token_stride, int num_kv_heads, int head_dim, const void* pairs, int pairs_64,
                               int64_t n_pairs, void* workspace, size_t workspace_bytes, int* err_flag, void* stream) {
  using namespace tq4;
  const int rc = check_caches(caches, num_caches, num_blocks, block_size, cache_block_stride, cache_token_stride, num_kv_heads, head_dim);
  if (rc != TQ4_OK) return rc;
  if (n_pairs < 0 || n_pairs > 0x7fffffff) return TQ4_ERR_INVALID_ARG;
  if (n_pairs == 0 || num_caches == 0) return TQ4_OK;
  if (!pairs) return TQ4_ERR_INVALID_ARG;
  const size_t need = tq4_copy_blocks_workspace_bytes(n_pairs, num_blocks);
  if (need && (!workspace || workspace_bytes < need)) return TQ4_ERR_WORKSPACE;
  if (need && ((uintptr_t)workspace & 3)) return TQ4_ERR_INVALID_ARG;
  cudaStream_t st = (cudaStream_t)stream;
  const int row_bytes = row_data_bytes(num_kv_heads, head_dim);
  CopyArgs a{};
  a.g = Geometry{num_blocks, cache_block_stride, cache_token_stride, block_size, 0};
  a.pairs = pairs;
  a.pairs_64 = pairs_64;
  a.n = n_pairs;
  a.err_flag = err_flag;
  if (need) {
    if (cudaMemsetAsync(workspace, 0xff, need, st) != cudaSuccess) return TQ4_ERR_CUDA;
    if (launch_kernel(claim_kernel, dim3((unsigned)((n_pairs + kThreads - 1) / kThreads)), dim3(kThreads), 0, st, false, a,
                      reinterpret_cast<unsigned*>(workspace)) != cudaSuccess)
      return TQ4_ERR_CUDA;
    TQ4_CHECK_LAUNCH();
    a.claim = reinterpret_cast<const unsigned*>(workspace);
  }
  for (int l0 = 0; l0 < num_caches; l0 += kMaxLayers) {
    Caches c{};
    a.layers = num_caches - l0 < kMaxLayers ? num_caches - l0 : kMaxLayers;
    for (int i = 0; i < a.layers; ++i) c.at[i] = caches[l0 + i];
    const int u = piece_of(c, a.layers, cache_block_stride, cache_token_stride, row_bytes);
    a.g.row_units = row_bytes / u;
    const int r = u == 16 ? launch_copy<16>(c, a, st) : u == 8 ? launch_copy<8>(c, a, st) : launch_copy<4>(c, a, st);
    if (r != TQ4_OK) return r;
  }
  return TQ4_OK;
}

extern "C" size_t tq4_compact_rows_workspace_bytes(int num_caches, int num_seqs, int keep_width, int num_kv_heads, int head_dim) {
  if (num_caches <= 0 || num_seqs <= 0 || keep_width <= tq4::kShortKeep || num_kv_heads <= 0 || head_dim <= 0) return 0;
  return tq4::compact_space(num_caches, num_seqs, keep_width, tq4::row_data_bytes(num_kv_heads, head_dim)).bytes;
}

extern "C" int tq4_compact_rows(uint8_t* const* caches, int num_caches, int64_t num_blocks, int block_size, int64_t cache_block_stride,
                                int64_t cache_token_stride, int num_kv_heads, int head_dim, const int32_t* block_table,
                                int64_t bt_stride, int64_t bt_width, int num_seqs, const int32_t* starts, const int32_t* keep,
                                int64_t keep_stride, int keep_width, const int32_t* keep_lens, int32_t* seq_lens_out, void* workspace,
                                size_t workspace_bytes, int* err_flag, void* stream) {
  using namespace tq4;
  const int rc = check_caches(caches, num_caches, num_blocks, block_size, cache_block_stride, cache_token_stride, num_kv_heads, head_dim);
  if (rc != TQ4_OK) return rc;
  if (num_seqs < 0 || keep_width < 0 || bt_width < 0) return TQ4_ERR_INVALID_ARG;
  if (num_seqs == 0 || num_caches == 0) return TQ4_OK;
  if (!block_table || !starts || !keep_lens || (keep_width > 0 && !keep)) return TQ4_ERR_INVALID_ARG;
  const size_t need = tq4_compact_rows_workspace_bytes(num_caches, num_seqs, keep_width, num_kv_heads, head_dim);
  if (need && (!workspace || workspace_bytes < need)) return TQ4_ERR_WORKSPACE;
  if (need && ((uintptr_t)workspace & 15)) return TQ4_ERR_INVALID_ARG;
  cudaStream_t st = (cudaStream_t)stream;
  const int row_bytes = row_data_bytes(num_kv_heads, head_dim);
  CompactArgs a{};
  a.g = Geometry{num_blocks, cache_block_stride, cache_token_stride, block_size, 0};
  a.table = block_table;
  a.table_stride = bt_stride;
  a.table_width = bt_width;
  a.first = starts;
  a.keep = keep;
  a.keep_stride = keep_stride;
  a.keep_width = keep_width;
  a.kept = keep_lens;
  a.lens_out = seq_lens_out;
  a.seqs = num_seqs;
  a.err_flag = err_flag;
  if (need) {
    const CompactSpace s = compact_space(num_caches, num_seqs, keep_width, row_bytes);
    unsigned char* w = reinterpret_cast<unsigned char*>(workspace);
    a.segments = s.segments;
    a.seg_rows = stage_rows(row_bytes);
    a.ticket = reinterpret_cast<int*>(w + s.ticket);
    a.valid = reinterpret_cast<int*>(w + s.valid);
    a.loaded = reinterpret_cast<int*>(w + s.loaded);
  }
  for (int l0 = 0; l0 < num_caches; l0 += kMaxLayers) {
    Caches c{};
    a.layers = num_caches - l0 < kMaxLayers ? num_caches - l0 : kMaxLayers;
    for (int i = 0; i < a.layers; ++i) c.at[i] = caches[l0 + i];
    const int u = piece_of(c, a.layers, cache_block_stride, cache_token_stride, row_bytes);
    a.g.row_units = row_bytes / u;
    const int r = u == 16 ? launch_compact<16>(c, a, row_bytes, st) : u == 8 ? launch_compact<8>(c, a, row_bytes, st)
                                                                             : launch_compact<4>(c, a, row_bytes, st);
    if (r != TQ4_OK) return r;
  }
  return TQ4_OK;
}
