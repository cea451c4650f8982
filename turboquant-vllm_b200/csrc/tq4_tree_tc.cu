// Attention of trees of drafted tokens over the packed TQ4 cache on the 5th-generation tensor cores, for sequences of few drafts
// (head_dim 64 to 128): the (draft, query head of the group) pairs of a sequence and KV head are the M = 128 rows of the MMAs.
//
// The mathematics is the prefill kernel's (tq4_prefill_tc.cu): queries times Pi, per 64-token tile S = Q K~^T, x key norm, masks, lazy
// online softmax, P = p * value norm, O += P V~, and O / l times Pi at the end.  What differs is what binds.  There a dequantised tile serves
// 256 rows; here it serves the rows of one tree, 8 to 128, so the bytes' way into the operands counts as much as the
// products.  Per tile of head_dim 128: 256 cycles of table lookups, 256 of operand stores and 256 (two terms: 512) of operand reads
// on the shared-memory pipe, 528 (1056) on the tensor pipe, and loads of the packed bytes, which through the load/store unit took
// as long as all of these (a dequantising warp spent 1300 - 1900 of 2800 cycles a tile issuing them).  Hence:
//   * the packed rows come by TMA boxes of 16 tokens, asked for by a warp of its own;
//   * two CTAs share an SM, of 256 tensor-memory columns and half the shared memory each: one's set-up, softmax and
//     rotations fill the other's waits.  One K~ buffer is enough: keys are written during the softmax of the tile before.  V~ has
//     two where there is room (all but two-term head_dim 128), which is worth 3 %;
//   * warps without a draft take no part.
// Measured (graph replays; in brackets single terms, mode 4; then the floor by bytes or operations), us: 8 drafts behind 1024 tokens of
// 28 / 4 heads of 128 25 (22), 0.1; 16 sequences of 300 to 8100 tokens, 5 to 24 drafts, 32 / 8 heads, fp16 108, 11.8; 64 of 4096 with
// 16 drafts, bf16 324 (225), 46; 8 of 65536 with 48 to 64 drafts, 32 / 32 heads of 96 1960 (1414), 268.  With two terms a CTA
// takes some 4300 cycles a tile at head_dim 128, where there is room for one stage of rows and one V~ buffer; the tensor pipe is busy for 39 %.
// What follows was measured with single terms.  A call of few tiles is its chain: 13 thousand cycles of search, queries and
// rotation, 6 of the first tile, 8 of un-rotation and stores.  In long ones a CTA takes 2900 cycles a tile, for
// keys and values (1200 and 1000) and the waits of the dequantising warps (750 with a wait for each of four barriers, 3050 in all and
// 231 us at 64 x 4096); the softmax warps need 1600 of them, the products 530.  The load/store pipe is
// 60 % busy with wavefronts and some 17 % more with operand reads and boxes: items of the same warps take twice as long with two
// CTAs as with one.  What took work off one of the groups moved it to the other, and none of it paid: rows of fewer than 64
// twice or four times among the 128, each with its share of a tile's columns, softmax 770 cycles a tile, 247 us instead of 234 at 64 x 4096; the
// norms by the softmax warps, 246; half of the values as well, 298; eight dequantising warps, 278; permutes for the values' table, 253.
// Roles: warps 0 - 3 softmax (a thread a row), 4 - 7 dequantisation, 8 the issuing thread, 9 the fetching lanes.  They meet at
// mbarriers; every wait is bounded as in the prefill kernel.
//
// FAST: the terms of queries, probabilities and Pi that 11 bits leave out stay out, half the tensor work.  For callers that ask for it
// (mode 4, bf16 queries): a rounding of 2^-12 of a query moves a score by that much of it, so the output's error grows with the scores,
// from 5e-4 of its norm to more than a bf16 output's own 1.7e-3 (tq4_tree.cu has figures).
#include <math_constants.h>

#include <cstdlib>

#include "tq4_tc.cuh"

namespace tq4 {
namespace {

constexpr int kSmx = 128, kDeq = 128;
constexpr int kThreads = kSmx + kDeq + 64;
constexpr int kIssueWarp = (kSmx + kDeq) / 32, kFetchWarp = kIssueWarp + 1;
constexpr int kGroup = 16;  // tokens of a box
constexpr int kMinTiles = 2;  // of a key part

template <int D, bool FAST>
struct Cfg {
  static constexpr int NC = (D + 63) / 64;                 // 64-coordinate blocks of a row
  static constexpr int NS = D / 32;                        // 16-byte segments of a packed row
  static constexpr int NIT = (kBN * NS + kDeq - 1) / kDeq;  // segments per dequantising thread
  static constexpr bool QLO = !FAST, QLO_SMEM = !FAST && D == 128;  // Q lo in shared memory where tensor memory has no room
  // tensor-memory columns: [S | P in place][Q hi][Q lo][O]
  static constexpr uint32_t kColS = 0, kColQ = 64, kColQlo = kColQ + D / 2;
  static constexpr uint32_t kColO = kColQ + (QLO && !QLO_SMEM ? D : D / 2);
  static constexpr uint32_t kCols = 256;
  static_assert(kColO + D <= kCols, "tensor memory");
  // shared memory, from a 1024-byte boundary
  static constexpr uint32_t kKv = NC * kBN * 128;          // K~ or V~ of a tile
  static constexpr int NVB = QLO_SMEM ? 1 : 2;             // V~ buffers, where there is room: values are written while the tile before is in its softmax
  // Pi's image.  Rotation: its hi term where K~ and V~ come to lie, its lo term (not FAST) where the tables do.  Un-rotation: the hi term in place of
  // the tables, which are read for the last time before the last weights are there, the lo term in place of K~ and V~.
  static constexpr uint32_t kImgPart = D * 128, kImgTerm = NC * kImgPart;
  static constexpr uint32_t kOffK = 0, kOffV = kKv, kOffLut = (1 + NVB) * kKv, kLut = 32768;
  static_assert(kImgTerm <= 2 * kKv && kImgTerm <= kLut, "room for Pi's image");
  static constexpr uint32_t kOffQlo = kOffLut + kLut;
  static constexpr uint32_t kOffRaw = kOffQlo + (QLO_SMEM ? NC * 128 * 128 : 0);
  // packed rows of a tile: K [64][D / 2], V [64][D / 2 + 16] (from the 16-byte boundary before it), the 16 bytes around each norm
  static constexpr uint32_t kVPitch = D / 2 + 16, kRawV = kBN * (D / 2), kRawKn = kRawV + kBN * kVPitch, kRawVn = kRawKn + kBN * 16;
  static constexpr uint32_t kRaw = kRawVn + kBN * 16;
  // stages of packed rows.  With two, keys and values of a tile are asked for, waited for and given back together; with one, apart, so that
  // the next keys are on their way while the values are being read
  static constexpr int kStages = QLO_SMEM ? 1 : 2;
  static constexpr bool kJoint = kStages == 2;
  static_assert(!kJoint || NVB == 2, "the keys' wait stands for the values'");
  static constexpr uint32_t kOffNorm = kOffRaw + kStages * kRaw;
  static constexpr uint32_t kSmem = kOffNorm + 2 * 2 * kBN * 4;
  // rows on their way out, padded against bank conflicts: 16-bit ones, or fp32 partials
  static constexpr uint32_t kOutPitch = 2 * D + 16, kPartPitch = 4 * D + 16;
  static_assert(128 * kPartPitch <= kOffNorm, "room for the partials");
  static constexpr int kDeqRegs = 56, kSmxRegs = 136;  // (together the 2 x 96 that the two groups of four warps are launched with)
  __host__ __device__ static constexpr uint32_t idesc(uint32_t n, bool b_mn) {  // kind::f16: fp16 operands, fp32 accumulator, M = 128
    return (1u << 4) | (b_mn ? 1u << 16 : 0u) | ((n >> 3) << 17) | ((128u >> 4) << 24);
  }
};

struct TreeArgs {
  const uint8_t* image;  // Pi's operand image
  int splits;            // key parts of a row, at most
  int slots;             // CTAs of a KV head that the parts are cut for
  int to_parts;          // leave partials for the merge kernel instead of writing the output
  float* part_o;         // [splits][rows][Hq][D] normalised, in the output's space
  float* part_m;         // [splits][rows][Hq] natural-log LSE
};

struct Bars {
  uint64_t rawk[2], rawv[2];          // packed keys and norms / values of a stage landed
  uint64_t rawk_free[2], rawv_free[2];  // ... and read
  uint64_t kready, vready[2];         // dequantising warps -> issuer: K~ / V~ (of a buffer) written
  uint64_t kfree, vfree;              // MMAs -> dequantising warps: ... read (vfree: where there is one buffer)
  uint64_t sready, pready;            // MMAs -> softmax: scores complete / softmax -> issuer: P written
  uint64_t img, aready, rot, qready;  // Pi's image landed / A operand of a rotation staged / rotation complete / queries in place
  uint64_t odone, drain;              // last MMA of the tile loop / of a dead CTA complete
};

__device__ __forceinline__ void box_load(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
               ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z) : "memory");
}

// A sequence: its rows [q0, q1) (q_end before the call's rows cut them), n blocks of RB of them; its length, and the t tiles of keys they see.
struct SeqShape {
  int q0, q_end, q1, seq_len, n, t;
};
__device__ __forceinline__ SeqShape sequence_shape(const AttnArgs& a, int RB, int s) {
  SeqShape x{0, 0, 0, 0, 0, 0};
  if (s >= a.sh.num_seqs) return x;
  x.q0 = max(__ldg(a.query_start_loc + s), 0);
  x.q_end = __ldg(a.query_start_loc + s + 1);
  x.seq_len = __ldg(a.seq_lens + s);
  x.q1 = min(x.q_end, a.sh.rows);
  x.n = x.q1 > x.q0 ? (x.q1 - x.q0 + RB - 1) / RB : 0;
  const int len = (int)min((long long)max(x.seq_len, 0), (long long)a.table_width * a.block_size), held = len - (x.q_end - x.q0);
  const int lo = a.sliding_window > 0 ? min(max(0, held - a.sliding_window), len) : 0;
  x.t = len > lo ? (len - lo / kBN * kBN + kBN - 1) / kBN : 0;
  return x;
}

// The fewest tiles a key part with which all parts of a KV head find a slot at once (a warp; `x`: the lane's sequence of the first 32; out of
// the way of the code that is run often).
__device__ __noinline__ int tiles_per_part(const AttnArgs& a, const TreeArgs& pa, int RB, int lane, int n0, int t0) {
  int longest = 0, blocks = 0;
  long long tiles = 0;
  for (int s0 = 0; s0 < a.sh.num_seqs; s0 += 32) {
    int n = n0, t = t0;
    if (s0 > 0) {
      const SeqShape x = sequence_shape(a, RB, s0 + lane);
      n = x.n;
      t = x.t;
    }
    longest = max(longest, __reduce_max_sync(0xffffffffu, n > 0 ? t : 0));
    blocks += __reduce_add_sync(0xffffffffu, n);
    const long long x = (long long)n * t;  // (in two sums of 32 lanes that 32 bits hold)
    tiles += ((long long)__reduce_add_sync(0xffffffffu, (unsigned)(x >> 20)) << 20) + __reduce_add_sync(0xffffffffu, (unsigned)x & 0xFFFFFu);
  }
  // (the parts of n blocks of t tiles are n t / per at least, and n more than that at most)
  int lo = max(kMinTiles, (longest + pa.splits - 1) / pa.splits), hi = max(lo, longest);
  lo = max(lo, (int)min((long long)hi, (tiles + pa.slots - 1) / pa.slots));
  if (blocks < pa.slots) hi = max(lo, (int)min((long long)hi, tiles / (pa.slots - blocks) + 1));
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    int parts = 0;
    for (int s0 = 0; s0 < a.sh.num_seqs; s0 += 32) {
      int n = n0, t = t0;
      if (s0 > 0) {
        const SeqShape x = sequence_shape(a, RB, s0 + lane);
        n = x.n;
        t = x.t;
      }
      parts += __reduce_add_sync(0xffffffffu, n * max(1, (t + mid - 1) / mid));
    }
    if (parts <= pa.slots) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}

template <int D, bool FAST>
__global__ void __launch_bounds__(kThreads, 2)
tree_tc_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_n,
               const __grid_constant__ AttnArgs a, const TreeArgs pa) {
  using C = Cfg<D, FAST>;
  constexpr int NIT = C::NIT;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  __shared__ __align__(8) Bars s_bars;
  __shared__ uint32_t s_tmem;
  __shared__ int s_info[8];        // sequence, first row and rows of the CTA; end of the sequence's rows, its length, their start; key part, parts
  __shared__ float s_cent[2][16];  // scaled centroids of K and V
  __shared__ int s_dead, s_bad;    // a wait gave up / some page id is out of range, or some norm is not finite
  __shared__ int s_badgrp[2];      // groups of the stage's tile whose page id is
  const AttnShape& sh = a.sh;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int kvh = (int)blockIdx.x % sh.Hkv, rowblk = (int)blockIdx.x / sh.Hkv, G = sh.G, RB = 128 / G;
  volatile int* dead = &s_dead;
  auto bar = [](const uint64_t& b) { return smem_addr(&b); };
  const uint32_t base = (smem_addr(smem_raw) + 1023u) & ~1023u;
  unsigned char* sm = smem_raw + (base - smem_addr(smem_raw));

  // ---- which rows and keys are this CTA's? -----------------------------------------------------------------------
  // A sequence's rows make n blocks of RB rows, its keys t tiles; in a call cut along the keys every block has ceil(t / per) parts, with
  // the fewest tiles a part, `per`, for which all parts find a slot at once: long sequences are cut into more.  (As many parts for all of
  // them: 16 of 300 to 8100 tokens 157 us where this took 115.)
  if (warp == 0) {
    const SeqShape own = sequence_shape(a, RB, lane);
    const int per = pa.to_parts ? tiles_per_part(a, pa, RB, lane, own.n, own.t) : 0x3fffffff;
    int acc = 0, found = -1, first = 0, nrows = 0;
    for (int s0 = 0; s0 < sh.num_seqs && found < 0; s0 += 32) {
      const SeqShape x = s0 == 0 ? own : sequence_shape(a, RB, s0 + lane);
      const int parts = max(1, (x.t + per - 1) / per), c = x.n * parts;
      int incl = c;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += up;
      }
      const int mine = rowblk - acc;
      const unsigned m = __ballot_sync(0xffffffffu, mine < incl);
      if (m) {
        const int w = __ffs(m) - 1;
        const int at = mine - (incl - c), b = at / parts;  // (lane w: its block)
        found = s0 + w;
        first = __shfl_sync(0xffffffffu, x.q0 + b * RB, w);
        nrows = __shfl_sync(0xffffffffu, min(RB, x.q1 - (x.q0 + b * RB)), w);
        if (lane == w) {
          s_info[3] = x.q_end;
          s_info[4] = x.seq_len;
          s_info[5] = x.q0;
          s_info[6] = at - b * parts;
          s_info[7] = parts;
        }
      }
      acc += __shfl_sync(0xffffffffu, incl, 31);
    }
    if (lane == 0) {
      s_info[0] = found;
      s_info[1] = found < 0 ? rowblk - acc : first;  // (without rows: which of the spare CTAs, and how many)
      s_info[2] = found < 0 ? (int)gridDim.x / sh.Hkv - acc : nrows;
      s_dead = 0;
      s_bad = 0;
    }
  }
  // byte -> half2 tables (centroid[hi nibble], centroid[lo nibble]) scaled onto the fp16 grid: one with a copy a lane, or, for two codebooks,
  // two with a copy for two lanes each
  auto build_tables = [&](int t) {
    bool one = true;
    for (int i = 0; i < 16; ++i) one = one && s_cent[0][i] == s_cent[1][i];
    uint4* lut = reinterpret_cast<uint4*>(sm + C::kOffLut);
#pragma unroll 4
    for (int i = t; i < (int)(C::kLut / 16); i += kDeq) {
      const int e = one ? i / 8 : i / 4, w = e >> 8, b = e & 255;
      const uint32_t v = pack_h2(s_cent[w][b >> 4], s_cent[w][b & 15]);
      lut[i] = make_uint4(v, v, v, v);
    }
  };
  if (warp >= kSmx / 32 && warp < kIssueWarp) {
    // (every warp of them makes the same entries of s_cent)
    const int w = lane >> 4, i = lane & 15;
    const float* cent = w ? a.v_centroids : a.k_centroids;
    s_cent[w][i] = i < (w ? a.n_v_centroids : a.n_k_centroids) ? __fmul_rn(w ? a.lut_scale_v : a.lut_scale_k, __ldg(cent + i)) : 0.f;
    __syncwarp();
    if (FAST) build_tables(tid - kSmx);
  }
  __syncthreads();
  const int seq = s_info[0], row0 = s_info[1], nrows = s_info[2];
  if (seq < 0) {  // the grid is an upper bound: ceil(rows / per CTA) + sequences, so at least one CTA is spare
    pdl_trigger();
    pdl_wait();
    // rows past the last offset belong to no sequence and see no key: zeros
    const int tail = min(max(a.query_start_loc[sh.num_seqs], 0), sh.rows);
    const float zero[4] = {0.f, 0.f, 0.f, 0.f};
    for (int r = tail + row0; r < sh.rows; r += nrows) {
      for (int i = tid; i < G * (D / 4); i += kThreads) {
        const int h = kvh * G + i / (D / 4), d = 4 * (i % (D / 4));
        if (!pa.to_parts)
          store4(a.out, a.out_dtype, (int64_t)r * a.out_token_stride + (int64_t)h * a.out_head_stride + d, zero);
        if (d > 0) continue;
        if (pa.to_parts)
          for (int p = 0; p < pa.splits; ++p) pa.part_m[((int64_t)p * sh.rows + r) * sh.Hq + h] = -CUDART_INF_F;
        else if (a.lse_out) a.lse_out[(int64_t)r * sh.Hq + h] = -CUDART_INF_F;
      }
    }
    return;
  }
  const int row_warps = (nrows * G + 31) / 32;  // softmax warps with rows
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      bar_init(bar(s_bars.rawk[i]), 1);
      bar_init(bar(s_bars.rawv[i]), 1);
      bar_init(bar(s_bars.rawk_free[i]), kDeq / 32);
      bar_init(bar(s_bars.rawv_free[i]), kDeq / 32);
      bar_init(bar(s_bars.vready[i]), kDeq / 32);
    }
    bar_init(bar(s_bars.kready), kDeq / 32);
    bar_init(bar(s_bars.kfree), 1);
    bar_init(bar(s_bars.vfree), 1);
    bar_init(bar(s_bars.sready), 1);
    bar_init(bar(s_bars.pready), row_warps);
    bar_init(bar(s_bars.img), 1);
    bar_init(bar(s_bars.aready), row_warps);
    bar_init(bar(s_bars.rot), 1);
    bar_init(bar(s_bars.qready), row_warps);
    bar_init(bar(s_bars.odone), 1);
    bar_init(bar(s_bars.drain), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_async();
  }
  if (warp == kIssueWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&s_tmem)), "r"(C::kCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  pdl_trigger();
  pdl_wait();  // the operand image of Pi; everything else was complete before the kernel in front started
  if (pa.to_parts && s_info[6] == 0) {  // the parts that these rows do not have
    const int parts = s_info[7];
    for (int i = tid; i < (pa.splits - parts) * nrows * G; i += kThreads) {
      const int p = i / (nrows * G), r = i - p * (nrows * G);
      pa.part_m[((int64_t)(parts + p) * sh.rows + row0 + r / G) * sh.Hq + kvh * G + r % G] = -CUDART_INF_F;
    }
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = s_tmem;

  // ---- keys the CTA needs -----------------------------------------------------------------------------------
  const int q_end = s_info[3], len = clamp_seq_len<true>(a, max(0, s_info[4])), held = len - (q_end - s_info[5]);  // (held: in front of the drafts)
  int t_first = 0, n_tiles = 0;
  {
    const int lo = a.sliding_window > 0 ? min(max(0, held - a.sliding_window), len) : 0;  // (a row's position is held - 1 or later)
    if (len > lo) {
      t_first = lo / kBN * kBN;
      n_tiles = (len - t_first + kBN - 1) / kBN;
      const int part = s_info[6], parts = s_info[7], per = (n_tiles + parts - 1) / parts;  // this part of the key range
      t_first += part * per * kBN;
      n_tiles = max(0, min(per, n_tiles - part * per));
    }
  }
  const RowLayout lay = row_layout(sh.Hkv, D);
  const int v_at = lay.v_idx + kvh * (D / 2), kn_at = lay.k_norm + 4 * kvh, vn_at = lay.v_norm + 4 * kvh;

  if (warp == kFetchWarp) {
    // ================= fetching lanes: a lane has one kind of box (keys, values, norms of either) of one group of 16 tokens =================
    const int grp = (lane >> 2) & 3, kind = lane & 3;
    const CUtensorMap* map = kind == 0 ? &map_k : kind == 1 ? &map_v : &map_n;
    const int x = kind == 0 ? lay.k_idx + kvh * (D / 2) : (kind == 1 ? v_at : kind == 2 ? kn_at : vn_at) & ~15;
    const uint32_t dst = base + C::kOffRaw +
                         (kind == 0 ? grp * kGroup * (D / 2) : kind == 1 ? C::kRawV + grp * kGroup * C::kVPitch
                                                                        : (kind == 2 ? C::kRawKn : C::kRawVn) + grp * kGroup * 16);
    const int32_t* bt = a.block_table + (int64_t)seq * a.bt_stride;
    const int bs = a.block_size, shift = (bs & (bs - 1)) == 0 ? __ffs(bs) - 1 : -1;
    auto page_of = [&](int j) -> int {
      const int pos = t_first + j * kBN + grp * kGroup;
      return j < n_tiles && pos < len && lane < 16 ? __ldg(bt + (shift >= 0 ? pos >> shift : pos / bs)) : 0;
    };
    int page = page_of(0), issued = 0;
    bool ok = true;
    for (int j = 0; j < n_tiles && ok; ++j) {
      const int st = j % C::kStages, u = j / C::kStages;
      const int pos = t_first + j * kBN + grp * kGroup, in = shift >= 0 ? pos & (bs - 1) : pos % bs;
      const bool want = lane < 16 && pos < len;
      const int next = page_of(j + 1);
      const bool bad = want && (unsigned)page >= (unsigned)a.num_blocks;
      if (bad && kind == 0) {  // reported, its tokens hidden; the box is filled with zeros
        if (a.err_flag) atomicOr(a.err_flag, TQ4_DEV_BAD_BLOCK);
        s_bad = 1;
      }
      const int groups = __popc(__ballot_sync(0xffffffffu, want)) / 4;
      const unsigned bads = __ballot_sync(0xffffffffu, bad && kind == 0);
      if (u > 0) ok = bar_wait(bar(C::kJoint ? s_bars.rawv_free[st] : s_bars.rawk_free[st]), (uint32_t)((u - 1) & 1), dead);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      if (lane == 0) {
        s_badgrp[st] = (int)((bads & 1) | (bads >> 3 & 2) | (bads >> 6 & 4) | (bads >> 9 & 8));
        expect_tx(bar(s_bars.rawk[st]), groups * kGroup * (D / 2 + 32 + (C::kJoint ? C::kVPitch : 0)));
      }
      __syncwarp();
      if (C::kJoint) {
        if (want) box_load(dst + st * C::kRaw, map, x, in, page, bar(s_bars.rawk[st]));
        issued = 2 * j + 1;  // (as keys)
        page = next;
        continue;
      }
      if (want && kind != 1) box_load(dst + st * C::kRaw, map, x, in, page, bar(s_bars.rawk[st]));
      if (u > 0) ok = bar_wait(bar(s_bars.rawv_free[st]), (uint32_t)((u - 1) & 1), dead);
      ok = __all_sync(0xffffffffu, ok);
      if (lane == 0 && ok) expect_tx(bar(s_bars.rawv[st]), groups * kGroup * C::kVPitch);
      __syncwarp();
      if (want && kind == 1 && ok) box_load(dst + st * C::kRaw, map, x, in, page, bar(s_bars.rawv[st]));
      issued = 2 * j + (ok ? 2 : 1);
      page = next;
    }
    // every box has landed before the CTA ends
    for (int st = 0; st < C::kStages; ++st) {
      const int nk = (issued + 1) / 2, nv = C::kJoint ? 0 : issued / 2;  // tiles whose keys / values were asked for
      const int uk = (nk - st + C::kStages - 1) / C::kStages, uv = (nv - st + C::kStages - 1) / C::kStages;  // ... into this stage
      if (uk > 0) bar_wait_own(bar(s_bars.rawk[st]), (uint32_t)((uk - 1) & 1), dead);
      if (uv > 0) bar_wait_own(bar(s_bars.rawv[st]), (uint32_t)((uv - 1) & 1), dead);
    }
  } else if (warp == kIssueWarp) {
    // ================= issuing thread =================
    if (n_tiles > 0 && elect_one_sync()) {
      bool ok = true;
      uint32_t img_n = 0, img_ph = 0;  // phases of Pi's image asked for / waited for
      const bool unrotate = !a.out_rotated;
      constexpr uint32_t kTerms = FAST ? 1 : 2;
      auto load_term = [&](int term, uint32_t to) { bulk_load(base + to, pa.image + term * C::kImgTerm, C::kImgTerm, bar(s_bars.img)); };
      // O = A * B: A = fp16 hi (and lo) terms at the S and Q columns, B = the image
      auto rotate = [&](bool unrot, bool a_lo) {
        ok = ok && bar_wait_own(bar(s_bars.img), img_ph & 1, dead);
        ++img_ph;
        ok = ok && bar_wait(bar(s_bars.aready), unrot ? 1u : 0u, dead);
        if (!ok) return;
        fence_after();
        constexpr uint32_t d = C::kColO;
        const uint32_t idesc = C::idesc(D, unrot), ihi = base + (unrot ? C::kOffLut : C::kOffK), ilo = base + (unrot ? C::kOffK : C::kOffLut);
#pragma unroll 1
        for (int s = 0; s < D / 16; ++s) {
          const uint32_t off = unrot ? 2048u * s : (s >> 2) * C::kImgPart + 32u * (s & 3);
          const uint64_t bh = make_desc(ihi + off, unrot ? C::kImgPart : 0), bl = make_desc(ilo + off, unrot ? C::kImgPart : 0);
          if (!FAST) mma_ta(tmem + d, tmem + C::kColS + 8 * s, bl, idesc, s > 0);
          if (a_lo) mma_ta(tmem + d, tmem + C::kColQ + 8 * s, bh, idesc, !FAST || s > 0);
          mma_ta(tmem + d, tmem + C::kColS + 8 * s, bh, idesc, !FAST || a_lo || s > 0);
        }
        mma_commit(bar(s_bars.rot));
      };
      ++img_n;
      expect_tx(bar(s_bars.img), kTerms * C::kImgTerm);
      load_term(0, C::kOffK);
      if (!FAST) load_term(1, C::kOffLut);
      rotate(false, !FAST && a.q_dtype == TQ4_F32);

      const uint64_t d_k = make_desc(base + C::kOffK, 0), d_v = make_desc(base + C::kOffV, kBN * 128);
      const uint64_t d_qlo = make_desc(base + C::kOffQlo, 0);
      constexpr uint32_t idS = C::idesc(kBN, false), idO = C::idesc(D, true);
      auto issue_s = [&]() {  // S = Q K~^T
#pragma unroll
        for (int s = 0; s < D / 16; ++s) {
          const uint64_t db = d_k + (uint64_t)(((s >> 2) * (kBN * 128) + 32 * (s & 3)) >> 4);
          if (C::QLO_SMEM) mma_sa(tmem + C::kColS, d_qlo + (uint64_t)(((s >> 2) * 16384 + 32 * (s & 3)) >> 4), db, idS, s > 0);
          else if (C::QLO) mma_ta(tmem + C::kColS, tmem + C::kColQlo + 8 * s, db, idS, s > 0);
          mma_ta(tmem + C::kColS, tmem + C::kColQ + 8 * s, db, idS, C::QLO || s > 0);
        }
        mma_commit(bar(s_bars.sready));
        mma_commit(bar(s_bars.kfree));  // (and of every product before)
      };
      auto issue_pv = [&](int j) {  // O += P V~
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          const uint64_t dv = d_v + (uint64_t)(((j % C::NVB) * C::kKv + 2048 * s) >> 4);
          const uint32_t ph = tmem + C::kColS + 16 * s;
          if (!FAST) mma_ta(tmem + C::kColO, ph + 8, dv, idO, j > 0 || s > 0);
          mma_ta(tmem + C::kColO, ph, dv, idO, !FAST || j > 0 || s > 0);
        }
        if (C::NVB == 1) mma_commit(bar(s_bars.vfree));
      };
      ok = ok && bar_wait(bar(s_bars.qready), 0u, dead);
      ok = ok && bar_wait(bar(s_bars.kready), 0u, dead);
      if (ok) {
        fence_after();
        issue_s();
      }
      for (int j = 0; j < n_tiles && ok; ++j) {
        ok = bar_wait(bar(s_bars.vready[j % C::NVB]), (uint32_t)((j / C::NVB) & 1), dead);
        if (ok && j == n_tiles - 1 && unrotate) {  // (the tables have been read)
          ++img_n;
          expect_tx(bar(s_bars.img), kTerms * C::kImgTerm);
          load_term(0, C::kOffLut);
        }
        ok = ok && bar_wait(bar(s_bars.pready), (uint32_t)(j & 1), dead);
        if (!ok) break;
        fence_after();
        issue_pv(j);
        if (j + 1 < n_tiles) {
          ok = bar_wait(bar(s_bars.kready), (uint32_t)((j + 1) & 1), dead);
          if (!ok) break;
          fence_after();
          issue_s();
        }
      }
      if (ok) {
        mma_commit(bar(s_bars.odone));
        ok = bar_wait_own(bar(s_bars.odone), 0u, dead);
        if (ok && unrotate) {
          if (!FAST) load_term(1, C::kOffK);  // (K~ and V~ have been read)
          rotate(true, true);
          if (ok) bar_wait_own(bar(s_bars.rot), 1u, dead);
        }
      }
      if (!ok) {  // (the CTA is dead)
        if (img_n != img_ph) {
          if (!FAST && img_n == 2) load_term(1, C::kOffLut);  // (the phase is one of two terms; the place does not matter any more)
          bar_wait_own(bar(s_bars.img), img_ph & 1, dead);
        }
        mma_commit(bar(s_bars.drain));
        bar_wait_own(bar(s_bars.drain), 0u, dead);
      }
    }
    __syncwarp();
  } else if (warp >= kSmx / 32) {
    // ================= dequantising warps =================
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::kDeqRegs));
    const int t = tid - kSmx;
    // item n of this thread: token and 16-byte segment of the packed row.  Eight lanes take 4 tokens x the 2 segments
    // of one 64-coordinate block: their operand stores (chunk ^ (token & 7)) fall into eight bank groups.
    auto item = [&](int n, int& tok, int& seg) -> bool {
      constexpr int NP = C::NS / 2;
      const int i = t + kDeq * n;
      if (i < 2 * kBN * NP) {
        const int r8 = i & 7, pg = i >> 4, pair = pg % NP, grp = pg / NP;
        tok = grp * 8 + 4 * ((i >> 3) & 1) + (r8 & 3);
        seg = 2 * pair + (r8 >> 2);
        return true;
      }
      tok = i - 2 * kBN * NP;
      seg = C::NS - 1;
      return (C::NS & 1) && tok < kBN;
    };
    bool ok = n_tiles > 0 && bar_wait(bar(s_bars.rot), 0u, dead);  // the image of Pi has been used
    bool one_table = true;
    for (int i = 0; i < 16; ++i) one_table = one_table && s_cent[0][i] == s_cent[1][i];
    if (!FAST) {  // tables in place of its lo term
      if (ok) build_tables(t);
      asm volatile("bar.sync 1, %0;" ::"n"(kDeq) : "memory");
    }
    const uint32_t entry = one_table ? 128 : 64;  // bytes of a byte's copies
    const uint32_t lut_k = base + C::kOffLut + (lane & (entry / 4 - 1)) * 4, lut_v = lut_k + (one_table ? 0u : 256 * entry);
    auto look = [&](uint32_t at) -> uint32_t {
      uint32_t y;
      asm volatile("ld.shared.b32 %0, [%1];" : "=r"(y) : "r"(at));
      return y;
    };
    auto expand = [&](const uint4& pk, uint32_t lut, uint32_t buf, int tok, int seg) {  // 16 bytes -> 32 fp16
      const uint32_t w[4] = {pk.x, pk.y, pk.z, pk.w};
      unsigned char* dst = sm + buf + (seg >> 1) * (kBN * 128);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const uint32_t x = w[c];
        const uint4 o = make_uint4(look(lut + __byte_perm(x, 0u, 0x4440) * entry), look(lut + __byte_perm(x, 0u, 0x4441) * entry),
                                   look(lut + __byte_perm(x, 0u, 0x4442) * entry), look(lut + (x >> 24) * entry));
        *reinterpret_cast<uint4*>(dst + swz(tok, (seg & 1) * 4 + c)) = o;
      }
    };
    const int v_off = v_at & 15, kn_off = kn_at & 15, vn_off = vn_at & 15;
    // two waits, in one round trip where both are over (in the kernel with one stage that is no gain: 16 ragged sequences 109 us, 108 without)
    auto wait_both = [&](bool second, const uint64_t& x, uint32_t px, const uint64_t& y, uint32_t py) -> bool {
      bool a = C::kJoint && bar_try(bar(x), px), b = !second || (C::kJoint && bar_try(bar(y), py));
      if (!a) a = bar_wait(bar(x), px, dead);
      if (!b) b = bar_wait(bar(y), py, dead);
      return __all_sync(0xffffffffu, a && b);
    };
    auto done = [&](uint64_t& written, const uint64_t* read) {
      fence_async();
      __syncwarp();
      if (lane == 0) {
        bar_arrive(bar(written));
        if (read) bar_arrive(bar(*read));
      }
    };
    for (int j = 0; j < n_tiles && ok; ++j) {
      const int st = j % C::kStages, u = j / C::kStages;
      const unsigned char* raw = sm + C::kOffRaw + st * C::kRaw;
      // ---- keys and norms ------------------------------------------------------------------------------------
      ok = wait_both(j > 0, s_bars.rawk[st], (uint32_t)(u & 1), s_bars.kfree, (uint32_t)((j - 1) & 1));
      if (!ok) break;
      if (t < kBN) {
        float* ns = reinterpret_cast<float*>(sm + C::kOffNorm) + (j & 1) * 2 * kBN;
        float kn = *reinterpret_cast<const float*>(raw + C::kRawKn + 16 * t + kn_off), vn = *reinterpret_cast<const float*>(raw + C::kRawVn + 16 * t + vn_off);
        const bool past = t_first + j * kBN + t >= len, bad = s_badgrp[st] >> (t / kGroup) & 1;
        // (positive, so that -inf times it stays -inf; what lies past the sequence is masked, whatever was there)
        const bool odd = !past && !bad && !(fabsf(kn) < CUDART_INF_F && fabsf(vn) < CUDART_INF_F);  // (a weight of zero times it is none)
        if (odd) s_bad = 1;
        ns[t] = past ? 1.f : bad ? kHidden : odd ? kNotFinite : fmaxf(kn, 1e-30f) * (1.f / kQGain);
        ns[kBN + t] = past || bad || odd ? 0.f : vn;
      }
#pragma unroll
      for (int n = 0; n < NIT; ++n) {
        int tok, seg;
        if (item(n, tok, seg)) expand(*reinterpret_cast<const uint4*>(raw + tok * (D / 2) + 16 * seg), lut_k, C::kOffK, tok, seg);
      }
      done(s_bars.kready, C::kJoint ? nullptr : &s_bars.rawk_free[st]);
      // ---- values ----------------------------------------------------------------------------------------------
      // (With two buffers: that the keys' buffer is free says that S of the tile before is complete, and with it the products with V~ that
      // were asked for in front of it, those of two tiles ago.)
      if (!C::kJoint) ok = wait_both(j >= C::NVB, s_bars.rawv[st], (uint32_t)(u & 1), s_bars.vfree, (uint32_t)((j / C::NVB - 1) & 1));
      if (!ok) break;
#pragma unroll
      for (int n = 0; n < NIT; ++n) {
        int tok, seg;
        if (item(n, tok, seg)) {
          const unsigned char* p = raw + C::kRawV + tok * C::kVPitch + 16 * seg + v_off;
          uint4 x;
          if (v_off == 0) {
            x = *reinterpret_cast<const uint4*>(p);
          } else {
            const uint32_t* w = reinterpret_cast<const uint32_t*>(p);
            x = make_uint4(w[0], w[1], w[2], w[3]);
          }
          expand(x, lut_v, C::kOffV + (j % C::NVB) * C::kKv, tok, seg);
        }
      }
      done(s_bars.vready[j % C::NVB], &s_bars.rawv_free[st]);
    }
  } else {
    // ================= softmax warps: a row per thread =================
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::kSmxRegs));
    if (warp < row_warps) {
      const int m = 32 * warp + lane, my_r = m / G, my_g = m - my_r * G;
      const bool live = my_r < RB && my_r < nrows;
      const int head = kvh * G + my_g, row = row0 + (live ? my_r : 0);
      const uint32_t tb = tmem + ((uint32_t)(32 * warp) << 16);
      const bool use = n_tiles > 0;
      auto arrive = [&](uint64_t& b) {  // this warp's share of a hand-over to the issuing thread
        fence_before();
        __syncwarp();
        if (lane == 0) bar_arrive(bar(b));
      };
      bool ok = true;
      float qexp = 1.f;  // what is left between a stored dot product and the score (1 unless the queries are very large or small)
      if (use) {
        // ---- rotate the queries: raw rows as fp16 terms, scaled by a power of two, times Pi ------------------------
        const int es = a.q_dtype == TQ4_F32 ? 4 : 2;
        const bool q_vec = ((uintptr_t)a.q % 16 == 0) && (a.q_token_stride * es) % 16 == 0 && (a.q_head_stride * es) % 16 == 0;
        const int64_t qi = (int64_t)row * a.q_token_stride + (int64_t)head * a.q_head_stride;
        float sc = 1.f, isc = 1.f, amax = 0.f;
        if (q_vec && es == 2) {  // all of a row's loads at once; the bits without the sign are in the order of the magnitudes
          const uint4* src = reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(a.q) + qi);
          const bool f16 = !FAST && a.q_dtype == TQ4_F16;  // (FAST: bf16)
          uint4 r[D / 8];
#pragma unroll
          for (int i = 0; i < D / 8; ++i) r[i] = live ? __ldg(src + i) : make_uint4(0u, 0u, 0u, 0u);
          uint32_t top = 0;
#pragma unroll
          for (int i = 0; i < D / 8; ++i)
            top = __vmaxu2(__vmaxu2(top, r[i].x & 0x7FFF7FFFu), __vmaxu2(r[i].y & 0x7FFF7FFFu, __vmaxu2(r[i].z & 0x7FFF7FFFu, r[i].w & 0x7FFF7FFFu)));
          float x0, x1;
          half_pair(top, f16, x0, x1);
          pow2_scale(fmaxf(x0, x1), sc, isc);
#pragma unroll
          for (int c = 0; c < D / 32; ++c) {
            uint32_t h[16];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint32_t w[4] = {r[4 * c + e].x, r[4 * c + e].y, r[4 * c + e].z, r[4 * c + e].w};
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                half_pair(w[k], f16, x0, x1);
                h[4 * e + k] = pack_h2(x0 * sc, x1 * sc);
              }
            }
            tmem_st16(tb + C::kColS + 16 * c, h);
          }
        } else {
#pragma unroll 1
          for (int pass = 0; pass < 2; ++pass) {
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
              float x[32];
#pragma unroll
              for (int e = 0; e < 32; ++e) x[e] = 0.f;
              if (live) load32(a.q, a.q_dtype, qi + 32 * c, q_vec, x);
              if (pass == 0) {
#pragma unroll
                for (int e = 0; e < 16; ++e) amax = max3(amax, fabsf(x[2 * e]), fabsf(x[2 * e + 1]));
              } else {
                uint32_t h[16], l[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) split2(x[2 * e] * sc, x[2 * e + 1] * sc, h[e], l[e]);
                tmem_st16(tb + C::kColS + 16 * c, h);
                if (a.q_dtype == TQ4_F32) tmem_st16(tb + C::kColQ + 16 * c, l);
              }
            }
            if (pass == 0) pow2_scale(amax, sc, isc);
          }
        }
        tmem_st_wait();
        arrive(s_bars.aready);
        ok = __all_sync(0xffffffffu, bar_wait(bar(s_bars.rot), 0u, dead));
        fence_after();
        // the rotated row times kQGain and what makes its dot products scores in the log2 domain (before the key norm), as fp16 terms; where
        // that could take the row out of fp16's range, the row keeps a power of two back (as in the prefill kernel)
        float f = isc * (a.scale_log2e / a.lut_scale_k);
        const int fe = (int)((__float_as_uint(fabsf(f)) >> 23) & 0xFFu) - 127;
        if (f != 0.f && (fe < -6 || fe > 3)) {
          const int ec = min(max(fe, -126), 126);
          qexp = __uint_as_float((uint32_t)(127 + ec) << 23);
          f *= __uint_as_float((uint32_t)(127 - ec) << 23);
        }
        f *= kQGain / 256.f;
#pragma unroll 1
        for (int c = 0; c < D / 32 && ok; ++c) {
          uint32_t v[32], h[16], l[16];
          tmem_ld_cols(tb + C::kColO + 32 * c, v);
#pragma unroll
          for (int e = 0; e < 16; ++e) split2(__uint_as_float(v[2 * e]) * f, __uint_as_float(v[2 * e + 1]) * f, h[e], l[e]);
          tmem_st16(tb + C::kColQ + 16 * c, h);
          if (FAST) continue;
          if (C::QLO_SMEM) {
            unsigned char* dst = sm + C::kOffQlo + ((32 * c) >> 6) * 16384;
#pragma unroll
            for (int i = 0; i < 4; ++i)
              *reinterpret_cast<uint4*>(dst + swz(m, (((32 * c) & 63) >> 3) + i)) = make_uint4(l[4 * i], l[4 * i + 1], l[4 * i + 2], l[4 * i + 3]);
          } else {
            tmem_st16(tb + C::kColQlo + 16 * c, l);
          }
        }
        tmem_st_wait();
        fence_async();
        arrive(s_bars.qready);
      }

      // ---- the tile loop --------------------------------------------------------------------------------
      int kv_lo = 0, kv_hi = 0x7fffffff;  // keys in front of the drafts that the row sees (a row that is not there: zeros, nothing to mask)
      const uint32_t* drafts = reinterpret_cast<const uint32_t*>(a.tree_mask) + (int64_t)row * a.tree_stride;
      if (live) {
        kv_hi = max(held, 0);
        if (a.sliding_window > 0) {
          int n = 0;
          for (int w = 0; w < a.tree_words; ++w) n += __popc(__ldg(drafts + w));
          kv_lo = min(max(0, held + n - a.sliding_window), kv_hi);
        }
      }
      // 32 bits of the row's mask from draft `k` on
      auto draft_bits = [&](int k) -> uint32_t {
        auto word = [&](int w) -> uint32_t { return (unsigned)w < (unsigned)a.tree_words ? __ldg(drafts + w) : 0u; };
        const int w = k >> 5;  // (k may be negative)
        return __funnelshift_r(word(w), word(w + 1), k & 31);
      };
      float m_run = -CUDART_INF_F, l_run = 0.f;
      const uint32_t scol = tb + C::kColS;
      for (int j = 0; use && j < n_tiles && ok; ++j) {
        const int t0 = t_first + j * kBN;  // first token
        ok = __all_sync(0xffffffffu, bar_wait(bar(s_bars.sready), (uint32_t)(j & 1), dead));
        if (!ok) break;
        fence_after();
        const float* ns = reinterpret_cast<const float*>(sm + C::kOffNorm) + (j & 1) * 2 * kBN;
        // dot x key norm x qscale - reference, exp2, x value norm, (split,) store in place; two columns per instruction.  The reference is updated
        // lazily, and looked at only after the fact: when some weight exceeds 2^8 (or the row has no reference yet) the tile is done
        // again from the scores, which stay in registers, with a new one.
        const int any_bad = *(volatile int*)&s_bad;  // (its latency beside the scores')
        uint32_t v[kBN];
        tmem_ld_cols(scol, v);
        bool seen = true;  // some key of the tile is visible
        if (!__all_sync(0xffffffffu, t0 >= kv_lo && kv_hi - kBN >= t0 && qexp == 1.f) || any_bad) {
          // hidden columns: a score of -inf (key norms are positive in shared memory)
          const int lo = min(max(kv_lo - t0, 0), kBN), hi = min(max(kv_hi - t0, 0), kBN);
          uint32_t vis[2];
          seen = false;
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            const int l = min(max(lo - 32 * w, 0), 32), h = min(max(hi - 32 * w, 0), 32);
            vis[w] = h > l ? (0xFFFFFFFFu >> (32 - (h - l))) << l : 0u;
            if (live) {  // (drafts of the sequence only)
              const int k = t0 + 32 * w - held, n = min(max(len - (t0 + 32 * w), 0), 32);
              if (n > 0 && k > -32) vis[w] |= draft_bits(k) & (0xFFFFFFFFu >> (32 - n));
            }
            if (any_bad)
              for (int i = 0; i < 32; ++i) {
                const float kn = ns[32 * w + i];
                if (kn == kHidden) vis[w] &= ~(1u << i);
                if (kn == kNotFinite && (vis[w] >> i & 1u)) l_run = CUDART_NAN_F;
              }
            seen = seen || vis[w];
          }
#pragma unroll
          for (int i = 0; i < kBN; ++i)
            v[i] = (vis[i >> 5] >> (i & 31)) & 1u ? __float_as_uint(__uint_as_float(v[i]) * qexp) : 0xFF800000u;
        }
        f2 ls2;
#pragma unroll 1
        for (int attempt = 0;; ++attempt) {
          const float m_neg = m_run == -CUDART_INF_F ? 0.f : -m_run;
          const f2 mn2 = pack2(m_neg, m_neg);
          float wmax = 0.f;
          ls2 = pack2(0.f, 0.f);
          // norms eight columns ahead of their use
          ulonglong2 kn[2][2], vn[2][2];
          auto load_norms = [&](int g) {
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              kn[g & 1][q] = *reinterpret_cast<const ulonglong2*>(ns + 8 * g + 4 * q);
              vn[g & 1][q] = *reinterpret_cast<const ulonglong2*>(ns + kBN + 8 * g + 4 * q);
            }
          };
          load_norms(0);
          f2 lsb = pack2(0.f, 0.f);
          uint32_t w16[16];  // P of 16 columns: eight words of hi, eight of lo
#pragma unroll
          for (int g = 0; g < kBN / 8; ++g) {
            if (g + 1 < kBN / 8) load_norms(g + 1);
            float x[8];
            f2 e[4];
#pragma unroll
            for (int p = 0; p < 4; ++p) {
              const int i = 8 * g + 2 * p;
              const f2 k2 = (p & 1) ? kn[g & 1][p >> 1].y : kn[g & 1][p >> 1].x;
              unpack2(fma2(pack2(__uint_as_float(v[i]), __uint_as_float(v[i + 1])), k2, mn2), x[2 * p], x[2 * p + 1]);
            }
#pragma unroll
            for (int p = 0; p < 4; ++p) e[p] = pack2(ex2_approx(x[2 * p]), ex2_approx(x[2 * p + 1]));
#pragma unroll
            for (int p = 0; p < 4; ++p) {
              f2& sum = (p & 1) ? lsb : ls2;
              sum = add2(sum, e[p]);
              const f2 v2 = (p & 1) ? vn[g & 1][p >> 1].y : vn[g & 1][p >> 1].x;
              unpack2(mul2(e[p], v2), x[2 * p], x[2 * p + 1]);
            }
            float2 f[4];
#pragma unroll
            for (int p = 0; p < 4; ++p) {
              wmax = max3(wmax, x[2 * p], x[2 * p + 1]);
              const __half2 h = __floats2half2_rn(x[2 * p], x[2 * p + 1]);
              w16[4 * (g & 1) + p] = *reinterpret_cast<const uint32_t*>(&h);
              f[p] = __half22float2(h);
            }
            if (!FAST) {
#pragma unroll
              for (int p = 0; p < 4; ++p) {
                float r0, r1;
                unpack2(fma2(pack2(f[p].x, f[p].y), pack2(-1.f, -1.f), pack2(x[2 * p], x[2 * p + 1])), r0, r1);
                w16[8 + 4 * (g & 1) + p] = pack_h2(r0, r1);
              }
            }
            if (g & 1) {
              if (FAST) tmem_st8(scol + 8 * (g - 1), *reinterpret_cast<const uint32_t(*)[8]>(w16));
              else tmem_st16(scol + 8 * (g - 1), w16);
            }
          }
          ls2 = add2(ls2, lsb);
          // (sums past 1e30: a value norm of zero hides an overflow from the weights)
          float e0, e1;
          unpack2(ls2, e0, e1);
          const bool need = attempt == 0 && (!(wmax <= 256.f) || !(e0 + e1 < 1e30f) || (seen && m_run == -CUDART_INF_F));
          if (!__any_sync(0xffffffffu, need)) break;
          // new reference: largest score of the tile, shifted by log2 of its value norm
          float mt = -CUDART_INF_F;
#pragma unroll
          for (int i = 0; i < kBN; i += 4) {
            const float4 k4 = *reinterpret_cast<const float4*>(ns + i), v4 = *reinterpret_cast<const float4*>(ns + kBN + i);
            mt = max3(mt, fmaf(__uint_as_float(v[i]), k4.x, fmaxf(lg2_approx(v4.x), -30.f)),
                      fmaf(__uint_as_float(v[i + 1]), k4.y, fmaxf(lg2_approx(v4.y), -30.f)));
            mt = max3(mt, fmaf(__uint_as_float(v[i + 2]), k4.z, fmaxf(lg2_approx(v4.z), -30.f)),
                      fmaf(__uint_as_float(v[i + 3]), k4.w, fmaxf(lg2_approx(v4.w), -30.f)));
          }
          const bool bump = need && mt > m_run;
          const float alpha = bump ? (m_run == -CUDART_INF_F ? 0.f : ex2_approx(m_run - mt)) : 1.f;
          if (bump) m_run = mt;
          l_run *= alpha;
          if (j > 0) {  // O: the scores of this tile were asked for behind the last products with V~, so no MMA is working on it
#pragma unroll 1
            for (int q = 0; q < D / 16; ++q) {
              uint32_t o[16];
              tmem_ld16_async(tb + C::kColO + 16 * q, o);
              tmem_ld16_wait(o);
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
              tmem_st16(tb + C::kColO + 16 * q, o);
            }
          }
        }
        tmem_st_wait();
        float s0, s1;
        unpack2(ls2, s0, s1);
        l_run += s0 + s1;
        arrive(s_bars.pready);
      }

      // ---- normalise, un-rotate, store ------------------------------------------------------------------
      bool have = use;
      if (use) {
        ok = __all_sync(0xffffffffu, ok && bar_wait(bar(s_bars.odone), 0u, dead));
        fence_after();
        have = ok && l_run != 0.f;  // (NaN: handed on)
      }
      const float inv = have ? 1.f / (a.lut_scale_v * l_run) : 0.f;
      const float lse = have ? (m_run + lg2_approx(l_run)) * 0.6931471805599453f : -CUDART_INF_F;
      const bool out_vec = (uintptr_t)a.out % 16 == 0 && a.out_token_stride % 8 == 0 && a.out_head_stride % 8 == 0;
      const int64_t oi = (int64_t)row * a.out_token_stride + (int64_t)head * a.out_head_stride;
      // rows leave through shared memory (of which everything is free now), from which the warp stores them whole; `to`: the element
      // at which a lane's row starts, -1: none
      auto store_rows = [&](uint32_t pitch, int row_bytes, void* out, int elem, int64_t to) {
        __syncwarp();
        const unsigned char* rows = sm + 32 * warp * pitch;
        const int pcs = row_bytes / 16;
#pragma unroll 4
        for (int i = lane; i < 32 * pcs; i += 32) {
          const int r = i / pcs, pc = i - r * pcs;
          const int64_t at = __shfl_sync(0xffffffffu, to, r);
          if (at >= 0)
            *reinterpret_cast<uint4*>(reinterpret_cast<unsigned char*>(out) + at * elem + 16 * pc) = *reinterpret_cast<const uint4*>(rows + r * pitch + 16 * pc);
        }
      };
      float f = inv;
      if (!a.out_rotated) {  // (parts, too: the merge is linear)
        float isc = 0.f;
        if (use) {
          float amax = 0.f, sc = 1.f;
#pragma unroll 1
          for (int pass = 0; pass < 2; ++pass) {
#pragma unroll 1
            for (int c = 0; c < D / 32 && ok; ++c) {
              uint32_t v[32];
              tmem_ld_cols(tb + C::kColO + 32 * c, v);
              if (pass == 0) {
#pragma unroll
                for (int e = 0; e < 16; ++e) amax = max3(amax, fabsf(__uint_as_float(v[2 * e])), fabsf(__uint_as_float(v[2 * e + 1])));
                continue;
              }
              uint32_t h[16], l[16];
#pragma unroll
              for (int e = 0; e < 16; ++e)
                split2(__uint_as_float(v[2 * e]) * inv * sc, __uint_as_float(v[2 * e + 1]) * inv * sc, h[e], l[e]);
              tmem_st16(tb + C::kColS + 16 * c, h);
              tmem_st16(tb + C::kColQ + 16 * c, l);
            }
            if (pass == 0) pow2_scale(amax * inv, sc, isc);
          }
          tmem_st_wait();
          arrive(s_bars.aready);
          ok = __all_sync(0xffffffffu, bar_wait(bar(s_bars.rot), 1u, dead)) && ok;
          fence_after();
        }
        f = have && ok ? isc * (1.f / 256.f) : 0.f;
      }
      const int64_t vec = ((int64_t)s_info[6] * sh.rows + row) * sh.Hq + head;
      const bool staged = pa.to_parts || (out_vec && a.out_dtype != TQ4_F32);
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        uint32_t v[32];
        if (use && ok) tmem_ld32(tb + C::kColO + 32 * c, v);
        if (live) {
          float y[32];
#pragma unroll
          for (int e = 0; e < 32; ++e) y[e] = f != 0.f ? __uint_as_float(v[e]) * f : 0.f;
          if (pa.to_parts) {
            float4* dst = reinterpret_cast<float4*>(sm + (uint32_t)m * C::kPartPitch + 128 * c);
#pragma unroll
            for (int e = 0; e < 8; ++e) dst[e] = make_float4(y[4 * e], y[4 * e + 1], y[4 * e + 2], y[4 * e + 3]);
          } else if (staged) {
            store32(sm + (uint32_t)m * C::kOutPitch, a.out_dtype, 32 * c, true, y);
          } else {
            store32(a.out, a.out_dtype, oi + 32 * c, out_vec, y);
          }
        }
      }
      if (pa.to_parts) store_rows(C::kPartPitch, 4 * D, pa.part_o, 4, live && have ? vec * D : -1);  // (an empty partial's sums are not read)
      else if (staged) store_rows(C::kOutPitch, 2 * D, a.out, 2, live ? oi : -1);
      if (live && pa.to_parts) pa.part_m[vec] = lse;
      else if (live && a.lse_out) a.lse_out[(int64_t)row * sh.Hq + head] = lse;
    }
  }
  fence_before();
  __syncthreads();
  if (s_dead && tid == 0 && a.err_flag) atomicOr(a.err_flag, TQ4_DEV_TIMEOUT);
  if (warp == kIssueWarp)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::kCols) : "memory");
}

// Map of the cache as [pages][tokens][bytes], in boxes of 16 tokens times `width` bytes.
bool cache_map(CUtensorMap& map, const AttnArgs& a, uint32_t width) {
  const EncodeTiledFn encode = encode_tiled_fn();
  if (!encode) return false;
  const cuuint64_t dims[3] = {(cuuint64_t)a.cache_token_stride, (cuuint64_t)a.block_size, (cuuint64_t)a.num_blocks};
  const cuuint64_t strides[2] = {(cuuint64_t)a.cache_token_stride, (cuuint64_t)a.cache_block_stride};
  const cuuint32_t box[3] = {width, (cuuint32_t)kGroup, 1}, steps[3] = {1, 1, 1};
  return encode(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<uint8_t*>(a.cache), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D, bool FAST>
int launch_t(const AttnArgs& a, const TreeArgs& pa, cudaStream_t st) {
  using C = Cfg<D, FAST>;
  constexpr int smem = (int)C::kSmem + 1024;
  static_assert(2 * (smem + 2048) <= 228 * 1024, "two CTAs an SM");
  if (!ensure_dynamic_smem<tree_tc_kernel<D, FAST>>(smem, true)) return TQ4_ERR_CUDA;
  CUtensorMap mk, mv, mn;
  if (!cache_map(mk, a, D / 2) || !cache_map(mv, a, C::kVPitch) || !cache_map(mn, a, 16)) return TQ4_ERR_CUDA;
  const int per_cta = 128 / a.sh.G;
  int64_t units = (int64_t)(a.sh.rows + per_cta - 1) / per_cta + a.sh.num_seqs;  // upper bound, with one spare
  if (pa.to_parts && units < pa.slots + 1) units = pa.slots + 1;
  const int64_t grid = units * a.sh.Hkv;
  if (grid > 0x7fffffff) return TQ4_ERR_UNSUPPORTED;
  if (launch_kernel(tree_tc_kernel<D, FAST>, dim3((unsigned)grid), dim3(kThreads), (size_t)smem, st, true, mk, mv, mn, a,
                    pa) != cudaSuccess)
    return TQ4_ERR_CUDA;
  TQ4_CHECK_LAUNCH();
  return TQ4_OK;
}

}  // namespace

// Boxes of 16 tokens need pages of whole boxes, and addresses and strides that are multiples of 16.
bool tree_few_supported(const AttnArgs& a) {
  return a.sh.D <= 128 && a.num_blocks > 0 && a.block_size % kGroup == 0 && ((uintptr_t)a.cache | a.cache_block_stride | a.cache_token_stride) % 16 == 0 &&
         a.cache_token_stride <= (1 << 30) && a.cache_block_stride >= a.cache_token_stride && encode_tiled_fn() != nullptr;
}

// CTAs of a KV head that run at once, two an SM.
int tree_few_slots(const AttnArgs& a) {
  const int s = 2 * sm_count() / a.sh.Hkv;
  return s < 1 ? 1 : s;
}

// Key parts of a row, at most: none where the sequences fill the SMs already.
int tree_few_splits(const AttnArgs& a, int64_t room) {
  const int per_cta = 128 / a.sh.G;
  const int64_t blocks = (a.sh.rows + per_cta - 1) / per_cta, units = blocks > a.sh.num_seqs ? blocks : a.sh.num_seqs;
  int64_t s = tree_few_slots(a);
  if (5 * units > 4 * s) return 1;  // (hardly any sequence would be cut, and all would go through the merge)
  const int64_t keys = a.sliding_window > 0 && a.sliding_window + kBN < a.max_keys ? a.sliding_window + kBN : a.max_keys;
  const int64_t tiles = (keys + kBN - 1) / kBN + 1;
  if (s > tiles / kMinTiles) s = tiles / kMinTiles;
  if (s > 64) s = 64;
  if (a.sh.rows > 0 && s > room / a.sh.rows) s = room / a.sh.rows;
  return s < 1 ? 1 : (int)s;
}

int launch_tree_few(const AttnArgs& a, cudaStream_t st, bool fast, int splits, bool to_parts, uint8_t* image, float* part_o, float* part_m) {
  const TreeArgs pa{image, splits, tree_few_slots(a), to_parts ? 1 : 0, part_o, part_m};
  const int rc = launch_pi_image(a.sh.D, a.rotation, image, st);
  if (rc != TQ4_OK) return rc;
  switch (a.sh.D) {
    case 64: return fast ? launch_t<64, true>(a, pa, st) : launch_t<64, false>(a, pa, st);
    case 96: return fast ? launch_t<96, true>(a, pa, st) : launch_t<96, false>(a, pa, st);
    case 128: return fast ? launch_t<128, true>(a, pa, st) : launch_t<128, false>(a, pa, st);
  }
  return TQ4_ERR_UNSUPPORTED;
}

}  // namespace tq4
