// Rotary positions of queries and keys, in front of the cache write: the pair (x, y) of frequency w at position p becomes
//   f (x cos a - y sin a,  y cos a + x sin a),   a = p w.
//
// The angle is kept in turns, as a 64-bit fixed-point fraction: F = frac(w / 2 pi) 2^64, made once per frequency in doubles, times
// the position modulo 2^64.  The product is exact whatever the position (the rounding of F moves a position of 10^6 by less than
// 2 pi 10^6 2^-53), where a product in floats is off by 2^-24 of the angle, 0.008 at position 131072.  The top 32 bits, as a signed
// number, are the turn in [-1/2, 1/2); sincospif takes it in fp32.
//
// Bound by HBM at many tokens, by one round trip to memory at few.  A block takes some tokens, or a share of one token's heads
// when there are few; its threads ask for their first vectors, then make the block's cosines and sines once for all heads, in
// shared memory, while those loads are on their way.
#include "tq4_common.cuh"

namespace tq4 {
namespace {

constexpr int kRotThreads = 256;
constexpr int kRotBatch = 4;      // vectors a thread has in flight
constexpr int kRotMaxDim = 1024;  // rotary dimensions

struct RotaryArgs {
  const void* x[2];  // queries, keys
  void* y[2];
  int64_t x_token_stride[2], x_head_stride[2], y_token_stride[2], y_head_stride[2];
  int heads[2];
  int64_t n_tokens;
  int rot, per_head;  // rotary dimensions; items of a head (turned ones first, then those handed through)
  int turned;         // ... of which turned
  int tokens;         // of a block
  const void* positions;
  int positions_64;
  const void* inv_freq;
  int inv_freq_64;
  float factor;
  int inverse;
};

template <typename T, int V>
struct alignas(V * sizeof(T) <= 16 ? V * sizeof(T) : 16) Chunk {
  T v[V];
};

// V elements of one type are moved at a time.  An item is the two chunks whose elements make V pairs (half layout: V i and
// rot / 2 + V i; interleaved: 2 V i and the one behind it), or one chunk of the dimensions that do not turn.
template <typename T, int V, bool INTERLEAVED>
__global__ void __launch_bounds__(kRotThreads) rotary_kernel(const RotaryArgs a) {
  extern __shared__ float s_cs[];  // [tokens][cos rot / 2, sin rot / 2]
  using C = Chunk<T, V>;
  const int half = a.rot / 2;
  const int64_t t0 = (int64_t)blockIdx.x * a.tokens;
  const int nt = (int)min((int64_t)a.tokens, a.n_tokens - t0);
  const int heads = a.heads[0] + a.heads[1], per_token = heads * a.per_head;
  // this block's share of the tokens' items
  const int all = nt * per_token, share = (all + (int)gridDim.y - 1) / (int)gridDim.y;
  const int i_end = min(all, ((int)blockIdx.y + 1) * share);

  C lo[kRotBatch], hi[kRotBatch];
  auto locate = [&](int i, int& tok, int& src, int& h, int& e) {
    tok = i / per_token;
    const int r = i - tok * per_token;
    h = r / a.per_head;
    e = r - h * a.per_head;
    src = h >= a.heads[0] ? 1 : 0;
    h -= src ? a.heads[0] : 0;
  };
  auto first_of = [&](int e) { return e >= a.turned ? a.rot + (e - a.turned) * V : INTERLEAVED ? 2 * V * e : V * e; };
  const int step = INTERLEAVED ? V : half;  // from an item's first chunk to its second
  auto load = [&](int i, C& x, C& y) {
    int tok, src, h, e;
    locate(i, tok, src, h, e);
    const T* p = reinterpret_cast<const T*>(a.x[src]) + (t0 + tok) * a.x_token_stride[src] + (int64_t)h * a.x_head_stride[src] + first_of(e);
    x = *reinterpret_cast<const C*>(p);
    if (e < a.turned) y = *reinterpret_cast<const C*>(p + step);
  };
  auto turn = [&](int i, const C& x, const C& y) {
    int tok, src, h, e;
    locate(i, tok, src, h, e);
    T* p = reinterpret_cast<T*>(a.y[src]) + (t0 + tok) * a.y_token_stride[src] + (int64_t)h * a.y_head_stride[src] + first_of(e);
    if (e >= a.turned) {
      *reinterpret_cast<C*>(p) = x;
      return;
    }
    const float* c = s_cs + tok * a.rot + V * e;
    const float* s = c + half;
    C u, w;
#pragma unroll
    for (int k = 0; k < V; ++k) {
      // pair k: elements k of the two chunks, or neighbours of the 2 V elements
      const float p0 = INTERLEAVED ? to_float<T>(2 * k < V ? x.v[(2 * k) % V] : y.v[(2 * k) % V]) : to_float<T>(x.v[k]);
      const float p1 = INTERLEAVED ? to_float<T>(2 * k + 1 < V ? x.v[(2 * k + 1) % V] : y.v[(2 * k + 1) % V]) : to_float<T>(y.v[k]);
      const T q0 = from_float<T>(fmaf(p0, c[k], -(p1 * s[k]))), q1 = from_float<T>(fmaf(p1, c[k], p0 * s[k]));
      if (!INTERLEAVED) {
        u.v[k] = q0;
        w.v[k] = q1;
      } else {
        (2 * k < V ? u : w).v[(2 * k) % V] = q0;
        (2 * k + 1 < V ? u : w).v[(2 * k + 1) % V] = q1;
      }
    }
    *reinterpret_cast<C*>(p) = u;
    *reinterpret_cast<C*>(p + step) = w;
  };

  int i = (int)blockIdx.y * share + (int)threadIdx.x;
#pragma unroll
  for (int b = 0; b < kRotBatch; ++b)
    if (i + b * kRotThreads < i_end) load(i + b * kRotThreads, lo[b], hi[b]);
  for (int k = threadIdx.x; k < nt * half; k += kRotThreads) {
    const int tok = k / half, j = k - tok * half;
    const int64_t pos = a.positions_64 ? reinterpret_cast<const int64_t*>(a.positions)[t0 + tok]
                                       : (int64_t)reinterpret_cast<const int32_t*>(a.positions)[t0 + tok];
    const double w = a.inv_freq_64 ? reinterpret_cast<const double*>(a.inv_freq)[j] : (double)reinterpret_cast<const float*>(a.inv_freq)[j];
    double turns = w * 0.15915494309189533577;  // 1 / (2 pi)
    turns -= floor(turns);
    const uint64_t frac = (uint64_t)(turns * 18446744073709551616.0) * (uint64_t)pos;
    float s, c;
    sincospif((float)(int32_t)(frac >> 32) * 0x1p-31f, &s, &c);
    if (!isfinite(w)) s = c = __int_as_float(0x7fffffff);
    s_cs[tok * a.rot + j] = c * a.factor;
    s_cs[tok * a.rot + half + j] = (a.inverse ? -s : s) * a.factor;
  }
  __syncthreads();
  for (; i < i_end; i += kRotBatch * kRotThreads) {
#pragma unroll
    for (int b = 0; b < kRotBatch; ++b)
      if (i + b * kRotThreads < i_end) turn(i + b * kRotThreads, lo[b], hi[b]);
    const int n = i + kRotBatch * kRotThreads;
#pragma unroll
    for (int b = 0; b < kRotBatch; ++b)
      if (n + b * kRotThreads < i_end) load(n + b * kRotThreads, lo[b], hi[b]);
  }
}

template <typename T, int V, bool INTERLEAVED>
int launch_rotary(RotaryArgs a, int head_dim, bool through, cudaStream_t st) {
  a.turned = a.rot / 2 / V;
  a.per_head = a.turned + (through ? (head_dim - a.rot) / V : 0);
  const int64_t per_token = (int64_t)(a.heads[0] + a.heads[1]) * a.per_head;
  if (per_token > (1 << 24)) return TQ4_ERR_UNSUPPORTED;
  // A batch of every thread's is a block's work, when there are blocks enough; few tokens: their heads are dealt out
  int tokens = (int)(kRotBatch * kRotThreads / per_token);
  const int64_t fill = 4 * (int64_t)sm_count();
  if (tokens > a.n_tokens / fill) tokens = (int)(a.n_tokens / fill);
  if (tokens > kRotMaxDim * 8 / a.rot) tokens = kRotMaxDim * 8 / a.rot;
  if (tokens < 1) tokens = 1;
  a.tokens = tokens;
  const int64_t blocks = (a.n_tokens + tokens - 1) / tokens;
  if (blocks > 0x7fffffff) return TQ4_ERR_UNSUPPORTED;
  int64_t split = fill / 2 / blocks;
  if (split > per_token / kRotThreads) split = per_token / kRotThreads;
  if (split < 1) split = 1;
  if (launch_kernel(rotary_kernel<T, V, INTERLEAVED>, dim3((unsigned)blocks, (unsigned)split), dim3(kRotThreads),
                    (size_t)tokens * a.rot * sizeof(float), st, false, a) != cudaSuccess)
    return TQ4_ERR_CUDA;
  TQ4_CHECK_LAUNCH();
  return TQ4_OK;
}

template <typename T>
int dispatch_rotary(const RotaryArgs& a, int head_dim, bool interleaved, bool through, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  bool vec = (a.rot / 2) % V == 0 && head_dim % V == 0;
  for (int s = 0; s < 2; ++s)
    if (a.heads[s] > 0)
      vec = vec && (((uintptr_t)a.x[s] | (uintptr_t)a.y[s]) & 15) == 0 &&
            (a.x_token_stride[s] | a.x_head_stride[s] | a.y_token_stride[s] | a.y_head_stride[s]) % V == 0;
  if (vec) return interleaved ? launch_rotary<T, V, true>(a, head_dim, through, st) : launch_rotary<T, V, false>(a, head_dim, through, st);
  return interleaved ? launch_rotary<T, 1, true>(a, head_dim, through, st) : launch_rotary<T, 1, false>(a, head_dim, through, st);
}

}  // namespace
}  // namespace tq4

extern "C" int tq4_rotary(const void* q, const void* k, int dtype, int64_t n_tokens, int num_q_heads, int num_k_heads,
                          int head_dim, const int64_t* q_strides, const int64_t* k_strides, const void* positions,
                          int positions_64, const void* inv_freq, int inv_freq_64, int rotary_dim, int interleaved,
                          float attention_factor, int inverse, void* q_out, void* k_out, const int64_t* q_out_strides,
                          const int64_t* k_out_strides, void* stream) {
  using namespace tq4;
  if (n_tokens < 0 || num_q_heads < 0 || num_k_heads < 0 || head_dim <= 0) return TQ4_ERR_INVALID_ARG;
  if (rotary_dim <= 0 || rotary_dim % 2 || rotary_dim > head_dim) return TQ4_ERR_INVALID_ARG;
  if (dtype < 0 || dtype > 2 || rotary_dim > kRotMaxDim) return TQ4_ERR_UNSUPPORTED;
  if (n_tokens == 0 || num_q_heads + num_k_heads == 0) return TQ4_OK;
  if (!positions || !inv_freq || (num_q_heads && (!q || !q_out || !q_strides || !q_out_strides)) ||
      (num_k_heads && (!k || !k_out || !k_strides || !k_out_strides)))
    return TQ4_ERR_INVALID_ARG;
  RotaryArgs a{};
  const void* x[2] = {q, k};
  void* y[2] = {q_out, k_out};
  const int64_t* xs[2] = {q_strides, k_strides};
  const int64_t* ys[2] = {q_out_strides, k_out_strides};
  const int heads[2] = {num_q_heads, num_k_heads};
  bool through = false;  // some output is not its input: the other dimensions are handed through
  for (int s = 0; s < 2; ++s) {
    a.heads[s] = heads[s];
    if (!heads[s]) continue;
    a.x[s] = x[s];
    a.y[s] = y[s];
    a.x_token_stride[s] = xs[s][0];
    a.x_head_stride[s] = xs[s][1];
    a.y_token_stride[s] = ys[s][0];
    a.y_head_stride[s] = ys[s][1];
    through = through || x[s] != y[s];
  }
  a.n_tokens = n_tokens;
  a.rot = rotary_dim;
  a.positions = positions;
  a.positions_64 = positions_64;
  a.inv_freq = inv_freq;
  a.inv_freq_64 = inv_freq_64;
  a.factor = attention_factor;
  a.inverse = inverse;
  through = through && rotary_dim < head_dim;
  cudaStream_t st = (cudaStream_t)stream;
  switch (dtype) {
    case TQ4_F32: return dispatch_rotary<float>(a, head_dim, interleaved != 0, through, st);
    case TQ4_F16: return dispatch_rotary<__half>(a, head_dim, interleaved != 0, through, st);
    default: return dispatch_rotary<__nv_bfloat16>(a, head_dim, interleaved != 0, through, st);
  }
}
