// Rotary positions of queries and keys, in front of the cache write: the pair (x, y) of frequency w at position p becomes
//   f (x cos a - y sin a,  y cos a + x sin a),   a = p w.
//
// The angle is kept in turns, as a 64-bit fixed-point fraction: F = frac(w / 2 pi) 2^64, made once per frequency in doubles, times
// the position modulo 2^64.  The product is exact whatever the position (the rounding of F moves a position of 10^6 by less than
// 2 pi 10^6 2^-53), where a product in floats is off by 2^-24 of the angle, 0.008 at position 131072.  The top 32 bits, as a signed
// number, are the turn in [-1/2, 1/2); sincospif takes it in fp32.
//
// Bound by HBM at many tokens (8 x 2048 of 32 / 8 heads of 128: 62 to 65 us, 5.2 TB/s read and written), by one round trip to memory at
// few (16 x 8: 2.6 us).  A block takes some tokens, or a share of one token's heads
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
  int rot, items;     // rotary dimensions; items of a head (turned ones first, then those handed through)
  int turned;         // ... of which turned
  int per_head;       // items of a head in a block
  int lanes;          // threads that share a token's item, each with every lanes-th head
  int pass, tokens;   // tokens of a block at a time, and in all
  const void* positions;
  int positions_64;
  const void* inv_freq;
  int inv_freq_64;
  float factor;
  int inverse;
};

// V elements as they are in memory: words of two 16-bit values or one float, or a single element
template <typename T, int V>
struct alignas(V * sizeof(T)) Chunk {
  static constexpr int kWords = V * sizeof(T) / 4;
  uint32_t w[kWords];
};
template <>
struct Chunk<__half, 1> { uint16_t w[1]; };
template <>
struct Chunk<__nv_bfloat16, 1> { uint16_t w[1]; };

__device__ __forceinline__ float2 unpack2(uint32_t w, __half) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
__device__ __forceinline__ float2 unpack2(uint32_t w, __nv_bfloat16) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}
__device__ __forceinline__ uint32_t pack2(float x, float y, __half) {
  const __half2 h = __floats2half2_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack2(float x, float y, __nv_bfloat16) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 turn2(float x, float y, float c, float s) { return make_float2(fmaf(x, c, -(y * s)), fmaf(y, c, x * s)); }

// The V pairs of two chunks, turned in place.
template <typename T, int V, bool INTERLEAVED>
__device__ __forceinline__ void turn(Chunk<T, V>& x, Chunk<T, V>& y, const float (&c)[V], const float (&s)[V]) {
  if constexpr (sizeof(T) == 4 && (V == 1 || !INTERLEAVED)) {
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const float2 r = turn2(__uint_as_float(x.w[k]), __uint_as_float(y.w[k]), c[k], s[k]);
      x.w[k] = __float_as_uint(r.x);
      y.w[k] = __float_as_uint(r.y);
    }
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int k = 0; k < V; ++k) {
      uint32_t* w = 2 * k < V ? x.w + 2 * k : y.w + (2 * k - V);
      const float2 r = turn2(__uint_as_float(w[0]), __uint_as_float(w[1]), c[k], s[k]);
      w[0] = __float_as_uint(r.x);
      w[1] = __float_as_uint(r.y);
    }
  } else if constexpr (V == 1) {
    const float2 r = turn2(unpack2(x.w[0], T()).x, unpack2(y.w[0], T()).x, c[0], s[0]);
    x.w[0] = (uint16_t)pack2(r.x, 0.f, T());
    y.w[0] = (uint16_t)pack2(r.y, 0.f, T());
  } else if constexpr (INTERLEAVED) {
#pragma unroll
    for (int k = 0; k < V; ++k) {
      uint32_t& w = k < V / 2 ? x.w[k] : y.w[k - V / 2];
      const float2 p = unpack2(w, T()), r = turn2(p.x, p.y, c[k], s[k]);
      w = pack2(r.x, r.y, T());
    }
  } else {
#pragma unroll
    for (int k = 0; k < V / 2; ++k) {
      const float2 p = unpack2(x.w[k], T()), q = unpack2(y.w[k], T());
      const float2 r0 = turn2(p.x, q.x, c[2 * k], s[2 * k]), r1 = turn2(p.y, q.y, c[2 * k + 1], s[2 * k + 1]);
      x.w[k] = pack2(r0.x, r1.x, T());
      y.w[k] = pack2(r0.y, r1.y, T());
    }
  }
}

// V elements of one type are moved at a time.  An item is the two chunks whose elements make V pairs (half layout: V i and
// rot / 2 + V i; interleaved: 2 V i and the one behind it), or one chunk of the dimensions that do not turn.  A thread has one item's
// place in some heads of a token, so what it needs of cosines and sines stays in its registers and nothing is divided on the way.
// (With the items of a token dealt out flat, two divisions a chunk, 8 x 2048 tokens of 32 / 8 heads took 123 us, bound by issue.)
template <typename T, int V, bool INTERLEAVED>
__global__ void __launch_bounds__(kRotThreads, 3) rotary_kernel(const RotaryArgs a) {
  extern __shared__ float s_cs[];  // [tokens][cos rot / 2, sin rot / 2]
  using C = Chunk<T, V>;
  const int half = a.rot / 2, tid = threadIdx.x;
  const int64_t t0 = (int64_t)blockIdx.x * a.tokens;
  const int nt = (int)min((int64_t)a.tokens, a.n_tokens - t0);
  const int per_token = a.lanes * a.per_head, slot = tid / per_token, r = tid - slot * per_token;
  const int lane = r / a.per_head, e = r - lane * a.per_head + (int)blockIdx.z * a.per_head;  // (items fastest: neighbours move neighbouring chunks)
  const bool act = slot < a.pass && e < a.items, turned = e < a.turned;
  const int at = !turned ? a.rot + (e - a.turned) * V : INTERLEAVED ? 2 * V * e : V * e;
  const int step = INTERLEAVED ? V : half;  // from an item's first chunk to its second
  const int heads = a.heads[0] + a.heads[1];
  C lo[kRotBatch], hi[kRotBatch];
  const T *xq, *xk;
  T *yq, *yk;
  auto token = [&](int t) {
    xq = reinterpret_cast<const T*>(a.x[0]) + (t0 + t) * a.x_token_stride[0] + at;
    xk = reinterpret_cast<const T*>(a.x[1]) + (t0 + t) * a.x_token_stride[1] + at;
    yq = reinterpret_cast<T*>(a.y[0]) + (t0 + t) * a.y_token_stride[0] + at;
    yk = reinterpret_cast<T*>(a.y[1]) + (t0 + t) * a.y_token_stride[1] + at;
  };
  auto load = [&](int h, C& x, C& y) {
    const int k = h - a.heads[0];
    const T* p = k < 0 ? xq + (int64_t)h * a.x_head_stride[0] : xk + (int64_t)k * a.x_head_stride[1];
    x = *reinterpret_cast<const C*>(p);
    if (turned) y = *reinterpret_cast<const C*>(p + step);
  };
  auto batch = [&](int h0) {
#pragma unroll
    for (int b = 0; b < kRotBatch; ++b)
      if (h0 + b * a.lanes < heads) load(h0 + b * a.lanes, lo[b], hi[b]);
  };
  const int first = lane + (int)blockIdx.y * kRotBatch * a.lanes, stride = (int)gridDim.y * kRotBatch * a.lanes;
  if (act && slot < nt && first < heads) {
    token(slot);
    batch(first);
  }
  // ---- the block's cosines and sines, while the first vectors are on their way -------------------------------
  for (int k = tid; k < nt * half; k += kRotThreads) {
    const int t = k / half, j = k - t * half;
    const double w = a.inv_freq_64 ? reinterpret_cast<const double*>(a.inv_freq)[j] : (double)reinterpret_cast<const float*>(a.inv_freq)[j];
    const int64_t pos = a.positions_64 ? reinterpret_cast<const int64_t*>(a.positions)[t0 + t]
                                       : (int64_t)reinterpret_cast<const int32_t*>(a.positions)[t0 + t];
    double turns = w * 0.15915494309189533577;  // 1 / (2 pi)
    turns -= floor(turns);
    const uint64_t frac = (uint64_t)(turns * 18446744073709551616.0) * (uint64_t)pos;
    float s, c;
    sincospif((float)(int32_t)(frac >> 32) * 0x1p-31f, &s, &c);
    if (!isfinite(w)) s = c = __int_as_float(0x7fffffff);
    s_cs[t * a.rot + j] = c * a.factor;
    s_cs[t * a.rot + half + j] = (a.inverse ? -s : s) * a.factor;
  }
  __syncthreads();
  if (!act) return;
  for (int t = slot; t < nt; t += a.pass) {
    float c[V], s[V];
    if (turned) {
#pragma unroll
      for (int k = 0; k < V; ++k) {
        c[k] = s_cs[t * a.rot + V * e + k];
        s[k] = s_cs[t * a.rot + half + V * e + k];
      }
    }
    for (int h0 = first; h0 < heads; h0 += stride) {
      if (t != slot || h0 != first) {
        if (h0 == first) token(t);
        batch(h0);
      }
#pragma unroll
      for (int b = 0; b < kRotBatch; ++b) {
        const int h = h0 + b * a.lanes, hk = h - a.heads[0];
        if (h >= heads) continue;
        T* p = hk < 0 ? yq + (int64_t)h * a.y_head_stride[0] : yk + (int64_t)hk * a.y_head_stride[1];
        if (turned) {
          turn<T, V, INTERLEAVED>(lo[b], hi[b], c, s);
          *reinterpret_cast<C*>(p + step) = hi[b];
        }
        *reinterpret_cast<C*>(p) = lo[b];
      }
    }
  }
}

template <typename T, int V, bool INTERLEAVED>
int launch_rotary(RotaryArgs a, int head_dim, bool through, cudaStream_t st) {
  a.turned = a.rot / 2 / V;
  a.items = a.turned + (through ? (head_dim - a.rot) / V : 0);
  a.per_head = a.items < kRotThreads ? a.items : kRotThreads;
  const int groups = (a.items + a.per_head - 1) / a.per_head;
  const int heads = a.heads[0] + a.heads[1], fit = kRotThreads / a.per_head;
  // Many tokens: a batch of heads for every thread, so that its cosines serve them all, and two passes of tokens a block.  Few: as many
  // threads a token as there are heads, and what a block cannot take dealt over several.
  const bool many = a.n_tokens * heads * a.per_head >= (int64_t)4 * kRotThreads * kRotBatch * sm_count();
  a.lanes = many ? (heads + kRotBatch - 1) / kRotBatch : heads;
  if (a.lanes > fit) a.lanes = fit;
  a.pass = fit / a.lanes;
  a.tokens = many ? 2 * a.pass : a.pass;
  while (a.tokens > 1 && a.tokens * a.rot > 8 * kRotMaxDim) --a.tokens;
  if (a.pass > a.tokens) a.pass = a.tokens;
  const int64_t blocks = (a.n_tokens + a.tokens - 1) / a.tokens;
  if (blocks > 0x7fffffff) return TQ4_ERR_UNSUPPORTED;
  const int split = many ? 1 : (heads + kRotBatch * a.lanes - 1) / (kRotBatch * a.lanes);
  if (split > 65535 || groups > 65535) return TQ4_ERR_UNSUPPORTED;
  if (launch_kernel(rotary_kernel<T, V, INTERLEAVED>, dim3((unsigned)blocks, (unsigned)split, (unsigned)groups), dim3(kRotThreads),
                    (size_t)a.tokens * a.rot * sizeof(float), st, false, a) != cudaSuccess)
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
