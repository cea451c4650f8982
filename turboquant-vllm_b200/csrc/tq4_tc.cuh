// What the kernels on the 5th-generation tensor cores of tq4_prefill_tc.cu and tq4_tree_tc.cu share: operand descriptors, MMAs, mbarriers
// with bounded waits, moves between tensor memory and registers, and conversions of rows.
#pragma once
#include "tq4_attention.cuh"

namespace tq4 {
namespace {

constexpr int kBN = 64;         // tokens per tile
constexpr float kHidden = 1e-33f;  // key norm in shared memory of a token whose page id is out of range
constexpr float kNotFinite = 2e-33f;  // ... of one that has an infinite or NaN norm (trees): NaN to the rows that see it, nothing to others
constexpr float kQGain = 64.f;     // factor of the queries' terms, its inverse in the key norms: keeps the lo terms normal numbers

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
// 16-byte chunk c of row `row` inside a [rows][128 B] block, 128-byte swizzle
__device__ __forceinline__ uint32_t swz(int row, int c) { return (uint32_t)(row * 128 + ((c ^ (row & 7)) << 4)); }
// operand descriptor, 128-byte swizzle, 8-row groups 1024 bytes apart; `lbo`: distance of the 64-element blocks
// of an MN-major operand (K-major: unused)
__device__ __forceinline__ uint64_t make_desc(uint32_t saddr, uint32_t lbo) {
  return (uint64_t)((saddr & 0x3FFFFu) >> 4) | ((uint64_t)(lbo ? lbo >> 4 : 1) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// D (tensor memory) (+)= A * B, A (128 rows x 16 fp16 = 8 columns) from tensor memory
__device__ __forceinline__ void mma_ta(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %5, %5, %5}, p;\n\t}"
      ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(acc ? 1u : 0u), "r"(0u)
      : "memory");
}
// the same with A from shared memory
__device__ __forceinline__ void mma_sa(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%5, %5, %5, %5}, p;\n\t}"
      ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc ? 1u : 0u), "r"(0u)
      : "memory");
}
__device__ __forceinline__ void mma_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(done) : "r"(bar), "r"(parity) : "memory");
  return done != 0;
}
// Bounded wait for another role: also gives up as soon as the CTA is marked dead; marks it itself otherwise.
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, volatile int* dead) {
  for (int it = 0; it < (1 << 22); ++it) {
    if (bar_try(bar, parity)) return true;
    if ((it & 1023) == 1023 && *dead) return false;
  }
  *dead = 1;
  return false;
}
// Bounded wait for copies or MMAs in flight, which no other role can hold up: a dead CTA sees them home, too.
__device__ __forceinline__ bool bar_wait_own(uint32_t bar, uint32_t parity, volatile int* dead) {
  for (int it = 0; it < (1 << 22); ++it)
    if (bar_try(bar, parity)) return true;
  *dead = 1;
  return false;
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
__device__ __forceinline__ void expect_tx(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool elect_one_sync() {
  uint32_t pred;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(pred));
  return pred != 0;
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// 32 consecutive 32-bit columns of this thread's tensor-memory lane (with the wait)
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, "
      "%14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
        "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]),
        "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]),
        "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(taddr)
      : "memory");
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
// 16 columns, without the wait; tmem_ld16_wait names the registers so that no use of them moves above it.  (No
// memory clobber on these: the compiler may move shared-memory loads across them.)
__device__ __forceinline__ void tmem_ld16_async(uint32_t taddr, uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, "
      "%14, %15}, [%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
        "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_ld16_wait(uint32_t (&v)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]),
                 "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15]));
}
// all 32 or 64 columns of a score tile, with the wait
template <int N>
__device__ __forceinline__ void tmem_ld_cols(uint32_t taddr, uint32_t (&v)[N]) {
#pragma unroll
  for (int h = 0; h < N / 16; ++h) tmem_ld16_async(taddr + 16 * h, *reinterpret_cast<uint32_t(*)[16]>(v + 16 * h));
#pragma unroll
  for (int h = 0; h < N / 16; ++h) tmem_ld16_wait(*reinterpret_cast<uint32_t(*)[16]>(v + 16 * h));
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&v)[8]) {  // (no wait)
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
               ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]));
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&v)[16]) {  // (no wait)
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16};"
      ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
        "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]));
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ float ex2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float lg2_approx(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float y;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}
// pairs of fp32 values in one 64-bit register: one instruction does both
typedef unsigned long long f2;
__device__ __forceinline__ f2 pack2(float lo, float hi) {
  f2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void unpack2(f2 v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ f2 mul2(f2 a, f2 b) {
  f2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f2 add2(f2 a, f2 b) {
  f2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) {
  f2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint32_t pack_h2(float lo, float hi) {
  __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&h);
}
// two values -> fp16 hi pair and fp16 pair of what the rounding left
__device__ __forceinline__ void split2(float x0, float x1, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(x0, x1);
  const float2 f = __half22float2(h);
  hi = *reinterpret_cast<const uint32_t*>(&h);
  lo = pack_h2(x0 - f.x, x1 - f.y);
}
// power of two that brings a value into [1, 2), and its inverse
__device__ __forceinline__ void pow2_scale(float amax, float& sc, float& isc) {
  sc = isc = 1.f;
  if (amax > 0.f && amax < CUDART_INF_F) {
    const int e = min(max((int)((__float_as_uint(amax) >> 23) & 0xFFu) - 127, -100), 100);
    sc = __uint_as_float((uint32_t)(127 - e) << 23);
    isc = __uint_as_float((uint32_t)(127 + e) << 23);
  }
}

// two packed 16-bit values
__device__ __forceinline__ void half_pair(uint32_t w, bool f16, float& x0, float& x1) {
  if (f16) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
    x0 = f.x; x1 = f.y;
  } else {
    x0 = __uint_as_float(w << 16); x1 = __uint_as_float(w & 0xFFFF0000u);
  }
}

// 32 consecutive elements i .. i + 31 of a typed tensor
__device__ __forceinline__ void load32(const void* q, int dtype, int64_t i, bool vec_ok, float (&x)[32]) {
  if (!vec_ok) {
#pragma unroll
    for (int e = 0; e < 32; ++e) x[e] = load_as_float(q, dtype, i + e);
    return;
  }
  if (dtype == TQ4_F32) {
    const float4* p = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(q) + i);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float4 v = __ldg(p + e);
      x[4 * e] = v.x; x[4 * e + 1] = v.y; x[4 * e + 2] = v.z; x[4 * e + 3] = v.w;
    }
    return;
  }
  const uint4* p = reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(q) + i);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const uint4 v = __ldg(p + e);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (dtype == TQ4_F16) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[k]));
        x[8 * e + 2 * k] = f.x; x[8 * e + 2 * k + 1] = f.y;
      } else {
        x[8 * e + 2 * k] = __uint_as_float(w[k] << 16);
        x[8 * e + 2 * k + 1] = __uint_as_float(w[k] & 0xFFFF0000u);
      }
    }
  }
}

// 32 consecutive outputs
__device__ __forceinline__ void store32(void* p, int dtype, int64_t i, bool vec_ok, const float (&y)[32]) {
  if (dtype != TQ4_F32 && vec_ok) {
    uint4* d = reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(p) + i);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      uint32_t w[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (dtype == TQ4_F16) {
          w[k] = pack_h2(y[8 * q + 2 * k], y[8 * q + 2 * k + 1]);
        } else {
          const __nv_bfloat162 h = __floats2bfloat162_rn(y[8 * q + 2 * k], y[8 * q + 2 * k + 1]);
          w[k] = *reinterpret_cast<const uint32_t*>(&h);
        }
      }
      d[q] = make_uint4(w[0], w[1], w[2], w[3]);
    }
    return;
  }
#pragma unroll
  for (int q = 0; q < 8; ++q) {
    const float t[4] = {y[4 * q], y[4 * q + 1], y[4 * q + 2], y[4 * q + 3]};
    store4(p, dtype, i + 4 * q, t);
  }
}

}  // namespace
}  // namespace tq4
