// Enough of a GPU to run the one-warp kernels of tq4_rows.cu on the host: 32 threads as the lanes of a block, one block after the other,
// bulk copies that land when their mbarrier is waited for, and waits that give up where a test says so.
#pragma once
#include <barrier>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <functional>
#include <memory>
#include <mutex>
#include <thread>
#include <unordered_map>
#include <vector>

#include "tq4.h"

#define __device__
#define __global__
#define __forceinline__ inline
#define __grid_constant__
#define __launch_bounds__(...)
#define __shared__ static
#define __align__(n) __attribute__((aligned(n)))

struct uint2 { uint32_t x, y; };
struct uint4 { uint32_t x, y, z, w; };
struct Dim { unsigned x, y, z; };
inline Dim blockIdx{}, blockDim{32, 1, 1}, gridDim{1, 1, 1};
inline thread_local Dim threadIdx{};

template <typename A, typename B>
std::common_type_t<A, B> min(A a, B b) { return a < b ? a : b; }
template <typename A, typename B>
std::common_type_t<A, B> max(A a, B b) { return a > b ? a : b; }

// ---- lanes ---------------------------------------------------------------------------------------
inline std::unique_ptr<std::barrier<>> g_lanes;
inline int64_t g_exchange[32];
inline std::mutex g_lock;

inline void __syncwarp() { g_lanes->arrive_and_wait(); }
inline void __syncthreads() { g_lanes->arrive_and_wait(); }
template <typename F>
auto with_all_lanes(int64_t mine, F&& read) {
  g_exchange[threadIdx.x] = mine;
  __syncwarp();
  const auto r = read();
  __syncwarp();
  return r;
}
inline unsigned __ballot_sync(unsigned, bool p) {
  return with_all_lanes(p, [] {
    unsigned m = 0;
    for (int i = 0; i < 32; ++i) m |= (unsigned)(g_exchange[i] != 0) << i;
    return m;
  });
}
inline int __any_sync(unsigned m, bool p) { return __ballot_sync(m, p) != 0; }
inline int __all_sync(unsigned m, bool p) { return __ballot_sync(m, p) == 0xffffffffu; }
inline int __syncthreads_or(int p) { return __any_sync(0xffffffffu, p != 0); }
template <typename T>
T __shfl_sync(unsigned, T v, int lane) {
  return with_all_lanes((int64_t)v, [&] { return (T)g_exchange[lane]; });
}
inline int __popc(unsigned x) { return __builtin_popcount(x); }
inline int __clz(unsigned x) { return x ? __builtin_clz(x) : 32; }
inline void __threadfence() {}
template <typename T>
T atomicAdd(T* p, T v) { std::lock_guard<std::mutex> l(g_lock); const T old = *p; *p += v; return old; }
template <typename T>
T atomicOr(T* p, T v) { std::lock_guard<std::mutex> l(g_lock); const T old = *p; *p |= v; return old; }
template <typename T>
T atomicMin(T* p, T v) { std::lock_guard<std::mutex> l(g_lock); const T old = *p; *p = v < old ? v : old; return old; }
inline uint32_t __cvta_generic_to_shared(const void*) { return 0; }
inline void pdl_trigger() {}
inline void pdl_wait() {}

// ---- bulk copies and mbarriers --------------------------------------------------------------------
struct Copy {
  uint32_t dst, bar;
  const void* src;
  uint32_t bytes;
};
struct Bar {
  int64_t pending = 0;  // bytes
  bool armed = false;
  unsigned phases = 0;  // complete
};
alignas(128) inline unsigned char g_rows[1 << 20];
inline std::unordered_map<uint32_t, Bar> g_bars;
inline std::vector<Copy> g_in_flight;
inline int g_looks[32];                              // waits of a lane in this block so far
inline std::function<bool(int lane, int look)> g_gives_up = [](int, int) { return false; };

inline uint32_t smem_of(const void* p) { return (uint32_t)(reinterpret_cast<const char*>(p) - reinterpret_cast<const char*>(g_rows)); }
inline unsigned char* at_smem(uint32_t a) { return g_rows + (int32_t)a; }
inline void bar_init(uint32_t bar) { std::lock_guard<std::mutex> l(g_lock); g_bars[bar] = Bar{}; }
inline void bar_fence() {}
inline void settle(Bar& b) {
  if (b.armed && b.pending == 0) {
    b.armed = false;
    ++b.phases;
  }
}
inline void bar_expect(uint32_t bar, uint32_t bytes) {
  std::lock_guard<std::mutex> l(g_lock);
  Bar& b = g_bars[bar];
  b.pending += bytes;
  b.armed = true;
  settle(b);
}
inline void bulk_in(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  std::lock_guard<std::mutex> l(g_lock);
  g_in_flight.push_back({dst, bar, src, bytes});
}
inline void bulk_out(void* dst, uint32_t src, uint32_t bytes) {
  std::lock_guard<std::mutex> l(g_lock);
  std::memcpy(dst, at_smem(src), bytes);
}
inline void bulk_commit() {}
template <int N>
void bulk_wait_read() {}
inline void bulk_wait_all() {}
inline bool bar_wait(uint32_t bar, uint32_t parity) {
  if (g_gives_up(threadIdx.x, g_looks[threadIdx.x]++)) return false;
  for (int it = 0; it < 1 << 16; ++it) {
    {
      std::lock_guard<std::mutex> l(g_lock);
      Bar& b = g_bars[bar];
      for (size_t i = 0; i < g_in_flight.size();) {
        const Copy c = g_in_flight[i];
        if (c.bar != bar) {
          ++i;
          continue;
        }
        std::memcpy(at_smem(c.dst), c.src, c.bytes);
        b.pending -= c.bytes;
        g_in_flight.erase(g_in_flight.begin() + i);
      }
      settle(b);
      if ((b.phases & 1) != parity) return true;
    }
    std::this_thread::yield();
  }
  return false;
}
inline void mark_set(int* mark) { std::lock_guard<std::mutex> l(g_lock); *mark = 1; }
inline bool mark_wait(const int* mark) { std::lock_guard<std::mutex> l(g_lock); return *mark != 0; }
inline void mark_fence() {}

// One block; says whether it left copies in flight behind.
template <typename F>
bool run_block(unsigned block, F&& kernel) {
  blockIdx = {block, 0, 0};
  g_lanes = std::make_unique<std::barrier<>>(32);
  g_in_flight.clear();
  std::memset(g_looks, 0, sizeof g_looks);
  std::vector<std::thread> lanes;
  for (unsigned i = 0; i < 32; ++i)
    lanes.emplace_back([&, i] {
      threadIdx = {i, 0, 0};
      kernel();
      g_lanes->arrive_and_drop();
    });
  for (auto& t : lanes) t.join();
  return g_in_flight.empty();
}
