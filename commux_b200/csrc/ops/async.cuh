#pragma once

// Asynchronous copies and barriers in shared memory (sm_100a), as the kernels
// that use TMA share them.

#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace async {

__device__ __forceinline__ std::uint32_t smem_u32(const void* p) {
  return static_cast<std::uint32_t>(__cvta_generic_to_shared(p));
}

__device__ __forceinline__ std::uint64_t gtimer() {
  std::uint64_t t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}

// Writes of this thread to shared memory become visible to TMA and the tensor core.
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// What the waits of a CTA share: once one gave up (it records that in the
// status word), the others return at once and every role leaves its loop.
struct Bound {
  volatile int* gave_up;  // shared memory, 0 at first
  unsigned* status;
  std::uint64_t limit_ns;
};

// The waits below take the barrier's address in shared memory.
template <bool kCluster>
__device__ __forceinline__ bool try_wait(std::uint32_t bar, unsigned parity) {
  unsigned done;
  if constexpr (kCluster)  // a barrier that the cluster's other CTAs arrive on
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n"
        " selp.b32 %0, 1, 0, p;\n}\n"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
  else
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
        " selp.b32 %0, 1, 0, p;\n}\n"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
  return done != 0;
}

template <bool kCluster>
__device__ __forceinline__ bool wait_here(std::uint32_t bar, unsigned parity, volatile int* gave_up, unsigned* status,
                                          std::uint64_t limit_ns) {
  std::uint64_t since = 0;
  while (!try_wait<kCluster>(bar, parity)) {  // which itself blocks for up to 4 us
    if (*gave_up != 0) return false;
    const std::uint64_t now = gtimer();
    if (since == 0) since = now;
    if (now - since >= limit_ns) {
      *gave_up = 1;
      if (status != nullptr) atomicExch(status, 1u);
      return false;
    }
  }
  return true;
}

template <bool kCluster>
__device__ __noinline__ bool wait_longer(std::uint32_t bar, unsigned parity, volatile int* gave_up, unsigned* status,
                                         std::uint64_t limit_ns) {
  return wait_here<kCluster>(bar, parity, gave_up, status, limit_ns);
}

// Short where the wait is over already: a lone thread that feeds the tensor core
// pays for every instruction between two products.
template <bool kCluster = false>
__device__ __forceinline__ bool wait(std::uint32_t bar, unsigned parity, const Bound& b) {
  if (try_wait<kCluster>(bar, parity)) return true;
  return wait_longer<kCluster>(bar, parity, b.gave_up, b.status, b.limit_ns);
}

// For a kernel without registers to spare: the call that wait() may make has every
// thread keep values in local memory, whether it is made or not.
template <bool kCluster = false>
__device__ __forceinline__ bool wait_inline(std::uint32_t bar, unsigned parity, const Bound& b) {
  return wait_here<kCluster>(bar, parity, b.gave_up, b.status, b.limit_ns);
}

// For blocks of a cluster whose last stores to each other's shared memory nobody
// waited for.
__device__ __forceinline__ void pause() {
  for (const std::uint64_t t0 = gtimer(); gtimer() - t0 < 1'000'000;) {
  }
}

__device__ __forceinline__ void arrive(std::uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}

__device__ __forceinline__ void init(std::uint32_t bar, unsigned count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}

__device__ __forceinline__ void expect_tx(std::uint32_t bar, unsigned bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}

__device__ __forceinline__ void load_2d(std::uint32_t dst, const CUtensorMap* map, int x, int y, std::uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
      "l"(reinterpret_cast<std::uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
      : "memory");
}

__device__ __forceinline__ void load_3d(std::uint32_t dst, const CUtensorMap* map, int x, int y, int z,
                                        std::uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
      "l"(reinterpret_cast<std::uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar)
      : "memory");
}

// The same by pointers.
__device__ __forceinline__ void mbar_init(std::uint64_t* bar, unsigned count) { init(smem_u32(bar), count); }
__device__ __forceinline__ void mbar_expect_tx(std::uint64_t* bar, unsigned bytes) { expect_tx(smem_u32(bar), bytes); }
__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, int x, int y, int z,
                                            std::uint64_t* bar) {
  load_3d(smem_u32(dst), map, x, y, z, smem_u32(bar));
}

// Bounded wait without a status; false if it gave up.
__device__ __forceinline__ bool mbar_wait(std::uint64_t* bar, unsigned parity, std::uint64_t limit_ns) {
  if (try_wait<false>(smem_u32(bar), parity)) return true;
  const std::uint64_t t0 = gtimer();
  while (!try_wait<false>(smem_u32(bar), parity)) {
    if (gtimer() - t0 > limit_ns) return false;
  }
  return true;
}

// A last wait, for a CTA's copies in flight before it ends. Copies arrive within
// microseconds; the bound, which no setting changes, is for a barrier that also
// counts arrivals of threads that gave up.
constexpr std::uint64_t kSettleNs = 20'000'000;
__device__ __forceinline__ void settle(std::uint32_t bar, unsigned parity) {
  for (const std::uint64_t t0 = gtimer(); !try_wait<false>(bar, parity) && gtimer() - t0 <= kSettleNs;) {
  }
}

// True in one lane of the warp.
__device__ __forceinline__ bool elect() {
  unsigned one;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.b32 %0, 1, 0, p;\n}\n" : "=r"(one));
  return one != 0;
}

// Place in a ring of n slots, and the parity of its round.
struct Place {
  unsigned slot = 0, round = 0;
  __device__ __forceinline__ void next(unsigned n) {
    if (++slot == n) {
      slot = 0;
      round ^= 1u;
    }
  }
};

}  // namespace async
