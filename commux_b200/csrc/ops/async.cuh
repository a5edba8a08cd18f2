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

__device__ __forceinline__ void mbar_init(std::uint64_t* bar, unsigned count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count) : "memory");
}

__device__ __forceinline__ void mbar_expect_tx(std::uint64_t* bar, unsigned bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes)
               : "memory");
}

__device__ __forceinline__ bool mbar_try_wait(std::uint64_t* bar, unsigned parity) {
  unsigned done;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
      " selp.b32 %0, 1, 0, p;\n}\n"
      : "=r"(done)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return done != 0;
}

// Bounded wait; false if it gave up.
__device__ __forceinline__ bool mbar_wait(std::uint64_t* bar, unsigned parity, std::uint64_t limit_ns) {
  if (mbar_try_wait(bar, parity)) return true;
  const std::uint64_t t0 = gtimer();
  while (!mbar_try_wait(bar, parity)) {
    if (gtimer() - t0 > limit_ns) return false;
  }
  return true;
}

__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, int x, int y, int z,
                                            std::uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<std::uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
      : "memory");
}

__device__ __forceinline__ void tma_load_2d(void* dst, const CUtensorMap* map, int x, int y, std::uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3}], [%4];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<std::uint64_t>(map)), "r"(x), "r"(y), "r"(smem_u32(bar))
      : "memory");
}

__device__ __forceinline__ void mbar_arrive(std::uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
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

__device__ __forceinline__ bool bounded_wait(std::uint64_t* bar, unsigned parity, const Bound& b) {
  if (mbar_try_wait(bar, parity)) return true;
  const std::uint64_t t0 = gtimer();
  while (!mbar_try_wait(bar, parity)) {
    if (*b.gave_up != 0) return false;
    if (gtimer() - t0 > b.limit_ns) {
      *b.gave_up = 1;
      if (b.status != nullptr) atomicExch(b.status, 1u);
      return false;
    }
  }
  return true;
}

}  // namespace async
