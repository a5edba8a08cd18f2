#pragma once

// Device helpers of the training operators: typed element access, reductions
// over a block, and the 8-bit form.

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "train.hpp"

namespace train {

__device__ __forceinline__ float load(const void* p, Type t, std::int64_t i) {
  if (t == Type::f32) return static_cast<const float*>(p)[i];
  if (t == Type::bf16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(static_cast<const __half*>(p)[i]);
}

__device__ __forceinline__ void store(void* p, Type t, std::int64_t i, float v) {
  if (t == Type::f32)
    static_cast<float*>(p)[i] = v;
  else if (t == Type::bf16)
    static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  else
    static_cast<__half*>(p)[i] = __float2half_rn(v);
}

// v rounded to type t
__device__ __forceinline__ float rounded(float v, Type t) {
  if (t == Type::f32) return v;
  if (t == Type::bf16) return __bfloat162float(__float2bfloat16_rn(v));
  return __half2float(__float2half_rn(v));
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

__device__ __forceinline__ float warp_max(float v) {  // NaN if a lane has one
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float u = __shfl_xor_sync(0xffffffffu, v, o);
    v = u > v || u != u ? u : v;
  }
  return v;
}

// Sum over the block (a multiple of 32 threads), in a fixed order, to every thread.
__device__ __forceinline__ float block_sum(float v, float* slots /* 32 floats */) {
  v = warp_sum(v);
  __syncthreads();  // the slots' last readers are done
  if ((threadIdx.x & 31) == 0) slots[threadIdx.x >> 5] = v;
  __syncthreads();
  const int warps = blockDim.x >> 5, lane = threadIdx.x & 31;
  return warp_sum(lane < warps ? slots[lane] : 0.0f);
}

__device__ __forceinline__ float block_max(float v, float* slots) {
  v = warp_max(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) slots[threadIdx.x >> 5] = v;
  __syncthreads();
  const int warps = blockDim.x >> 5, lane = threadIdx.x & 31;
  return warp_max(lane < warps ? slots[lane] : -INFINITY);
}

// Scale byte of a group from the bits of its largest magnitude (a NaN's bits
// are above an infinity's, so a maximum over the bits keeps both). The step is
// the smallest power of two s >= 2^-126 with 127 s >= big: 127 = 1.984375 * 64,
// whose mantissa is 0x7e0000, so adding 0x1ffff carries into the exponent
// exactly where the mantissa is above that.
__device__ __forceinline__ unsigned scale_of(unsigned big) {
  if (big >= 0x7f800000u) return 255u;
  const int e = static_cast<int>((big + 0x1ffffu) >> 23) - 6;
  return static_cast<unsigned>(max(e, 1));
}

// 1 / 2^(e-127), a normal number (e is at most 249: no group needs a larger step)
__device__ __forceinline__ float inverse_step(unsigned e) { return __uint_as_float((254u - e) << 23); }
// 2^(e-127); NaN for 255
__device__ __forceinline__ float step_of(unsigned e) {
  return __uint_as_float(e == 255u ? 0x7fffffffu : e << 23);
}

__device__ __forceinline__ int quantise(float v, unsigned e) {
  // x / s is exact, so this is rint(x / s), |.| <= 127. At the largest step,
  // 2^122, 64 would stand for 2^128, an infinity: 63 stands in.
  const int q = e == 255u ? 0 : __float2int_rn(v * inverse_step(e));
  return e == 249u ? max(-63, min(63, q)) : q;
}

// The scale byte of the 32 values that a warp holds, one in each lane.
__device__ __forceinline__ unsigned warp_scale(float v) {
  return scale_of(__reduce_max_sync(0xffffffffu, __float_as_uint(v) & 0x7fffffffu));
}

}  // namespace train
