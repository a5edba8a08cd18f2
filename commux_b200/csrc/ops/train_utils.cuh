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

// Element types of the kernels that are compiled for each of them.
template <typename T>
struct Elem;
template <>
struct Elem<float> {
  static constexpr Type kType = Type::f32;
  static __device__ __forceinline__ float get(float v) { return v; }
  static __device__ __forceinline__ float put(float v) { return v; }
};
template <>
struct Elem<__nv_bfloat16> {
  static constexpr Type kType = Type::bf16;
  static __device__ __forceinline__ float get(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __nv_bfloat16 put(float v) { return __float2bfloat16_rn(v); }
  static __device__ __forceinline__ float2 get2(unsigned w) {
    return {__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)};
  }
  static __device__ __forceinline__ unsigned put2(float a, float b) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const unsigned*>(&v);
  }
};
template <>
struct Elem<__half> {
  static constexpr Type kType = Type::f16;
  static __device__ __forceinline__ float get(__half v) { return __half2float(v); }
  static __device__ __forceinline__ __half put(float v) { return __float2half_rn(v); }
  static __device__ __forceinline__ float2 get2(unsigned w) { return __half22float2(*reinterpret_cast<__half2*>(&w)); }
  static __device__ __forceinline__ unsigned put2(float a, float b) {
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const unsigned*>(&v);
  }
};

// The raw bits of 8 neighbours, on a 16-byte boundary: one or two wide loads
// that can be in flight before their first use.
template <typename T>
struct Eight {
  uint4 w;
  __device__ __forceinline__ void load(const T* p) { w = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void zero() { w = uint4{0, 0, 0, 0}; }
  __device__ __forceinline__ void get(float (&v)[8]) const {
    const unsigned u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = Elem<T>::get2(u[i]);
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  }
  __device__ __forceinline__ void put(const float (&v)[8]) {
    w = uint4{Elem<T>::put2(v[0], v[1]), Elem<T>::put2(v[2], v[3]), Elem<T>::put2(v[4], v[5]),
              Elem<T>::put2(v[6], v[7])};
  }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<uint4*>(p) = w; }
};
template <>
struct Eight<float> {
  float4 a, b;
  __device__ __forceinline__ void load(const float* p) {
    a = reinterpret_cast<const float4*>(p)[0];
    b = reinterpret_cast<const float4*>(p)[1];
  }
  __device__ __forceinline__ void zero() { a = b = float4{0, 0, 0, 0}; }
  __device__ __forceinline__ void get(float (&v)[8]) const {
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  }
  __device__ __forceinline__ void put(const float (&v)[8]) {
    a = float4{v[0], v[1], v[2], v[3]};
    b = float4{v[4], v[5], v[6], v[7]};
  }
  __device__ __forceinline__ void store(float* p) const {
    reinterpret_cast<float4*>(p)[0] = a;
    reinterpret_cast<float4*>(p)[1] = b;
  }
};

// Rows that can be read 8 elements at a time.
inline bool by_eight(const void* p, std::int64_t ld, std::int64_t cols) {
  return cols % 8 == 0 && ld % 8 == 0 && reinterpret_cast<std::uintptr_t>(p) % 16 == 0;
}

// Calls f with a value of the element type that t names.
template <typename F>
void with_type(Type t, F f) {
  if (t == Type::f32)
    f(float());
  else if (t == Type::bf16)
    f(__nv_bfloat16());
  else
    f(__half());
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

// x / s is exact, so rint(x / s) is the low part of x / s + 1.5 * 2^23, rounded
// once: its low byte is the value's. At the largest step, 2^122, 64 would stand
// for 2^128, an infinity: 63 stands in. Nothing is held for a group without steps.
__device__ __forceinline__ unsigned quantised(float v, unsigned e) {
  float n = v * inverse_step(e);
  if (e >= 249u) n = e == 255u ? 0.0f : fminf(fmaxf(n, -63.0f), 63.0f);
  return __float_as_uint(n + 12582912.0f);
}

__device__ __forceinline__ unsigned low_bytes(unsigned a, unsigned b, unsigned c, unsigned d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

__device__ __forceinline__ unsigned magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// 8 neighbours of a row to four lanes of a group: its scale byte to all four,
// this lane's 8 values as bytes.
__device__ __forceinline__ unsigned pack_eight(const float (&v)[8], uint2& q) {
  unsigned big = magnitude(v[0]);
#pragma unroll
  for (int i = 1; i < 8; ++i) big = max(big, magnitude(v[i]));
  big = max(big, __shfl_xor_sync(0xffffffffu, big, 1));
  big = max(big, __shfl_xor_sync(0xffffffffu, big, 2));
  const unsigned e = scale_of(big);
  unsigned n[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) n[i] = quantised(v[i], e);
  q.x = low_bytes(n[0], n[1], n[2], n[3]);
  q.y = low_bytes(n[4], n[5], n[6], n[7]);
  return e;
}

// 8 held values
__device__ __forceinline__ void unpack_eight(uint2 q, unsigned e, float (&v)[8]) {
  const float s = step_of(e);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const unsigned word = (i < 4 ? q.x : q.y) ^ 0x80808080u;  // u = value + 128 in a byte
    v[i] = (__uint_as_float(__byte_perm(word, 0x4b000000u, 0x7540u + (i & 3))) - 8388736.0f) * s;
  }
}

// The scale byte of the 32 values that a warp holds, one in each lane.
__device__ __forceinline__ unsigned warp_scale(float v) {
  return scale_of(__reduce_max_sync(0xffffffffu, magnitude(v)));
}

}  // namespace train
