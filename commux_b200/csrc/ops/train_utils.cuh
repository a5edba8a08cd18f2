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

// Two fp32 operations in one instruction.
__device__ __forceinline__ float2 both(float v) { return {v, v}; }
__device__ __forceinline__ float2 add2(float2 a, float2 b) { return __fadd2_rn(a, b); }
__device__ __forceinline__ float2 mul2(float2 a, float2 b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) { return __ffma2_rn(a, b, c); }

// 2^x and 1/x to about two units of the last place; results (and arguments)
// under 2^-126 become 0.
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float inverse_fast(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float larger(float a, float b) {  // NaN if either is
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
__device__ __forceinline__ float larger(float a, float b, float c) {
  float y;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}

// Element types of the kernels that are compiled for each of them.
template <typename T>
struct Elem;
template <>
struct Elem<float> {
  static constexpr Type kType = Type::f32;
  static __device__ __forceinline__ float put(float v) { return v; }
  static __device__ __forceinline__ float2 rounded2(float2 v) { return v; }
};
template <>
struct Elem<__nv_bfloat16> {
  static constexpr Type kType = Type::bf16;
  static __device__ __forceinline__ __nv_bfloat16 put(float v) { return __float2bfloat16_rn(v); }
  static __device__ __forceinline__ float2 get2(unsigned w) {
    return {__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)};
  }
  static __device__ __forceinline__ unsigned put2(float2 v) {
    const __nv_bfloat162 r = __floats2bfloat162_rn(v.x, v.y);
    return *reinterpret_cast<const unsigned*>(&r);
  }
  static __device__ __forceinline__ unsigned larger2(unsigned a, unsigned b) {  // NaN if either is
    const __nv_bfloat162 r =
        __hmax2_nan(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
    return *reinterpret_cast<const unsigned*>(&r);
  }
  static __device__ __forceinline__ float2 rounded2(float2 v) { return get2(put2(v)); }
};
template <>
struct Elem<__half> {
  static constexpr Type kType = Type::f16;
  static __device__ __forceinline__ __half put(float v) { return __float2half_rn(v); }
  static __device__ __forceinline__ float2 get2(unsigned w) { return __half22float2(*reinterpret_cast<__half2*>(&w)); }
  static __device__ __forceinline__ unsigned put2(float2 v) {
    const __half2 r = __floats2half2_rn(v.x, v.y);
    return *reinterpret_cast<const unsigned*>(&r);
  }
  static __device__ __forceinline__ unsigned larger2(unsigned a, unsigned b) {  // NaN if either is
    const __half2 r = __hmax2_nan(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const unsigned*>(&r);
  }
  static __device__ __forceinline__ float2 rounded2(float2 v) { return get2(put2(v)); }
};

// A thread's part of a row: the 8 elements from column c, a multiple of 8, as
// four pairs; a warp's lanes hold parts that follow each other. Columns past
// the row's end read as 0 (or as get()'s fill) and are not written.
//
// kAligned: rows are whole numbers of parts on 16-byte boundaries. Otherwise a
// row begins `shift` elements after such a boundary, a part lies across two
// vectors (three of fp32), and the registers are shifted: loads stay 16 bytes
// wide, and a store's vector takes its first elements from the lane before.
// The 16 bytes around a row's ends belong to the row's allocation, which
// starts and ends on such a boundary; what is not the row's is masked.
template <typename T, bool kAligned>
struct Part {
  static constexpr int kWords = sizeof(T) * 2;                // of 8 elements
  static constexpr int E = 16 / sizeof(T);                    // elements of a vector
  static constexpr int kVectors = 8 / E + (kAligned ? 0 : 1);
  unsigned w[4 * kVectors];
  int shift, left;  // left: columns from c to the row's end

  static __device__ __forceinline__ int shift_of(const T* row) {
    return static_cast<int>(reinterpret_cast<std::uintptr_t>(row) & 15) / static_cast<int>(sizeof(T));
  }

  __device__ __forceinline__ void load(const T* row, int c, int cols) {
    shift = kAligned ? 0 : shift_of(row);
    left = cols - c;
    const uint4* from = reinterpret_cast<const uint4*>(row + c - shift);
#pragma unroll
    for (int k = 0; k < kVectors; ++k) {
      uint4 v = {0, 0, 0, 0};
      // a vector that holds an element of the part
      const bool some = kAligned ? left > 0 : left > 0 && k * E - shift < min(left, 8);
      if (some) v = from[k];
      w[4 * k] = v.x, w[4 * k + 1] = v.y, w[4 * k + 2] = v.z, w[4 * k + 3] = v.w;
    }
  }

  // `fill`: what columns past the end of an unaligned row become
  __device__ __forceinline__ void get(float2 (&v)[4], float fill = 0.0f) const {
    unsigned u[4 * kVectors];
#pragma unroll
    for (int i = 0; i < 4 * kVectors; ++i) u[i] = w[i];
    if constexpr (!kAligned) {
      const int words = shift * static_cast<int>(sizeof(T)) / 4;
      if constexpr (4 * kVectors >= kWords + 3) {
#pragma unroll
        for (int i = 0; i < kWords + 2; ++i)
          if (i + 2 < 4 * kVectors) u[i] = words & 2 ? u[i + 2] : u[i];
#pragma unroll
        for (int i = 0; i < kWords + 1; ++i)
          if (i + 1 < 4 * kVectors) u[i] = words & 1 ? u[i + 1] : u[i];
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 4) {
        v[i] = float2{__uint_as_float(u[2 * i]), __uint_as_float(u[2 * i + 1])};
      } else if constexpr (kAligned) {
        v[i] = Elem<T>::get2(u[i]);
      } else {
        v[i] = Elem<T>::get2(__funnelshift_r(u[i], u[i + 1], (shift & 1) * 16));
      }
    }
    if (!kAligned && left < 8) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (2 * i >= left) v[i].x = fill;
        if (2 * i + 1 >= left) v[i].y = fill;
      }
    }
  }

  // Every lane of the warp calls this. `joined`: the lane before holds the part
  // before c of the same row; `last`: the lane after does not hold the next.
  static __device__ __forceinline__ void store(T* row, int c, int cols, const float2 (&v)[4], bool joined, bool last) {
    unsigned own[kWords];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 4) {
        own[2 * i] = __float_as_uint(v[i].x);
        own[2 * i + 1] = __float_as_uint(v[i].y);
      } else {
        own[i] = Elem<T>::put2(v[i]);
      }
    }
    if constexpr (kAligned) {
      if (c >= cols) return;
#pragma unroll
      for (int k = 0; k < kWords / 4; ++k)
        reinterpret_cast<uint4*>(row + c)[k] = uint4{own[4 * k], own[4 * k + 1], own[4 * k + 2], own[4 * k + 3]};
    } else {
      const int shift = shift_of(row);
      // the 4 words before the part, then the part: the vectors begin `shift` elements before c
      unsigned u[kWords + 4];
#pragma unroll
      for (int i = 0; i < 4; ++i) u[i] = __shfl_up_sync(0xffffffffu, own[kWords - 4 + i], 1);
#pragma unroll
      for (int i = 0; i < kWords; ++i) u[4 + i] = own[i];
      const int back = E - shift, words = back * static_cast<int>(sizeof(T)) / 4;  // 1 to 4 whole words on
#pragma unroll
      for (int i = 0; i < kWords; ++i) u[i] = words & 4 ? u[i + 4] : u[i];
      if (!(words & 4)) {
#pragma unroll
        for (int i = 0; i < kWords + 2; ++i) u[i] = words & 2 ? u[i + 2] : u[i];
#pragma unroll
        for (int i = 0; i < kWords + 1; ++i) u[i] = words & 1 ? u[i + 1] : u[i];
      }
      if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int i = 0; i < kWords; ++i) u[i] = __funnelshift_r(u[i], u[i + 1], (back & 1) * 16);
      }
      // elements [from, to) of the vectors are to be written
      const int from = joined ? 0 : shift, to = cols - c + shift;
      T* at = row + c - shift;
#pragma unroll
      for (int k = 0; k < kWords / 4; ++k) {
        if (k * E >= from && (k + 1) * E <= to) {
          reinterpret_cast<uint4*>(at)[k] = uint4{u[4 * k], u[4 * k + 1], u[4 * k + 2], u[4 * k + 3]};
        } else {
#pragma unroll
          for (int i = k * E; i < (k + 1) * E; ++i)
            if (i >= from && i < to) put_element(at + i, u, i);
        }
      }
      if (last) {  // nobody takes the part's end over
#pragma unroll
        for (int i = 1; i < 8; ++i)
          if (i >= 8 - shift && c + i < cols) put_element(row + c + i, own, i);
      }
    }
  }

  static __device__ __forceinline__ void put_element(T* to, const unsigned* u, int i) {
    if constexpr (sizeof(T) == 4)
      *reinterpret_cast<unsigned*>(to) = u[i];
    else
      *reinterpret_cast<unsigned short*>(to) = static_cast<unsigned short>(u[i / 2] >> (16 * (i & 1)));
  }
};

// Rows of whole parts on 16-byte boundaries.
inline bool aligned_rows(const void* p, std::int64_t ld, std::int64_t cols) {
  return cols % 8 == 0 && ld % 8 == 0 && reinterpret_cast<std::uintptr_t>(p) % 16 == 0;
}

// Lets a kernel use more than 48 KB of shared memory: an attribute of the kernel
// on each device, set at its first use there.
template <auto kKernel>
cudaError_t allow_shared(int bytes) {
  static std::atomic<std::uint64_t> done{0};
  int device = 0;
  cudaError_t rc = cudaGetDevice(&device);
  if (rc != cudaSuccess) return rc;
  const std::uint64_t bit = 1ull << (device & 63);
  if (device < 64 && (done.load(std::memory_order_relaxed) & bit) != 0) return cudaSuccess;
  rc = cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (rc == cudaSuccess && device < 64) done.fetch_or(bit, std::memory_order_relaxed);
  return rc;
}

// What an occupancy query answered, by device and a small key; 0: not asked yet.
// An answer that fails is not kept, and its error is not left to the next check.
template <int kKeys>
class Occupancy {
 public:
  template <typename F>
  int get(int key, F query) {
    int device = 0;
    if (cudaGetDevice(&device) != cudaSuccess || device >= kDevices) device = -1;
    std::atomic<int>* at = device < 0 ? nullptr : &known_[device][key];
    int n = at != nullptr ? at->load(std::memory_order_relaxed) : 0;
    if (n > 0) return n;
    if (query(&n) != cudaSuccess || n < 1) {
      cudaGetLastError();
      return 0;
    }
    if (at != nullptr) at->store(n, std::memory_order_relaxed);
    return n;
  }

 private:
  static constexpr int kDevices = 16;
  std::atomic<int> known_[kDevices][kKeys]{};
};

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

__device__ __forceinline__ unsigned low_bytes(float a, float b, float c, float d) {
  return __byte_perm(__byte_perm(__float_as_uint(a), __float_as_uint(b), 0x0040),
                     __byte_perm(__float_as_uint(c), __float_as_uint(d), 0x0040), 0x5410);
}

// The 8-bit form of a group that four lanes hold: its scale byte, and this
// lane's 8 values as bytes. x / s is exact, so rint(x / s) is the low part of
// x / s + 1.5 * 2^23, rounded once: its low byte is the value's.
__device__ __forceinline__ unsigned pack_eight(const float2 (&v)[4], uint2& q) {
  float top = larger(larger(fabsf(v[0].x), fabsf(v[0].y), fabsf(v[1].x)), fabsf(v[1].y), fabsf(v[2].x));
  top = larger(larger(top, fabsf(v[2].y), fabsf(v[3].x)), fabsf(v[3].y));
  top = larger(top, __shfl_xor_sync(0xffffffffu, top, 1));
  top = larger(top, __shfl_xor_sync(0xffffffffu, top, 2));
  const unsigned e = scale_of(__float_as_uint(top) & 0x7fffffffu);
  const float inv = inverse_step(e);
  float2 n[4];
  if (e < 249u) {
#pragma unroll
    for (int i = 0; i < 4; ++i) n[i] = fma2(v[i], both(inv), both(12582912.0f));
  } else {
    // At the largest step, 2^122, 64 would stand for 2^128, an infinity: 63
    // stands in. Nothing is held for a group without steps.
    const float m = e == 255u ? 0.0f : inv;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      n[i] = float2{fminf(fmaxf(v[i].x * m, -63.0f), 63.0f) * (e != 255u) + 12582912.0f,
                    fminf(fmaxf(v[i].y * m, -63.0f), 63.0f) * (e != 255u) + 12582912.0f};
  }
  q.x = low_bytes(n[0].x, n[0].y, n[1].x, n[1].y);
  q.y = low_bytes(n[2].x, n[2].y, n[3].x, n[3].y);
  return e;
}

// 8 held values. A byte u = value + 128 in the low bits of 2^23's mantissa is
// 2^23 + u.
__device__ __forceinline__ void unpack_eight(uint2 q, unsigned e, float2 (&v)[4]) {
  const float s = step_of(e);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const unsigned word = (i < 2 ? q.x : q.y) ^ 0x80808080u, at = 0x7540u + 2 * (i & 1);
    const float2 f = {__uint_as_float(__byte_perm(word, 0x4b000000u, at)),
                      __uint_as_float(__byte_perm(word, 0x4b000000u, at + 1))};
    v[i] = mul2(add2(f, both(-8388736.0f)), both(s));
  }
}

// For the kernels that give a lane one element of a group: the scale byte of a
// warp's 32 values, and a value's byte (in the low bits).
__device__ __forceinline__ unsigned warp_scale(float v) {
  return scale_of(__reduce_max_sync(0xffffffffu, __float_as_uint(v) & 0x7fffffffu));
}
__device__ __forceinline__ unsigned quantised(float v, unsigned e) {
  float n = v * inverse_step(e);
  if (e >= 249u) n = e == 255u ? 0.0f : fminf(fmaxf(n, -63.0f), 63.0f);
  return __float_as_uint(n + 12582912.0f);
}

}  // namespace train
