// Layer norm, forward and backward, of a residual stream:
//   s = x + r,  h = (s - mean) / sqrt(var + eps),  y = w h + b
//   dx = rstd (g - mean(g) - h mean(g h)) + ds with g = w dy,
//   dw = sum over rows of dy h,  db = sum over rows of dy.
// The mean is the sum's quotient, off by its roundings, and what s - mean sums up
// to (a second pass over the row) corrects it. The variance is the mean square of
// s - mean, less that correction's, and not a difference of moments. So a large
// mean costs no accuracy, and a constant row has no variance.
// HBM-bound: about 10 operations an element.

#include <atomic>
#include <type_traits>

#include "train_utils.cuh"

namespace train {

namespace {

// Both passes hold a row in registers, so it is read once: `group` threads (whole
// warps) share it, each with one or two parts of 8 neighbours, and groups walk
// over rows. A thread keeps its columns from row to row, so the weights, and the
// backward pass's sums of dw and db, stay on the SM, and the next row is on its way
// while one is worked on. Arithmetic is on pairs of elements. What bounds both next to
// the memory is how many rows are under way (registers) and the instructions: converting
// 16-bit values, the group's reductions and the 8-bit form cost as many as the norm
// itself. 32768 rows of 4096 bf16 take 108 us forward (5.0 TB/s; 104 without the
// correction of the mean), 139 with the 8-bit form (4.8 TB/s), and 157 backward from it
// with the join of the columns' sums (4.3 TB/s).
constexpr int kMaxGroup = 512;
constexpr int kBlock = 256;  // threads of a block of several groups, about

__host__ __device__ inline std::int64_t held_groups(std::int64_t cols) { return (cols + kGroup - 1) / kGroup; }

// A part of a vector over the columns, of a type known at run time.
template <bool kAligned>
__device__ __forceinline__ void load_any(const void* p, Type t, int c, int cols, float2 (&v)[4]) {
  if (t == Type::f32) {
    Part<float, kAligned> k;
    k.load(static_cast<const float*>(p), c, cols);
    k.get(v);
  } else if (t == Type::bf16) {
    Part<__nv_bfloat16, kAligned> k;
    k.load(static_cast<const __nv_bfloat16*>(p), c, cols);
    k.get(v);
  } else {
    Part<__half, kAligned> k;
    k.load(static_cast<const __half*>(p), c, cols);
    k.get(v);
  }
}

__device__ __forceinline__ void sync_group(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id + 1), "r"(threads) : "memory");
}

// The sum of a value over a row's threads, in a fixed order, to all of them.
// `slots` (one for each of the group's warps) may be used again after another
// sum with other slots.
__device__ __forceinline__ float group_sum(float v, int group, int id, float* slots) {
  v = warp_sum(v);
  if (group == 32) return v;
  const int lane = threadIdx.x & 31, warps = group >> 5;
  if (lane == 0) slots[(threadIdx.x >> 5) - id * warps] = v;
  sync_group(id, group);
  v = lane < warps ? slots[lane] : 0.0f;
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);  // 16 warps at most
  return __shfl_sync(0xffffffffu, v, 0);
}

// The same of two values at the price of little more than one: after a first
// exchange the lower half of a warp sums one of them and the upper half the other.
__device__ __forceinline__ float2 group_sum2(float2 v, int group, int id, float* slots /* 32 */) {
  const int lane = threadIdx.x & 31, warps = group >> 5;
  const bool upper = lane >= 16;
  float mine = upper ? v.y : v.x;
  mine += __shfl_xor_sync(0xffffffffu, upper ? v.x : v.y, 16);
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
  if (group > 32) {
    if ((lane & 15) == 0) slots[lane + (threadIdx.x >> 5) - id * warps] = mine;
    sync_group(id, group);
    mine = (lane & 15) < warps ? slots[lane] : 0.0f;
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
  }
  return {__shfl_sync(0xffffffffu, mine, 0), __shfl_sync(0xffffffffu, mine, 16)};
}

struct None {};

// The tensors of a row as they are loaded. S: the residual's type, or None.
template <typename X, typename S, bool kAligned, int kParts>
struct FwdRow {
  Part<X, kAligned> x[kParts];
  Part<S, kAligned> r[kParts];
  __device__ __forceinline__ void load(const NormFwd& a, std::int64_t row, int group, int t) {
    const int cols = static_cast<int>(a.cols);
#pragma unroll
    for (int n = 0; n < kParts; ++n)
      x[n].load(static_cast<const X*>(a.x.p) + row * a.x.ld, (n * group + t) * 8, cols);
#pragma unroll
    for (int n = 0; n < kParts; ++n)
      r[n].load(static_cast<const S*>(a.r.p) + row * a.r.ld, (n * group + t) * 8, cols);
  }
};
template <typename X, bool kAligned, int kParts>
struct FwdRow<X, None, kAligned, kParts> {
  Part<X, kAligned> x[kParts];
  __device__ __forceinline__ void load(const NormFwd& a, std::int64_t row, int group, int t) {
#pragma unroll
    for (int n = 0; n < kParts; ++n)
      x[n].load(static_cast<const X*>(a.x.p) + row * a.x.ld, (n * group + t) * 8, static_cast<int>(a.cols));
  }
};

template <typename X, typename Y, typename S, bool kAligned, int kParts>
__global__ void __launch_bounds__(kMaxGroup) norm_fwd(const NormFwd a, const int group) {
  extern __shared__ float4 params[];
  __shared__ float slots[kMaxGroup / 32], slots2[32 * (kMaxGroup / 64)];  // a group of one warp uses none
  const int id = threadIdx.x / group, t = threadIdx.x - id * group, ids = blockDim.x / group, lane = threadIdx.x & 31;
  const int cols = static_cast<int>(a.cols), ng = static_cast<int>(held_groups(a.cols));
  const float inv = 1.0f / static_cast<float>(cols);
  const bool joined = lane > 0, last = lane == 31;
  const std::int64_t stride = static_cast<std::int64_t>(gridDim.x) * ids;
  std::int64_t row = static_cast<std::int64_t>(blockIdx.x) * ids + id;
  FwdRow<X, S, kAligned, kParts> in;
  if (row < a.rows) in.load(a, row, group, t);
  // Weights (0) and biases (1) of a thread's columns: one part's in registers, two
  // parts' in shared memory (in two halves), so that twice as many rows are under way.
  float2 kept[2][4];
  auto at = [&](int which, int n, int half) { return params + ((which * kParts + n) * 2 + half) * group + t; };
#pragma unroll
  for (int n = 0; n < kParts; ++n) {
    float2 w[4], b[4] = {};
    load_any<kAligned>(a.w, a.wt, (n * group + t) * 8, cols, w);
    if (a.b != nullptr) load_any<kAligned>(a.b, a.wt, (n * group + t) * 8, cols, b);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (kParts == 1) {
        kept[0][i] = w[i], kept[1][i] = b[i];
      } else if (id == 0 && i % 2 == 0) {
        *at(0, n, i / 2) = float4{w[i].x, w[i].y, w[i + 1].x, w[i + 1].y};
        *at(1, n, i / 2) = float4{b[i].x, b[i].y, b[i + 1].x, b[i + 1].y};
      }
    }
  }
  if (kParts > 1) __syncthreads();
  for (; row < a.rows; row += stride) {
    float2 v[kParts][4];
#pragma unroll
    for (int n = 0; n < kParts; ++n) {
      in.x[n].get(v[n]);
      if constexpr (!std::is_same<S, None>::value) {
        float2 r[4];
        in.r[n].get(r);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[n][i] = Elem<X>::rounded2(add2(v[n][i], r[i]));
      }
    }
    if (row + stride < a.rows) in.load(a, row + stride, group, t);
    float2 sum = {0.0f, 0.0f}, rest = {0.0f, 0.0f}, sq = {0.0f, 0.0f};
#pragma unroll
    for (int n = 0; n < kParts; ++n) {
      if constexpr (!std::is_same<S, None>::value)
        Part<X, kAligned>::store(static_cast<X*>(a.s) + row * a.cols, (n * group + t) * 8, cols, v[n], joined, last);
#pragma unroll
      for (int i = 0; i < 4; ++i) sum = add2(sum, v[n][i]);  // 0 past the row's end
    }
    const float mean = group_sum(sum.x + sum.y, group, id, slots + id * (group >> 5)) * inv;
#pragma unroll
    for (int n = 0; n < kParts; ++n) {
      const int left = cols - (n * group + t) * 8;
#pragma unroll
      for (int i = 0; i < 4; ++i) v[n][i] = add2(v[n][i], both(-mean));
      if (left < 8) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (2 * i >= left) v[n][i].x = 0.0f;
          if (2 * i + 1 >= left) v[n][i].y = 0.0f;
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        rest = add2(rest, v[n][i]);
        sq = fma2(v[n][i], v[n][i], sq);
      }
    }
    const float2 joined2 = group_sum2(float2{rest.x + rest.y, sq.x + sq.y}, group, id, slots2 + id * 32);
    const float off = joined2.x * inv, var = larger(joined2.y * inv - off * off, 0.0f);
    const float rstd = rsqrtf(var + a.eps);
    if (t == 0 && a.rstd != nullptr) {
      a.rstd[row] = rstd;
      if (a.mean != nullptr) a.mean[row] = mean + off;
    }
#pragma unroll
    for (int n = 0; n < kParts; ++n) {
      const int c = (n * group + t) * 8;
#pragma unroll
      for (int i = 0; i < 4; ++i) v[n][i] = fma2(v[n][i], both(rstd), both(-off * rstd));
      if (a.q != nullptr) {
        if (cols - c < 8) {  // zeros past the row's end
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (c + 2 * i >= cols) v[n][i].x = 0.0f;
            if (c + 2 * i + 1 >= cols) v[n][i].y = 0.0f;
          }
        }
        uint2 q;
        const unsigned e = pack_eight(v[n], q);
        if (c < ng * kGroup) {
          *reinterpret_cast<uint2*>(a.q + row * ng * kGroup + c) = q;
          if ((threadIdx.x & 3) == 0) a.scale[row * ng + c / kGroup] = static_cast<std::uint8_t>(e);
        }
      }
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        float2* to = v[n] + 2 * half;
        if constexpr (kParts == 1) {
          to[0] = fma2(to[0], kept[0][2 * half], kept[1][2 * half]);
          to[1] = fma2(to[1], kept[0][2 * half + 1], kept[1][2 * half + 1]);
        } else {
          const float4 w = *at(0, n, half), b = *at(1, n, half);
          to[0] = fma2(to[0], float2{w.x, w.y}, float2{b.x, b.y});
          to[1] = fma2(to[1], float2{w.z, w.w}, float2{b.z, b.w});
        }
      }
      Part<Y, kAligned>::store(static_cast<Y*>(a.y) + row * a.cols, c, cols, v[n], joined, last);
    }
  }
}

// The tensors of a row of the backward pass. kHeld: the normalised input comes
// from its 8-bit form; kSum: a gradient of the stream is added.
template <typename X, typename Y, bool kAligned, bool kHeld, bool kSum, int kParts>
struct BwdRow {
  Part<Y, kAligned> dy[kParts];
  Part<X, kAligned> s[kHeld ? 1 : kParts], ds[kSum ? kParts : 1];
  uint2 q[kHeld ? kParts : 1];  // 8 held values
  unsigned e[kHeld ? kParts : 1];
  float mean, rstd;

  __device__ __forceinline__ void load(const NormBwd& a, std::int64_t row, int group, int t) {
    const int cols = static_cast<int>(a.cols);
#pragma unroll
    for (int n = 0; n < kParts; ++n)
      dy[n].load(static_cast<const Y*>(a.dy.p) + row * a.dy.ld, (n * group + t) * 8, cols);
    if constexpr (kSum) {
#pragma unroll
      for (int n = 0; n < kParts; ++n)
        ds[n].load(static_cast<const X*>(a.ds.p) + row * a.ds.ld, (n * group + t) * 8, cols);
    }
    rstd = a.rstd[row];
    if constexpr (!kHeld) {
      mean = a.mean[row];
#pragma unroll
      for (int n = 0; n < kParts; ++n)
        s[n].load(static_cast<const X*>(a.s.p) + row * a.s.ld, (n * group + t) * 8, cols);
    } else {
      const int ng = static_cast<int>(held_groups(a.cols));
#pragma unroll
      for (int n = 0; n < kParts; ++n) {
        const int c = (n * group + t) * 8;
        q[n] = uint2{0, 0};
        e[n] = 1;
        if (c < cols) {
          q[n] = *reinterpret_cast<const uint2*>(a.q + row * ng * kGroup + c);
          e[n] = a.scale[row * ng + c / kGroup];
        }
      }
    }
  }

  // 0 past the row's end: -mean * rstd there would meet a dy of 0, but it can be
  // infinite where no normalised value of the row is
  __device__ __forceinline__ void normalised(int n, float2 (&h)[4]) const {
    if constexpr (kHeld) {
      unpack_eight(q[n], e[n], h);
    } else {
      s[n].get(h, mean);
      const float m = kAligned && s[n].left <= 0 ? 0.0f : mean;
#pragma unroll
      for (int i = 0; i < 4; ++i) h[i] = mul2(add2(h[i], both(-m)), both(rstd));
    }
  }
};

// A block adds its groups' sums of the columns up in shared memory and leaves one
// partial sum of each column, and norm_join adds those.
template <typename X, typename Y, bool kAligned, bool kHeld, bool kSum, int kParts>
__global__ void __launch_bounds__(kMaxGroup) norm_bwd(const NormBwd a, const int group, float* part) {
  extern __shared__ float sums[];  // [2][cols], where a block has more than one group
  __shared__ float slots[2][32 * (kMaxGroup / 32)];
  const int id = threadIdx.x / group, t = threadIdx.x - id * group, ids = blockDim.x / group, lane = threadIdx.x & 31;
  const int cols = static_cast<int>(a.cols);
  const float inv = 1.0f / static_cast<float>(cols);
  const std::int64_t stride = static_cast<std::int64_t>(gridDim.x) * ids;
  std::int64_t row = static_cast<std::int64_t>(blockIdx.x) * ids + id;
  BwdRow<X, Y, kAligned, kHeld, kSum, kParts> in;
  if (row < a.rows) in.load(a, row, group, t);
  float2 dw[kParts][4] = {}, db[kParts][4] = {}, w[kParts][4];
#pragma unroll
  for (int n = 0; n < kParts; ++n) load_any<kAligned>(a.w, a.wt, (n * group + t) * 8, cols, w[n]);
  for (unsigned turn = 0; row < a.rows; row += stride, turn ^= 1u) {
    float2 g[kParts][4], h[kParts][4], ds[kSum ? kParts : 1][4], c1 = {0.0f, 0.0f}, c2 = {0.0f, 0.0f};
#pragma unroll
    for (int n = 0; n < kParts; ++n) {
      in.normalised(n, h[n]);
      in.dy[n].get(g[n]);
      if constexpr (kSum) in.ds[n].get(ds[n]);
    }
    const float rstd = in.rstd;
    if (row + stride < a.rows) in.load(a, row + stride, group, t);
#pragma unroll
    for (int n = 0; n < kParts; ++n) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        dw[n][i] = fma2(g[n][i], h[n][i], dw[n][i]);
        db[n][i] = add2(db[n][i], g[n][i]);
        g[n][i] = mul2(g[n][i], w[n][i]);  // 0 past the row's end
        c1 = add2(c1, g[n][i]);
        c2 = fma2(g[n][i], h[n][i], c2);
      }
    }
    const float2 c = group_sum2(float2{c1.x + c1.y, c2.x + c2.y}, group, id, slots[turn] + id * 32);
    const float2 k0 = both(-c.x * inv), k1 = both(-c.y * inv), r = both(rstd);
#pragma unroll
    for (int n = 0; n < kParts; ++n) {
      const int at = (n * group + t) * 8;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        g[n][i] = mul2(fma2(h[n][i], k1, add2(g[n][i], k0)), r);
        if constexpr (kSum) g[n][i] = add2(g[n][i], ds[n][i]);
      }
      Part<X, kAligned>::store(static_cast<X*>(a.dx) + row * a.cols, at, cols, g[n], lane > 0, lane == 31);
      if constexpr (!std::is_same<X, Y>::value) {
        if (a.dr != nullptr)
          Part<Y, kAligned>::store(static_cast<Y*>(a.dr) + row * a.cols, at, cols, g[n], lane > 0, lane == 31);
      }
    }
  }
  if (part == nullptr) return;
  float* to = part + static_cast<std::int64_t>(blockIdx.x) * 2 * cols;
  for (int k = 0; k < ids; ++k) {  // group after group
    if (id == k) {
#pragma unroll
      for (int n = 0; n < kParts; ++n) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int at = (n * group + t) * 8 + i;
          if (at >= cols) continue;
          const float dwi = i & 1 ? dw[n][i / 2].y : dw[n][i / 2].x, dbi = i & 1 ? db[n][i / 2].y : db[n][i / 2].x;
          (k + 1 < ids ? sums : to)[at] = (k > 0 ? sums[at] : 0.0f) + dwi;
          (k + 1 < ids ? sums : to)[cols + at] = (k > 0 ? sums[cols + at] : 0.0f) + dbi;
        }
      }
    }
    if (k + 1 < ids) __syncthreads();
  }
}

// dw and db from `parts` partial sums [parts][2][cols], in a fixed order.
constexpr int kJoin = 32;
__global__ void __launch_bounds__(32 * kJoin) norm_join(const float* part, int parts, std::int64_t cols, void* dw,
                                                        void* db, Type t) {
  __shared__ float sums[kJoin][33];
  const std::int64_t col = static_cast<std::int64_t>(blockIdx.x) * 32 + threadIdx.x;
  float v = 0.0f;
  if (col < cols)
#pragma unroll 4
    for (int k = threadIdx.y; k < parts; k += kJoin) v += part[(2ll * k + blockIdx.y) * cols + col];
  sums[threadIdx.y][threadIdx.x] = v;
  __syncthreads();
  // 32 sums of a column each, joined by the warp that owns the column
  v = warp_sum(sums[threadIdx.x][threadIdx.y]);
  const std::int64_t mine = static_cast<std::int64_t>(blockIdx.x) * 32 + threadIdx.y;
  void* to = blockIdx.y == 0 ? dw : db;
  if (threadIdx.x == 0 && mine < cols && to != nullptr) store(to, t, mine, v);
}

// --- rows too long for registers, and rare pairs of types: a block sweeps a row several times ---

constexpr int kSweep = 256;

__global__ void __launch_bounds__(kSweep) norm_fwd_sweep(const NormFwd a) {
  __shared__ float slots[32];
  const int lane = threadIdx.x & 31;
  const std::int64_t ng = (a.cols + kGroup - 1) / kGroup;
  for (std::int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const std::int64_t xo = row * a.x.ld, oo = row * a.cols;
    auto stream = [&](std::int64_t i) {
      const float v = load(a.x.p, a.x.t, xo + i);
      return a.r.p != nullptr ? rounded(v + load(a.r.p, a.r.t, row * a.r.ld + i), a.x.t) : v;
    };
    float sum = 0.0f;
    for (std::int64_t i = threadIdx.x; i < a.cols; i += kSweep) {
      const float v = stream(i);
      if (a.s != nullptr) store(a.s, a.x.t, oo + i, v);
      sum += v;
    }
    const float mean = block_sum(sum, slots) / static_cast<float>(a.cols);
    float rest = 0.0f, sq = 0.0f;
    for (std::int64_t i = threadIdx.x; i < a.cols; i += kSweep) {
      const float d = stream(i) - mean;
      rest += d;
      sq += d * d;
    }
    const float off = block_sum(rest, slots) / static_cast<float>(a.cols);
    const float var = larger(block_sum(sq, slots) / static_cast<float>(a.cols) - off * off, 0.0f);
    const float rstd = rsqrtf(var + a.eps);
    if (threadIdx.x == 0) {
      if (a.mean != nullptr) a.mean[row] = mean + off;
      if (a.rstd != nullptr) a.rstd[row] = rstd;
    }
    for (std::int64_t i = threadIdx.x; i < ng * kGroup; i += kSweep) {  // whole warps
      float h = 0.0f;
      if (i < a.cols) {
        h = (stream(i) - mean - off) * rstd;
        const float y = h * load(a.w, a.wt, i) + (a.b != nullptr ? load(a.b, a.wt, i) : 0.0f);
        store(a.y, a.yt, oo + i, y);
      }
      if (a.q != nullptr) {
        const unsigned e = warp_scale(h);
        a.q[row * ng * kGroup + i] = static_cast<std::int8_t>(quantised(h, e));
        if (lane == 0) a.scale[row * ng + i / kGroup] = static_cast<std::uint8_t>(e);
      }
    }
  }
}

__device__ __forceinline__ float normalised(const NormBwd& a, std::int64_t row, std::int64_t i, std::int64_t ng,
                                            float mean, float rstd) {
  if (a.q != nullptr)
    return static_cast<float>(a.q[row * ng * kGroup + i]) * step_of(a.scale[row * ng + i / kGroup]);
  return (load(a.s.p, a.s.t, row * a.s.ld + i) - mean) * rstd;
}

__global__ void __launch_bounds__(kSweep) norm_bwd_sweep(const NormBwd a) {
  __shared__ float slots[32];
  const std::int64_t ng = (a.cols + kGroup - 1) / kGroup;
  for (std::int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const float mean = a.q != nullptr ? 0.0f : a.mean[row], rstd = a.rstd[row];
    float c1 = 0.0f, c2 = 0.0f;
    for (std::int64_t i = threadIdx.x; i < a.cols; i += kSweep) {
      const float g = load(a.dy.p, a.dy.t, row * a.dy.ld + i) * load(a.w, a.wt, i);
      c1 += g;
      c2 += g * normalised(a, row, i, ng, mean, rstd);
    }
    c1 = block_sum(c1, slots) / static_cast<float>(a.cols);
    c2 = block_sum(c2, slots) / static_cast<float>(a.cols);
    for (std::int64_t i = threadIdx.x; i < a.cols; i += kSweep) {
      const float g = load(a.dy.p, a.dy.t, row * a.dy.ld + i) * load(a.w, a.wt, i);
      float dx = rstd * (g - c1 - normalised(a, row, i, ng, mean, rstd) * c2);
      if (a.ds.p != nullptr) dx += load(a.ds.p, a.ds.t, row * a.ds.ld + i);
      store(a.dx, a.xt, row * a.cols + i, dx);
      if (a.dr != nullptr) store(a.dr, a.rt, row * a.cols + i, dx);
    }
  }
}

constexpr int kColRows = 8;  // rows in flight of a column block

// Partial sums over a share of the rows: part[share][2][cols] (dw, db).
__global__ void __launch_bounds__(32 * kColRows) norm_bwd_columns(const NormBwd a, float* part) {
  __shared__ float sw[kColRows][33], sb[kColRows][33];
  const std::int64_t ng = (a.cols + kGroup - 1) / kGroup;
  const std::int64_t col = static_cast<std::int64_t>(blockIdx.x) * 32 + threadIdx.x;
  const std::int64_t share = (a.rows + gridDim.y - 1) / gridDim.y;
  const std::int64_t first = blockIdx.y * share, last = min(first + share, a.rows);
  float dw = 0.0f, db = 0.0f;
  if (col < a.cols) {
    for (std::int64_t row = first + threadIdx.y; row < last; row += kColRows) {
      const float dy = load(a.dy.p, a.dy.t, row * a.dy.ld + col);
      dw += dy * normalised(a, row, col, ng, a.q != nullptr ? 0.0f : a.mean[row], a.rstd[row]);
      db += dy;
    }
  }
  sw[threadIdx.y][threadIdx.x] = dw;
  sb[threadIdx.y][threadIdx.x] = db;
  __syncthreads();
  if (threadIdx.y == 0 && col < a.cols) {
    for (int k = 1; k < kColRows; ++k) {
      dw += sw[k][threadIdx.x];
      db += sb[k][threadIdx.x];
    }
    part[2ll * blockIdx.y * a.cols + col] = dw;
    part[(2ll * blockIdx.y + 1) * a.cols + col] = db;
  }
}

// The stream's type, the norm's and the residual's: one type, or a 32-bit stream
// with a norm of 16 bits (autocast) and a residual of either. Others are swept.
bool paired(Type x, Type y) { return x == y || x == Type::f32; }
template <typename F>
void with_pair(Type x, Type y, F f) {
  if (x == Type::f32)
    with_type(y, [&](auto e) { f(float(), e); });
  else if (x == Type::bf16)
    f(__nv_bfloat16(), __nv_bfloat16());
  else
    f(__half(), __half());
}

bool aligned(const void* p, std::int64_t ld, std::int64_t cols) { return p == nullptr || aligned_rows(p, ld, cols); }

// A row's threads and how many rows a block and the GPU work on at once.
struct Walk {
  bool aligned;
  int parts, group, ids;  // parts 0: the row is too long, or its types are rare
};

// Two parts a thread halve the cost of a row's sums, where `two` says that their
// registers allow it, unless a row then leaves much more of its last warp idle (768
// columns are 96 threads of one part, or 48 of 64 of two).
Walk walk_of(std::int64_t cols, bool aligned, bool types, bool two) {
  Walk p{};
  p.aligned = aligned;
  if (!types || cols > 16 * kMaxGroup) return p;
  const int warps1 = static_cast<int>((cols + 255) / 256), warps2 = static_cast<int>((cols + 511) / 512);
  p.parts = cols > 8 * kMaxGroup || (two && 2 * warps2 * 4 <= warps1 * 5) ? 2 : 1;
  p.group = 32 * (p.parts == 1 ? warps1 : warps2);
  p.ids = p.group < kBlock ? kBlock / p.group : 1;
  return p;
}

// Blocks that fill the GPU, or fewer where a group would have under `least` rows.
// No more than run at once: the rest would walk over their rows after the others.
template <auto kKernel>
int blocks_of(const Walk& p, std::int64_t rows, int least, int shared) {
  // blocks of an SM, by the warps of a group: for one kernel they give a block's threads and its shared memory
  static Occupancy<kMaxGroup / 32 + 1> known;
  const int found = known.get(p.group / 32, [&](int* n) {
    return cudaOccupancyMaxActiveBlocksPerMultiprocessor(n, kKernel, p.group * p.ids, shared);
  });
  const int fit = found > 0 ? found : 1;
  const std::int64_t most = static_cast<std::int64_t>(sm_count()) * fit;
  const std::int64_t each = static_cast<std::int64_t>(least) * p.ids, want = (rows + each - 1) / each;
  return static_cast<int>(want < most ? want : most);
}

Walk walk_of(const NormBwd& a) {
  const bool all = aligned(a.dy.p, a.dy.ld, a.cols) && aligned(a.ds.p, a.ds.ld, a.cols) &&
                   aligned(a.s.p, a.s.ld, a.cols) && aligned(a.w, a.cols, a.cols);
  // One part or two: 112 or 89 us for 65536 rows of 1024 bf16, 110 or 83 from the 8-bit
  // form. With a gradient of the stream as well two spill (181 or 276 us for 16384 rows
  // of 4096 fp32), and unaligned rows have registers for two from the 8-bit form only
  // (253 or 359 us for 32768 rows of 3001 bf16, 312 or 294). Rows over 4096 take two
  // all the same: sweeps are slower yet (16384 rows of 8192 fp32 with a gradient of the
  // stream 591 or 2175 us, 8192 of 6001 476 or 749, 16384 of 6001 bf16 without 392 or 1435).
  const bool two = a.ds.p == nullptr && (all || a.q != nullptr);
  return walk_of(a.cols, all, paired(a.xt, a.dy.t) && (a.dr == nullptr || a.rt == a.dy.t), two);
}

// Shares of the rows of a sweep over the columns.
int sweep_shares(const NormBwd& a) {
  const std::int64_t blocks = (a.cols + 31) / 32, want = (8ll * sm_count() + blocks - 1) / blocks;
  const std::int64_t most = (a.rows + 63) / 64;
  return static_cast<int>(want < most ? want : most);
}

constexpr int kMostPartials = 16;  // blocks an SM: 2 * 16 * 148 sums of a column at most

constexpr int kParamBytes = 2 * 16 * static_cast<int>(sizeof(float));  // of a thread's two parts

template <auto kKernel>
cudaError_t go_fwd(const NormFwd& a, const Walk& p, cudaStream_t stream) {
  const int shared = p.parts == 1 ? 0 : kParamBytes * p.group;
  if (shared > 0) {
    const cudaError_t rc = allow_shared<kKernel>(kParamBytes * kMaxGroup);
    if (rc != cudaSuccess) return rc;
  }
  kKernel<<<blocks_of<kKernel>(p, a.rows, 1, shared), p.group * p.ids, shared, stream>>>(a, p.group);
  return cudaSuccess;
}

template <typename X, typename Y, typename S>
cudaError_t launch_fwd(const NormFwd& a, const Walk& p, cudaStream_t stream) {
  if (p.aligned)
    return p.parts == 1 ? go_fwd<norm_fwd<X, Y, S, true, 1>>(a, p, stream)
                        : go_fwd<norm_fwd<X, Y, S, true, 2>>(a, p, stream);
  return p.parts == 1 ? go_fwd<norm_fwd<X, Y, S, false, 1>>(a, p, stream)
                      : go_fwd<norm_fwd<X, Y, S, false, 2>>(a, p, stream);
}

template <auto kKernel>
int go_bwd(const NormBwd& a, const Walk& p, float* part, cudaStream_t stream) {
  const int shared = p.ids > 1 ? 2 * 8 * static_cast<int>(sizeof(float)) * p.parts * p.group : 0;
  int blocks = blocks_of<kKernel>(p, a.rows, 4, shared);
  if (blocks > kMostPartials * sm_count()) blocks = kMostPartials * sm_count();
  kKernel<<<blocks, p.group * p.ids, shared, stream>>>(a, p.group, part);
  return blocks;
}

template <typename X, typename Y, bool kAligned, bool kHeld, bool kSum>
int launch_bwd(const NormBwd& a, const Walk& p, float* part, cudaStream_t stream) {
  return p.parts == 1 ? go_bwd<norm_bwd<X, Y, kAligned, kHeld, kSum, 1>>(a, p, part, stream)
                      : go_bwd<norm_bwd<X, Y, kAligned, kHeld, kSum, 2>>(a, p, part, stream);
}

}  // namespace

cudaError_t norm_forward(const NormFwd& a, cudaStream_t stream) {
  const bool all = aligned(a.x.p, a.x.ld, a.cols) && aligned(a.r.p, a.r.ld, a.cols) && aligned(a.w, a.cols, a.cols) &&
                   aligned(a.b, a.cols, a.cols);
  // One part or two: 133 or 109 us for 32768 rows of 4096 bf16; unaligned rows, 125 or
  // 141 us for 65536 of 1001 bf16, but 162 or 115 us for 32768 of fp32 with a residual.
  const Walk p = walk_of(a.cols, all, paired(a.x.t, a.yt) && (a.r.p == nullptr || a.r.t == a.x.t || a.r.t == a.yt),
                         all || a.x.t == Type::f32);
  cudaError_t rc = cudaSuccess;
  if (p.parts == 0) {
    const std::int64_t most = 32ll * sm_count();
    norm_fwd_sweep<<<static_cast<unsigned>(a.rows < most ? a.rows : most), kSweep, 0, stream>>>(a);
  } else {
    with_pair(a.x.t, a.yt, [&](auto x, auto y) {
      using X = decltype(x);
      using Y = decltype(y);
      if (a.r.p == nullptr)
        rc = launch_fwd<X, Y, None>(a, p, stream);
      else if (a.r.t == a.x.t)
        rc = launch_fwd<X, Y, X>(a, p, stream);
      else
        rc = launch_fwd<X, Y, Y>(a, p, stream);
    });
  }
  if (rc != cudaSuccess) return rc;
  commux_ops::g_launches++;
  return cudaGetLastError();
}

std::int64_t norm_backward_work(const NormBwd& a) {
  const Walk p = walk_of(a);
  if (p.parts == 0) return 2ll * sweep_shares(a) * a.cols;
  const std::int64_t most = static_cast<std::int64_t>(kMostPartials) * sm_count();
  const std::int64_t want = (a.rows + 4ll * p.ids - 1) / (4ll * p.ids);
  return 2 * (want < most ? want : most) * a.cols;
}

cudaError_t norm_backward(const NormBwd& a, cudaStream_t stream) {
  const Walk p = walk_of(a);
  const bool columns = a.dw != nullptr || a.db != nullptr;
  int parts = 0;
  if (p.parts == 0) {
    const std::int64_t most = 32ll * sm_count();
    norm_bwd_sweep<<<static_cast<unsigned>(a.rows < most ? a.rows : most), kSweep, 0, stream>>>(a);
    commux_ops::g_launches++;
    if (columns) {
      parts = sweep_shares(a);
      norm_bwd_columns<<<dim3(static_cast<unsigned>((a.cols + 31) / 32), parts), dim3(32, kColRows), 0, stream>>>(
          a, a.work);
      commux_ops::g_launches++;
    }
  } else {
    with_pair(a.xt, a.dy.t, [&](auto x, auto y) {
      using X = decltype(x);
      using Y = decltype(y);
      float* part = columns ? a.work : nullptr;
      auto sum = [&](auto aligned, auto held) {
        constexpr bool kAligned = decltype(aligned)::value, kHeld = decltype(held)::value;
        parts = a.ds.p != nullptr ? launch_bwd<X, Y, kAligned, kHeld, true>(a, p, part, stream)
                                  : launch_bwd<X, Y, kAligned, kHeld, false>(a, p, part, stream);
      };
      auto held = [&](auto aligned) {
        a.q != nullptr ? sum(aligned, std::true_type()) : sum(aligned, std::false_type());
      };
      p.aligned ? held(std::true_type()) : held(std::false_type());
    });
    commux_ops::g_launches++;
  }
  if (columns) {
    norm_join<<<dim3(static_cast<unsigned>((a.cols + 31) / 32), 2), dim3(32, kJoin), 0, stream>>>(
        a.work, parts, a.cols, a.dw, a.db, a.wt);
    commux_ops::g_launches++;
  }
  return cudaGetLastError();
}

int sm_count() {
  static std::atomic<int> known[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev >= 64) return 148;
  int n = known[dev].load(std::memory_order_relaxed);
  if (n == 0) {
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) n = 148;
    known[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}

}  // namespace train
