// Layer norm, forward and backward, of a residual stream:
//   s = x + r,  h = (s - mean) / sqrt(var + eps),  y = w h + b
//   dx = rstd (g - mean(g) - h mean(g h)) + ds with g = w dy,
//   dw = sum over rows of dy h,  db = sum over rows of dy.
// The variance is the mean square of s - mean (a second pass over the row),
// not a difference of moments, so a large mean costs no accuracy.
// HBM-bound: about 10 operations an element.

#include "train_utils.cuh"

namespace train {

namespace {

// Both passes hold a row in registers, so it is read once: `group` threads (whole
// warps) share it, each with a few parts of 8 neighbours. Sums, products and the
// 8-bit form work on pairs of elements: a third of the instructions of a first
// version with one element at a time, which they bound.
constexpr int kMaxGroup = 512;

__host__ __device__ inline std::int64_t held_groups(std::int64_t cols) { return (cols + kGroup - 1) / kGroup; }

// A part of a tensor whose type is known at run time alone (the weights, the
// residual: their branches are the same for the whole grid).
template <bool kAligned>
__device__ __forceinline__ void load_any(const void* p, Type t, std::int64_t at, int c, int cols, float2 (&v)[4]) {
  if (t == Type::f32) {
    Part<float, kAligned> k;
    k.load(static_cast<const float*>(p) + at, c, cols);
    k.get(v);
  } else if (t == Type::bf16) {
    Part<__nv_bfloat16, kAligned> k;
    k.load(static_cast<const __nv_bfloat16*>(p) + at, c, cols);
    k.get(v);
  } else {
    Part<__half, kAligned> k;
    k.load(static_cast<const __half*>(p) + at, c, cols);
    k.get(v);
  }
}

template <bool kAligned>
__device__ __forceinline__ void store_any(void* p, Type t, std::int64_t at, int c, int cols, const float2 (&v)[4],
                                          bool joined, bool last) {
  if (t == Type::f32)
    Part<float, kAligned>::store(static_cast<float*>(p) + at, c, cols, v, joined, last);
  else if (t == Type::bf16)
    Part<__nv_bfloat16, kAligned>::store(static_cast<__nv_bfloat16*>(p) + at, c, cols, v, joined, last);
  else
    Part<__half, kAligned>::store(static_cast<__half*>(p) + at, c, cols, v, joined, last);
}

__device__ __forceinline__ void sync_group(int id, int threads) {
  if (threads > 32)
    asm volatile("bar.sync %0, %1;" ::"r"(id + 1), "r"(threads) : "memory");
}

// Sums of two values over a row's threads, in a fixed order. `slots` (one for
// each warp) may be used again after another sum with other slots.
__device__ __forceinline__ float2 group_sum(float2 v, int group, int id, float2* slots) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    v = add2(v, float2{__shfl_xor_sync(0xffffffffu, v.x, o), __shfl_xor_sync(0xffffffffu, v.y, o)});
  if (group == 32) return v;
  const int lane = threadIdx.x & 31, warps = group >> 5;
  if (lane == 0) slots[(threadIdx.x >> 5) % warps] = v;
  sync_group(id, group);
  v = lane < warps ? slots[lane] : float2{0.0f, 0.0f};
#pragma unroll
  for (int o = 8; o > 0; o >>= 1)  // 16 warps at most
    v = add2(v, float2{__shfl_xor_sync(0xffffffffu, v.x, o), __shfl_xor_sync(0xffffffffu, v.y, o)});
  return {__shfl_sync(0xffffffffu, v.x, 0), __shfl_sync(0xffffffffu, v.y, 0)};
}

// --- forward: one row to a group of threads, 256 threads or one row a block ---

constexpr int kFwdParts = 4;

template <typename X, typename Y, bool kAligned>
__global__ void __launch_bounds__(kMaxGroup) norm_fwd(const NormFwd a, const int group) {
  __shared__ float2 slots[2][32];
  const int id = threadIdx.x / group, t = threadIdx.x - id * group, lane = threadIdx.x & 31;
  const std::int64_t row = static_cast<std::int64_t>(blockIdx.x) * (blockDim.x / group) + id;
  if (row >= a.rows) return;  // a whole group
  const int cols = static_cast<int>(a.cols);
  const std::int64_t out = row * a.cols;
  const X* x = static_cast<const X*>(a.x.p) + row * a.x.ld;
  float2 v[kFwdParts][4];
  {
    Part<X, kAligned> k[kFwdParts];
#pragma unroll
    for (int n = 0; n < kFwdParts; ++n) k[n].load(x, (n * group + t) * 8, cols);
#pragma unroll
    for (int n = 0; n < kFwdParts; ++n) k[n].get(v[n]);
  }
  const bool joined = lane > 0, last = lane == 31;
  if (a.r.p != nullptr) {
#pragma unroll
    for (int n = 0; n < kFwdParts; ++n) {
      if (n * group * 8 >= cols) break;
      const int c = (n * group + t) * 8;
      float2 r[4];
      load_any<kAligned>(a.r.p, a.r.t, row * a.r.ld, c, cols, r);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[n][i] = Elem<X>::rounded2(add2(v[n][i], r[i]));
      Part<X, kAligned>::store(static_cast<X*>(a.s) + out, c, cols, v[n], joined, last);
    }
  }
  float2 sum = {0.0f, 0.0f}, sq = {0.0f, 0.0f};
#pragma unroll
  for (int n = 0; n < kFwdParts; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) sum = add2(sum, v[n][i]);  // 0 past the row's end
  const float inv = 1.0f / static_cast<float>(cols);
  sum = group_sum(sum, group, id, slots[0] + id * (group >> 5));
  const float mean = (sum.x + sum.y) * inv;
#pragma unroll
  for (int n = 0; n < kFwdParts; ++n) {
    const int left = cols - (n * group + t) * 8;
    if (left >= 8) {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[n][i] = add2(v[n][i], both(-mean));
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        v[n][i] = float2{2 * i < left ? v[n][i].x - mean : 0.0f, 2 * i + 1 < left ? v[n][i].y - mean : 0.0f};
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) sq = fma2(v[n][i], v[n][i], sq);
  }
  sq = group_sum(sq, group, id, slots[1] + id * (group >> 5));
  const float rstd = rsqrtf((sq.x + sq.y) * inv + a.eps);
  if (t == 0) {
    if (a.mean != nullptr) a.mean[row] = mean;
    if (a.rstd != nullptr) a.rstd[row] = rstd;
  }
  const int ng = static_cast<int>(held_groups(a.cols));
#pragma unroll
  for (int n = 0; n < kFwdParts; ++n) {
    if (n * group * 8 >= cols) break;
    const int c = (n * group + t) * 8;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[n][i] = mul2(v[n][i], both(rstd));
    if (a.q != nullptr) {
      uint2 q;
      const unsigned e = pack_eight(v[n], q);
      if (c < ng * kGroup) {
        *reinterpret_cast<uint2*>(a.q + row * ng * kGroup + c) = q;
        if ((threadIdx.x & 3) == 0) a.scale[row * ng + c / kGroup] = static_cast<std::uint8_t>(e);
      }
    }
    float2 w[4], b[4] = {};
    load_any<kAligned>(a.w, a.wt, 0, c, cols, w);
    if (a.b != nullptr) load_any<kAligned>(a.b, a.wt, 0, c, cols, b);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[n][i] = fma2(v[n][i], w[i], b[i]);
    Part<Y, kAligned>::store(static_cast<Y*>(a.y) + out, c, cols, v[n], joined, last);
  }
}

// --- backward: groups of threads walk over rows ---
//
// A thread keeps its columns from row to row, so their parts of dw and db stay
// in registers; a block adds its groups' parts up in shared memory and leaves
// one partial sum of each column, and norm_join adds those. The next row is on
// its way while one is worked on.

template <typename X, typename Y, bool kAligned, bool kHeld, int kParts>
struct BwdRow {
  Part<Y, kAligned> dy[kParts];
  Part<X, kAligned> s[kHeld ? 1 : kParts];
  uint2 q[kHeld ? kParts : 1];  // 8 held values
  unsigned e[kHeld ? kParts : 1];
  float mean, rstd;

  __device__ __forceinline__ void load(const NormBwd& a, std::int64_t row, int group, int t) {
    const int cols = static_cast<int>(a.cols);
    const Y* from = static_cast<const Y*>(a.dy.p) + row * a.dy.ld;
#pragma unroll
    for (int n = 0; n < kParts; ++n) dy[n].load(from, (n * group + t) * 8, cols);
    rstd = a.rstd[row];
    if constexpr (!kHeld) {
      mean = a.mean[row];
      const X* x = static_cast<const X*>(a.s.p) + row * a.s.ld;
#pragma unroll
      for (int n = 0; n < kParts; ++n) s[n].load(x, (n * group + t) * 8, cols);
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

  // past the row's end 0 (packed) or -mean * rstd, which meets a dy of 0
  __device__ __forceinline__ void normalised(int n, float2 (&h)[4]) const {
    if constexpr (kHeld) {
      unpack_eight(q[n], e[n], h);
    } else {
      s[n].get(h);
#pragma unroll
      for (int i = 0; i < 4; ++i) h[i] = mul2(add2(h[i], both(-mean)), both(rstd));
    }
  }
};

template <typename X, typename Y, bool kAligned, bool kHeld, int kParts>
__global__ void __launch_bounds__(kMaxGroup) norm_bwd(const NormBwd a, const int group, float* part) {
  extern __shared__ float sums[];  // [2][cols], where a block has more than one group
  __shared__ float2 slots[2][32];
  const int id = threadIdx.x / group, t = threadIdx.x - id * group, ids = blockDim.x / group, lane = threadIdx.x & 31;
  const int cols = static_cast<int>(a.cols);
  const float inv = 1.0f / static_cast<float>(cols);
  float2 dw[kParts][4] = {}, db[kParts][4] = {}, w[kParts][4];
#pragma unroll
  for (int n = 0; n < kParts; ++n) load_any<kAligned>(a.w, a.wt, 0, (n * group + t) * 8, cols, w[n]);
  const std::int64_t stride = static_cast<std::int64_t>(gridDim.x) * ids;
  std::int64_t row = static_cast<std::int64_t>(blockIdx.x) * ids + id;
  BwdRow<X, Y, kAligned, kHeld, kParts> next;
  if (row < a.rows) next.load(a, row, group, t);
  for (unsigned turn = 0; row < a.rows; row += stride, turn ^= 1u) {
    const BwdRow<X, Y, kAligned, kHeld, kParts> now = next;
    if (row + stride < a.rows) next.load(a, row + stride, group, t);
    float2 g[kParts][4], h[kParts][4], c1 = {0.0f, 0.0f}, c2 = {0.0f, 0.0f};
#pragma unroll
    for (int n = 0; n < kParts; ++n) {
      now.normalised(n, h[n]);
      now.dy[n].get(g[n]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        dw[n][i] = fma2(g[n][i], h[n][i], dw[n][i]);
        db[n][i] = add2(db[n][i], g[n][i]);
        g[n][i] = mul2(g[n][i], w[n][i]);  // 0 past the row's end
        c1 = add2(c1, g[n][i]);
        c2 = fma2(g[n][i], h[n][i], c2);
      }
    }
    const float2 c = group_sum(float2{c1.x + c1.y, c2.x + c2.y}, group, id, slots[turn] + id * (group >> 5));
    const float2 k0 = both(-c.x * inv), k1 = both(-c.y * inv), r = both(now.rstd);
#pragma unroll
    for (int n = 0; n < kParts; ++n) {
      const int at = (n * group + t) * 8;
#pragma unroll
      for (int i = 0; i < 4; ++i) g[n][i] = mul2(fma2(h[n][i], k1, add2(g[n][i], k0)), r);
      if (a.ds.p != nullptr) {
        Part<X, kAligned> k;
        float2 ds[4];
        k.load(static_cast<const X*>(a.ds.p) + row * a.ds.ld, at, cols);
        k.get(ds);
#pragma unroll
        for (int i = 0; i < 4; ++i) g[n][i] = add2(g[n][i], ds[i]);
      }
      Part<X, kAligned>::store(static_cast<X*>(a.dx) + row * a.cols, at, cols, g[n], lane > 0, lane == 31);
      if (a.dr != nullptr) store_any<kAligned>(a.dr, a.rt, row * a.cols, at, cols, g[n], lane > 0, lane == 31);
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
    float sq = 0.0f;
    for (std::int64_t i = threadIdx.x; i < a.cols; i += kSweep) {
      const float d = stream(i) - mean;
      sq += d * d;
    }
    const float rstd = rsqrtf(block_sum(sq, slots) / static_cast<float>(a.cols) + a.eps);
    if (threadIdx.x == 0) {
      if (a.mean != nullptr) a.mean[row] = mean;
      if (a.rstd != nullptr) a.rstd[row] = rstd;
    }
    for (std::int64_t i = threadIdx.x; i < ng * kGroup; i += kSweep) {  // whole warps
      float h = 0.0f;
      if (i < a.cols) {
        h = (stream(i) - mean) * rstd;
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

// The stream's type and the norm's: one type, or a 32-bit stream with a norm of
// 16 bits (autocast). Other pairs are swept.
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

// How the backward pass is laid out.
struct BwdPlan {
  bool aligned;
  int parts, group, ids, blocks;  // parts 0: sweeps, with `blocks` row shares
};

bool aligned(const void* p, std::int64_t ld, std::int64_t cols) { return p == nullptr || aligned_rows(p, ld, cols); }

// Threads of a group that hold `cols` in up to `parts` parts each.
int group_of(std::int64_t cols, int parts) {
  return static_cast<int>((cols + 8 * parts * 32 - 1) / (8 * parts * 32)) * 32;
}

BwdPlan plan_of(const NormBwd& a) {
  BwdPlan p{};
  p.aligned = aligned(a.dy.p, a.dy.ld, a.cols) && aligned(a.ds.p, a.ds.ld, a.cols) && aligned(a.s.p, a.s.ld, a.cols) &&
              aligned(a.w, a.cols, a.cols);
  // One part a thread keeps the registers (two sums and two values for each
  // element) near 80 and the loads of many rows in flight; long rows take two.
  p.parts = a.cols <= 8 * kMaxGroup ? 1 : a.cols <= 16 * kMaxGroup ? 2 : 0;
  if (!paired(a.xt, a.dy.t)) p.parts = 0;
  const int sms = sm_count();
  if (p.parts == 0) {
    const std::int64_t blocks = (a.cols + 31) / 32, want = (8ll * sms + blocks - 1) / blocks, most = (a.rows + 63) / 64;
    p.blocks = static_cast<int>(want < most ? want : most);
    return p;
  }
  p.group = group_of(a.cols, p.parts);
  p.ids = p.group < 384 ? 384 / p.group : 1;
  // two blocks an SM, or fewer where a group would have under four rows
  const std::int64_t want = (a.rows + 4ll * p.ids - 1) / (4ll * p.ids);
  p.blocks = static_cast<int>(want < 2 * sms ? want : 2 * sms);
  return p;
}

template <typename X, typename Y, bool kAligned, bool kHeld>
void launch_bwd(const NormBwd& a, const BwdPlan& p, float* part, cudaStream_t stream) {
  const int threads = p.group * p.ids;
  const std::size_t smem = p.ids > 1 ? 2 * sizeof(float) * a.cols : 0;
  if (p.parts == 1)
    norm_bwd<X, Y, kAligned, kHeld, 1><<<p.blocks, threads, smem, stream>>>(a, p.group, part);
  else
    norm_bwd<X, Y, kAligned, kHeld, 2><<<p.blocks, threads, smem, stream>>>(a, p.group, part);
}

}  // namespace

cudaError_t norm_forward(const NormFwd& a, cudaStream_t stream) {
  if (a.cols > 8 * kFwdParts * kMaxGroup || !paired(a.x.t, a.yt)) {
    const std::int64_t most = 32ll * sm_count();
    norm_fwd_sweep<<<static_cast<unsigned>(a.rows < most ? a.rows : most), kSweep, 0, stream>>>(a);
  } else {
    const bool all = aligned(a.x.p, a.x.ld, a.cols) && aligned(a.r.p, a.r.ld, a.cols) &&
                     aligned(a.w, a.cols, a.cols) && aligned(a.b, a.cols, a.cols);
    const int group = group_of(a.cols, kFwdParts), ids = group < 256 ? 256 / group : 1;
    const unsigned blocks = static_cast<unsigned>((a.rows + ids - 1) / ids);
    with_pair(a.x.t, a.yt, [&](auto x, auto y) {
      using X = decltype(x);
      using Y = decltype(y);
      if (all)
        norm_fwd<X, Y, true><<<blocks, group * ids, 0, stream>>>(a, group);
      else
        norm_fwd<X, Y, false><<<blocks, group * ids, 0, stream>>>(a, group);
    });
  }
  commux_ops::g_launches++;
  return cudaGetLastError();
}

std::int64_t norm_backward_work(const NormBwd& a) { return 2ll * plan_of(a).blocks * a.cols; }

cudaError_t norm_backward(const NormBwd& a, cudaStream_t stream) {
  const BwdPlan p = plan_of(a);
  const bool columns = a.dw != nullptr || a.db != nullptr;
  if (p.parts == 0) {
    const std::int64_t most = 32ll * sm_count();
    norm_bwd_sweep<<<static_cast<unsigned>(a.rows < most ? a.rows : most), kSweep, 0, stream>>>(a);
    commux_ops::g_launches++;
    if (columns) {
      norm_bwd_columns<<<dim3(static_cast<unsigned>((a.cols + 31) / 32), p.blocks), dim3(32, kColRows), 0, stream>>>(
          a, a.work);
      commux_ops::g_launches++;
    }
  } else {
    with_pair(a.xt, a.dy.t, [&](auto x, auto y) {
      using X = decltype(x);
      using Y = decltype(y);
      float* part = columns ? a.work : nullptr;
      if (p.aligned && a.q != nullptr)
        launch_bwd<X, Y, true, true>(a, p, part, stream);
      else if (p.aligned)
        launch_bwd<X, Y, true, false>(a, p, part, stream);
      else if (a.q != nullptr)
        launch_bwd<X, Y, false, true>(a, p, part, stream);
      else
        launch_bwd<X, Y, false, false>(a, p, part, stream);
    });
    commux_ops::g_launches++;
  }
  if (columns) {
    norm_join<<<dim3(static_cast<unsigned>((a.cols + 31) / 32), 2), dim3(32, kJoin), 0, stream>>>(
        a.work, p.blocks, a.cols, a.dw, a.db, a.wt);
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
