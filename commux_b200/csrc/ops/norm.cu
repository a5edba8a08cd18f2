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

// Both passes hold a row in registers, 8 elements of it to a chunk and a few
// chunks to a thread, so a row is read once; `group` threads (whole warps) share
// it. Where the rows allow it a chunk is 8 neighbours (wide loads and stores),
// else 8 elements `group` apart (a warp's lanes on 32 neighbours), so that any
// length, stride and alignment keeps whole cache lines. A warp holds whole groups
// of the 8-bit form in both.
constexpr int kMaxGroup = 512;

__host__ __device__ inline std::int64_t held_groups(std::int64_t cols) { return (cols + kGroup - 1) / kGroup; }

template <typename T, bool kVec>
struct Chunk {
  Eight<T> w;
  __device__ __forceinline__ void load(const T* row, int c, int, int cols) {
    if (c < cols)
      w.load(row + c);
    else
      w.zero();
  }
  __device__ __forceinline__ void get(float (&v)[8]) const { w.get(v); }
  static __device__ __forceinline__ void store(T* row, int c, int, int cols, const float (&v)[8]) {
    if (c >= cols) return;
    Eight<T> o;
    o.put(v);
    o.store(row + c);
  }
};
template <typename T>
struct Chunk<T, false> {
  T w[8];
  __device__ __forceinline__ void load(const T* row, int c, int apart, int cols) {
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = c + i * apart < cols ? row[c + i * apart] : Elem<T>::put(0.0f);
  }
  __device__ __forceinline__ void get(float (&v)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = Elem<T>::get(w[i]);
  }
  static __device__ __forceinline__ void store(T* row, int c, int apart, int cols, const float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i * apart < cols) row[c + i * apart] = Elem<T>::put(v[i]);
  }
};

// A chunk of a tensor whose type is known at run time alone (the weights, the
// residual: their branches are the same for the whole grid).
template <bool kVec>
__device__ __forceinline__ void load_any(const void* p, Type t, std::int64_t at, int c, int apart, int cols,
                                         float (&v)[8]) {
  if (t == Type::f32) {
    Chunk<float, kVec> k;
    k.load(static_cast<const float*>(p) + at, c, apart, cols);
    k.get(v);
  } else if (t == Type::bf16) {
    Chunk<__nv_bfloat16, kVec> k;
    k.load(static_cast<const __nv_bfloat16*>(p) + at, c, apart, cols);
    k.get(v);
  } else {
    Chunk<__half, kVec> k;
    k.load(static_cast<const __half*>(p) + at, c, apart, cols);
    k.get(v);
  }
}

template <bool kVec>
__device__ __forceinline__ void store_any(void* p, Type t, std::int64_t at, int c, int apart, int cols,
                                          const float (&v)[8]) {
  if (t == Type::f32)
    Chunk<float, kVec>::store(static_cast<float*>(p) + at, c, apart, cols, v);
  else if (t == Type::bf16)
    Chunk<__nv_bfloat16, kVec>::store(static_cast<__nv_bfloat16*>(p) + at, c, apart, cols, v);
  else
    Chunk<__half, kVec>::store(static_cast<__half*>(p) + at, c, apart, cols, v);
}

// First element of this thread's chunk n, and whether element i is in the row.
template <bool kVec>
__device__ __forceinline__ int chunk_at(int n, int group, int t) {
  return kVec ? (n * group + t) * 8 : n * 8 * group + t;
}
template <bool kVec>
__device__ __forceinline__ bool in_row(int c, int i, int apart, int cols) {
  return kVec ? c < cols : c + i * apart < cols;
}

__device__ __forceinline__ void sync_group(int id, int threads) {
  if (threads > 32)
    asm volatile("bar.sync %0, %1;" ::"r"(id + 1), "r"(threads) : "memory");
}

// Sums of two values over a row's threads, in a fixed order. `slots` (one for
// each warp) may be used again after another sum with other slots.
__device__ __forceinline__ float2 group_sum(float a, float b, int group, int id, float2* slots) {
  a = warp_sum(a);
  b = warp_sum(b);
  if (group == 32) return {a, b};
  const int lane = threadIdx.x & 31, warps = group >> 5;
  if (lane == 0) slots[(threadIdx.x >> 5) % warps] = float2{a, b};
  sync_group(id, group);
  const float2 v = lane < warps ? slots[lane] : float2{0.0f, 0.0f};
  return {warp_sum(v.x), warp_sum(v.y)};
}

// A chunk's 8-bit form at its place in the row.
template <bool kVec>
__device__ __forceinline__ void pack_chunk(const float (&h)[8], std::int8_t* q, std::uint8_t* scale, int c, int apart,
                                           int padded) {
  if (kVec) {
    uint2 v;
    const unsigned e = pack_eight(h, v);
    if (c < padded) {
      *reinterpret_cast<uint2*>(q + c) = v;
      if ((threadIdx.x & 3) == 0) scale[c / kGroup] = static_cast<std::uint8_t>(e);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const unsigned e = warp_scale(h[i]);
      const int at = c + i * apart;
      if (at < padded) {
        q[at] = static_cast<std::int8_t>(quantised(h[i], e));
        if ((threadIdx.x & 31) == 0) scale[at / kGroup] = static_cast<std::uint8_t>(e);
      }
    }
  }
}

// --- forward: one row to a group of threads, 256 threads or one row a block ---

constexpr int kFwdChunks = 4;

template <typename X, typename Y, bool kVec>
__global__ void __launch_bounds__(kMaxGroup) norm_fwd(const NormFwd a, const int group) {
  __shared__ float2 slots[2][32];
  const int id = threadIdx.x / group, t = threadIdx.x - id * group;
  const std::int64_t row = static_cast<std::int64_t>(blockIdx.x) * (blockDim.x / group) + id;
  if (row >= a.rows) return;  // a whole group
  const int cols = static_cast<int>(a.cols), apart = group;
  const std::int64_t out = row * a.cols;
  const X* x = static_cast<const X*>(a.x.p) + row * a.x.ld;
  float v[kFwdChunks][8];
  {
    Chunk<X, kVec> k[kFwdChunks];
#pragma unroll
    for (int n = 0; n < kFwdChunks; ++n) k[n].load(x, chunk_at<kVec>(n, group, t), apart, cols);
#pragma unroll
    for (int n = 0; n < kFwdChunks; ++n) k[n].get(v[n]);
  }
  if (a.r.p != nullptr) {
#pragma unroll
    for (int n = 0; n < kFwdChunks; ++n) {
      const int c = chunk_at<kVec>(n, group, t);
      float r[8];
      load_any<kVec>(a.r.p, a.r.t, row * a.r.ld, c, apart, cols, r);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[n][i] = Elem<X>::get(Elem<X>::put(v[n][i] + r[i]));
      Chunk<X, kVec>::store(static_cast<X*>(a.s) + out, c, apart, cols, v[n]);
    }
  }
  float sum = 0.0f, sq = 0.0f;
#pragma unroll
  for (int n = 0; n < kFwdChunks; ++n)
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += v[n][i];  // 0 past the row's end
  const float inv = 1.0f / static_cast<float>(cols);
  const float mean = group_sum(sum, 0.0f, group, id, slots[0] + id * (group >> 5)).x * inv;
#pragma unroll
  for (int n = 0; n < kFwdChunks; ++n) {
    const int c = chunk_at<kVec>(n, group, t);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      v[n][i] = in_row<kVec>(c, i, apart, cols) ? v[n][i] - mean : 0.0f;
      sq += v[n][i] * v[n][i];
    }
  }
  const float rstd = rsqrtf(group_sum(sq, 0.0f, group, id, slots[1] + id * (group >> 5)).x * inv + a.eps);
  if (t == 0) {
    if (a.mean != nullptr) a.mean[row] = mean;
    if (a.rstd != nullptr) a.rstd[row] = rstd;
  }
  const int padded = static_cast<int>(held_groups(a.cols)) * kGroup;
#pragma unroll
  for (int n = 0; n < kFwdChunks; ++n) {
    const int c = chunk_at<kVec>(n, group, t);
    if (n > 0 && chunk_at<kVec>(n, group, 0) >= cols) break;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[n][i] *= rstd;
    if (a.q != nullptr)
      pack_chunk<kVec>(v[n], a.q + row * padded, a.scale + row * (padded / kGroup), c, apart, padded);
    float w[8], b[8] = {};
    load_any<kVec>(a.w, a.wt, 0, c, apart, cols, w);
    if (a.b != nullptr) load_any<kVec>(a.b, a.wt, 0, c, apart, cols, b);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[n][i] = v[n][i] * w[i] + b[i];
    Chunk<Y, kVec>::store(static_cast<Y*>(a.y) + out, c, apart, cols, v[n]);
  }
}

// --- backward: groups of threads walk over rows ---
//
// A thread keeps its columns from row to row, so their parts of dw and db stay
// in registers; a block adds its groups' parts up in shared memory and leaves
// one partial sum of each column, and norm_join adds those. The next row is on
// its way while one is worked on.

template <typename X, typename Y, bool kVec, bool kHeld, int kChunks>
struct BwdRow {
  Chunk<Y, kVec> dy[kChunks];
  Chunk<X, kVec> s[kHeld ? 1 : kChunks];
  uint2 q[kHeld ? kChunks : 1];  // 8 held values
  unsigned e[kHeld ? kChunks : 1][kVec ? 1 : 8];
  float mean, rstd;

  __device__ __forceinline__ void load(const NormBwd& a, std::int64_t row, int group, int t) {
    const int cols = static_cast<int>(a.cols);
    const Y* from = static_cast<const Y*>(a.dy.p) + row * a.dy.ld;
#pragma unroll
    for (int n = 0; n < kChunks; ++n) dy[n].load(from, chunk_at<kVec>(n, group, t), group, cols);
    rstd = a.rstd[row];
    if constexpr (!kHeld) {
      mean = a.mean[row];
      const X* x = static_cast<const X*>(a.s.p) + row * a.s.ld;
#pragma unroll
      for (int n = 0; n < kChunks; ++n) s[n].load(x, chunk_at<kVec>(n, group, t), group, cols);
    } else {
      const int ng = static_cast<int>(held_groups(a.cols));
      const std::int8_t* held = a.q + row * ng * kGroup;
      const std::uint8_t* scale = a.scale + row * ng;
#pragma unroll
      for (int n = 0; n < kChunks; ++n) {
        const int c = chunk_at<kVec>(n, group, t);
        q[n] = uint2{0, 0};
        if constexpr (kVec) {
          e[n][0] = 1;
          if (c < cols) {
            q[n] = *reinterpret_cast<const uint2*>(held + c);
            e[n][0] = scale[c / kGroup];
          }
        } else {
          unsigned b[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int at = c + i * group;
            b[i] = 0;
            e[n][i] = 1;
            if (at < cols) {
              b[i] = static_cast<std::uint8_t>(held[at]);
              e[n][i] = scale[at / kGroup];
            }
          }
          q[n] = uint2{low_bytes(b[0], b[1], b[2], b[3]), low_bytes(b[4], b[5], b[6], b[7])};
        }
      }
    }
  }

  __device__ __forceinline__ void normalised(const NormBwd& a, int n, int c, int group, float (&h)[8]) const {
    if constexpr (!kHeld) {
      s[n].get(h);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        h[i] = in_row<kVec>(c, i, group, static_cast<int>(a.cols)) ? (h[i] - mean) * rstd : 0.0f;
    } else if constexpr (kVec) {
      unpack_eight(q[n], e[n][0], h);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        h[i] = static_cast<float>(static_cast<std::int8_t>((i < 4 ? q[n].x : q[n].y) >> (8 * (i & 3)))) *
               step_of(e[n][i]);
    }
  }
};

template <typename X, typename Y, bool kVec, bool kHeld, int kChunks>
__global__ void __launch_bounds__(kMaxGroup) norm_bwd(const NormBwd a, const int group, float* part) {
  extern __shared__ float sums[];  // [2][cols], where a block has more than one group
  __shared__ float2 slots[2][32];
  const int id = threadIdx.x / group, t = threadIdx.x - id * group, ids = blockDim.x / group;
  const int cols = static_cast<int>(a.cols);
  const float inv = 1.0f / static_cast<float>(cols);
  float dw[kChunks][8] = {}, db[kChunks][8] = {}, w[kChunks][8];
#pragma unroll
  for (int n = 0; n < kChunks; ++n) load_any<kVec>(a.w, a.wt, 0, chunk_at<kVec>(n, group, t), group, cols, w[n]);
  const std::int64_t stride = static_cast<std::int64_t>(gridDim.x) * ids;
  std::int64_t row = static_cast<std::int64_t>(blockIdx.x) * ids + id;
  BwdRow<X, Y, kVec, kHeld, kChunks> next;
  if (row < a.rows) next.load(a, row, group, t);
  for (unsigned turn = 0; row < a.rows; row += stride, turn ^= 1u) {
    const BwdRow<X, Y, kVec, kHeld, kChunks> now = next;
    if (row + stride < a.rows) next.load(a, row + stride, group, t);
    float g[kChunks][8], h[kChunks][8], c1 = 0.0f, c2 = 0.0f;
#pragma unroll
    for (int n = 0; n < kChunks; ++n) {
      const int c = chunk_at<kVec>(n, group, t);
      now.normalised(a, n, c, group, h[n]);
      now.dy[n].get(g[n]);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        dw[n][i] += g[n][i] * h[n][i];
        db[n][i] += g[n][i];
        g[n][i] *= w[n][i];  // 0 past the row's end, and so is h
        c1 += g[n][i];
        c2 += g[n][i] * h[n][i];
      }
    }
    const float2 c = group_sum(c1, c2, group, id, slots[turn] + id * (group >> 5));
    c1 = c.x * inv;
    c2 = c.y * inv;
#pragma unroll
    for (int n = 0; n < kChunks; ++n) {
      const int at = chunk_at<kVec>(n, group, t);
#pragma unroll
      for (int i = 0; i < 8; ++i) g[n][i] = now.rstd * (g[n][i] - c1 - h[n][i] * c2);
      if (a.ds.p != nullptr) {
        Chunk<X, kVec> k;
        float ds[8];
        k.load(static_cast<const X*>(a.ds.p) + row * a.ds.ld, at, group, cols);
        k.get(ds);
#pragma unroll
        for (int i = 0; i < 8; ++i) g[n][i] += ds[i];
      }
      Chunk<X, kVec>::store(static_cast<X*>(a.dx) + row * a.cols, at, group, cols, g[n]);
      if (a.dr != nullptr) store_any<kVec>(a.dr, a.rt, row * a.cols, at, group, cols, g[n]);
    }
  }
  if (part == nullptr) return;
  float* to = part + static_cast<std::int64_t>(blockIdx.x) * 2 * cols;
  for (int k = 0; k < ids; ++k) {  // group after group
    if (id == k) {
#pragma unroll
      for (int n = 0; n < kChunks; ++n) {
        const int c = chunk_at<kVec>(n, group, t);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int at = kVec ? c + i : c + i * group;
          if (at >= cols) continue;
          const float w = (k > 0 ? sums[at] : 0.0f) + dw[n][i], b = (k > 0 ? sums[cols + at] : 0.0f) + db[n][i];
          (k + 1 < ids ? sums : to)[at] = w;
          (k + 1 < ids ? sums : to)[cols + at] = b;
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
  bool vec;
  int chunks, group, ids, blocks;  // chunks 0: sweeps, with `blocks` row shares
};

bool by_chunks(const Rows& r, std::int64_t cols) { return r.p == nullptr || by_eight(r.p, r.ld, cols); }

// Threads of a group that hold `cols` in up to `chunks` chunks each.
int group_of(std::int64_t cols, int chunks) {
  return static_cast<int>((cols + 8 * chunks * 32 - 1) / (8 * chunks * 32)) * 32;
}

BwdPlan plan_of(const NormBwd& a) {
  BwdPlan p{};
  p.vec = by_chunks(a.dy, a.cols) && by_chunks(a.ds, a.cols) && by_chunks(a.s, a.cols) &&
          by_eight(a.w, a.cols, a.cols);
  // One chunk a thread keeps the registers (two sums and two values for each
  // element) near 80 and the loads of many rows in flight; long rows take more.
  p.chunks = a.cols <= 8 * kMaxGroup ? 1 : a.cols <= 16 * kMaxGroup ? 2 : 0;
  if (!paired(a.xt, a.dy.t)) p.chunks = 0;
  const int sms = sm_count();
  if (p.chunks == 0) {
    const std::int64_t blocks = (a.cols + 31) / 32, want = (8ll * sms + blocks - 1) / blocks, most = (a.rows + 63) / 64;
    p.blocks = static_cast<int>(want < most ? want : most);
    return p;
  }
  p.group = group_of(a.cols, p.chunks);
  p.ids = p.group < 384 ? 384 / p.group : 1;
  // two blocks an SM, or fewer where a group would have under four rows
  const std::int64_t want = (a.rows + 4ll * p.ids - 1) / (4ll * p.ids);
  p.blocks = static_cast<int>(want < 2 * sms ? want : 2 * sms);
  return p;
}

template <typename X, typename Y, bool kVec, bool kHeld>
void launch_bwd(const NormBwd& a, const BwdPlan& p, float* part, cudaStream_t stream) {
  const int threads = p.group * p.ids;
  const std::size_t smem = p.ids > 1 ? 2 * sizeof(float) * a.cols : 0;
  if (p.chunks == 1)
    norm_bwd<X, Y, kVec, kHeld, 1><<<p.blocks, threads, smem, stream>>>(a, p.group, part);
  else
    norm_bwd<X, Y, kVec, kHeld, 2><<<p.blocks, threads, smem, stream>>>(a, p.group, part);
}

}  // namespace

cudaError_t norm_forward(const NormFwd& a, cudaStream_t stream) {
  if (a.cols > 8 * kFwdChunks * kMaxGroup || !paired(a.x.t, a.yt)) {
    const std::int64_t most = 32ll * sm_count();
    norm_fwd_sweep<<<static_cast<unsigned>(a.rows < most ? a.rows : most), kSweep, 0, stream>>>(a);
  } else {
    const bool vec = by_chunks(a.x, a.cols) && by_chunks(a.r, a.cols) && by_eight(a.w, a.cols, a.cols) &&
                     by_chunks(Rows{a.b, a.cols, a.wt}, a.cols);
    const int group = group_of(a.cols, kFwdChunks), ids = group < 256 ? 256 / group : 1;
    const unsigned blocks = static_cast<unsigned>((a.rows + ids - 1) / ids);
    with_pair(a.x.t, a.yt, [&](auto x, auto y) {
      using X = decltype(x);
      using Y = decltype(y);
      if (vec)
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
  if (p.chunks == 0) {
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
      if (p.vec && a.q != nullptr)
        launch_bwd<X, Y, true, true>(a, p, part, stream);
      else if (p.vec)
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
