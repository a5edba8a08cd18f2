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

constexpr int kThreads = 256;

// A block takes a row at a time and sweeps it three times.
__global__ void __launch_bounds__(kThreads) norm_fwd_sweep(const NormFwd a) {
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
    for (std::int64_t i = threadIdx.x; i < a.cols; i += kThreads) {
      const float v = stream(i);
      if (a.s != nullptr) store(a.s, a.x.t, oo + i, v);
      sum += v;
    }
    const float mean = block_sum(sum, slots) / static_cast<float>(a.cols);
    float sq = 0.0f;
    for (std::int64_t i = threadIdx.x; i < a.cols; i += kThreads) {
      const float d = stream(i) - mean;
      sq += d * d;
    }
    const float rstd = rsqrtf(block_sum(sq, slots) / static_cast<float>(a.cols) + a.eps);
    if (threadIdx.x == 0) {
      if (a.mean != nullptr) a.mean[row] = mean;
      if (a.rstd != nullptr) a.rstd[row] = rstd;
    }
    for (std::int64_t i = threadIdx.x; i < ng * kGroup; i += kThreads) {  // whole warps
      float h = 0.0f;
      if (i < a.cols) {
        h = (stream(i) - mean) * rstd;
        const float y = h * load(a.w, a.wt, i) + (a.b != nullptr ? load(a.b, a.wt, i) : 0.0f);
        store(a.y, a.yt, oo + i, y);
      }
      if (a.q != nullptr) {
        const unsigned e = warp_scale(h);
        a.q[row * ng * kGroup + i] = static_cast<std::int8_t>(quantise(h, e));
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

__global__ void __launch_bounds__(kThreads) norm_bwd_sweep(const NormBwd a) {
  __shared__ float slots[32];
  const std::int64_t ng = (a.cols + kGroup - 1) / kGroup;
  for (std::int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const float mean = a.q != nullptr ? 0.0f : a.mean[row], rstd = a.rstd[row];
    float c1 = 0.0f, c2 = 0.0f;
    for (std::int64_t i = threadIdx.x; i < a.cols; i += kThreads) {
      const float g = load(a.dy.p, a.dy.t, row * a.dy.ld + i) * load(a.w, a.wt, i);
      c1 += g;
      c2 += g * normalised(a, row, i, ng, mean, rstd);
    }
    c1 = block_sum(c1, slots) / static_cast<float>(a.cols);
    c2 = block_sum(c2, slots) / static_cast<float>(a.cols);
    for (std::int64_t i = threadIdx.x; i < a.cols; i += kThreads) {
      const float g = load(a.dy.p, a.dy.t, row * a.dy.ld + i) * load(a.w, a.wt, i);
      float dx = rstd * (g - c1 - normalised(a, row, i, ng, mean, rstd) * c2);
      if (a.ds.p != nullptr) dx += load(a.ds.p, a.ds.t, row * a.ds.ld + i);
      store(a.dx, a.xt, row * a.cols + i, dx);
      if (a.dr != nullptr) store(a.dr, a.rt, row * a.cols + i, dx);
    }
  }
}

constexpr int kColRows = 8;  // rows in flight of a column block

// Partial sums over a share of the rows: part[2][gridDim.y][cols] (dw, db).
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
    part[blockIdx.y * a.cols + col] = dw;
    part[(gridDim.y + blockIdx.y) * a.cols + col] = db;
  }
}

// dw and db from `parts` partial sums of each column, in a fixed order.
__global__ void __launch_bounds__(32 * kColRows) norm_bwd_join(const float* part, int parts, std::int64_t cols,
                                                               void* dw, void* db, Type t) {
  __shared__ float sums[kColRows][33];
  const std::int64_t col = static_cast<std::int64_t>(blockIdx.x) * 32 + threadIdx.x;
  const float* from = part + static_cast<std::int64_t>(blockIdx.y) * parts * cols;
  float v = 0.0f;
  if (col < cols)
    for (int k = threadIdx.y; k < parts; k += kColRows) v += from[k * cols + col];
  sums[threadIdx.y][threadIdx.x] = v;
  __syncthreads();
  void* to = blockIdx.y == 0 ? dw : db;
  if (threadIdx.y == 0 && col < cols && to != nullptr) {
    for (int k = 1; k < kColRows; ++k) v += sums[k][threadIdx.x];
    store(to, t, col, v);
  }
}

int column_parts(const NormBwd& a) {
  // enough row shares to fill the GPU, no share under 64 rows
  const std::int64_t blocks = (a.cols + 31) / 32, want = (8ll * sm_count() + blocks - 1) / blocks;
  const std::int64_t most = (a.rows + 63) / 64;
  return static_cast<int>(want < most ? want : most);
}

}  // namespace

cudaError_t norm_forward(const NormFwd& a, cudaStream_t stream) {
  const std::int64_t most = 32ll * sm_count();
  norm_fwd_sweep<<<static_cast<unsigned>(a.rows < most ? a.rows : most), kThreads, 0, stream>>>(a);
  commux_ops::g_launches++;
  return cudaGetLastError();
}

std::int64_t norm_backward_work(const NormBwd& a) { return 2ll * column_parts(a) * a.cols; }

cudaError_t norm_backward(const NormBwd& a, cudaStream_t stream) {
  const std::int64_t most = 32ll * sm_count();
  norm_bwd_sweep<<<static_cast<unsigned>(a.rows < most ? a.rows : most), kThreads, 0, stream>>>(a);
  commux_ops::g_launches++;
  if (a.dw != nullptr || a.db != nullptr) {
    const int parts = column_parts(a);
    const unsigned blocks = static_cast<unsigned>((a.cols + 31) / 32);
    norm_bwd_columns<<<dim3(blocks, parts), dim3(32, kColRows), 0, stream>>>(a, a.work);
    norm_bwd_join<<<dim3(blocks, 2), dim3(32, kColRows), 0, stream>>>(a.work, parts, a.cols, a.dw, a.db, a.wt);
    commux_ops::g_launches += 2;
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
