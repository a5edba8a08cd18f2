// Weight gradient of a linear layer whose input was kept in 8 bits:
//   dw[o][i] = sum_t dy[t][o] X[t][i],  db[o] = sum_t dy[t][o].
// X is q s, or w (q s) + b after a norm, for which
//   dw[o][i] = w[i] sum_t dy[t][o] (q s)[t][i] + b[i] db[o],
// so the norm's weight and bias enter once at the end.

#include "train_utils.cuh"

namespace train {

namespace {

constexpr int kTile = 64;  // outputs of a block, both ways
constexpr int kStep = 16;  // tokens of a step
constexpr int kThreads = 256;

__global__ void __launch_bounds__(kThreads) wgrad_tile(const Wgrad8 a, const float* db) {
  __shared__ float sy[kStep][kTile], sx[kStep][kTile];
  const std::int64_t ng = (a.cols + kGroup - 1) / kGroup;
  const std::int64_t o0 = static_cast<std::int64_t>(blockIdx.y) * kTile, i0 = static_cast<std::int64_t>(blockIdx.x) * kTile;
  const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
  float acc[4][4] = {};
  for (std::int64_t t0 = 0; t0 < a.rows; t0 += kStep) {
    for (int k = threadIdx.x; k < kStep * kTile; k += kThreads) {
      const std::int64_t t = t0 + k / kTile, o = o0 + k % kTile, i = i0 + k % kTile;
      sy[k / kTile][k % kTile] = t < a.rows && o < a.outs ? load(a.dy.p, a.dy.t, t * a.dy.ld + o) : 0.0f;
      sx[k / kTile][k % kTile] = t < a.rows && i < a.cols ? static_cast<float>(a.q[t * ng * kGroup + i]) *
                                                                step_of(a.scale[t * ng + i / kGroup])
                                                          : 0.0f;
    }
    __syncthreads();
    for (int k = 0; k < kStep; ++k)
      for (int y = 0; y < 4; ++y)
        for (int x = 0; x < 4; ++x) acc[y][x] += sy[k][ty + 16 * y] * sx[k][tx + 16 * x];
    __syncthreads();
  }
  for (int y = 0; y < 4; ++y) {
    for (int x = 0; x < 4; ++x) {
      const std::int64_t o = o0 + ty + 16 * y, i = i0 + tx + 16 * x;
      if (o >= a.outs || i >= a.cols) continue;
      float v = acc[y][x];
      if (a.w != nullptr) v *= load(a.w, a.wt, i);
      if (a.b != nullptr) v += load(a.b, a.wt, i) * db[o];
      store(a.dw, a.dwt, o * a.cols + i, v);
    }
  }
}

// db and, for the norm's bias, its 32-bit form; a block to 32 outputs
__global__ void __launch_bounds__(kThreads) dy_columns(const Wgrad8 a, float* sum) {
  __shared__ float sums[kThreads / 32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const std::int64_t o = static_cast<std::int64_t>(blockIdx.x) * 32 + lane;
  float v = 0.0f;
  if (o < a.outs)
    for (std::int64_t t = warp; t < a.rows; t += kThreads / 32) v += load(a.dy.p, a.dy.t, t * a.dy.ld + o);
  sums[warp][lane] = v;
  __syncthreads();
  if (warp == 0 && o < a.outs) {
    for (int k = 1; k < kThreads / 32; ++k) v += sums[k][lane];
    sum[o] = v;
    if (a.db != nullptr) store(a.db, a.dwt, o, v);
  }
}

}  // namespace

std::int64_t wgrad8_work(const Wgrad8& a) { return a.outs * static_cast<std::int64_t>(sizeof(float)); }

cudaError_t wgrad8(const Wgrad8& a, cudaStream_t stream) {
  float* db = static_cast<float*>(a.work);
  if (a.db != nullptr || a.b != nullptr) {
    dy_columns<<<static_cast<unsigned>((a.outs + 31) / 32), kThreads, 0, stream>>>(a, db);
    commux_ops::g_launches++;
  }
  const dim3 grid(static_cast<unsigned>((a.cols + kTile - 1) / kTile),
                  static_cast<unsigned>((a.outs + kTile - 1) / kTile));
  wgrad_tile<<<grid, kThreads, 0, stream>>>(a, db);
  commux_ops::g_launches++;
  return cudaGetLastError();
}

}  // namespace train
