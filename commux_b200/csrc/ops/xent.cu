// Softmax cross entropy of rows of logits with its gradient:
//   m = max_j x_j, s = sum_j exp(x_j - m);  loss = log s + (m - x_target)
//   dx_j = (exp(x_j - m) / s - [j = target]) gout (/ number of rows that count).
// HBM-bound: an element is read and its gradient written, with one exponential
// between. m and s stay apart (m + log s would lose s beside a large m, as in a
// row of the type's lowest value), and x_j - m comes before the product with
// log2(e), which such a value would overflow. A row of only -inf has no
// softmax: its loss and gradient are NaN, as is every row with NaN or +inf.

#include "train_utils.cuh"

namespace train {

namespace {

constexpr int kThreads = 512;
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ bool bad_target(const Xent& a, std::int64_t t) { return t < 0 || t >= a.cols; }

// work[0] = number of rows that count
__global__ void __launch_bounds__(1024) count_rows(const Xent a) {
  __shared__ float slots[32];
  int n = 0;
  for (std::int64_t r = threadIdx.x; r < a.rows; r += 1024) n += a.target[r] != a.ignore;
  // counts of a thread are exact in 32 bits, sums of them up to 2^24 and then rounded once each
  const float sum = block_sum(static_cast<float>(n), slots);
  if (threadIdx.x == 0) a.work[0] = sum;
}

// dx of a row from its maximum, its sum and the factor of its gradient
__device__ __forceinline__ void write_row(const Xent& a, std::int64_t row, float m, float s, std::int64_t target,
                                          float f, bool counts) {
  const float inv = 1.0f / s;
  const bool bad = counts && bad_target(a, target);
  for (std::int64_t i = threadIdx.x; i < a.cols; i += blockDim.x) {
    float d = 0.0f;
    if (counts) {
      d = exp2f((load(a.x.p, a.x.t, row * a.x.ld + i) - m) * kLog2e) * inv;
      if (i == target) d -= 1.0f;
      d = bad ? __int_as_float(0x7fffffff) : d * f;
    }
    store(a.dx, a.x.t, row * a.cols + i, d);
  }
}

__global__ void __launch_bounds__(kThreads) xent_sweep(const Xent a) {
  __shared__ float slots[32];
  const float count = a.reduction == 1 ? a.work[0] : 1.0f;
  float* losses = a.reduction == 0 ? a.loss : a.work + 1;
  for (std::int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const std::int64_t target = a.target[row];
    const bool counts = target != a.ignore;
    float m = -INFINITY, s = 0.0f, loss = 0.0f;
    if (counts) {
      for (std::int64_t i = threadIdx.x; i < a.cols; i += kThreads) {
        const float v = load(a.x.p, a.x.t, row * a.x.ld + i);
        m = v > m || v != v ? v : m;
      }
      m = block_max(m, slots);
      for (std::int64_t i = threadIdx.x; i < a.cols; i += kThreads)
        s += exp2f((load(a.x.p, a.x.t, row * a.x.ld + i) - m) * kLog2e);
      s = block_sum(s, slots);
      loss = bad_target(a, target) ? __int_as_float(0x7fffffff)
                                   : logf(s) + (m - load(a.x.p, a.x.t, row * a.x.ld + target));
    }
    if (threadIdx.x == 0) {
      losses[row] = loss;
      a.stats[row] = m;
      a.stats[a.rows + row] = s;
    }
    if (a.dx != nullptr) write_row(a, row, m, s, target, 1.0f / count, counts);
  }
}

// mean or sum of the rows' losses, in a fixed order
__global__ void __launch_bounds__(1024) join_losses(const Xent a) {
  __shared__ float slots[32];
  float v = 0.0f;
  for (std::int64_t r = threadIdx.x; r < a.rows; r += 1024) v += a.work[1 + r];
  v = block_sum(v, slots);
  if (threadIdx.x == 0) *a.loss = a.reduction == 1 ? v / a.work[0] : v;
}

__global__ void __launch_bounds__(kThreads) xent_again(const Xent a, const float* gout, bool have_unit) {
  if (have_unit && *gout == 1.0f) return;
  const float count = a.reduction == 1 ? a.work[0] : 1.0f;
  for (std::int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const std::int64_t target = a.target[row];
    write_row(a, row, a.stats[row], a.stats[a.rows + row], target,
              (a.reduction == 0 ? gout[row] : *gout) / count, target != a.ignore);
  }
}

unsigned grid_of(std::int64_t rows) {
  const std::int64_t most = 16ll * sm_count();
  return static_cast<unsigned>(rows < 1 ? 1 : rows < most ? rows : most);
}

}  // namespace

std::int64_t xent_work(std::int64_t rows) { return 1 + rows; }

cudaError_t xent_forward(const Xent& a, cudaStream_t stream) {
  if (a.reduction == 1) count_rows<<<1, 1024, 0, stream>>>(a), commux_ops::g_launches++;
  xent_sweep<<<grid_of(a.rows), kThreads, 0, stream>>>(a);
  commux_ops::g_launches++;
  if (a.reduction != 0) join_losses<<<1, 1024, 0, stream>>>(a), commux_ops::g_launches++;
  return cudaGetLastError();
}

cudaError_t xent_backward(const Xent& a, const float* gout, bool have_unit, cudaStream_t stream) {
  xent_again<<<grid_of(a.rows), kThreads, 0, stream>>>(a, gout, have_unit);
  commux_ops::g_launches++;
  return cudaGetLastError();
}

}  // namespace train
