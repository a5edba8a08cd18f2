// Activation checkpoints in 8 bits: packing, unpacking, and GELU with its
// input kept in that form. All are HBM-bound: an element costs its own bytes
// plus 33/32 of a byte for each 8-bit copy.
//
// A group's step is a power of two, so x / s and q s are exact, the packing is
// the same on every path, and q s (7 significant bits) is exact in bf16: a
// tensor core multiplies it without a second rounding. Against the best step
// that costs at most one bit of the eight.

#include "train_utils.cuh"

namespace train {

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;

// tanh form: x (1 + tanh u) / 2 = x / (1 + exp(-2u)), 2u = k (x + c x^3). The
// quotient keeps its relative accuracy where the sum 1 + tanh u cancels.
constexpr float kK = 1.5957691216057308f;  // 2 sqrt(2 / pi)
constexpr float kC = 0.044715f;

__device__ __forceinline__ float gelu(float x, bool tanh_form) {
  if (tanh_form) {
    // exp(-2u) is infinite only where x < -6, and x / inf is the limit 0
    return __fdividef(x, 1.0f + __expf(-kK * (x + kC * x * x * x)));
  }
  return 0.5f * x * (1.0f + erff(x * 0.70710678118654752f));
}

__device__ __forceinline__ float gelu_slope(float x, bool tanh_form) {
  if (tanh_form) {
    // the slope is 0 or 1 to every bit beyond +-20; the clamp keeps x^2 finite, and a NaN
    x = x > 20.0f ? 20.0f : x < -20.0f ? -20.0f : x;
    const float sig = __fdividef(1.0f, 1.0f + __expf(-kK * (x + kC * x * x * x)));
    return sig + x * sig * (1.0f - sig) * kK * (1.0f + 3.0f * kC * x * x);
  }
  return 0.5f * (1.0f + erff(x * 0.70710678118654752f)) + x * 0.39894228040143268f * __expf(-0.5f * x * x);
}

// One warp to a group of a row, one lane to an element: any length, stride and type.
template <typename Body>
__device__ __forceinline__ void each_group(std::int64_t rows, std::int64_t cols, Body body) {
  const std::int64_t ng = (cols + kGroup - 1) / kGroup, total = rows * ng;
  const int lane = threadIdx.x & 31;
  for (std::int64_t g = static_cast<std::int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5); g < total;
       g += static_cast<std::int64_t>(gridDim.x) * kWarps) {
    const std::int64_t row = g / ng, col = (g - row * ng) * kGroup + lane;
    body(row, col, g, g * kGroup + lane, col < cols);
  }
}

__device__ __forceinline__ void pack_lane(float v, std::int8_t* q, std::uint8_t* scale, std::int64_t g,
                                          std::int64_t at) {
  const unsigned e = warp_scale(v);
  q[at] = static_cast<std::int8_t>(quantise(v, e));
  if ((threadIdx.x & 31) == 0) scale[g] = static_cast<std::uint8_t>(e);
}

__global__ void __launch_bounds__(kThreads) pack_groups(Rows x, std::int8_t* q, std::uint8_t* scale,
                                                        std::int64_t rows, std::int64_t cols) {
  each_group(rows, cols, [&](std::int64_t row, std::int64_t col, std::int64_t g, std::int64_t at, bool in) {
    pack_lane(in ? load(x.p, x.t, row * x.ld + col) : 0.0f, q, scale, g, at);
  });
}

__global__ void __launch_bounds__(kThreads) unpack_groups(const std::int8_t* q, const std::uint8_t* scale,
                                                          const void* w, const void* b, Type wt, void* out, Type t,
                                                          std::int64_t rows, std::int64_t cols) {
  each_group(rows, cols, [&](std::int64_t row, std::int64_t col, std::int64_t g, std::int64_t at, bool in) {
    if (!in) return;
    float v = static_cast<float>(q[at]) * step_of(scale[g]);
    // 65504 may be held as 2^16, which float16 has no finite value for
    if (t == Type::f16 && w == nullptr && fabsf(v) == 65536.0f) v = copysignf(65504.0f, v);
    if (w != nullptr) v *= load(w, wt, col);
    if (b != nullptr) v += load(b, wt, col);
    store(out, t, row * cols + col, v);
  });
}

__global__ void __launch_bounds__(kThreads) gelu_fwd_groups(const GeluFwd a) {
  each_group(a.rows, a.cols, [&](std::int64_t row, std::int64_t col, std::int64_t g, std::int64_t at, bool in) {
    const float x = in ? load(a.x.p, a.x.t, row * a.x.ld + col) : 0.0f;
    const float y = gelu(x, a.tanh_form);  // 0 at 0
    if (a.q != nullptr) pack_lane(x, a.q, a.scale, g, at);
    if (a.yq != nullptr) pack_lane(y, a.yq, a.yscale, g, at);
    if (in) store(a.y, a.x.t, row * a.cols + col, y);
  });
}

__global__ void __launch_bounds__(kThreads) gelu_bwd_groups(const GeluBwd a) {
  each_group(a.rows, a.cols, [&](std::int64_t row, std::int64_t col, std::int64_t g, std::int64_t at, bool in) {
    if (!in) return;
    const float h = static_cast<float>(a.q[at]) * step_of(a.scale[g]);
    store(a.dx, a.dy.t, row * a.cols + col, load(a.dy.p, a.dy.t, row * a.dy.ld + col) * gelu_slope(h, a.tanh_form));
  });
}

unsigned grid_of(std::int64_t rows, std::int64_t cols) {
  const std::int64_t want = (rows * groups(cols) + kWarps - 1) / kWarps, most = 64ll * sm_count();
  return static_cast<unsigned>(want < most ? want : most);
}

}  // namespace

cudaError_t pack8(Rows x, std::int8_t* q, std::uint8_t* scale, std::int64_t rows, std::int64_t cols,
                  cudaStream_t stream) {
  pack_groups<<<grid_of(rows, cols), kThreads, 0, stream>>>(x, q, scale, rows, cols);
  commux_ops::g_launches++;
  return cudaGetLastError();
}

cudaError_t unpack8(const std::int8_t* q, const std::uint8_t* scale, const void* w, const void* b, Type wt, void* out,
                    Type t, std::int64_t rows, std::int64_t cols, cudaStream_t stream) {
  unpack_groups<<<grid_of(rows, cols), kThreads, 0, stream>>>(q, scale, w, b, wt, out, t, rows, cols);
  commux_ops::g_launches++;
  return cudaGetLastError();
}

cudaError_t gelu8_forward(const GeluFwd& a, cudaStream_t stream) {
  gelu_fwd_groups<<<grid_of(a.rows, a.cols), kThreads, 0, stream>>>(a);
  commux_ops::g_launches++;
  return cudaGetLastError();
}

cudaError_t gelu8_backward(const GeluBwd& a, cudaStream_t stream) {
  gelu_bwd_groups<<<grid_of(a.rows, a.cols), kThreads, 0, stream>>>(a);
  commux_ops::g_launches++;
  return cudaGetLastError();
}

}  // namespace train
