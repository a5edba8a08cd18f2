#pragma once

// Training operators (sm_100a): what the bindings (train.cpp) hand to the
// kernels. No torch types here, so the kernels compile without ATen; every
// launch function enqueues on the given stream, and returns the first
// CUDA error.
//
// Matrices are rows of `cols` adjacent elements; `ld*` is the distance
// between rows in elements. Outputs without an ld are contiguous.

#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>

namespace train {

enum class Type : int { f32 = 0, bf16 = 1, f16 = 2 };

// 8-bit form of a matrix: groups of kGroup neighbours of a row share a scale.
// q is [rows][groups * kGroup] (zeros past the row's end), scale [rows][groups].
// A scale byte e stands for 2^(e-127), 1 <= e <= 249; 255 marks a group that
// held an infinity or NaN and stands for NaN throughout.
constexpr int kGroup = 32;
inline std::int64_t groups(std::int64_t cols) { return (cols + kGroup - 1) / kGroup; }

struct Rows {  // one operand: typed pointer, row distance
  const void* p = nullptr;
  std::int64_t ld = 0;
  Type t = Type::f32;
};

// s = x + residual (rounded to x's type; s = x without a residual),
// y = (s - mean) * rstd * w + b. Optional (null): r, s, b, mean, rstd, q.
struct NormFwd {
  Rows x, r;
  const void* w;
  const void* b;
  Type wt;
  void* s;
  void* y;
  Type yt;
  std::int8_t* q;
  std::uint8_t* scale;
  float *mean, *rstd;
  std::int64_t rows, cols;
  float eps;
};
cudaError_t norm_forward(const NormFwd& a, cudaStream_t stream);

// Gradients of the above. The normalised input comes from s, mean and rstd, or
// from its 8-bit form (q not null). ds (the gradient of s) may be null; dr is
// written when not null (a residual of another type than x). dw and db (of
// type wt) may be null; `work` holds norm_backward_work() floats.
struct NormBwd {
  Rows dy, ds, s;
  const std::int8_t* q;
  const std::uint8_t* scale;
  const float *mean, *rstd;
  const void* w;
  Type wt;
  void* dx;
  Type xt;
  void* dr;
  Type rt;
  void *dw, *db;
  float* work;
  std::int64_t rows, cols;
};
std::int64_t norm_backward_work(const NormBwd& a);
cudaError_t norm_backward(const NormBwd& a, cudaStream_t stream);

cudaError_t pack8(Rows x, std::int8_t* q, std::uint8_t* scale, std::int64_t rows, std::int64_t cols,
                  cudaStream_t stream);
// out: [rows][cols] of type t; values times w plus b (both null: as held)
cudaError_t unpack8(const std::int8_t* q, const std::uint8_t* scale, const void* w, const void* b, Type wt, void* out,
                    Type t, std::int64_t rows, std::int64_t cols, cudaStream_t stream);

// y = gelu(x); unless null, x's 8-bit form to (q, scale) and y's to (yq, yscale)
struct GeluFwd {
  Rows x;
  void* y;  // of x's type
  std::int8_t* q;
  std::uint8_t* scale;
  std::int8_t* yq;
  std::uint8_t* yscale;
  std::int64_t rows, cols;
  bool tanh_form;
};
cudaError_t gelu8_forward(const GeluFwd& a, cudaStream_t stream);

struct GeluBwd {
  Rows dy;
  const std::int8_t* q;
  const std::uint8_t* scale;
  void* dx;  // of dy's type
  std::int64_t rows, cols;
  bool tanh_form;
};
cudaError_t gelu8_backward(const GeluBwd& a, cudaStream_t stream);

// dw[o][i] = sum_t dy[t][o] X[t][i], db[o] = sum_t dy[t][o], where X is the
// 8-bit form, or w * it + b (w, b: the weight and bias of the norm it came from)
struct Wgrad8 {
  Rows dy;
  const std::int8_t* q;
  const std::uint8_t* scale;
  const void *w, *b;
  Type wt;
  void *dw, *db;  // db may be null
  Type dwt, dbt;
  void* work;  // wgrad8_work() bytes, 16-byte aligned
  std::int64_t rows, cols, outs;
};
std::int64_t wgrad8_work(const Wgrad8& a);
cudaError_t wgrad8(const Wgrad8& a, cudaStream_t stream);

// Softmax cross entropy of rows of logits. reduction 0: a loss for each row,
// 1: their mean over the rows that are not ignored, 2: their sum. `loss` is
// [rows] or a scalar; `stats` (each row's maximum, then each row's sum of
// exponentials) is kept for xent_backward. With `dx` (of
// the logits' type) the gradient for an upstream gradient of one is written
// in the same call (reductions 1 and 2). A target outside [0, cols) that is
// not ignore_index makes its row's loss and gradient NaN.
struct Xent {
  Rows x;
  const std::int64_t* target;
  std::int64_t ignore;
  int reduction;
  float* loss;
  float* stats;
  void* dx;
  float* work;  // xent_work() floats: first the number of rows that count
  std::int64_t rows, cols;
};
std::int64_t xent_work(std::int64_t rows);
cudaError_t xent_forward(const Xent& a, cudaStream_t stream);
// dx = gout * gradient, where gout is a device scalar (reductions 1 and 2) or
// [rows] (reduction 0). `have_unit`: dx holds the gradient for gout = 1 and
// nothing is written when that is what gout is.
cudaError_t xent_backward(const Xent& a, const float* gout, bool have_unit, cudaStream_t stream);

int sm_count();  // of the current device

}  // namespace train

namespace commux_ops {

extern std::atomic<std::int64_t> g_launches;  // kernels this extension launched

// Host-mapped status word (nonzero after a bounded wait in a kernel gave up)
// and its device address.
unsigned* status_word(unsigned** dev);
bool wait_gave_up();             // whether the status word says so, without one made for it
std::uint64_t wait_limit_ns();  // bound of every wait in a kernel (COMMUX_KERNEL_WAIT_MS)

}  // namespace commux_ops
