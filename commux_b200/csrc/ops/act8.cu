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
constexpr int kUnroll = 4;  // independent loads of a thread

// tanh form: x (1 + tanh u) / 2 = x / (1 + exp(-2u)), 2u = k (x + c x^3). The
// quotient keeps its relative accuracy where the sum 1 + tanh u cancels.
constexpr float kK = 1.5957691216057308f;  // 2 sqrt(2 / pi)
constexpr float kC = 0.044715f;

template <bool kTanh>
__device__ __forceinline__ float gelu(float x) {
  if (kTanh) {
    // exp(-2u) is infinite only where x < -6, and x / inf is the limit 0
    return __fdividef(x, 1.0f + __expf(-kK * (x + kC * x * x * x)));
  }
  return 0.5f * x * (1.0f + erff(x * 0.70710678118654752f));
}

template <bool kTanh>
__device__ __forceinline__ float gelu_slope(float x) {
  if (kTanh) {
    // the slope is 0 or 1 to every bit beyond +-20; the clamp keeps x^2 finite, and a NaN
    x = x > 20.0f ? 20.0f : x < -20.0f ? -20.0f : x;
    const float sig = __fdividef(1.0f, 1.0f + __expf(-kK * (x + kC * x * x * x)));
    return sig + x * sig * (1.0f - sig) * kK * (1.0f + 3.0f * kC * x * x);
  }
  return 0.5f * (1.0f + erff(x * 0.70710678118654752f)) + x * 0.39894228040143268f * __expf(-0.5f * x * x);
}

// What a pass does with values: the four passes differ in that alone, and each
// runs in the two arrangements below. `In` and `Out` are the element types of
// its tensors; a pass reads a tensor (kReads) or an 8-bit form (kHeld) or both.
struct Args {
  Rows x;                                        // kReads
  const std::int8_t* q;                          // kHeld
  const std::uint8_t* scale;
  void* y;                                       // unless null
  std::int8_t *q1, *q2;                          // forms to write, unless null
  std::uint8_t *scale1, *scale2;
  const void *w, *b;                             // unpack: the norm's
  Type wt;
  std::int64_t rows, cols;
};

struct Pack {
  static constexpr bool kReads = true, kHeld = false;
  template <typename T>
  static __device__ __forceinline__ void apply(const Args&, std::int64_t, float x, float, float& y, float& f1, float&) {
    y = 0.0f;
    f1 = x;
  }
};

struct Unpack {
  static constexpr bool kReads = false, kHeld = true;
  template <typename T>
  static __device__ __forceinline__ void apply(const Args& a, std::int64_t col, float, float h, float& y, float&,
                                               float&) {
    // 65504 may be held as 2^16, which float16 has no finite value for
    if (Elem<T>::kType == Type::f16 && a.w == nullptr && fabsf(h) == 65536.0f) h = copysignf(65504.0f, h);
    if (a.w != nullptr && col < a.cols) h *= load(a.w, a.wt, col);
    if (a.b != nullptr && col < a.cols) h += load(a.b, a.wt, col);
    y = h;
  }
};

template <bool kTanh>
struct GeluForward {
  static constexpr bool kReads = true, kHeld = false;
  template <typename T>
  static __device__ __forceinline__ void apply(const Args&, std::int64_t, float x, float, float& y, float& f1,
                                               float& f2) {
    y = gelu<kTanh>(x);  // 0 at 0, so the padding of a row's last group stays 0
    f1 = x;
    f2 = y;
  }
};

template <bool kTanh>
struct GeluBackward {
  static constexpr bool kReads = true, kHeld = true;
  template <typename T>
  static __device__ __forceinline__ void apply(const Args&, std::int64_t, float x, float h, float& y, float&, float&) {
    y = x * gelu_slope<kTanh>(h);
  }
};

// Rows that can be read by eight: a thread takes 8 neighbours, four threads a
// group. kFlat: the rows follow each other without a gap or a partial group,
// so the matrix is one row.
template <typename T, typename Pass, bool kFlat>
__global__ void __launch_bounds__(kThreads) by_vectors(const Args a) {
  const std::int64_t ng = (a.cols + kGroup - 1) / kGroup, total = a.rows * ng * 4;
  const std::int64_t first = static_cast<std::int64_t>(blockIdx.x) * (kThreads * kUnroll) + threadIdx.x;
  Eight<T> in[kUnroll];
  uint2 held[kUnroll];
  unsigned e[kUnroll];
  std::int64_t xo[kUnroll], yo[kUnroll], col[kUnroll];
  bool some[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const std::int64_t v = first + u * kThreads;
    std::int64_t row = 0;
    if (!kFlat) row = total < (1ll << 31) ? static_cast<unsigned>(v) / static_cast<unsigned>(ng * 4) : v / (ng * 4);
    col[u] = (v - row * ng * 4) * 8;
    xo[u] = row * a.x.ld + col[u];
    yo[u] = row * a.cols + col[u];
    some[u] = v < total && col[u] < a.cols;
    in[u].zero();
    held[u] = uint2{0, 0};
    e[u] = 1;
    if (Pass::kReads && some[u]) in[u].load(static_cast<const T*>(a.x.p) + xo[u]);
    if (Pass::kHeld && some[u]) {
      held[u] = *reinterpret_cast<const uint2*>(a.q + v * 8);
      e[u] = a.scale[v >> 2];
    }
  }
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const std::int64_t v = first + u * kThreads;
    float x[8], h[8], y[8], f1[8], f2[8];
    if (Pass::kReads) in[u].get(x);
    if (Pass::kHeld) unpack_eight(held[u], e[u], h);
#pragma unroll
    for (int i = 0; i < 8; ++i) Pass::template apply<T>(a, col[u] + i, x[i], h[i], y[i], f1[i], f2[i]);
    if (a.y != nullptr && some[u]) {
      Eight<T> out;
      out.put(y);
      out.store(static_cast<T*>(a.y) + yo[u]);
    }
    if (a.q1 != nullptr) {
      uint2 q;
      const unsigned s = pack_eight(f1, q);
      if (v < total) {
        *reinterpret_cast<uint2*>(a.q1 + v * 8) = q;
        if ((threadIdx.x & 3) == 0) a.scale1[v >> 2] = static_cast<std::uint8_t>(s);
      }
    }
    if (a.q2 != nullptr) {
      uint2 q;
      const unsigned s = pack_eight(f2, q);
      if (v < total) {
        *reinterpret_cast<uint2*>(a.q2 + v * 8) = q;
        if ((threadIdx.x & 3) == 0) a.scale2[v >> 2] = static_cast<std::uint8_t>(s);
      }
    }
  }
}

// Any rows: a warp takes kUnroll groups that follow each other, a lane an
// element of each. Index (32 bits where the counts allow) divides once a warp.
template <typename T, typename Pass, typename Index>
__global__ void __launch_bounds__(kThreads) by_lanes(const Args a) {
  const int lane = threadIdx.x & 31;
  const Index ng = static_cast<Index>((a.cols + kGroup - 1) / kGroup), total = static_cast<Index>(a.rows) * ng;
  const Index first = (static_cast<Index>(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5)) * kUnroll;
  if (first >= total) return;
  Index row = first / ng, at = first - row * ng;
  T in[kUnroll] = {};
  std::int8_t held[kUnroll];
  unsigned e[kUnroll];
  std::int64_t yo[kUnroll], col[kUnroll];
  bool some[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    col[u] = static_cast<std::int64_t>(at) * kGroup + lane;
    yo[u] = static_cast<std::int64_t>(row) * a.cols + col[u];
    some[u] = first + u < total && col[u] < a.cols;
    held[u] = 0;
    e[u] = 1;
    if (Pass::kReads && some[u]) in[u] = static_cast<const T*>(a.x.p)[static_cast<std::int64_t>(row) * a.x.ld + col[u]];
    if (Pass::kHeld && some[u]) {
      held[u] = a.q[static_cast<std::int64_t>(first + u) * kGroup + lane];
      e[u] = a.scale[first + u];
    }
    if (++at == ng) at = 0, ++row;
  }
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    if (first + u >= total) break;  // the same for a warp
    float y = 0.0f, f1 = 0.0f, f2 = 0.0f;
    Pass::template apply<T>(a, col[u], some[u] ? Elem<T>::get(in[u]) : 0.0f,
                            static_cast<float>(held[u]) * step_of(e[u]), y, f1, f2);
    if (a.y != nullptr && some[u]) static_cast<T*>(a.y)[yo[u]] = Elem<T>::put(y);
    const std::int64_t g = first + u;
    if (a.q1 != nullptr) {
      const unsigned s = warp_scale(f1);
      a.q1[g * kGroup + lane] = static_cast<std::int8_t>(quantised(f1, s));
      if (lane == 0) a.scale1[g] = static_cast<std::uint8_t>(s);
    }
    if (a.q2 != nullptr) {
      const unsigned s = warp_scale(f2);
      a.q2[g * kGroup + lane] = static_cast<std::int8_t>(quantised(f2, s));
      if (lane == 0) a.scale2[g] = static_cast<std::uint8_t>(s);
    }
  }
}

template <typename T, typename Pass>
cudaError_t launch(const Args& a, cudaStream_t stream) {
  const std::int64_t total = a.rows * groups(a.cols);
  const auto blocks = [](std::int64_t work, std::int64_t each) { return static_cast<unsigned>((work + each - 1) / each); };
  if (by_eight(a.x.p, a.x.ld, a.cols)) {
    const unsigned n = blocks(total * 4, kThreads * kUnroll);
    if (a.cols % kGroup == 0 && (a.x.ld == a.cols || a.rows == 1) && a.w == nullptr) {
      Args one = a;
      one.rows = 1;
      one.cols = a.rows * a.cols;
      by_vectors<T, Pass, true><<<n, kThreads, 0, stream>>>(one);
    } else {
      by_vectors<T, Pass, false><<<n, kThreads, 0, stream>>>(a);
    }
  } else {
    const unsigned n = blocks(total, kThreads / 32 * kUnroll);
    if (total < (1ll << 30))
      by_lanes<T, Pass, unsigned><<<n, kThreads, 0, stream>>>(a);
    else
      by_lanes<T, Pass, std::int64_t><<<n, kThreads, 0, stream>>>(a);
  }
  commux_ops::g_launches++;
  return cudaGetLastError();
}

template <typename Pass>
cudaError_t launch(const Args& a, Type t, cudaStream_t stream) {
  cudaError_t rc = cudaSuccess;
  with_type(t, [&](auto e) { rc = launch<decltype(e), Pass>(a, stream); });
  return rc;
}

}  // namespace

cudaError_t pack8(Rows x, std::int8_t* q, std::uint8_t* scale, std::int64_t rows, std::int64_t cols,
                  cudaStream_t stream) {
  Args a{};
  a.x = x;
  a.q1 = q;
  a.scale1 = scale;
  a.rows = rows;
  a.cols = cols;
  return launch<Pack>(a, x.t, stream);
}

cudaError_t unpack8(const std::int8_t* q, const std::uint8_t* scale, const void* w, const void* b, Type wt, void* out,
                    Type t, std::int64_t rows, std::int64_t cols, cudaStream_t stream) {
  Args a{};
  a.x = Rows{out, cols, t};  // the arrangement goes by what is written
  a.q = q;
  a.scale = scale;
  a.y = out;
  a.w = w;
  a.b = b;
  a.wt = wt;
  a.rows = rows;
  a.cols = cols;
  return launch<Unpack>(a, t, stream);
}

cudaError_t gelu8_forward(const GeluFwd& g, cudaStream_t stream) {
  Args a{};
  a.x = g.x;
  a.y = g.y;
  a.q1 = g.q;
  a.scale1 = g.scale;
  a.q2 = g.yq;
  a.scale2 = g.yscale;
  a.rows = g.rows;
  a.cols = g.cols;
  return g.tanh_form ? launch<GeluForward<true>>(a, g.x.t, stream) : launch<GeluForward<false>>(a, g.x.t, stream);
}

cudaError_t gelu8_backward(const GeluBwd& g, cudaStream_t stream) {
  Args a{};
  a.x = g.dy;
  a.q = g.q;
  a.scale = g.scale;
  a.y = g.dx;
  a.rows = g.rows;
  a.cols = g.cols;
  return g.tanh_form ? launch<GeluBackward<true>>(a, g.dy.t, stream) : launch<GeluBackward<false>>(a, g.dy.t, stream);
}

}  // namespace train
