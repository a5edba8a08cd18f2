// Activation checkpoints in 8 bits: packing, unpacking, and GELU with its
// input kept in that form. All are HBM-bound: an element costs its own bytes
// plus 33/32 of a byte for each 8-bit copy. 8192 x 3072 bf16: GELU with two copies
// 25.9 us (5.9 TB/s), its backward pass 21.9 us (5.8), unpacking 12.5 us (6.1);
// 4099 x 10001 fp32, exact form, 73 us and 69 us (5.1; 68 and 65 with a shorter fit, of
// absolute accuracy). Two exponential-unit operations an element keep that unit 50 to
// 60 % busy beside the memory.
//
// A group's step is a power of two, so x / s and q s are exact, the packing is
// the same on every path, and q s (7 significant bits) is exact in bf16: a
// tensor core multiplies it without a second rounding. Against the best step
// that costs at most one bit of the eight.

#include <type_traits>

#include "train_utils.cuh"

namespace train {

namespace {

constexpr int kThreads = 256;

// tanh form: x (1 + tanh u) / 2 = x / (1 + exp(-2u)), 2u = k (x + c x^3). The
// quotient keeps its relative accuracy where the sum 1 + tanh u cancels. exp(-2u)
// is infinite only where x < -6, and x / inf is the limit 0. The constants carry
// the log2(e) of the exponential.
constexpr float kK = 1.5957691216057308f;  // 2 sqrt(2 / pi)
constexpr float kC = 0.044715f;
constexpr float kE = 1.4426950408889634f;

__device__ __forceinline__ float2 sigmoid2(float2 x, float2 sq) {  // 1 / (1 + exp(-k x (1 + c x^2)))
  const float2 z = mul2(x, fma2(sq, both(-kK * kC * kE), both(-kK * kE)));
  const float2 d = add2(float2{exp2_fast(z.x), exp2_fast(z.y)}, both(1.0f));
  return {inverse_fast(d.x), inverse_fast(d.y)};
}

// exact form: Phi(-|x|) = t P(t) exp(-z^2), z = |x| / sqrt(2), t = 1 / (1 + 0.55 z). The
// variable t is that of Hastings (Abramowitz and Stegun, Handbook of Mathematical
// Functions, 7.1.26). P, of degree 9, is a minimax fit in relative error, 7e-9 in exact
// arithmetic and 3e-8 with its coefficients rounded, so the tail of a negative x keeps
// its accuracy as well: fp32 results are off by 5e-8 in norm, gradients by 6.5e-8
// (7.1.26 itself, 1.5e-7 absolute, left 1.1e-7, and up to 1.5e-3 of a value in the tail,
// three half units of float16). exp(-z^2) is also the density that the slope needs.
// For a positive x, Phi is 1 - that.
struct Normal {
  float2 cdf, bell;  // Phi(x), exp(-x^2 / 2)
};
__device__ __forceinline__ Normal normal(float2 x) {
  constexpr float kFit[10] = {0.155146043f,   0.155331775f, 0.129409972f,  0.101025455f, -0.0474978568f,
                              0.181981957f,   -0.426716751f, 0.390624953f, -0.16832934f, 0.0290237965f};
  const float2 z = {fabsf(x.x) * 0.70710678118654752f, fabsf(x.y) * 0.70710678118654752f};
  const float2 d = fma2(z, both(0.55f), both(1.0f)), t = {inverse_fast(d.x), inverse_fast(d.y)};
  float2 s = both(kFit[9]);
#pragma unroll
  for (int i = 8; i >= 0; --i) s = fma2(t, s, both(kFit[i]));
  const float2 y = mul2(mul2(z, z), both(-kE));
  Normal n;
  n.bell = float2{exp2_fast(y.x), exp2_fast(y.y)};
  s = mul2(mul2(s, t), n.bell);
  n.cdf = float2{x.x > 0.0f ? 1.0f - s.x : s.x, x.y > 0.0f ? 1.0f - s.y : s.y};
  return n;
}

template <bool kTanh>
__device__ __forceinline__ float2 gelu(float2 x) {
  if constexpr (kTanh) return mul2(x, sigmoid2(x, mul2(x, x)));
  return mul2(x, normal(x).cdf);
}

template <bool kTanh>
__device__ __forceinline__ float2 gelu_slope(float2 x) {
  if constexpr (kTanh) {
    // beyond +-20 the slope is 0 or 1 to every bit; the bound keeps x^2 finite
    float2 sq = mul2(x, x);
    sq = float2{fminf(sq.x, 400.0f), fminf(sq.y, 400.0f)};
    const float2 sig = sigmoid2(x, sq);
    const float2 rest = fma2(sig, both(-1.0f), both(1.0f));
    return fma2(mul2(x, sig), mul2(rest, fma2(sq, both(3.0f * kC * kK), both(kK))), sig);
  }
  const Normal n = normal(x);
  return fma2(mul2(x, both(0.39894228040143268f)), n.bell, n.cdf);
}

// What a pass does with its values; the passes differ in that alone. A pass
// reads a tensor x (kReads), an 8-bit form h (kHeld) or both, writes a tensor y
// (kWrites) and the 8-bit forms of x and y that it is asked for.
struct Args {
  Rows x;
  const std::int8_t* q;
  const std::uint8_t* scale;
  void* y;
  std::int8_t *xq, *yq;
  std::uint8_t *xscale, *yscale;
  const void *w, *b;  // unpack: the norm's weight and bias
  Type wt;
  std::int64_t rows, cols;
};

struct Pack {
  static constexpr bool kReads = true, kHeld = false, kWrites = false;
  template <typename T, typename Col>
  static __device__ __forceinline__ void apply(const Args&, Col, const float2 (&)[4], const float2 (&)[4],
                                               float2 (&)[4]) {}
};

template <bool kAffine>
struct Unpack {
  static constexpr bool kReads = false, kHeld = true, kWrites = true;
  template <typename T, typename Col>
  static __device__ __forceinline__ void apply(const Args& a, Col c, const float2 (&)[4], const float2 (&h)[4],
                                               float2 (&y)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      y[i] = h[i];
      if constexpr (kAffine) {
        const Col at = c + 2 * i;
        const bool one = at < a.cols, two = at + 1 < a.cols;
        y[i] = mul2(y[i], float2{one ? train::load(a.w, a.wt, at) : 0.0f, two ? train::load(a.w, a.wt, at + 1) : 0.0f});
        if (a.b != nullptr)
          y[i] = add2(y[i],
                      float2{one ? train::load(a.b, a.wt, at) : 0.0f, two ? train::load(a.b, a.wt, at + 1) : 0.0f});
      } else if constexpr (Elem<T>::kType == Type::f16) {
        // 65504 may be held as 2^16, which float16 has no finite value for
        if (fabsf(y[i].x) == 65536.0f) y[i].x = copysignf(65504.0f, y[i].x);
        if (fabsf(y[i].y) == 65536.0f) y[i].y = copysignf(65504.0f, y[i].y);
      }
    }
  }
};

template <bool kTanh>
struct GeluForward {
  static constexpr bool kReads = true, kHeld = false, kWrites = true;
  template <typename T, typename Col>
  static __device__ __forceinline__ void apply(const Args&, Col, const float2 (&x)[4], const float2 (&)[4],
                                               float2 (&y)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = gelu<kTanh>(x[i]);  // 0 at 0, as past a row's end
  }
};

template <bool kTanh>
struct GeluBackward {
  static constexpr bool kReads = true, kHeld = true, kWrites = true;
  template <typename T, typename Col>
  static __device__ __forceinline__ void apply(const Args&, Col, const float2 (&x)[4], const float2 (&h)[4],
                                               float2 (&y)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = mul2(x[i], gelu_slope<kTanh>(h[i]));
  }
};

__device__ __forceinline__ void pack_part(const float2 (&v)[4], std::int8_t* q, std::uint8_t* scale, std::int64_t part,
                                          bool in) {
  uint2 bytes;
  const unsigned e = pack_eight(v, bytes);
  if (!in) return;
  *reinterpret_cast<uint2*>(q + part * 8) = bytes;
  if ((threadIdx.x & 3) == 0) scale[part >> 2] = static_cast<std::uint8_t>(e);
}

// A thread takes a few parts of 8 elements; four threads hold a group. kFlat:
// the rows are whole groups without gaps, so the matrix is one long row (and
// no index is divided); otherwise Index counts parts through the rows, and a
// column has as many bits.
constexpr int unroll_of(bool aligned) { return aligned ? 4 : 2; }  // independent loads, as the registers allow

template <typename T, typename Pass, bool kFlat, bool kAligned, typename Index>
__global__ void __launch_bounds__(kThreads) eights(const Args a) {
  constexpr int kUnroll = unroll_of(kAligned);
  const Index per = static_cast<Index>((a.cols + kGroup - 1) / kGroup * 4);  // parts of a row
  const Index total = static_cast<Index>(a.rows) * per;
  const Index first = static_cast<Index>(blockIdx.x) * (kThreads * kUnroll) + threadIdx.x;
  using Col = std::conditional_t<sizeof(Index) == 4, int, std::int64_t>;
  const Col cols = kFlat ? 8 : static_cast<Col>(a.cols);  // flat: a part is a row of its own
  Part<T, kAligned> in[Pass::kReads ? kUnroll : 1];
  uint2 held[kUnroll];
  unsigned e[kUnroll];
  Index row[kUnroll];
  Col col[kUnroll];
  // a part's place in its row, for Part, whose columns are ints
  auto near = [&](Col c) { return sizeof(Col) == 4 ? static_cast<int>(c) : 0; };
  auto ends = [&](Col c) { return static_cast<int>(sizeof(Col) == 4 ? cols : min(cols - c, Col{64})); };
  auto skip = [&](Col c) { return sizeof(Col) == 4 ? Col{0} : c; };
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const Index part = first + u * kThreads;
    const bool some = part < total;
    row[u] = kFlat ? part : part / per;
    col[u] = kFlat ? 0 : static_cast<Col>(part - row[u] * per) * 8;
    if (!some) col[u] = cols;  // past the end: reads 0, writes nothing
    if (Pass::kReads) {
      const std::int64_t at = some ? (kFlat ? static_cast<std::int64_t>(part) * 8 : row[u] * a.x.ld) : 0;
      in[u].load(static_cast<const T*>(a.x.p) + at + skip(col[u]), near(col[u]), ends(col[u]));
    }
    if (Pass::kHeld) {
      held[u] = uint2{0, 0};
      e[u] = 1;
      if (some) {
        held[u] = *reinterpret_cast<const uint2*>(a.q + static_cast<std::int64_t>(part) * 8);
        e[u] = a.scale[part >> 2];
      }
    }
  }
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const Index part = first + u * kThreads;
    float2 x[4], h[4], y[4];
    if (Pass::kReads) in[u].get(x);
    if (Pass::kHeld) unpack_eight(held[u], e[u], h);
    Pass::template apply<T>(a, col[u], x, h, y);
    if (Pass::kWrites) {
      const bool some = part < total;
      T* to = static_cast<T*>(a.y) + (some ? (kFlat ? static_cast<std::int64_t>(part) * 8 : row[u] * a.cols) : 0);
      const int lane = threadIdx.x & 31;
      Part<T, kAligned>::store(to + skip(col[u]), near(col[u]), ends(col[u]), y, lane > 0 && col[u] > 0 && some,
                               some && (lane == 31 || part + 1 == total || col[u] + 8 >= static_cast<Col>(per) * 8));
    }
    if (Pass::kReads && a.xq != nullptr) pack_part(x, a.xq, a.xscale, part, part < total);
    if (Pass::kReads && a.yq != nullptr) pack_part(y, a.yq, a.yscale, part, part < total);
  }
}

template <typename T, typename Pass>
cudaError_t launch(const Args& a, cudaStream_t stream) {
  const std::int64_t parts = a.rows * groups(a.cols) * 4;
  // 32 bits count the parts, and the columns of a row (a few past its end too)
  const bool few = parts < (1ll << 30), small = few && a.cols < (1ll << 31) - 64;
  const bool whole = few && aligned_rows(a.x.p, a.x.ld, a.cols);
  const bool flat = whole && a.cols % kGroup == 0 && (a.x.ld == a.cols || a.rows == 1) && a.w == nullptr;
  const bool aligned = flat || (whole && small);
  const std::int64_t each = kThreads * unroll_of(aligned);
  const unsigned blocks = static_cast<unsigned>((parts + each - 1) / each);
  if (flat)
    eights<T, Pass, true, true, unsigned><<<blocks, kThreads, 0, stream>>>(a);
  else if (aligned)
    eights<T, Pass, false, true, unsigned><<<blocks, kThreads, 0, stream>>>(a);
  else if (small)
    eights<T, Pass, false, false, unsigned><<<blocks, kThreads, 0, stream>>>(a);
  else
    eights<T, Pass, false, false, std::int64_t><<<blocks, kThreads, 0, stream>>>(a);
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
  a.xq = q;
  a.xscale = scale;
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
  return w != nullptr ? launch<Unpack<true>>(a, t, stream) : launch<Unpack<false>>(a, t, stream);
}

cudaError_t gelu8_forward(const GeluFwd& g, cudaStream_t stream) {
  Args a{};
  a.x = g.x;
  a.y = g.y;
  a.xq = g.q;
  a.xscale = g.scale;
  a.yq = g.yq;
  a.yscale = g.yscale;
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
