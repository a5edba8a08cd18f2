// Softmax cross entropy of rows of logits with its gradient:
//   m = max_j x_j, s = sum_j exp(x_j - m);  loss = log s + (m - x_target)
//   dx_j = (exp(x_j - m) / s - [j = target]) gout (/ number of rows that count).
// HBM-bound: an element is read and its gradient written, with one exponential
// between. m and s stay apart (m + log s would lose s beside a large m, as in a
// row of the type's lowest value), and x_j - m comes before the product with
// log2(e), which such a value would overflow. A row of only -inf has no
// softmax: its loss and gradient are NaN, as is every row with NaN or +inf.
//
// A row is read once and lives in the registers of its threads, 32 elements
// each, from the maximum to the gradient. Rows up to 16 K elements have a block
// of their own and many blocks an SM, so that some load while others compute.
// Longer rows fill an SM's registers; there one block of 1024 threads walks
// over rows, whose elements come through shared memory by bulk copies that run
// ahead of it, and up to 8 blocks (a cluster) share a row that is longer still
// or one of few.

#include <cooperative_groups.h>

#include <type_traits>

#include "async.cuh"
#include "train_utils.cuh"

namespace train {

namespace {

constexpr float kLog2e = 1.4426950408889634f;

// The largest value of a warp; NaN if there is one.
__device__ __forceinline__ float largest(float v) {
  float m;
  asm("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(v));
  return m;
}

constexpr int kEach = 32;      // elements of a thread
constexpr int kSweep = 512;

__device__ __forceinline__ float nan_value() { return __int_as_float(0x7fffffff); }
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

// mean or sum of the rows' losses, in a fixed order
__global__ void __launch_bounds__(1024) join_losses(const Xent a) {
  __shared__ float slots[32];
  float v = 0.0f;
  for (std::int64_t r = threadIdx.x; r < a.rows; r += 1024) v += a.work[1 + r];
  v = block_sum(v, slots);
  if (threadIdx.x == 0) *a.loss = a.reduction == 1 ? v / a.work[0] : v;
}

// The target's logit; NaN where the target names none.
__device__ __forceinline__ float target_logit(const Xent& a, std::int64_t row, std::int64_t target) {
  return bad_target(a, target) ? nan_value() : load(a.x.p, a.x.t, row * a.x.ld + target);
}

// What is known of a row once its maximum and sum are (one thread).
__device__ __forceinline__ void finish_row(const Xent& a, std::int64_t row, std::int64_t target, float logit, float m,
                                           float s) {
  const float loss = target != a.ignore ? logf(s) + (m - logit) : 0.0f;
  (a.reduction == 0 ? a.loss : a.work + 1)[row] = loss;
  a.stats[row] = m;
  a.stats[a.rows + row] = s;
}

// A row's elements in registers: each thread has kEach / E vectors of E = 16
// bytes' worth, `threads` vectors apart. Vectors start on 16-byte boundaries: a
// row that does not begins `shift` elements into its first one. The 16 bytes
// around a row's first and last element belong to its allocation (which starts
// and ends on such a boundary), and what is not the row's is masked. Arithmetic
// is on pairs of elements: with one at a time the instructions, and not the
// memory, bounded the kernel (27 an element; 298 us for 8192 rows of 32000).
template <typename T>
struct Row {
  static constexpr int E = 16 / sizeof(T), kVectors = kEach / E;
  float2 v[kEach / 2];

  __device__ __forceinline__ void take(int k, uint4 w) {
    float2* p = v + k * (E / 2);
    if constexpr (sizeof(T) == 4) {
      p[0] = float2{__uint_as_float(w.x), __uint_as_float(w.y)};
      p[1] = float2{__uint_as_float(w.z), __uint_as_float(w.w)};
    } else {
      p[0] = Elem<T>::get2(w.x), p[1] = Elem<T>::get2(w.y), p[2] = Elem<T>::get2(w.z), p[3] = Elem<T>::get2(w.w);
    }
  }

  __device__ __forceinline__ float max() const {
    float m = larger(v[0].x, v[0].y);
#pragma unroll
    for (int i = 1; i < kEach / 2; ++i) m = larger(m, v[i].x, v[i].y);
    return m;
  }

  __device__ __forceinline__ float exponentials(float m) {
    float2 s = {0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < kEach / 2; ++i) {
      const float2 z = mul2(add2(v[i], both(-m)), both(kLog2e));
      v[i] = float2{exp2_fast(z.x), exp2_fast(z.y)};
      s = add2(s, v[i]);
    }
    return s.x + s.y;
  }
};

// A row part of `cols` elements that starts `shift` elements into vector 0:
// which elements of vector `at` are the part's.
template <int E>
struct Span {
  int from, to;
  __device__ __forceinline__ Span(int at, int shift, int cols)
      : from(at == 0 ? shift : 0), to(min(E, shift + cols - at * E)) {}
  __device__ __forceinline__ bool none() const { return to <= 0; }
  __device__ __forceinline__ bool all() const { return from == 0 && to == E; }
};

template <typename T>
__device__ __forceinline__ uint4 minus_infinities() {
  const unsigned w = sizeof(T) == 4 ? 0xff800000u : Elem<T>::kType == Type::bf16 ? 0xff80ff80u : 0xfc00fc00u;
  return {w, w, w, w};
}

// What is not the part's in the first and last vector of a part becomes -inf, in
// the shared memory that this thread alone reads it from. (In registers every
// vector of every thread would pay for the test of each element.)
template <typename T>
__device__ __forceinline__ void blank(uint4* vector, Span<Row<T>::E> s) {
  T* v = reinterpret_cast<T*>(vector);
#pragma unroll 1
  for (int i = 0; i < Row<T>::E; ++i)
    if (i < s.from || i >= s.to) v[i] = Elem<T>::put(-INFINITY);
}

// Gradient of a row part, to dx, but for what the target takes from its own.
// Where dx has the logits' shift (`aligned`) its vectors are those of the
// registers. `spare`: shared memory of this thread. kWhole: there is no shift
// and no part of a vector, here and in the logits.
template <typename T, bool kWhole>
__device__ __forceinline__ void write_part(T* dx, Row<T>& r, int cols, int shift, bool aligned, int threads, int t,
                                           float scale, uint4* spare) {
  constexpr int E = Row<T>::E;
#pragma unroll
  for (int k = 0; k < Row<T>::kVectors; ++k) {
    const int at = k * threads + t;
    if (at * E >= shift + cols) break;
    float2* v = r.v + k * (E / 2);
#pragma unroll
    for (int i = 0; i < E / 2; ++i) v[i] = mul2(v[i], both(scale));
    uint4 w;
    if constexpr (sizeof(T) == 4)
      w = uint4{__float_as_uint(v[0].x), __float_as_uint(v[0].y), __float_as_uint(v[1].x), __float_as_uint(v[1].y)};
    else
      w = uint4{Elem<T>::put2(v[0]), Elem<T>::put2(v[1]), Elem<T>::put2(v[2]), Elem<T>::put2(v[3])};
    T* out = dx + at * E - shift;
    if constexpr (kWhole) {
      *reinterpret_cast<uint4*>(out) = w;
      continue;
    }
    const Span<E> span(at, shift, cols);
    if (aligned && span.all()) {
      *reinterpret_cast<uint4*>(out) = w;
    } else {
      *spare = w;
      const T* from = reinterpret_cast<const T*>(spare);
#pragma unroll 1
      for (int i = span.from; i < span.to; ++i) out[i] = from[i];
    }
  }
}

// A row part's gradient; `owner`: this thread holds the target, `logit` is its
// value. The target's element is written over by the thread that wrote it.
template <typename T, bool kWhole>
__device__ __forceinline__ void write_row_part(const Xent& a, Row<T>& r, std::int64_t row, int first, int cols,
                                               int shift, bool aligned, int threads, int t, std::int64_t target,
                                               bool owner, float logit, float m, float s, float f, uint4* spare) {
  T* dx = static_cast<T*>(a.dx) + row * a.cols + first;
  if (target == a.ignore) {  // zeros, whatever the row holds
#pragma unroll
    for (int i = 0; i < kEach / 2; ++i) r.v[i] = float2{0.0f, 0.0f};
    write_part<T, kWhole>(dx, r, cols, shift, aligned, threads, t, 0.0f, spare);
    return;
  }
  const bool bad = bad_target(a, target);
  const float scale = bad ? nan_value() : f * (1.0f / s);
  write_part<T, kWhole>(dx, r, cols, shift, aligned, threads, t, scale, spare);
  if (owner && !bad)
    static_cast<T*>(a.dx)[row * a.cols + target] = Elem<T>::put(exp2_fast((logit - m) * kLog2e) * scale - f);
}

// The thread (of a row's part) that holds the target; the first one where no
// element is the target, so that somebody writes the loss.
template <int E>
__device__ __forceinline__ int owner_of(const Xent& a, std::int64_t target, int shift, int threads) {
  return target == a.ignore || bad_target(a, target) ? 0 : static_cast<int>((target + shift) / E % threads);
}

__device__ __forceinline__ int shift_of(const void* p, int size) {
  return static_cast<int>(reinterpret_cast<std::uintptr_t>(p) % 16) / size;
}

// --- rows up to kEach * 512: a block (or a warp of one) to a row ---

template <typename T>
__global__ void __launch_bounds__(512) xent_rows(const Xent a, const int group) {
  __shared__ float slots[2][32];
  __shared__ uint4 spare[512];
  constexpr int E = Row<T>::E;
  const int id = threadIdx.x / group, t = threadIdx.x - id * group, warps = group >> 5, lane = t & 31;
  const std::int64_t row = static_cast<std::int64_t>(blockIdx.x) * (blockDim.x / group) + id;
  if (row >= a.rows) return;  // whole warps; a row of more than one has the block alone
  const int cols = static_cast<int>(a.cols);
  const T* x = static_cast<const T*>(a.x.p) + row * a.x.ld;
  const int shift = shift_of(x, sizeof(T));
  const std::int64_t target = a.target[row];
  const bool owner = t == owner_of<E>(a, target, shift, group);
  const float logit = owner ? target_logit(a, row, target) : 0.0f;  // on its way early
  Row<T> r;
  uint4 w[Row<T>::kVectors];
#pragma unroll
  for (int k = 0; k < Row<T>::kVectors; ++k) {
    const int at = k * group + t;
    w[k] = minus_infinities<T>();
    if (at * E < shift + cols) w[k] = *reinterpret_cast<const uint4*>(x - shift + at * E);
  }
#pragma unroll
  for (int k = 0; k < Row<T>::kVectors; ++k) {
    const Span<E> span(k * group + t, shift, cols);
    if (!span.all() && !span.none()) {
      spare[threadIdx.x] = w[k];
      blank<T>(&spare[threadIdx.x], span);
      w[k] = spare[threadIdx.x];
    }
    r.take(k, w[k]);
  }
  float m = largest(r.max());
  if (warps > 1) {
    if (lane == 0) slots[0][t >> 5] = m;
    __syncthreads();
    m = largest(lane < warps ? slots[0][lane] : -INFINITY);
  }
  float s = warp_sum(r.exponentials(m));
  if (warps > 1) {
    if (lane == 0) slots[1][t >> 5] = s;
    __syncthreads();
    s = warp_sum(lane < warps ? slots[1][lane] : 0.0f);
  }
  if (owner) finish_row(a, row, target, logit, m, s);
  if (a.dx != nullptr) {
    const bool aligned = shift_of(static_cast<T*>(a.dx) + row * a.cols, sizeof(T)) == shift;
    write_row_part<T, false>(a, r, row, 0, cols, shift, aligned, group, t, target, owner, logit, m, s,
                      1.0f / (a.reduction == 1 ? a.work[0] : 1.0f), &spare[threadIdx.x]);
  }
}

// --- longer rows: blocks of 1024 threads, clusters of `kC` to a row ---

constexpr int kLong = 1024;
constexpr int kPiece = kLong * 16;           // bytes of one vector a thread, one bulk copy
constexpr int kRing = 12;                    // pieces in shared memory
constexpr int kRingBytes = kRing * kPiece;

__device__ __forceinline__ void bulk_load(void* dst, const void* src, unsigned bytes, std::uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
          async::smem_u32(dst)),
      "l"(src), "r"(bytes), "r"(async::smem_u32(bar))
      : "memory");
}

// Leaves v in the shared memory of block `rank` of the cluster, at its copy of
// `to`, and counts its 4 bytes on that block's copy of `bar`. Unlike a cluster
// barrier it does not wait for this thread's stores of gradients to arrive
// (which cost 8 us a row).
__device__ __forceinline__ void send(float* to, std::uint64_t* bar, int rank, float v) {
  std::uint32_t at, there;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(async::smem_u32(to)), "r"(rank));
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(async::smem_u32(bar)), "r"(rank));
  asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.b32 [%0], %1, [%2];" ::"r"(at),
               "r"(__float_as_uint(v)), "r"(there)
               : "memory");
}

template <typename T, int kC, bool kWhole>
__global__ void __launch_bounds__(kLong, 1) xent_long(const Xent a, unsigned* status, std::uint64_t limit_ns) {
  extern __shared__ __align__(128) unsigned char ring[];
  __shared__ std::uint64_t full[kRing], joined[2][2];
  __shared__ float slots[2][32], ranks[2][2][8];
  __shared__ uint4 spare[kLong];
  __shared__ int gave_up;
  constexpr int E = Row<T>::E, kV = Row<T>::kVectors;
  namespace cg = cooperative_groups;
  const int t = threadIdx.x, lane = t & 31;
  int rank = 0;
  if constexpr (kC > 1) rank = cg::this_cluster().block_rank();
  const std::int64_t clusters = gridDim.x / kC, mine = blockIdx.x / kC;
  // this block's part of every row; parts begin on whole vectors of the columns
  const std::int64_t share = ((a.cols + kC - 1) / kC + E - 1) / E * E;
  const int first = static_cast<int>(share * rank);
  const int cols = static_cast<int>(a.cols - first < share ? (a.cols > first ? a.cols - first : 0) : share);
  if (t == 0) {
    for (int i = 0; i < kRing; ++i) async::mbar_init(&full[i], 1);
    if constexpr (kC > 1)
      for (int i = 0; i < 4; ++i) async::mbar_init(&joined[i >> 1][i & 1], 1);
    gave_up = 0;
    async::fence_async();
  }
  __syncthreads();
  if constexpr (kC > 1) cg::this_cluster().sync();  // every block has started: its shared memory can be written
  const async::Bound bound{&gave_up, status, limit_ns};
  auto part = [&](std::int64_t row) { return static_cast<const T*>(a.x.p) + row * a.x.ld + first; };
  // Pieces are numbered through the rows; piece n goes to slot n % kRing. Every
  // row of this block has the same pieces but for one that a shift may add.
  auto vectors = [&](std::int64_t row) {
    return kWhole ? cols / E : cols == 0 ? 0 : (shift_of(part(row), sizeof(T)) + cols + E - 1) / E;
  };
  auto pieces = [&](std::int64_t row) { return (vectors(row) + kLong - 1) / kLong; };
  unsigned issued = 0, used = 0;
  std::int64_t ahead = mine;  // the row, and its piece, to ask for next
  int piece = 0;
  auto request = [&] {  // thread 0: pieces while they find room
    while (ahead < a.rows) {
      const T* x = part(ahead);
      const char* from = reinterpret_cast<const char*>(x - shift_of(x, sizeof(T)));
      const int n = pieces(ahead), bytes = vectors(ahead) * 16;
      for (; piece < n; ++piece, ++issued) {
        if (issued == used + kRing) return;
        const unsigned slot = issued % kRing;
        const unsigned size = min(kPiece, bytes - piece * kPiece);
        async::mbar_expect_tx(&full[slot], size);
        bulk_load(ring + slot * kPiece, from + piece * kPiece, size, &full[slot]);
      }
      ahead += clusters;
      piece = 0;
    }
  };
  if (t == 0) request();
  const float f = 1.0f / (a.reduction == 1 ? a.work[0] : 1.0f);
  // A value of each of the cluster's blocks to all of them. Slots and barriers
  // come in two sets: a block that is a row ahead writes to the other one, and
  // it cannot be two ahead.
  unsigned round = 0;
  auto exchange = [&](int which, float v) {
    const unsigned set = round & 1u;
    if (t == 0) async::mbar_expect_tx(&joined[set][which], kC * 4);
    if (t < kC) send(&ranks[set][which][rank], &joined[set][which], t, v);
    async::wait(async::smem_u32(&joined[set][which]), round >> 1 & 1u, bound);
    return ranks[set][which][lane & (kC - 1)];
  };
  for (std::int64_t row = mine; row < a.rows; row += clusters, ++round) {
    const int n = pieces(row), shift = kWhole ? 0 : shift_of(part(row), sizeof(T));
    const std::int64_t target = a.target[row];
    // the part that holds the target, or the first one where none does
    const bool here = target == a.ignore || bad_target(a, target) ? rank == 0 : target >= first && target - first < cols;
    const bool owner = here && t == owner_of<E>(a, target, shift - first, kLong);
    const float logit = owner ? target_logit(a, row, target) : 0.0f;  // on its way early
    Row<T> r;
#pragma unroll
    for (int k = 0; k < kV; ++k) {
      uint4 w = minus_infinities<T>();
      if (k < n) {
        const unsigned slot = (used + k) % kRing;
        async::wait(async::smem_u32(&full[slot]), (used + k) / kRing & 1u, bound);
        uint4* vector = reinterpret_cast<uint4*>(ring + slot * kPiece) + t;
        const Span<E> span(k * kLong + t, shift, cols);
        if (kWhole) {
          if ((k * kLong + t) * E < cols) w = *vector;
        } else if (!span.none()) {
          if (!span.all()) {
            blank<T>(vector, span);
            async::fence_async();  // the slot's next copy comes after these writes
          }
          w = *vector;
        }
      }
      r.take(k, w);
    }
    used += n;
    float m = largest(r.max());
    if (lane == 0) slots[0][t >> 5] = m;
    __syncthreads();  // and every thread has its elements: their pieces are free
    if (t == 0) {
      async::fence_async();
      request();
    }
    m = largest(slots[0][lane]);
    if constexpr (kC > 1) m = largest(exchange(0, m));
    float s = warp_sum(r.exponentials(m));
    if (lane == 0) slots[1][t >> 5] = s;
    __syncthreads();
    s = warp_sum(slots[1][lane]);
    if constexpr (kC > 1) {
      const float part = exchange(1, s);
      s = warp_sum(lane < kC ? part : 0.0f);
    }
    if (owner) finish_row(a, row, target, logit, m, s);
    if (a.dx != nullptr) {
      const bool aligned = kWhole || shift_of(static_cast<T*>(a.dx) + row * a.cols + first, sizeof(T)) == shift;
      write_row_part<T, kWhole>(a, r, row, first, cols, shift, aligned, kLong, t, target, owner, logit, m, s, f, &spare[t]);
    }
  }
  // shared memory outlives the copies, and what other blocks send, also where a wait gave up
  if (t == 0 && gave_up != 0)
    for (unsigned n = used; n < issued; ++n) async::settle(async::smem_u32(&full[n % kRing]), n / kRing & 1u, limit_ns);
  if constexpr (kC > 1) cg::this_cluster().sync();
}

// --- rows longer than a cluster's registers, and gradients formed again ---

// dx of a row from its maximum, its sum and the factor of its gradient
__device__ __forceinline__ void write_row(const Xent& a, std::int64_t row, float m, float s, std::int64_t target,
                                          float f, bool counts) {
  const float inv = 1.0f / s;
  const bool bad = counts && bad_target(a, target);
  for (std::int64_t i = threadIdx.x; i < a.cols; i += blockDim.x) {
    float d = 0.0f;
    if (counts) {
      d = exp2_fast((load(a.x.p, a.x.t, row * a.x.ld + i) - m) * kLog2e) * inv;
      if (i == target) d -= 1.0f;
      d = bad ? nan_value() : d * f;
    }
    store(a.dx, a.x.t, row * a.cols + i, d);
  }
}

__global__ void __launch_bounds__(kSweep) xent_sweep(const Xent a) {
  __shared__ float slots[32];
  const float count = a.reduction == 1 ? a.work[0] : 1.0f;
  for (std::int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const std::int64_t target = a.target[row];
    float m = -INFINITY, s = 0.0f;
    if (target != a.ignore) {
      for (std::int64_t i = threadIdx.x; i < a.cols; i += kSweep) m = larger(m, load(a.x.p, a.x.t, row * a.x.ld + i));
      m = block_max(m, slots);
      for (std::int64_t i = threadIdx.x; i < a.cols; i += kSweep)
        s += exp2_fast((load(a.x.p, a.x.t, row * a.x.ld + i) - m) * kLog2e);
      s = block_sum(s, slots);
    }
    if (threadIdx.x == 0) finish_row(a, row, target, target_logit(a, row, target), m, s);
    if (a.dx != nullptr) write_row(a, row, m, s, target, 1.0f / count, target != a.ignore);
  }
}

__global__ void __launch_bounds__(kSweep) xent_again(const Xent a, const float* gout, bool have_unit) {
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

template <typename T, int kC, bool kWhole>
cudaError_t launch_long(const Xent& a, cudaStream_t stream) {
  const auto kernel = xent_long<T, kC, kWhole>;
  const cudaError_t rc = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRingBytes);
  if (rc != cudaSuccess) return rc;
  const std::int64_t most = sm_count() / kC;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>((a.rows < most ? a.rows : most) * kC));
  cfg.blockDim = dim3(kLong);
  cfg.dynamicSmemBytes = kRingBytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = kC;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  unsigned* status = nullptr;
  commux_ops::status_word(&status);
  return cudaLaunchKernelEx(&cfg, kernel, a, status, commux_ops::wait_limit_ns());
}

template <typename T>
cudaError_t launch_rows(const Xent& a, cudaStream_t stream) {
  constexpr int E = Row<T>::E;
  const std::int64_t need = a.cols + E - 1;  // with the longest shift
  if (need <= kEach * 512) {
    const int group = static_cast<int>((need + kEach * 32 - 1) / (kEach * 32)) * 32;
    const int ids = group == 32 ? 4 : 1;
    xent_rows<T><<<static_cast<unsigned>((a.rows + ids - 1) / ids), group * ids, 0, stream>>>(a, group);
    return cudaSuccess;
  }
  // the fewest blocks that hold a row, and more where the rows leave SMs idle
  int c = 1;
  const int most = kEach * kLong - E;
  while (c < 8 && ((a.cols + c - 1) / c + E > most || a.rows * c * 2 <= sm_count())) c *= 2;
  if ((a.cols + c - 1) / c + E > most) {
    xent_sweep<<<grid_of(a.rows), kSweep, 0, stream>>>(a);
    return cudaSuccess;
  }
  const bool whole = a.cols % E == 0 && a.x.ld % E == 0 && reinterpret_cast<std::uintptr_t>(a.x.p) % 16 == 0;
  auto go = [&](auto blocks) {
    constexpr int kC = decltype(blocks)::value;
    return whole ? launch_long<T, kC, true>(a, stream) : launch_long<T, kC, false>(a, stream);
  };
  return c == 1   ? go(std::integral_constant<int, 1>())
         : c == 2 ? go(std::integral_constant<int, 2>())
         : c == 4 ? go(std::integral_constant<int, 4>())
                  : go(std::integral_constant<int, 8>());
}

}  // namespace

std::int64_t xent_work(std::int64_t rows) { return 1 + rows; }

cudaError_t xent_forward(const Xent& a, cudaStream_t stream) {
  if (a.reduction == 1) count_rows<<<1, 1024, 0, stream>>>(a), commux_ops::g_launches++;
  if (a.rows > 0) {
    cudaError_t rc = cudaSuccess;
    with_type(a.x.t, [&](auto e) { rc = launch_rows<decltype(e)>(a, stream); });
    if (rc != cudaSuccess) return rc;
    commux_ops::g_launches++;
  }
  if (a.reduction != 0) join_losses<<<1, 1024, 0, stream>>>(a), commux_ops::g_launches++;
  return cudaGetLastError();
}

cudaError_t xent_backward(const Xent& a, const float* gout, bool have_unit, cudaStream_t stream) {
  xent_again<<<grid_of(a.rows), kSweep, 0, stream>>>(a, gout, have_unit);
  commux_ops::g_launches++;
  return cudaGetLastError();
}

}  // namespace train
