// Softmax cross entropy of rows of logits with its gradient:
//   m = max_j x_j, s = sum_j exp(x_j - m);  loss = log s + (m - x_target)
//   dx_j = (exp(x_j - m) / s - [j = target]) gout (/ number of rows that count).
// HBM-bound: an element is read and its gradient written, with one exponential
// between. m and s stay apart (m + log s would lose s beside a large m, as in a
// row of the type's lowest value), and x_j - m comes before the product with
// log2(e), which such a value would overflow. A row of only -inf has no
// softmax: its loss and gradient are NaN, as is every row with NaN or +inf.
//
// A row is read once. Short rows live in the registers of a warp or a small
// block, 32 elements a thread, from the maximum to the gradient, with many blocks
// an SM, so that some load while others compute. Longer ones come through shared
// memory by bulk copies that run ahead of blocks which walk over rows, and up to 8
// blocks (a cluster) share a row that is longer still or one of few.

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
__device__ __forceinline__ void finish_row(const Xent& a, std::int64_t row, bool ignored, float logit, float m,
                                           float s) {
  (a.reduction == 0 ? a.loss : a.work + 1)[row] = ignored ? 0.0f : logf(s) + (m - logit);
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

  // The largest element of a vector, NaN if it has one. 16-bit elements are
  // compared two at a time, before they are widened.
  static __device__ __forceinline__ float max(uint4 w) {
    if constexpr (sizeof(T) == 4) {
      return larger(larger(__uint_as_float(w.x), __uint_as_float(w.y)),
                    larger(__uint_as_float(w.z), __uint_as_float(w.w)));
    } else {
      const unsigned m = Elem<T>::larger2(Elem<T>::larger2(w.x, w.y), Elem<T>::larger2(w.z, w.w));
      const float2 f = Elem<T>::get2(m);
      return larger(f.x, f.y);
    }
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

// The first and the last vector of a part, in functions of their own: inlined,
// every vector of every thread would pay for the test of each element.

// What is not the part's becomes -inf.
template <typename T>
__device__ __noinline__ uint4 blanked(uint4 w, int from, int to) {
  constexpr int E = Row<T>::E;
  unsigned u[4] = {w.x, w.y, w.z, w.w};
  const uint4 none = minus_infinities<T>();
#pragma unroll
  for (int i = 0; i < E; ++i) {
    if (i >= from && i < to) continue;
    if constexpr (E == 4)
      u[i] = none.x;
    else
      u[i / 2] = i & 1 ? (u[i / 2] & 0xffffu) | (none.x & 0xffff0000u) : (u[i / 2] & 0xffff0000u) | (none.x & 0xffffu);
  }
  return {u[0], u[1], u[2], u[3]};
}

// Elements [from, to) of a vector, one by one.
template <typename T>
__device__ __noinline__ void store_some(T* out, uint4 w, int from, int to) {
  constexpr int E = Row<T>::E;
  const unsigned u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < E; ++i) {
    if (i < from || i >= to) continue;
    if constexpr (E == 4)
      reinterpret_cast<unsigned*>(out)[i] = u[i];
    else
      reinterpret_cast<unsigned short*>(out)[i] = static_cast<unsigned short>(u[i / 2] >> (16 * (i & 1)));
  }
}

// Gradient of a row part, to dx, but for what the target takes from its own.
// Where dx has the logits' shift (`aligned`) its vectors are those of the
// registers.
template <typename T>
__device__ __forceinline__ void write_part(T* dx, Row<T>& r, int cols, int shift, bool aligned, int threads, int t,
                                           float scale) {
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
    const Span<E> span(at, shift, cols);
    if (aligned && span.all())
      *reinterpret_cast<uint4*>(out) = w;
    else
      store_some<T>(out, w, span.from, span.to);
  }
}

// A row part's gradient; `owner`: this thread holds the target, `logit` is its
// value. The target's element is written over by the thread that wrote it.
template <typename T>
__device__ __forceinline__ void write_row_part(const Xent& a, Row<T>& r, std::int64_t row, int first, int cols,
                                               int shift, bool aligned, int threads, int t, std::int64_t target,
                                               bool owner, float logit, float m, float s, float f) {
  T* dx = static_cast<T*>(a.dx) + row * a.cols + first;
  if (target == a.ignore) {  // zeros, whatever the row holds
#pragma unroll
    for (int i = 0; i < kEach / 2; ++i) r.v[i] = float2{0.0f, 0.0f};
    write_part<T>(dx, r, cols, shift, aligned, threads, t, 0.0f);
    return;
  }
  const bool bad = bad_target(a, target);
  const float scale = bad ? nan_value() : f * (1.0f / s);
  write_part<T>(dx, r, cols, shift, aligned, threads, t, scale);
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

// --- rows up to 32 * 128: a block (or a warp of one) to a row ---

constexpr int kRowThreads = 128;

template <typename T>
__global__ void __launch_bounds__(kRowThreads) xent_rows(const Xent a, const int group) {
  __shared__ float slots[2][32];
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
    if (!span.all() && !span.none()) w[k] = blanked<T>(w[k], span.from, span.to);
    r.take(k, w[k]);
  }
  float m = -INFINITY;
#pragma unroll
  for (int k = 0; k < Row<T>::kVectors; ++k) m = larger(m, Row<T>::max(w[k]));
  m = largest(m);
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
  if (owner) finish_row(a, row, target == a.ignore, logit, m, s);
  if (a.dx != nullptr) {
    const bool aligned = shift_of(static_cast<T*>(a.dx) + row * a.cols, sizeof(T)) == shift;
    write_row_part<T>(a, r, row, 0, cols, shift, aligned, group, t, target, owner, logit, m, s,
                      1.0f / (a.reduction == 1 ? a.work[0] : 1.0f));
  }
}

// --- longer rows: a block of `kThreads` walks over rows, clusters of `kC` blocks share one ---
//
// A block has 64 bytes a thread of every row, an SM 1024 threads in one, two or
// four blocks: the smallest that holds a row, so that more rows are under way. One
// barrier a row: while a row's sum is joined, so is the next row's maximum, and then
// each thread writes its vectors of the one and fills the registers with the
// exponentials of the other, vector by vector. Stores, conversions and exponentials,
// each of which would bound a phase of its own, run side by side (with two barriers
// and a phase for each, 211 us for 8192 rows of 32000 bf16). The next row stays in
// shared memory until then, its maximum and its exponentials read it from there.
//
// A row's chain (wait, maximum, barrier, two reductions) and the instructions bound
// it next to the memory: 8192 rows of 32000 bf16 with their gradient take 192 us with the
// small kernels before and after (5.5 TB/s); 208 us with 32001 columns; 1024 rows of
// 128001 in clusters of 4 take 151.

constexpr int kLong = 1024;    // threads of an SM
constexpr int kVectors = 4;    // 16-byte vectors of a thread
constexpr int kBuffers = 3;    // rows in shared memory
constexpr int buffer_bytes(int threads) { return kVectors * threads * 16; }

__device__ __forceinline__ void bulk_load(void* dst, const void* src, unsigned bytes, std::uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
          async::smem_u32(dst)),
      "l"(src), "r"(bytes), "r"(async::smem_u32(bar))
      : "memory");
}

// Leaves v in the shared memory of block `rank` of the cluster, at its copy of
// `to`, and counts its bytes on that block's copy of `bar`. Unlike a cluster
// barrier it does not wait for this thread's stores of gradients to arrive
// (which cost 8 us a row).
__device__ __forceinline__ void send(float2* to, std::uint64_t* bar, int rank, float2 v) {
  std::uint32_t at, there;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(async::smem_u32(to)), "r"(rank));
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(async::smem_u32(bar)), "r"(rank));
  const unsigned long long w = static_cast<unsigned long long>(__float_as_uint(v.y)) << 32 | __float_as_uint(v.x);
  asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.b64 [%0], %1, [%2];" ::"r"(at), "l"(w),
               "r"(there)
               : "memory");
}

// A block's part of every row: parts begin on whole vectors of the columns.
template <int E, int kC>
struct Share {
  int first, cols;
  __device__ __forceinline__ Share(std::int64_t all, int rank) {
    const std::int64_t share = ((all + kC - 1) / kC + E - 1) / E * E;
    first = static_cast<int>(share * rank);
    cols = static_cast<int>(all - first < share ? (all > first ? all - first : 0) : share);
  }
};

// Rows that a block did not finish, since a wait gave up in its turn `left` (from 1):
// NaN in its part of their gradients, in their losses and in what a later pass reads.
// The turn before that one's row was not finished either.
template <typename T, int kC>
__device__ __forceinline__ void poison(const Xent& a, int left) {
  const Share<16 / sizeof(T), kC> part(a.cols, blockIdx.x % kC);
  const int clusters = gridDim.x / kC;
  for (std::int64_t row = blockIdx.x / kC + (left > 1 ? left - 2ll : 0) * clusters; row < a.rows; row += clusters) {
    T* dx = static_cast<T*>(a.dx) + row * a.cols + part.first;
    for (int i = threadIdx.x; a.dx != nullptr && i < part.cols; i += blockDim.x) dx[i] = Elem<T>::put(nan_value());
    if (threadIdx.x == 0) finish_row(a, row, false, nan_value(), nan_value(), nan_value());
  }
}

// kWhole: every row lies in whole vectors. Where one does not, its buffer holds
// other rows' elements before and after its own. The warp that owns such a vector
// overwrites them with -inf, so that all threads may take all vectors as they are
// (with tests of each vector and a warp for what is left over: 259 us for 8192 rows
// of 32001 bf16), and writes that vector of the gradient element by element.
template <typename T, int kThreads, int kC, bool kWhole>
__global__ void __launch_bounds__(kThreads, kLong / kThreads)
    xent_long(const Xent a, unsigned* status, std::uint64_t limit_ns) {
  constexpr int kPiece = kThreads * 16;  // bytes of one vector a thread, one bulk copy
  constexpr int kBuffer = buffer_bytes(kThreads), kWarps = kThreads / 32;
  extern __shared__ __align__(128) unsigned char buffers[];
  __shared__ std::uint64_t full[kBuffers], joined[2];
  __shared__ float2 slots[2][kWarps], ranks[2][8];  // (sum of a row, maximum of the next)
  __shared__ float factors[2];                      // of a row's gradient
  __shared__ uint4 ends[2];                         // a gradient's first and last vector
  __shared__ int gave_up, left_at;  // left_at: the turn, from 1, in which a wait gave up
  // What single warps keep from row to row is in shared memory too: registers
  // would hold it in every thread, and the exponentials need them.
  __shared__ struct {
    const char* x;  // the row that is asked for next
    std::int64_t row;
    unsigned slot, round;  // its buffer, and the parity of that buffer's turn
  } asked;
  __shared__ struct {
    std::int64_t target, next_target[2];  // of the row that is finished next
    float f, m, logit;
    float last_grad;  // the target's gradient of the row before, and its place
    T* last_at;
  } note;
  constexpr int E = 16 / sizeof(T);
  namespace cg = cooperative_groups;
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  // What one thread or a few do for a row is spread over warps, since a barrier
  // waits for the slowest: the first sees to a row's first vector, and of the last
  // two one asks for rows and one writes down the loss and the target's gradient.
  const bool asks = warp == kWarps - 2, notes = warp == kWarps - 1;
  int rank = 0;
  if constexpr (kC > 1) rank = cg::this_cluster().block_rank();
  const int clusters = gridDim.x / kC;
  const Share<E, kC> part(a.cols, rank);
  const int first = part.first, cols = part.cols;
  const int vectors = cols == 0 ? 0 : kWhole ? cols / E : (cols + 2 * E - 2) / E;  // that a part may touch
  // vectors of this warp's threads
  const int mine = (vectors - warp * 32 + kThreads - 1) / kThreads;
  if (t == 0) {
    for (int i = 0; i < kBuffers; ++i) async::mbar_init(&full[i], 1);
    if constexpr (kC > 1)
      for (int i = 0; i < 2; ++i) async::mbar_init(&joined[i], 1);
    gave_up = left_at = 0;
  }
  // what no row fills, up to a whole warp's vectors
  for (int i = 0; i < kBuffers; ++i)
    for (int v = cols / E + t; v < (vectors + 31) / 32 * 32; v += kThreads)
      reinterpret_cast<uint4*>(buffers + i * kBuffer)[v] = minus_infinities<T>();
  async::fence_async();
  __syncthreads();
  if constexpr (kC > 1) cg::this_cluster().sync();  // every block has started: its shared memory can be written
  const async::Bound bound{&gave_up, status, limit_ns};
  // Inlined: the long way of a wait as a call has every thread keep values in local
  // memory (208 or 222 us for 8192 rows of 32001 bf16, 192 either way of 32000, 120 or
  // 118 for 1024 rows of 128000).
  auto wait = [&](std::uint64_t& bar, unsigned parity, int turn) {
    if (!async::wait_inline<>(async::smem_u32(&bar), parity, bound)) left_at = turn + 1;
  };
  // Whether the block leaves in this turn. Asked after a barrier behind the turn's
  // waits, so that all threads leave: one that is a turn ahead may have given up there.
  auto leaves = [&](int turn) { return left_at != 0 && left_at <= turn + 1; };

  // a row's part: of the logits, and of dx, whose rows lie alike to their vectors
  const int row0 = blockIdx.x / kC;
  const int turns = row0 < a.rows ? static_cast<int>((a.rows - row0 + clusters - 1) / clusters) : 0;
  const char* x0 = reinterpret_cast<const char*>(static_cast<const T*>(a.x.p) + row0 * a.x.ld + first);

  auto request = [&] {  // one warp: a row, a lane to a piece of it
    if (asked.row >= a.rows) return;
    const char* from = asked.x;
    const unsigned slot = asked.slot;
    const int skip = kWhole ? 0 : static_cast<int>(reinterpret_cast<std::uintptr_t>(from) & 15);
    const int bytes = cols == 0 ? 0 : (skip + cols * static_cast<int>(sizeof(T)) + 15) & ~15;
    __syncwarp();
    if (lane == 0) {
      async::mbar_expect_tx(&full[slot], bytes);
      asked.x = from + clusters * a.x.ld * static_cast<std::int64_t>(sizeof(T));
      asked.row += clusters;
      asked.slot = slot + 1 < kBuffers ? slot + 1 : 0;
      if (asked.slot == 0) asked.round ^= 1u;
    }
    __syncwarp();
    const int left = bytes - lane * kPiece;
    if (lane < kVectors && left > 0)
      bulk_load(buffers + slot * kBuffer + lane * kPiece, from - skip + lane * kPiece, min(left, kPiece), &full[slot]);
  };
  if (asks) {
    if (lane == 0) {
      asked.x = x0;
      asked.row = row0;
      asked.slot = asked.round = 0;
    }
    __syncwarp();
    for (int i = 0; i < kBuffers; ++i) request();
  }

  // elements before a part in its first vector
  const int shift0 = kWhole ? 0 : shift_of(x0, sizeof(T)), shift_step = static_cast<int>(clusters * a.x.ld % E);
  auto shift_at = [&](int turn) { return kWhole ? 0 : (shift0 + turn * shift_step) & (E - 1); };

  // Whether a vector is one of this warp's.
  auto holds = [&](int at) { return (at & (kThreads - 1)) >> 5 == warp; };
  // a part ends in one of two vectors
  const bool heads = !kWhole && warp == 0, tails = !kWhole && (holds(cols / E) || holds(cols / E + 1));

  // The sum (x) and the maximum (y) of the blocks of a row, to all threads.
  auto join = [&](int turn, float sum, float top) {
    const int set = turn & 1;
    sum = warp_sum(sum);
    top = largest(top);
    if (lane == 0) slots[set][warp] = float2{sum, top};
    __syncthreads();  // also: nobody reads the finished row's buffer any more
    float2 v = slots[set][lane & (kWarps - 1)];
    v = float2{warp_sum(lane < kWarps ? v.x : 0.0f), largest(v.y)};
    if constexpr (kC > 1) {
      // slots and barriers come in two sets: a block that is a row ahead writes to
      // the other one, and it cannot be two ahead
      if (leaves(turn)) v = float2{nan_value(), nan_value()};  // the other blocks' rows are not what they should be
      if (t == 0) async::mbar_expect_tx(&joined[set], kC * 8);
      if (t < kC) send(&ranks[set][rank], &joined[set], t, v);
      // what the other blocks stored is acquired from the cluster, not from this block
      if (t == 0 && !async::wait_inline<true>(async::smem_u32(&joined[set]), turn >> 1 & 1, bound)) left_at = turn + 1;
      __syncthreads();
      v = ranks[set][lane & (kC - 1)];
      v = float2{warp_sum(lane < kC ? v.x : 0.0f), largest(v.y)};
    }
    return v;
  };

  // The next row's target is asked for a turn before it is used.
  auto ask_target = [&](int turn) {
    if (turn < turns)
      asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(async::smem_u32(&note.next_target[turn & 1])),
                   "l"(a.target + row0 + static_cast<std::int64_t>(turn) * clusters)
                   : "memory");
  };
  if (notes && lane == 0) {
    ask_target(0);
    note.target = a.ignore;
    note.f = 1.0f / (a.reduction == 1 ? a.work[0] : 1.0f);
    note.m = note.logit = 0.0f;
    note.last_at = nullptr;
  }
  __syncwarp();
  auto counts = [&](std::int64_t target) { return target != a.ignore && !bad_target(a, target); };
  auto owns = [&](std::int64_t target) { return counts(target) && target >= first && target - first < cols; };
  // The target's gradient takes the place of what another thread wrote a turn ago,
  // on the other side of a barrier.
  auto late = [&] {
    if (lane == 0 && note.last_at != nullptr) *note.last_at = Elem<T>::put(note.last_grad);
  };

  float2 e[kVectors][E / 2];  // exponentials of the row that is finished next
  float sum = 0.0f;
  T* dx = static_cast<T*>(a.dx) + (row0 - clusters) * a.cols + first;  // of the row that is finished
  // the first turn has no row to finish, the last none to begin
  int turn = 0;
  for (;; ++turn) {
    const bool more = turn < turns;
    const int set = turn & 1;
    const unsigned third = static_cast<unsigned>(turn) / kBuffers, slot = turn - third * kBuffers;
    const uint4* in = reinterpret_cast<const uint4*>(buffers + slot * kBuffer) + t;
    float top = -INFINITY;
    if (more) {
      // one lane of a warp asks: a thousand threads at a barrier are served one by one
      if (lane == 0) wait(full[slot], third & 1u, turn);
      __syncwarp();
      if (heads || tails) {
        // what is not the part's in its first vector, and from its end to the last one
        const int before = shift_at(turn), end = before + cols + lane;
        T* row = reinterpret_cast<T*>(buffers + slot * kBuffer);
        if (heads && lane < before) row[lane] = Elem<T>::put(-INFINITY);
        if (tails && end < vectors * E && holds(end / E)) row[end] = Elem<T>::put(-INFINITY);
        __syncwarp();
      }
#pragma unroll
      for (int k = 0; k < kVectors; ++k)
        if (k < mine) top = larger(top, Row<T>::max(in[k * kThreads]));
    }
    if (notes && lane == 0)
      factors[set] = note.target == a.ignore ? 0.0f : bad_target(a, note.target) ? nan_value() : note.f;
    const float2 v = join(turn, sum, top);
    if (leaves(turn)) break;
    if (asks && turn > 0) {
      async::fence_async();
      request();
    }
    const bool write = turn > 0 && a.dx != nullptr;
    const float factor = factors[set], scale = factor * inverse_fast(v.x);
    // whole vectors of the finished row, the first one with what comes before the part
    const int shift = shift_at(turn - 1), whole = (shift + cols) / E;
    uint4* out = reinterpret_cast<uint4*>(dx - shift) + t;
    float2 part_sum = {0.0f, 0.0f};
#pragma unroll
    for (int k = 0; k < kVectors; ++k) {
      if (k >= mine) break;
      if (write) {
        uint4 w = {0, 0, 0, 0};
        if (factor != 0.0f) {  // else an ignored row: zeros, whatever it holds
          if constexpr (sizeof(T) == 4) {
            const float2 p = mul2(e[k][0], both(scale)), q = mul2(e[k][1], both(scale));
            w = uint4{__float_as_uint(p.x), __float_as_uint(p.y), __float_as_uint(q.x), __float_as_uint(q.y)};
          } else {
            w = uint4{Elem<T>::put2(mul2(e[k][0], both(scale))), Elem<T>::put2(mul2(e[k][1], both(scale))),
                      Elem<T>::put2(mul2(e[k][2], both(scale))), Elem<T>::put2(mul2(e[k][3], both(scale)))};
          }
        }
        const int at = k * kThreads + t;
        if (at < whole && (kWhole || at > 0 || shift == 0))
          out[k * kThreads] = w;
        else if (!kWhole && (at == 0 || at == whole))
          ends[at > 0] = w;
      }
      if (more) {
        const uint4 w = in[k * kThreads];
        float2 z[E / 2];
        if constexpr (sizeof(T) == 4) {
          z[0] = float2{__uint_as_float(w.x), __uint_as_float(w.y)};
          z[1] = float2{__uint_as_float(w.z), __uint_as_float(w.w)};
        } else {
          z[0] = Elem<T>::get2(w.x), z[1] = Elem<T>::get2(w.y), z[2] = Elem<T>::get2(w.z), z[3] = Elem<T>::get2(w.w);
        }
#pragma unroll
        for (int i = 0; i < E / 2; ++i) {
          const float2 y = mul2(add2(z[i], both(-v.y)), both(kLog2e));
          e[k][i] = float2{exp2_fast(y.x), exp2_fast(y.y)};
          part_sum = add2(part_sum, e[k][i]);
        }
      }
    }
    if (write && (heads || tails)) {
      __syncwarp();
      T* row = dx - shift;
      if (heads && (shift > 0 || whole == 0) && lane < E && lane >= shift && lane < shift + cols)
        row[lane] = reinterpret_cast<const T*>(ends)[lane];
      if (tails && whole > 0 && holds(whole) && lane < shift + cols - whole * E)
        row[whole * E + lane] = reinterpret_cast<const T*>(ends + 1)[lane];
      __syncwarp();
    }
    if (notes) {
      late();
      if (lane == 0) {
        note.last_at = nullptr;
        const std::int64_t row = row0 + static_cast<std::int64_t>(turn) * clusters;
        if (turn > 0) {
          const bool owner = owns(note.target);
          // the first block where no block has the target
          if (owner || (rank == 0 && !counts(note.target)))
            finish_row(a, row - clusters, note.target == a.ignore, note.logit, note.m, v.x);
          if (write && owner) {
            note.last_at = dx + (note.target - first);
            note.last_grad = exp2_fast((note.logit - note.m) * kLog2e) * scale - factor;
          }
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        const std::int64_t target = note.next_target[set];
        ask_target(turn + 1);
        note.m = v.y;
        note.target = target;
        note.logit = more && owns(target)
                         ? load(buffers + slot * kBuffer, Elem<T>::kType, shift_at(turn) + target - first)
                         : nan_value();
      }
    }
    if (!more) break;
    sum = part_sum.x + part_sum.y;
    dx += clusters * a.cols;
  }
  __syncthreads();
  if (notes) late();
  // shared memory outlives the copies, and what other blocks send, also where a wait gave up
  if (left_at != 0) {
    asm volatile("cp.async.wait_all;" ::: "memory");
    if (t == 0) {
      for (unsigned i = 0; i < kBuffers; ++i)
        async::settle(async::smem_u32(&full[i]), i < asked.slot ? asked.round : asked.round ^ 1u);
      if constexpr (kC > 1) async::pause();
    }
    __syncthreads();
  }
  if constexpr (kC > 1) cg::this_cluster().sync();
  // after whatever the row's other blocks wrote
  if (left_at != 0) poison<T, kC>(a, left_at);
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
    if (threadIdx.x == 0) finish_row(a, row, target == a.ignore, target_logit(a, row, target), m, s);
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

template <typename T, int kThreads, int kC, bool kWhole>
cudaError_t launch_long(const Xent& a, cudaStream_t stream) {
  const auto kernel = xent_long<T, kThreads, kC, kWhole>;
  constexpr int kBytes = kBuffers * buffer_bytes(kThreads);
  const cudaError_t rc = allow_shared<xent_long<T, kThreads, kC, kWhole>>(kBytes);
  if (rc != cudaSuccess) return rc;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(sm_count() / kC * kC));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kBytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = kC;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  // The clusters that run at once (an SM count of a GPU part need not be a
  // multiple of kC): one more would wait for another to finish all its rows.
  static Occupancy<1> known;
  int most = kC == 1 ? 0 : known.get(0, [&](int* n) { return cudaOccupancyMaxActiveClusters(n, kernel, &cfg); });
  if (most == 0) most = sm_count() * (kLong / kThreads) / kC;
  cfg.gridDim = dim3(static_cast<unsigned>((a.rows < most ? a.rows : most) * kC));
  unsigned* status = nullptr;
  commux_ops::status_word(&status);
  return cudaLaunchKernelEx(&cfg, kernel, a, status, commux_ops::wait_limit_ns());
}

template <typename T>
cudaError_t launch_rows(const Xent& a, cudaStream_t stream) {
  constexpr int E = Row<T>::E;
  const std::int64_t need = a.cols + E - 1;  // with the longest shift
  if (need <= kEach * kRowThreads) {
    const int group = static_cast<int>((need + kEach * 32 - 1) / (kEach * 32)) * 32;
    const int ids = group == 32 ? 4 : 1;
    xent_rows<T><<<static_cast<unsigned>((a.rows + ids - 1) / ids), group * ids, 0, stream>>>(a, group);
    return cudaSuccess;
  }
  const bool whole = a.cols % E == 0 && a.x.ld % E == 0 && reinterpret_cast<std::uintptr_t>(a.x.p) % 16 == 0;
  if (a.dx != nullptr && !(a.x.ld % E == a.cols % E && reinterpret_cast<std::uintptr_t>(a.x.p) % 16 ==
                                                           reinterpret_cast<std::uintptr_t>(a.dx) % 16)) {
    // rows of dx lie otherwise to their vectors than the logits' (a slice of a wider tensor at an odd place)
    xent_sweep<<<grid_of(a.rows), kSweep, 0, stream>>>(a);
    return cudaSuccess;
  }
  auto go = [&](auto threads, auto blocks) {
    constexpr int kThreads = decltype(threads)::value, kC = decltype(blocks)::value;
    return whole ? launch_long<T, kThreads, kC, true>(a, stream) : launch_long<T, kThreads, kC, false>(a, stream);
  };
  const std::integral_constant<int, 1> one;
  // Many rows: the smallest block that holds one. Where the rows leave SMs idle,
  // or a row is longer than a block's, more blocks to a row.
  const bool few = a.rows * 2 <= sm_count();
  if (!few && need <= kVectors * 256 * E) return go(std::integral_constant<int, 256>(), one);
  if (!few && need <= kVectors * 512 * E) return go(std::integral_constant<int, 512>(), one);
  int c = 1;
  const int most = kVectors * kLong * E - E;
  while (c < 8 && ((a.cols + c - 1) / c + E > most || a.rows * c * 2 <= sm_count())) c *= 2;
  if ((a.cols + c - 1) / c + E > most) {
    xent_sweep<<<grid_of(a.rows), kSweep, 0, stream>>>(a);
    return cudaSuccess;
  }
  const std::integral_constant<int, kLong> all;
  return c == 1   ? go(all, one)
         : c == 2 ? go(all, std::integral_constant<int, 2>())
         : c == 4 ? go(all, std::integral_constant<int, 4>())
                  : go(all, std::integral_constant<int, 8>());
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
