// Weight gradient of a linear layer whose input was kept in 8 bits:
//   dw[o][i] = sum_t dy[t][o] X[t][i],  db[o] = sum_t dy[t][o].
// X is q s, or w (q s) + b after a norm, for which
//   dw[o][i] = w[i] sum_t dy[t][o] (q s)[t][i] + b[i] db[o],
// so the norm's weight and bias enter once at the end.
//
// Tensor-core bound: 2 rows cols outs operations on bf16 operands with fp32
// sums. q s is exact in bf16 (see act8.cu), so the 8-bit form is widened on its
// way into shared memory, and only 33/32 bytes an element are read. dy enters
// as 1, 2 or 3 bf16 terms (bf16, fp16, fp32: 8, 11, 24 significant bits, each
// term the next 8 of them), so the products are exact for every type.

#include <cuda.h>

#include "async.cuh"
#include "train_utils.cuh"

namespace train {

namespace {

// A CTA's tile of dw and its step over tokens. 256 x 256 fp32 sums fill the
// 512 columns of tensor memory (two M = 128 halves side by side), and each
// widened X tile feeds two products, which halves the widening per product.
constexpr int kM = 256, kN = 256, kK = 64;
constexpr int kStages = 3;                // dy and 8-bit tiles in flight
constexpr int kWide = 2;                  // widened tiles
constexpr int kBox = 64 * kK * 2;         // a 64-wide bf16 box of a step
constexpr int kBytesA = kM * kK * 2, kBytesQ = kN * kK, kBytesB = kN * kK * 2;
constexpr int kBytesS = kK * (kN / kGroup) * 4;  // a step's steps (scales) as floats
constexpr int kOffQ = kStages * kBytesA, kOffB = kOffQ + kStages * kBytesQ, kOffS = kOffB + kWide * kBytesB;
constexpr int kOffBars = kOffS + kStages * kBytesS;
constexpr int kSmem = kOffBars + 256 + 1024;  // and room to align
constexpr int kConvert = 8;               // widening warps, which also write the results
constexpr int kColumn = 4;                // warps that sum dy's columns
constexpr int kScale = 2;                 // warps that fetch scales, a lane to a token
constexpr int kThreads = 32 * (2 + kConvert + kColumn + kScale);
constexpr int kSlot = kM * kN + kM;       // floats of a partial tile: sums, then db

// Steps of all tiles in a row are dealt out evenly to the CTAs: a CTA's range
// may begin and end inside a tile. A tile that one CTA holds whole is written
// at once, the others' parts go to slots that wgrad_join adds up in order.
struct Plan {
  std::int64_t rows, cols, outs, groups;
  int tiles_n, tiles, steps, ctas, planes;
  __host__ __device__ std::int64_t begin(int cta) const {
    return static_cast<std::int64_t>(tiles) * steps * cta / ctas;
  }
};

struct Out {
  void *dw, *db;
  Type dwt;
  const void *w, *b;
  Type wt;
  float* slots;
};

__device__ __forceinline__ void write_dw(const Plan& p, const Out& out, std::int64_t o, std::int64_t i, float v,
                                         float db) {
  if (out.w != nullptr) v *= load(out.w, out.wt, i);
  if (out.b != nullptr) v += load(out.b, out.wt, i) * db;
  store(out.dw, out.dwt, o * p.cols + i, v);
}

// Two neighbouring bytes (of u = q + 128) times the step, as two bf16. A byte
// in the low bits of 2^23's mantissa is 2^23 + u; less 2^23 + 128 that is q,
// and q s has its low 16 bits clear, so its upper half is the bf16.
__device__ __forceinline__ unsigned widen2(unsigned word, int at, float2 step) {
  const unsigned sel = 0x7540u + static_cast<unsigned>(at);
  const float2 u = {__uint_as_float(__byte_perm(word, 0x4b000000u, sel)),
                    __uint_as_float(__byte_perm(word, 0x4b000000u, sel + 1))};
  const float2 v = mul2(add2(u, both(-8388736.0f)), step);
  return __byte_perm(__float_as_uint(v.x), __float_as_uint(v.y), 0x7632);
}

// Both operands have their M or N elements adjacent: blocks of 64 elements
// (128-byte rows, one for each token, 128-byte swizzle), kBox bytes from one
// block to the next, 1024 bytes from 8 tokens to the next 8.
__device__ __forceinline__ std::uint64_t operand(std::uint32_t smem) {
  return static_cast<std::uint64_t>((smem & 0x3ffffu) >> 4) | static_cast<std::uint64_t>(kBox >> 4) << 16 |
         static_cast<std::uint64_t>(1024 >> 4) << 32 | 1ull << 46 | 2ull << 61;
}

// fp32 sums of bf16 products, both operands M/N-major, M = 128
__device__ __forceinline__ unsigned mma_form(int n) {
  return 1u << 4 | 1u << 7 | 1u << 10 | 1u << 15 | 1u << 16 | static_cast<unsigned>(n >> 3) << 17 | (128u >> 4) << 24;
}

__device__ __forceinline__ void mma(std::uint32_t d, std::uint64_t a, std::uint64_t b, unsigned form, bool add) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(form), "r"(static_cast<unsigned>(add))
      : "memory");
}

__device__ __forceinline__ void commit(std::uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
                   async::smem_u32(bar))
               : "memory");
}

__device__ __forceinline__ void load_sums(float (&v)[32], std::uint32_t at) {
  unsigned r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(at));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}

struct Segment {  // a CTA's part of a tile
  int tile, first, last;  // steps [first, last)
  bool whole, head;
  int m0, n0, halves, boxes, n;
};

__device__ __forceinline__ Segment segment(const Plan& p, std::int64_t at, std::int64_t begin, std::int64_t end) {
  Segment s;
  s.tile = static_cast<int>(at / p.steps);
  s.first = static_cast<int>(at - static_cast<std::int64_t>(s.tile) * p.steps);
  const std::int64_t left = end - at;
  s.last = left < p.steps - s.first ? s.first + static_cast<int>(left) : p.steps;
  s.whole = s.first == 0 && s.last == p.steps;
  s.head = at == begin;
  s.m0 = s.tile / p.tiles_n * kM;
  s.n0 = s.tile % p.tiles_n * kN;
  const std::int64_t m = p.outs - s.m0, n = p.cols - s.n0;
  s.boxes = m >= kM ? kM / 64 : static_cast<int>((m + 63) / 64);
  s.halves = s.boxes > 2 ? 2 : 1;
  s.n = n >= kN ? kN : static_cast<int>((n + 15) / 16 * 16);
  return s;
}

__global__ void __launch_bounds__(kThreads, 1)
    wgrad_tiles(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_q, const Plan p,
                const Out out, const std::uint8_t* scale, unsigned* status, std::uint64_t limit_ns) {
  extern __shared__ unsigned char raw[];
  unsigned char* smem = raw + ((1024u - (async::smem_u32(raw) & 1023u)) & 1023u);
  std::uint64_t* bars = reinterpret_cast<std::uint64_t*>(smem + kOffBars);
  std::uint64_t *full_a = bars, *empty_a = bars + 3, *full_q = bars + 6, *empty_q = bars + 9, *full_b = bars + 12,
                *empty_b = bars + 14, *sums_full = bars + 16, *sums_empty = bars + 17, *column_full = bars + 18,
                *drained = bars + 19;
  std::uint32_t* tmem_at = reinterpret_cast<std::uint32_t*>(bars + 20);
  volatile int* gave_up = reinterpret_cast<volatile int*>(bars + 21);
  __shared__ float column[kM];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const async::Bound bound{gave_up, status, limit_ns};

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      async::mbar_init(&full_a[s], 1);
      async::mbar_init(&empty_a[s], 1 + kColumn);
      async::mbar_init(&full_q[s], 1 + kScale);
      async::mbar_init(&empty_q[s], kConvert);
    }
    for (int s = 0; s < kWide; ++s) {
      async::mbar_init(&full_b[s], kConvert);
      async::mbar_init(&empty_b[s], 1);
    }
    async::mbar_init(sums_full, 1);
    async::mbar_init(sums_empty, kConvert);
    async::mbar_init(column_full, kColumn);
    async::mbar_init(drained, 1);
    *gave_up = 0;
    async::fence_async();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(async::smem_u32(tmem_at))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const std::uint32_t tmem = *tmem_at;

  const std::int64_t begin = p.begin(blockIdx.x), end = p.begin(blockIdx.x + 1);
  // db of a tile's rows: wanted by the tiles of the first column block, and by
  // all where the norm's bias multiplies it
  auto sums_columns = [&](const Segment& s) { return out.b != nullptr || (out.db != nullptr && s.n0 == 0); };

  if (warp == 0) {  // --- loads
    if (lane == 0) {
      unsigned ia = 0, iq = 0;
      bool ok = true;
      for (std::int64_t at = begin; ok && at < end;) {
        const Segment s = segment(p, at, begin, end);
        for (int k = s.first; ok && k < s.last; ++k) {
          const int t0 = k * kK;
          unsigned st = iq % kStages;
          ok = async::bounded_wait(&empty_q[st], iq / kStages & 1u ^ 1u, bound);
          if (!ok) break;
          async::mbar_expect_tx(&full_q[st], kBytesQ);
          async::tma_load_2d(smem + kOffQ + st * kBytesQ, &map_q, s.n0, t0, &full_q[st]);
          ++iq;
          for (int pl = 0; pl < p.planes; ++pl) {
            st = ia % kStages;
            ok = async::bounded_wait(&empty_a[st], ia / kStages & 1u ^ 1u, bound);
            if (!ok) break;
            async::mbar_expect_tx(&full_a[st], s.boxes * kBox);
            for (int b = 0; b < s.boxes; ++b)
              async::tma_load_3d(smem + st * kBytesA + b * kBox, &map_a, s.m0 + 64 * b, t0, pl, &full_a[st]);
            ++ia;
          }
        }
        at += s.last - s.first;
      }
      // the CTA's shared memory outlives the copies also where a wait gave up
      for (unsigned i = ia > kStages ? ia - kStages : 0; !ok && i < ia; ++i)
        async::mbar_wait(&full_a[i % kStages], i / kStages & 1u, limit_ns);
      for (unsigned i = iq > kStages ? iq - kStages : 0; !ok && i < iq; ++i)
        async::mbar_wait(&full_q[i % kStages], i / kStages & 1u, limit_ns);
    }
  } else if (warp == 1) {  // --- products
    if (lane == 0) {
      unsigned ia = 0, ib = 0, seg = 0;
      bool ok = true;
      for (std::int64_t at = begin; ok && at < end; ++seg) {
        const Segment s = segment(p, at, begin, end);
        const unsigned form = mma_form(s.n);
        ok = async::bounded_wait(sums_empty, seg & 1u ^ 1u, bound);
        for (int k = s.first; ok && k < s.last; ++k) {
          const unsigned sb = ib % kWide;
          ok = async::bounded_wait(&full_b[sb], ib / kWide & 1u, bound);
          for (int pl = 0; ok && pl < p.planes; ++pl) {
            const unsigned sa = ia % kStages;
            ok = async::bounded_wait(&full_a[sa], ia / kStages & 1u, bound);
            if (!ok) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const std::uint64_t a = operand(async::smem_u32(smem + sa * kBytesA));
            const std::uint64_t b = operand(async::smem_u32(smem + kOffB + sb * kBytesB));
            for (int h = 0; h < s.halves; ++h)
#pragma unroll
              for (int kk = 0; kk < kK / 16; ++kk)  // 16 tokens are 2048 bytes of every block
                mma(tmem + h * kN, a + (h * 2 * kBox + kk * 2048 >> 4), b + (kk * 2048 >> 4), form,
                    k != s.first || pl != 0 || kk != 0);
            commit(&empty_a[sa]);
            ++ia;
          }
          if (ok) commit(&empty_b[sb]);
          ++ib;
        }
        if (ok) commit(sums_full);
        at += s.last - s.first;
      }
      if (!ok) {  // products in flight read shared memory and write tensor memory
        commit(drained);
        async::mbar_wait(drained, 0, limit_ns);
      }
    }
  } else if (warp < 2 + kConvert) {  // --- widening, and the results
    const int cw = warp - 2, unit = lane & 15, row0 = cw * 2 + (lane >> 4);
    const int block = unit >> 2, odd = block & 1;
    unsigned i = 0, seg = 0;
    bool ok = true;
    for (std::int64_t at = begin; ok && at < end; ++seg) {
      const Segment s = segment(p, at, begin, end);
      const bool busy = unit * 16 < s.n;
      for (int k = s.first; k < s.last; ++k, ++i) {
        const unsigned sq = i % kStages, sb = i % kWide;
        ok = async::bounded_wait(&full_q[sq], i / kStages & 1u, bound) &&
             async::bounded_wait(&empty_b[sb], i / kWide & 1u ^ 1u, bound);
        if (!__all_sync(0xffffffffu, ok)) {
          ok = false;
          break;
        }
        const unsigned char* from = smem + kOffQ + sq * kBytesQ;
        const float* steps = reinterpret_cast<const float*>(smem + kOffS + sq * kBytesS) + (unit >> 1);
        unsigned char* to = smem + kOffB + sb * kBytesB + block * kBox;
        if (busy) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int r = j * 16 + row0;
            uint4 v = *reinterpret_cast<const uint4*>(from + r * kN + unit * 16);
            v.x ^= 0x80808080u, v.y ^= 0x80808080u, v.z ^= 0x80808080u, v.w ^= 0x80808080u;
            const float2 step = both(steps[r * (kN / kGroup)]);
            const uint4 lo = {widen2(v.x, 0, step), widen2(v.x, 2, step), widen2(v.y, 0, step), widen2(v.y, 2, step)};
            const uint4 hi = {widen2(v.z, 0, step), widen2(v.z, 2, step), widen2(v.w, 0, step), widen2(v.w, 2, step)};
            // odd blocks write their halves the other way round: the 8 lanes of
            // a store then meet 8 different 16-byte columns of the banks
            const int u = (unit & 3) * 2;
            unsigned char* row = to + r * 128;
            *reinterpret_cast<uint4*>(row + (((u + odd) ^ (r & 7)) << 4)) = odd ? hi : lo;
            *reinterpret_cast<uint4*>(row + (((u + 1 - odd) ^ (r & 7)) << 4)) = odd ? lo : hi;
          }
        }
        async::fence_async();
        __syncwarp();
        if (lane == 0) {
          async::mbar_arrive(&empty_q[sq]);
          async::mbar_arrive(&full_b[sb]);
        }
      }
      if (!ok) break;
      ok = async::bounded_wait(sums_full, seg & 1u, bound) && async::bounded_wait(column_full, seg & 1u, bound);
      if (!__all_sync(0xffffffffu, ok)) {
        ok = false;
        break;
      }
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      // A warp reads the lanes (rows) of its quarter; a block of 32 x 32 is
      // turned round in the widened tiles' memory, which nothing reads now, so
      // that every store is one row of 32 neighbours.
      const int quarter = warp & 3, h = cw >> 2;
      float* turn = reinterpret_cast<float*>(smem + kOffB) + cw * 32 * 33;
      const int rows0 = h * 128 + quarter * 32;
      float* slot = out.slots + (2 * static_cast<std::int64_t>(blockIdx.x) + (s.head ? 0 : 1)) * kSlot;
      if (h < s.halves) {
        for (int c = 0; c * 32 < s.n; ++c) {
          float v[32];
          load_sums(v, tmem + (static_cast<std::uint32_t>(quarter * 32) << 16) + h * kN + c * 32);
#pragma unroll
          for (int j = 0; j < 32; ++j) turn[lane * 33 + j] = v[j];
          __syncwarp();
          const std::int64_t i0 = s.n0 + c * 32 + lane;
          if (s.whole) {
            for (int r = 0; r < 32; ++r) {
              const std::int64_t o = s.m0 + rows0 + r;
              if (o < p.outs && i0 < p.cols) write_dw(p, out, o, i0, turn[r * 33 + lane], column[rows0 + r]);
            }
          } else {
#pragma unroll 8
            for (int r = 0; r < 32; ++r) slot[(rows0 + r) * kN + c * 32 + lane] = turn[r * 33 + lane];
          }
          __syncwarp();
        }
        if ((s.whole ? s.n0 == 0 && out.db != nullptr : true) && sums_columns(s)) {
          const std::int64_t o = s.m0 + rows0 + lane;
          if (!s.whole)
            slot[kM * kN + rows0 + lane] = column[rows0 + lane];
          else if (o < p.outs)
            store(out.db, out.dwt, o, column[rows0 + lane]);
        }
      }
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) async::mbar_arrive(sums_empty);
      at += s.last - s.first;
      // every warp has read its `turn` before any widens the next tile
      ok = async::bounded_wait(sums_empty, seg & 1u, bound);
      ok = __all_sync(0xffffffffu, ok);
    }
  } else if (warp >= 2 + kConvert + kColumn) {  // --- scales
    // They are bytes at any alignment, which TMA cannot fetch; the widening warps
    // spent more than half of their time on waiting for their own loads of them.
    // Two steps are on their way while one is written.
    const int token = (warp - 2 - kConvert - kColumn) * 32 + lane;
    constexpr int kEach = kN / kGroup;
    unsigned i = 0;
    bool ok = true;
    for (std::int64_t at = begin; ok && at < end;) {
      const Segment s = segment(p, at, begin, end);
      const int some = static_cast<int>(p.groups - s.n0 / kGroup < kEach ? p.groups - s.n0 / kGroup : kEach);
      unsigned ahead[2][kEach];
      auto fetch = [&](int k, unsigned (&e)[kEach]) {
        const std::int64_t t = static_cast<std::int64_t>(k) * kK + token;
        const std::uint8_t* from = scale + t * p.groups + s.n0 / kGroup;
        const bool in = k < s.last && t < p.rows;
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
          e[j] = 1;
          if (in && j < some) e[j] = from[j];
        }
      };
      fetch(s.first, ahead[0]);
      fetch(s.first + 1, ahead[1]);
      auto put = [&](int k, unsigned (&e)[kEach]) {
        const unsigned sq = i % kStages;
        ok = async::bounded_wait(&empty_q[sq], i / kStages & 1u ^ 1u, bound);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) return;
        float4* to = reinterpret_cast<float4*>(smem + kOffS + sq * kBytesS) + token * (kEach / 4);
        to[0] = float4{step_of(e[0]), step_of(e[1]), step_of(e[2]), step_of(e[3])};
        to[1] = float4{step_of(e[4]), step_of(e[5]), step_of(e[6]), step_of(e[7])};
        fetch(k + 2, e);
        __syncwarp();
        if (lane == 0) async::mbar_arrive(&full_q[sq]);
        ++i;
      };
      for (int k = s.first; ok && k < s.last; k += 2) {
        put(k, ahead[0]);
        if (ok && k + 1 < s.last) put(k + 1, ahead[1]);
      }
      at += s.last - s.first;
    }
  } else {  // --- sums of dy's columns
    const int c = (warp - 2 - kConvert) * 32 + lane;  // columns 2c and 2c + 1 of the tile
    const int block = c >> 5, unit = (c & 31) >> 2, in = (c & 3) * 4;
    unsigned i = 0, seg = 0;
    bool ok = true;
    for (std::int64_t at = begin; ok && at < end; ++seg) {
      const Segment s = segment(p, at, begin, end);
      const bool busy = sums_columns(s) && block < s.boxes;
      float v0 = 0.0f, v1 = 0.0f;
      for (std::int64_t k = static_cast<std::int64_t>(s.last - s.first) * p.planes; k > 0; --k, ++i) {
        const unsigned sa = i % kStages;
        ok = async::bounded_wait(&full_a[sa], i / kStages & 1u, bound);
        if (!__all_sync(0xffffffffu, ok)) {
          ok = false;
          break;
        }
        if (busy) {
          // a step's 64 tokens are added up first: a sum over many tokens then
          // has one rounding of its own size for each step, not for each token
          const unsigned char* from = smem + sa * kBytesA + block * kBox + in;
          float a0 = 0.0f, a1 = 0.0f;
#pragma unroll 16
          for (int t = 0; t < kK; ++t) {
            const unsigned w = *reinterpret_cast<const unsigned*>(from + t * 128 + ((unit ^ (t & 7)) << 4));
            a0 += __uint_as_float(w << 16);
            a1 += __uint_as_float(w & 0xffff0000u);
          }
          v0 += a0;
          v1 += a1;
        }
        __syncwarp();
        if (lane == 0) async::mbar_arrive(&empty_a[sa]);
      }
      // the last tile's sums have been read once its results are out
      ok = ok && async::bounded_wait(sums_empty, seg & 1u ^ 1u, bound);
      if (!__all_sync(0xffffffffu, ok)) break;
      column[2 * c] = v0;
      column[2 * c + 1] = v1;
      __syncwarp();
      if (lane == 0) async::mbar_arrive(column_full);
      at += s.last - s.first;
    }
  }
  __syncwarp();
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

// Tiles whose steps several CTAs shared: their parts in the order of the steps.
// A block takes kJoinRows rows of a tile, a thread four neighbours of a few rows.
constexpr int kJoinRows = 16;
constexpr int kJoinThreads = 256;
__global__ void __launch_bounds__(kJoinThreads) wgrad_join(const Plan p, const Out out) {
  __shared__ int parts, first_slot;
  __shared__ float column[kJoinRows];
  const int tile = blockIdx.x, m0 = tile / p.tiles_n * kM, n0 = tile % p.tiles_n * kN, r0 = blockIdx.y * kJoinRows;
  if (m0 + r0 >= p.outs) return;
  if (threadIdx.x == 0) {
    const std::int64_t lo = static_cast<std::int64_t>(tile) * p.steps, hi = lo + p.steps;
    int c = static_cast<int>(lo * p.ctas / (static_cast<std::int64_t>(p.tiles) * p.steps));
    while (p.begin(c + 1) <= lo) ++c;  // the quotient rounds down twice
    // the first part is a CTA's last one unless the CTA begins with it; every
    // later part is its CTA's first
    first_slot = 2 * c + (p.begin(c) >= lo ? 0 : 1);
    int n = 1;
    while (p.begin(c + n) < hi && c + n < p.ctas) ++n;
    parts = n;
  }
  __syncthreads();
  const int n = parts, s0 = first_slot;
  if (n == 1) return;
  auto slot = [&](int k) { return out.slots + static_cast<std::int64_t>(k == 0 ? s0 : (s0 / 2 + k) * 2) * kSlot; };
  if (out.b != nullptr || (out.db != nullptr && n0 == 0)) {
    if (threadIdx.x < kJoinRows) {
      const int r = r0 + threadIdx.x;
      float db = 0.0f;
      for (int k = 0; k < n; ++k) db += slot(k)[kM * kN + r];
      column[threadIdx.x] = db;
      if (n0 == 0 && out.db != nullptr && m0 + r < p.outs) store(out.db, out.dwt, m0 + r, db);
    }
    __syncthreads();
  }
  constexpr int kPass = kJoinThreads * 4 / kN;  // rows that the block reads at once
  const int col = threadIdx.x % (kN / 4) * 4, row = r0 + threadIdx.x / (kN / 4);
  float4 v[kJoinRows / kPass] = {};
#pragma unroll 2
  for (int k = 0; k < n; ++k) {
    const float* from = slot(k) + row * kN + col;
#pragma unroll
    for (int j = 0; j < kJoinRows / kPass; ++j) {
      const float4 w = *reinterpret_cast<const float4*>(from + j * kPass * kN);
      v[j].x += w.x, v[j].y += w.y, v[j].z += w.z, v[j].w += w.w;
    }
  }
#pragma unroll
  for (int j = 0; j < kJoinRows / kPass; ++j) {
    const int r = row + j * kPass;
    const std::int64_t o = m0 + r, i = n0 + col;
    if (o >= p.outs || i >= p.cols) continue;
    const float db = out.b != nullptr ? column[r - r0] : 0.0f;
    if (out.dwt == Type::f32 && out.w == nullptr && p.cols % 4 == 0) {
      *reinterpret_cast<float4*>(static_cast<float*>(out.dw) + o * p.cols + i) = v[j];
      continue;
    }
    write_dw(p, out, o, i, v[j].x, db);
    if (i + 1 < p.cols) write_dw(p, out, o, i + 1, v[j].y, db);
    if (i + 2 < p.cols) write_dw(p, out, o, i + 2, v[j].z, db);
    if (i + 3 < p.cols) write_dw(p, out, o, i + 3, v[j].w, db);
  }
}

// dy as `planes` bf16 terms, [planes][rows][ld]: each term the leading 8 bits of
// what the terms before it left (cut off, not rounded, so no term overflows).
__global__ void __launch_bounds__(256) wgrad_terms(Rows dy, __nv_bfloat16* to, int planes, std::int64_t rows,
                                                   std::int64_t outs, std::int64_t ld) {
  const std::int64_t n = rows * ld;
  for (std::int64_t at = blockIdx.x * 256ll + threadIdx.x; at < n; at += gridDim.x * 256ll) {
    const std::int64_t t = at / ld, o = at - t * ld;
    float v = o < outs ? load(dy.p, dy.t, t * dy.ld + o) : 0.0f;
    for (int p = 0; p < planes; ++p) {
      const bool finite = (__float_as_uint(v) & 0x7f800000u) != 0x7f800000u;
      // a NaN whose bits are all in the lower half stays one
      const unsigned bits = v != v ? 0x7fc00000u : __float_as_uint(v) & 0xffff0000u;
      to[p * n + at] = __ushort_as_bfloat16(static_cast<unsigned short>(bits >> 16));
      v = finite ? v - __uint_as_float(bits) : 0.0f;
    }
  }
}

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_tiled() {
  static const EncodeTiledFn fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q = cudaDriverEntryPointSymbolNotFound;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      f = nullptr;
    return reinterpret_cast<EncodeTiledFn>(f);
  }();
  return fn;
}

// TMA reads dy itself where it is bf16 with rows on 16-byte boundaries.
bool as_it_is(const Wgrad8& a) {
  return a.dy.t == Type::bf16 && reinterpret_cast<std::uintptr_t>(a.dy.p) % 16 == 0 && a.dy.ld % 8 == 0 &&
         a.dy.ld >= a.outs;
}

int planes_of(Type t) { return t == Type::bf16 ? 1 : t == Type::f16 ? 2 : 3; }

Plan plan_of(const Wgrad8& a) {
  Plan p;
  p.rows = a.rows;
  p.cols = a.cols;
  p.outs = a.outs;
  p.groups = groups(a.cols);
  p.planes = planes_of(a.dy.t);
  p.tiles_n = static_cast<int>((a.cols + kN - 1) / kN);
  p.tiles = static_cast<int>((a.outs + kM - 1) / kM) * p.tiles_n;
  p.steps = static_cast<int>((a.rows + kK - 1) / kK);
  // One CTA an SM. Where whole shares of the tiles fill nearly all of them,
  // every CTA has one part of one tile; otherwise parts may cross tiles. No
  // tile is cut into parts under 4 steps, which cost about what a CTA's start
  // and end do.
  const int sms = sm_count();
  const std::int64_t total = static_cast<std::int64_t>(p.tiles) * p.steps;
  std::int64_t n = p.tiles <= sms && sms / p.tiles * p.tiles * 10 >= sms * 9 ? sms / p.tiles * p.tiles : sms;
  const std::int64_t most = (total + 3) / 4 > p.tiles ? (total + 3) / 4 : p.tiles;
  if (n > most) n = most;
  p.ctas = static_cast<int>(n);
  return p;
}

std::int64_t slots_bytes(const Plan& p) { return 2ll * p.ctas * kSlot * static_cast<std::int64_t>(sizeof(float)); }
std::int64_t terms_ld(const Wgrad8& a) { return (a.outs + 7) / 8 * 8; }

}  // namespace

std::int64_t wgrad8_work(const Wgrad8& a) {
  const Plan p = plan_of(a);
  return slots_bytes(p) + (as_it_is(a) ? 0 : 2ll * p.planes * a.rows * terms_ld(a));
}

cudaError_t wgrad8(const Wgrad8& a, cudaStream_t stream) {
  const EncodeTiledFn encode = encode_tiled();
  if (encode == nullptr) return cudaErrorNotSupported;
  const Plan p = plan_of(a);
  const void* dy = a.dy.p;
  std::int64_t ld = a.dy.ld;
  if (!as_it_is(a)) {
    auto* terms = reinterpret_cast<__nv_bfloat16*>(static_cast<char*>(a.work) + slots_bytes(p));
    ld = terms_ld(a);
    const std::int64_t want = (a.rows * ld + 255) / 256, most = 32ll * sm_count();
    wgrad_terms<<<static_cast<unsigned>(want < most ? want : most), 256, 0, stream>>>(a.dy, terms, p.planes, a.rows,
                                                                                     a.outs, ld);
    commux_ops::g_launches++;
    dy = terms;
  }
  CUtensorMap map_a, map_q;
  const cuuint32_t one[3] = {1, 1, 1};
  const cuuint64_t dim_a[3] = {static_cast<cuuint64_t>(a.outs), static_cast<cuuint64_t>(a.rows),
                               static_cast<cuuint64_t>(p.planes)};
  const cuuint64_t stride_a[2] = {static_cast<cuuint64_t>(ld) * 2, static_cast<cuuint64_t>(ld) * 2 * a.rows};
  const cuuint32_t box_a[3] = {64, kK, 1};
  const cuuint64_t dim_q[2] = {static_cast<cuuint64_t>(p.groups) * kGroup, static_cast<cuuint64_t>(a.rows)};
  const cuuint64_t stride_q[1] = {static_cast<cuuint64_t>(p.groups) * kGroup};
  const cuuint32_t box_q[2] = {kN, kK};
  if (encode(&map_a, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(dy), dim_a, stride_a, box_a, one,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS ||
      encode(&map_q, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<std::int8_t*>(a.q), dim_q, stride_q, box_q, one,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
    return cudaErrorInvalidValue;
  const cudaError_t set = cudaFuncSetAttribute(wgrad_tiles, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
  if (set != cudaSuccess) return set;
  const Out out{a.dw, a.db, a.dwt, a.w, a.b, a.wt, static_cast<float*>(a.work)};
  unsigned* status = nullptr;
  commux_ops::status_word(&status);
  wgrad_tiles<<<p.ctas, kThreads, kSmem, stream>>>(map_a, map_q, p, out, a.scale, status, commux_ops::wait_limit_ns());
  commux_ops::g_launches++;
  bool joined = false;
  for (int c = 1; c < p.ctas && !joined; ++c) joined = p.begin(c) % p.steps != 0;
  if (joined) {
    wgrad_join<<<dim3(p.tiles, kM / kJoinRows), kJoinThreads, 0, stream>>>(p, out);
    commux_ops::g_launches++;
  }
  return cudaGetLastError();
}

}  // namespace train
