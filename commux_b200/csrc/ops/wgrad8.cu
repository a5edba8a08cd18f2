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
// term the next 8 of them), so the products are exact for every type. The terms
// are further tokens of the same sums, the smallest terms first.
//
// 16384 tokens, 4096 x 4096: 451 us for the tiles (1.22 PFLOP/s) and 28 us to join
// partial tiles; 8192 tokens, 768 x 3072, fp32 results: 51 and 7 us. 4096 tokens, 4096 x
// 4096: 348 us in fp16 (two terms, 0.79 PFLOP/s of them) and 485 in fp32 (three, 0.85).

#include <cuda.h>

#include "async.cuh"
#include "tensor_map.hpp"
#include "train_utils.cuh"

namespace train {

namespace {

// Two CTAs (a cluster, on neighbouring SMs) share a tile of dw and each product:
// both hold 128 rows of an M = 256 half, and each widens half of the columns, so
// an operand is brought and widened once for both. What bounds such a tile next
// to the products is shared memory: a token's tiles are written by TMA, read and
// written by the widening and read by the products. That is 24 cycles of 128
// bytes for 16 cycles of products on one CTA's 256 x 256 tile (which ran at half
// of the products' rate), and 16 for 16 here. The 2 x 256 columns of a CTA's sums
// fill tensor memory.
constexpr int kM = 512, kN = 256, kK = 64;    // a pair's tile, tokens of a step
constexpr int kStages = 4;                    // dy and 8-bit tiles in flight
constexpr int kWide = 3;                      // widened tiles
constexpr int kDone = 12;                     // steps of which it is known whether they were read
constexpr int kBox = 64 * kK * 2;             // a 64-wide bf16 box of a step
constexpr int kOwnN = kN / 2;                 // columns that a CTA widens, at most
constexpr int kBytesA = kM / 2 * kK * 2, kBytesQ = kOwnN * kK, kBytesB = kOwnN * kK * 2;
constexpr int kBytesS = kK * (kOwnN / kGroup) * 4;  // a step's scales as pairs of bf16
constexpr int kOffQ = kStages * kBytesA, kOffB = kOffQ + kStages * kBytesQ, kOffS = kOffB + kWide * kBytesB;
constexpr int kOffBars = kOffS + kStages * kBytesS;
constexpr int kBarBytes = 512;
constexpr int kSmem = kOffBars + kBarBytes + 1024;  // and room to align
constexpr int kConvert = 8;                   // widening warps, which also write the results
constexpr int kColumn = 4;                    // warps that sum dy's columns
constexpr int kScale = kK / 32;               // warps that fetch scales, a lane to a token
constexpr int kThreads = 32 * (2 + kConvert + kColumn + kScale);
constexpr int kSlot = kM * kN + kM;           // floats of a partial tile: sums, then db

// Steps of all tiles in a row are dealt out evenly to the pairs: a pair's range
// may begin and end inside a tile. A tile that one pair holds whole is written
// at once, the others' parts go to slots that wgrad_join adds up in order.
//
// Tensor memory's fp32 sums are cut off, not rounded, at every 16 tokens, so a sum
// of products of one sign shrinks with its length: by 1.8e-6, 5.5e-5 and 1.2e-3 of
// itself over 1536, 16384 and 200000 tokens. Results are therefore summed over `cut`
// steps of dy's leading term at most in there, and a part's sums of those are added
// up, rounded, in its slot: 1536 tokens for fp32 results, 8 and 32 times as many for
// fp16 and bf16, whose sums then shrink by less than a tenth of half their unit. The
// lower terms come first: what cuts off sums of theirs is 2^-8 of that, where between the leading
// terms' products each of them would cut off the whole sum once more (1.7e-5 over
// 1536 tokens of fp32, 2.1e-3 over 200000 of fp16).
constexpr int kCut = 1536 / kK;
struct Plan {
  std::int64_t rows, cols, outs, groups;
  int tiles_n, tiles, pairs, cut, slots;  // slots of a pair
  int span, lower, steps;                 // steps of one term of dy, of all but the leading one, of all
  __host__ __device__ std::int64_t begin(int pair) const {
    return static_cast<std::int64_t>(tiles) * steps * pair / pairs;
  }
};

struct Out {
  void *dw, *db;
  Type dwt, dbt;
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

// Two neighbouring values times their step, as two bf16. In bf16, 0x4300 and the
// low 7 bits of q are 128 + (q mod 128), 0x4300 and its sign bit are 128 or 256;
// the difference is q, and a power of two times it is exact.
__device__ __forceinline__ unsigned widen2(unsigned word, unsigned at, __nv_bfloat162 step) {
  const unsigned p = __byte_perm(word, 0x43434343u, at), low = p & 0xff7fff7fu, sign = p & 0xff80ff80u;
  const __nv_bfloat162 q = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&low),
                                   *reinterpret_cast<const __nv_bfloat162*>(&sign));
  const __nv_bfloat162 v = __hmul2(q, step);
  return *reinterpret_cast<const unsigned*>(&v);
}

// A scale byte's step as a pair of bf16.
__device__ __forceinline__ unsigned step_pair(unsigned e) {
  const unsigned s = e == 255u ? 0x7fffu : e << 7;
  return s << 16 | s;
}

// Both operands have their M or N elements adjacent: blocks of 64 elements
// (128-byte rows, one for each token, 128-byte swizzle), kBox bytes from one
// block to the next, 1024 bytes from 8 tokens to the next 8. The low word of a
// descriptor holds the address and the first distance, the high word the rest.
__device__ __forceinline__ unsigned operand(std::uint32_t smem) {
  return (smem & 0x3ffffu) >> 4 | static_cast<unsigned>(kBox >> 4) << 16;
}
constexpr unsigned kOperandHigh = 1024 >> 4 | 1u << 14 | 2u << 29;

// fp32 sums of bf16 products, both operands M/N-major, M = 256 over the pair
__device__ __forceinline__ unsigned mma_form(int n) {
  return 1u << 4 | 1u << 7 | 1u << 10 | 1u << 15 | 1u << 16 | static_cast<unsigned>(n >> 3) << 17 | (256u >> 4) << 24;
}

__device__ __forceinline__ void mma(std::uint32_t d, unsigned a, unsigned b, unsigned form, unsigned add) {
  asm volatile(
      "{\n .reg .pred p;\n .reg .b64 x, y;\n setp.ne.u32 p, %4, 0;\n mov.b64 x, {%1, %5};\n mov.b64 y, {%2, %5};\n"
      " tcgen05.mma.cta_group::2.kind::f16 [%0], x, y, %3, p;\n}\n" ::"r"(d),
      "r"(a), "r"(b), "r"(form), "r"(add), "r"(kOperandHigh)
      : "memory");
}

// One half's products of a step; `add` 0: the first of them begins the sums.
__device__ __forceinline__ void mma_step(std::uint32_t d, unsigned a, unsigned b, unsigned form, unsigned add) {
  mma(d, a, b, form, add);
#pragma unroll
  for (int kk = 1; kk < kK / 16; ++kk) mma(d, a + kk * (2048 >> 4), b + kk * (2048 >> 4), form, 1);  // 16 tokens on
}

// Arrives on this barrier in both CTAs once the products issued so far are done.
__device__ __forceinline__ void commit(std::uint32_t bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
      "h"(static_cast<std::uint16_t>(3))
      : "memory");
}

// Four neighbours of a row of dw, those that are in it.
__device__ __forceinline__ void write_four(const Plan& p, const Out& out, std::int64_t o, std::int64_t i, float4 v,
                                           float db) {
  if (o >= p.outs || i >= p.cols) return;
  if (out.dwt == Type::f32 && out.w == nullptr && p.cols % 4 == 0) {
    *reinterpret_cast<float4*>(static_cast<float*>(out.dw) + o * p.cols + i) = v;
    return;
  }
#pragma unroll 1
  for (int k = 0; k < 4 && i + k < p.cols; ++k)
    write_dw(p, out, o, i + k, k == 0 ? v.x : k == 1 ? v.y : k == 2 ? v.z : v.w, db);
}

__device__ __forceinline__ void sync_pair() {
  asm volatile("barrier.cluster.arrive.aligned;\nbarrier.cluster.wait.aligned;" ::: "memory");
}

// The address of CTA 0's copy of a barrier, and an arrival there. What this CTA's
// threads wrote to its shared memory for the products has passed a proxy fence
// before: they are in the memory that the tensor core reads, and no other thread
// reads them. A release over the cluster for each step would wait for more than
// that (64 or 82 us for 8192 tokens, 768 -> 3072; 530 or 800 for 16384, 4096 -> 4096).
__device__ __forceinline__ std::uint32_t leaders(std::uint32_t bar) {
  std::uint32_t there;
  asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(there) : "r"(bar));
  return there;
}
__device__ __forceinline__ void arrive_there(std::uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
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

// Where a step's tokens and their term of dy are.
struct Step {
  int tile, term;
  __device__ __forceinline__ Step(const Plan& p, int k) : tile(k % p.span), term(p.lower / p.span - k / p.span) {}
  __device__ __forceinline__ void next(const Plan& p) {
    if (++tile == p.span) {
      tile = 0;
      --term;
    }
  }
};

struct Segment {  // what a pair sums up in one go: (a cut of) its part of a tile
  int tile, first, last;  // steps [first, last)
  bool whole;             // the part is all of the tile
  bool begins, ends;      // the part's first and last cut
  int slot;               // the part's: 0 at the pair's begin, 1 at its end, 2 between
  int m0, n0, halves, n;  // n: columns of the products, a multiple of 64
};

__device__ __forceinline__ Segment segment(const Plan& p, std::int64_t at, std::int64_t begin, std::int64_t end) {
  Segment s;
  s.tile = static_cast<int>(at / p.steps);
  const std::int64_t tile0 = static_cast<std::int64_t>(s.tile) * p.steps;
  const int now = static_cast<int>(at - tile0);
  const int part0 = begin > tile0 ? static_cast<int>(begin - tile0) : 0;
  const int part1 = end < tile0 + p.steps ? static_cast<int>(end - tile0) : p.steps;
  // steps of the leading term are cut; what comes before them belongs to the first cut
  const int lead = part0 > p.lower ? part0 : p.lower, cuts = part1 > lead ? (part1 - lead + p.cut - 1) / p.cut : 1;
  const int size = (part1 - lead + cuts - 1) / cuts, last = (now > lead ? now : lead) + size;
  s.first = now;
  s.last = last < part1 ? last : part1;
  s.whole = part0 == 0 && part1 == p.steps;
  s.begins = now == part0;
  s.ends = s.last == part1;
  s.slot = s.whole ? 2 : tile0 + part0 == begin ? 0 : 1;
  s.m0 = s.tile / p.tiles_n * kM;
  s.n0 = s.tile % p.tiles_n * kN;
  const std::int64_t n = p.cols - s.n0;
  s.halves = p.outs - s.m0 > kM / 2 ? 2 : 1;
  s.n = n >= kN ? kN : static_cast<int>((n + 63) / 64 * 64);
  return s;
}

// Row of the tile of a CTA's local row (0 to 255): 128 of each half
__device__ __forceinline__ int tile_row(int local, int rank) { return (local >> 7) * 256 + rank * 128 + (local & 127); }

// NaN in a CTA's rows of its pair's tiles, or parts of tiles, of which some were not summed up.
__device__ __noinline__ void poison(const Plan& p, const Out& out, std::int64_t begin, std::int64_t end, int pair,
                                    int rank) {
  const float nan = __int_as_float(0x7fffffff);
  for (std::int64_t at = begin; at < end;) {
    const Segment s = segment(p, at, begin, end);
    float* slot = out.slots + (static_cast<std::int64_t>(p.slots) * pair + s.slot) * kSlot;
    for (int k = threadIdx.x; k < kM / 2 * kN; k += kThreads) {
      const int row = tile_row(k / kN, rank), col = k % kN;
      const std::int64_t o = s.m0 + row, i = s.n0 + col;
      if (!s.whole)
        slot[row * kN + col] = nan;
      else if (o < p.outs && i < p.cols)
        store(out.dw, out.dwt, o * p.cols + i, nan);
      if (col > 0) continue;
      if (!s.whole)
        slot[kM * kN + row] = nan;
      else if (o < p.outs && s.n0 == 0 && out.db != nullptr)
        store(out.db, out.dbt, o, nan);
    }
    const std::int64_t tile_end = static_cast<std::int64_t>(s.tile + 1) * p.steps;
    at = tile_end < end ? tile_end : end;
  }
}

// One barrier tells the products that everything of a step is there and another
// that it was read: the thread that issues the products is the narrowest place of
// the kernel (it cost twice the products' time with a wait for each tile).
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    wgrad_tiles(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_q, const Plan p,
                const Out out, const std::uint8_t* scale, unsigned* status, std::uint64_t limit_ns) {
  extern __shared__ unsigned char raw[];
  unsigned char* smem = raw + ((1024u - (async::smem_u32(raw) & 1023u)) & 1023u);
  // Barriers, by their addresses. In both CTAs: tiles of its own, steps whose tiles
  // were read (done), results. Used in CTA 0, which issues the products: full_b (both
  // have widened, and have their dy tiles), sums_empty (both have the results).
  const std::uint32_t base = async::smem_u32(smem), bars = base + kOffBars;
  const std::uint32_t full_a = bars, empty_a = full_a + 8 * kStages, full_q = empty_a + 8 * kStages,
                      empty_q = full_q + 8 * kStages, full_b = empty_q + 8 * kStages, sums_full = full_b + 8 * kWide,
                      sums_empty = sums_full + 8, turned = sums_full + 16, column_full = sums_full + 24,
                      drained = sums_full + 32, done = sums_full + 40;
  constexpr int kAfter = kOffBars + 8 * (4 * kStages + kWide + 5 + kDone);
  std::uint32_t* tmem_at = reinterpret_cast<std::uint32_t*>(smem + kAfter);
  volatile int* gave_up = reinterpret_cast<volatile int*>(smem + kAfter + 8);
  static_assert((4 * kStages + kWide + 7 + kDone) * 8 <= kBarBytes, "barriers");
  static_assert(kConvert * 32 * 32 * 4 <= kWide * kBytesB, "the results are turned round in the widened tiles");
  __shared__ float column[kM / 2];
  __shared__ int others_gave_up;  // in the other CTA
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int pair = static_cast<int>(blockIdx.x >> 1), rank = static_cast<int>(blockIdx.x & 1);
  const async::Bound bound{gave_up, status, limit_ns};

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      async::init(full_a + 8 * s, 1);
      async::init(empty_a + 8 * s, kColumn);
      async::init(full_q + 8 * s, 1 + kScale);
      async::init(empty_q + 8 * s, kConvert);
    }
    for (int s = 0; s < kWide; ++s) async::init(full_b + 8 * s, 2 * kConvert);
    async::init(sums_full, 1);
    async::init(sums_empty, 2 * kConvert);
    async::init(turned, kConvert);
    async::init(column_full, kColumn);
    async::init(drained, 1);
    for (int s = 0; s < kDone; ++s) async::init(done + 8 * s, 1);
    *gave_up = others_gave_up = 0;
    async::fence_async();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(async::smem_u32(tmem_at))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  sync_pair();  // both CTAs have their barriers and their tensor memory
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const std::uint32_t tmem = *tmem_at;

  const std::int64_t begin = p.begin(pair), end = p.begin(pair + 1);
  // db of a tile's rows: wanted by the tiles of the first column block, and by
  // all where the norm's bias multiplies it
  auto sums_columns = [&](const Segment& s) { return out.b != nullptr || (out.db != nullptr && s.n0 == 0); };

  if (warp == 0) {  // --- loads
    // All lanes go through the loop and one issues, here and for the products: the
    // addresses then stay in the warp's uniform registers.
    const bool chosen = async::elect();
    async::Place place, freed;  // freed: the step whose read frees this one's dy tile
    std::int64_t loaded_a = 0, loaded_q = 0;
    bool ok = true;
    for (std::int64_t at = begin; ok && at < end;) {
      const Segment s = segment(p, at, begin, end);
      const int n0 = s.n0 + rank * (s.n / 2);
      // boxes that hold rows of dw; what the others' memory holds meets only sums
      // that are not written
      int m[4], boxes = 0;
      for (int b = 0; b < 4; ++b) {
        m[b] = s.m0 + tile_row(64 * b, rank);
        boxes += m[b] < p.outs;
      }
      Step step(p, s.first);
      for (int k = s.first; k < s.last; ++k) {
        ok = __all_sync(0xffffffffu, async::wait(empty_q + 8 * place.slot, place.round ^ 1u, bound));
        if (!ok) break;
        if (chosen) {
          async::expect_tx(full_q + 8 * place.slot, kBytesQ);
          async::load_2d(base + kOffQ + place.slot * kBytesQ, &map_q, n0, step.tile * kK, full_q + 8 * place.slot);
        }
        ++loaded_q;
        ok = async::wait(empty_a + 8 * place.slot, place.round ^ 1u, bound);
        if (loaded_a >= kStages) {
          ok = ok && async::wait(done + 8 * freed.slot, freed.round, bound);
          freed.next(kDone);
        }
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        if (chosen) {
          async::expect_tx(full_a + 8 * place.slot, boxes * kBox);
#pragma unroll
          for (int b = 0; b < 4; ++b)
            if (m[b] < p.outs)
              async::load_3d(base + place.slot * kBytesA + b * kBox, &map_a, m[b], step.tile * kK, step.term,
                             full_a + 8 * place.slot);
        }
        ++loaded_a;
        place.next(kStages);
        step.next(p);
      }
      at += s.last - s.first;
    }
    // the CTA's shared memory outlives the copies, also where a wait gave up, here or elsewhere
    for (std::int64_t i = loaded_a > kStages ? loaded_a - kStages : 0; i < loaded_a; ++i)
      async::settle(full_a + 8 * static_cast<unsigned>(i % kStages), static_cast<unsigned>(i / kStages) & 1u);
    for (std::int64_t i = loaded_q > kStages ? loaded_q - kStages : 0; i < loaded_q; ++i)
      async::settle(full_q + 8 * static_cast<unsigned>(i % kStages), static_cast<unsigned>(i / kStages) & 1u);
  } else if (warp == 1 && rank == 1) {  // CTA 0 issues the products of both
  } else if (warp == 1) {  // --- products
    const bool chosen = async::elect();
    async::Place ia, ib, steps;
    unsigned seg = 0;
    bool ok = true;
    const unsigned a0 = operand(base), b0 = operand(base + kOffB);
    for (std::int64_t at = begin; ok && at < end; ++seg) {
      const Segment s = segment(p, at, begin, end);
      const unsigned form = mma_form(s.n);
      ok = __all_sync(0xffffffffu, async::wait<true>(sums_empty, seg & 1u ^ 1u, bound));
      unsigned add = 0;
      for (int k = s.first; ok && k < s.last; ++k) {
        ok = __all_sync(0xffffffffu, async::wait<true>(full_b + 8 * ib.slot, ib.round, bound));
        if (!ok) break;
        const unsigned a = a0 + ia.slot * (kBytesA >> 4), b = b0 + ib.slot * (kBytesB >> 4);
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        if (chosen) {
          mma_step(tmem, a, b, form, add);
          if (s.halves == 2) mma_step(tmem + kN, a + (2 * kBox >> 4), b, form, add);
          commit(done + 8 * steps.slot);
        }
        add = 1;
        ia.next(kStages);
        ib.next(kWide);
        steps.next(kDone);
      }
      if (ok && chosen) commit(sums_full);
      at += s.last - s.first;
    }
  } else if (warp < 2 + kConvert) {  // --- widening, and the results
    // A warp takes two tokens' 128 columns at a time, a lane 8 of them: 8 bytes
    // in, one 16-byte column of a swizzled row out, both without bank conflicts.
    const int cw = warp - 2, in = lane & 15, block = in >> 3, unit = in & 7, row0 = cw * 2 + (lane >> 4);
    const std::uint32_t leaders_b = leaders(full_b), leaders_sums = leaders(sums_empty);
    async::Place iq, ib, freed;
    unsigned seg = 0, widened = 0;
    bool ok = true;
    for (std::int64_t at = begin; ok && at < end; ++seg) {
      const Segment s = segment(p, at, begin, end);
      const bool busy = in * 8 < s.n / 2;
      for (int k = s.first; k < s.last; ++k) {
        ok = async::wait(full_q + 8 * iq.slot, iq.round, bound);
        if (widened < kWide) {
          ++widened;
        } else {
          ok = ok && async::wait(done + 8 * freed.slot, freed.round, bound);
          freed.next(kDone);
        }
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        const unsigned char* from = smem + kOffQ + iq.slot * kBytesQ + in * 8;
        const unsigned* steps = reinterpret_cast<const unsigned*>(smem + kOffS + iq.slot * kBytesS) + (in >> 2);
        unsigned char* to = smem + kOffB + ib.slot * kBytesB + block * kBox;
        if (busy) {
          constexpr int kTurns = kK / (2 * kConvert);
          uint2 v[kTurns];
          unsigned two[kTurns];
#pragma unroll
          for (int j = 0; j < kTurns; ++j) {
            const int r = j * 2 * kConvert + row0;
            v[j] = *reinterpret_cast<const uint2*>(from + r * kOwnN);
            two[j] = steps[r * (kOwnN / kGroup)];
          }
#pragma unroll
          for (int j = 0; j < kTurns; ++j) {
            const int r = j * 2 * kConvert + row0;
            const __nv_bfloat162 step = *reinterpret_cast<const __nv_bfloat162*>(&two[j]);
            *reinterpret_cast<uint4*>(to + r * 128 + ((unit ^ (r & 7)) << 4)) =
                uint4{widen2(v[j].x, 0x4140u, step), widen2(v[j].x, 0x4342u, step), widen2(v[j].y, 0x4140u, step),
                      widen2(v[j].y, 0x4342u, step)};
          }
        }
        async::fence_async();
        __syncwarp();
        if (lane == 0) {
          async::arrive(empty_q + 8 * iq.slot);
          // one warp's arrival stands for dy's tile too; its places are the 8-bit
          // tile's. The others have arrived long before.
          if (cw == 0) ok = async::wait(full_a + 8 * iq.slot, iq.round, bound);
          if (ok) arrive_there(leaders_b + 8 * ib.slot);
        }
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        iq.next(kStages);
        ib.next(kWide);
      }
      if (!ok) break;
      ok = async::wait(sums_full, seg & 1u, bound) && async::wait(column_full, seg & 1u, bound);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      // A warp reads the lanes (rows) of its quarter; a block of 32 x 32 is turned
      // round in the widened tiles' memory, which nothing reads now, so that a
      // store is 4 rows of 32 neighbours. A thread has the same places in every
      // segment, so it finds its own earlier sums in the slot.
      const int quarter = warp & 3, h = cw >> 2;
      float4* turn = reinterpret_cast<float4*>(smem + kOffB) + cw * 32 * 8;
      const int local0 = h * 128 + quarter * 32, rows0 = tile_row(local0, rank);
      float* slot = out.slots + (static_cast<std::int64_t>(p.slots) * pair + s.slot) * kSlot;
      const bool last = s.ends && s.whole;
      if (h < s.halves) {
        for (int c = 0; c * 32 < s.n; ++c) {
          float v[32];
          load_sums(v, tmem + (static_cast<std::uint32_t>(quarter * 32) << 16) + h * kN + c * 32);
          const int sub = lane >> 3, four = lane & 7;
          float4* place = reinterpret_cast<float4*>(slot + (rows0 + sub) * kN + c * 32) + four;
          float4 w[8] = {};
          if (!s.begins) {
#pragma unroll
            for (int j = 0; j < 8; ++j) w[j] = place[j * kN];
          }
#pragma unroll
          for (int j = 0; j < 8; ++j)
            turn[lane * 8 + (j ^ (lane & 7))] = float4{v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]};
          __syncwarp();
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int r = j * 4 + sub;
            float4* mine = &turn[r * 8 + (four ^ (r & 7))];
            const float4 u = *mine;
            w[j] = float4{w[j].x + u.x, w[j].y + u.y, w[j].z + u.z, w[j].w + u.w};
            if (!last)
              place[j * kN] = w[j];
            else
              *mine = w[j];
          }
          if (last) {
            // not unrolled: a small product spends its time on fetching instructions
#pragma unroll 1
            for (int r = sub; r < 32; r += 4)
              write_four(p, out, s.m0 + rows0 + r, s.n0 + c * 32 + four * 4, turn[r * 8 + (four ^ (r & 7))],
                         column[local0 + r]);
          }
          __syncwarp();
        }
        if (s.ends && sums_columns(s) && (s.n0 == 0 || !s.whole)) {
          const std::int64_t o = s.m0 + rows0 + lane;
          if (!s.whole)
            slot[kM * kN + rows0 + lane] = column[local0 + lane];
          else if (o < p.outs && out.db != nullptr)
            store(out.db, out.dbt, o, column[local0 + lane]);
        }
      }
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) {
        async::arrive(turned);
        arrive_there(leaders_sums);
      }
      at += s.last - s.first;
      // every warp has read its `turn` before any widens the next tile
      ok = __all_sync(0xffffffffu, async::wait(turned, seg & 1u, bound));
    }
  } else if (warp >= 2 + kConvert + kColumn) {  // --- scales
    // They are bytes at any alignment, which TMA cannot fetch. Two steps are on
    // their way while one is written.
    const int token = (warp - 2 - kConvert - kColumn) * 32 + lane;
    constexpr int kEach = kOwnN / kGroup;
    async::Place iq;
    bool ok = true;
    for (std::int64_t at = begin; ok && at < end;) {
      const Segment s = segment(p, at, begin, end);
      const std::int64_t group = (s.n0 + rank * (s.n / 2)) / kGroup, left = p.groups - group;
      const int some = static_cast<int>(left < kEach ? left : kEach);
      unsigned ahead[2][kEach];
      Step step(p, s.first);  // what is fetched next
      auto fetch = [&](int k, unsigned (&e)[kEach]) {
        const std::int64_t t = static_cast<std::int64_t>(step.tile) * kK + token;
        step.next(p);
        const std::uint8_t* from = scale + t * p.groups + group;
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
        ok = __all_sync(0xffffffffu, async::wait(empty_q + 8 * iq.slot, iq.round ^ 1u, bound));
        if (!ok) return;
        static_assert(kEach == 4, "a token's scales are one vector");
        reinterpret_cast<uint4*>(smem + kOffS + iq.slot * kBytesS)[token] =
            uint4{step_pair(e[0]), step_pair(e[1]), step_pair(e[2]), step_pair(e[3])};
        fetch(k + 2, e);
        __syncwarp();
        if (lane == 0) async::arrive(full_q + 8 * iq.slot);
        iq.next(kStages);
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
    async::Place ia;
    unsigned seg = 0;
    bool ok = true;
    float v0 = 0.0f, v1 = 0.0f;
    for (std::int64_t at = begin; ok && at < end; ++seg) {
      const Segment s = segment(p, at, begin, end);
      const bool busy = sums_columns(s) && s.m0 + tile_row(64 * block, rank) < p.outs;
      if (s.begins) v0 = v1 = 0.0f;  // a part's cuts go on
      for (int k = s.first; k < s.last; ++k) {
        ok = __all_sync(0xffffffffu, async::wait(full_a + 8 * ia.slot, ia.round, bound));
        if (!ok) break;
        if (busy) {
          // a step's 64 tokens are added up first: a sum over many tokens then
          // has one rounding of its own size for each step, not for each token
          const unsigned char* from = smem + ia.slot * kBytesA + block * kBox + in;
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
        if (lane == 0) async::arrive(empty_a + 8 * ia.slot);
        ia.next(kStages);
      }
      // the last tile's sums have been read once its results are out
      ok = __all_sync(0xffffffffu, ok && async::wait(turned, seg & 1u ^ 1u, bound));
      if (!ok) break;
      column[2 * c] = v0;
      column[2 * c + 1] = v1;
      __syncwarp();
      if (lane == 0) async::arrive(column_full);
      at += s.last - s.first;
    }
  }
  __syncwarp();
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0 && *gave_up != 0) {
    std::uint32_t there;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(async::smem_u32(&others_gave_up)), "r"(rank ^ 1));
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(there), "r"(1) : "memory");
  }
  sync_pair();  // neither CTA's memory is in use by the other, unless a wait gave up
  if (*gave_up != 0 || *const_cast<volatile int*>(&others_gave_up) != 0) {
    // products in flight read shared memory and write tensor memory of both CTAs
    if (warp == 1) {
      if (rank == 0 && async::elect()) commit(drained);  // the thread that issued them
      __syncwarp();
      async::settle(drained, 0);
    }
    poison(p, out, begin, end, pair, rank);
    sync_pair();
  }
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

// Tiles whose steps several pairs shared: their parts in the order of the steps.
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
    int c = static_cast<int>(lo * p.pairs / (static_cast<std::int64_t>(p.tiles) * p.steps));
    while (p.begin(c + 1) <= lo) ++c;  // the quotient rounds down twice
    // the first part is a pair's last one unless the pair begins with it; every
    // later part is its pair's first
    first_slot = p.slots * c + (p.begin(c) >= lo ? 0 : 1);
    int n = 1;
    while (p.begin(c + n) < hi && c + n < p.pairs) ++n;
    parts = n;
  }
  __syncthreads();
  const int n = parts, s0 = first_slot;
  if (n == 1) return;
  auto slot = [&](int k) {
    return out.slots + static_cast<std::int64_t>(k == 0 ? s0 : (s0 / p.slots + k) * p.slots) * kSlot;
  };
  if (out.b != nullptr || (out.db != nullptr && n0 == 0)) {
    if (threadIdx.x < kJoinRows) {
      const int r = r0 + threadIdx.x;
      float db = 0.0f;
      for (int k = 0; k < n; ++k) db += slot(k)[kM * kN + r];
      column[threadIdx.x] = db;
      if (n0 == 0 && out.db != nullptr && m0 + r < p.outs) store(out.db, out.dbt, m0 + r, db);
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
    write_four(p, out, o, i, v[j], out.b != nullptr ? column[r - r0] : 0.0f);
  }
}

// dy as `terms` bf16 terms, [terms][rows][ld]: each term the leading 8 bits of
// what the terms before it left (cut off, not rounded, so no term overflows).
__global__ void __launch_bounds__(256) wgrad_terms(Rows dy, __nv_bfloat16* to, int terms, std::int64_t rows,
                                                   std::int64_t outs, std::int64_t ld) {
  const std::int64_t n = rows * ld;
  for (std::int64_t at = blockIdx.x * 256ll + threadIdx.x; at < n; at += gridDim.x * 256ll) {
    const std::int64_t t = at / ld, o = at - t * ld;
    float v = o < outs ? load(dy.p, dy.t, t * dy.ld + o) : 0.0f;
    for (int p = 0; p < terms; ++p) {
      const bool finite = (__float_as_uint(v) & 0x7f800000u) != 0x7f800000u;
      // a NaN whose bits are all in the lower half stays one
      const unsigned bits = v != v ? 0x7fc00000u : __float_as_uint(v) & 0xffff0000u;
      to[p * n + at] = __ushort_as_bfloat16(static_cast<unsigned short>(bits >> 16));
      v = finite ? v - __uint_as_float(bits) : 0.0f;
    }
  }
}

// TMA reads dy itself where it is bf16 with rows on 16-byte boundaries.
bool as_it_is(const Wgrad8& a) {
  return a.dy.t == Type::bf16 && reinterpret_cast<std::uintptr_t>(a.dy.p) % 16 == 0 && a.dy.ld % 8 == 0 &&
         a.dy.ld >= a.outs;
}

int terms_of(Type t) { return t == Type::bf16 ? 1 : t == Type::f16 ? 2 : 3; }

Plan plan_of(const Wgrad8& a) {
  Plan p;
  p.rows = a.rows;
  p.cols = a.cols;
  p.outs = a.outs;
  p.groups = groups(a.cols);
  p.tiles_n = static_cast<int>((a.cols + kN - 1) / kN);
  p.tiles = static_cast<int>((a.outs + kM - 1) / kM) * p.tiles_n;
  p.span = static_cast<int>((a.rows + kK - 1) / kK);
  p.lower = (terms_of(a.dy.t) - 1) * p.span;
  p.steps = p.lower + p.span;
  // One CTA an SM. Where whole shares of the tiles fill nearly all of them,
  // every pair has one part of one tile; otherwise parts may cross tiles. No
  // tile is cut into parts under 4 steps, which cost about what a pair's start
  // and end do.
  const int most_pairs = sm_count() / 2;
  const std::int64_t total = static_cast<std::int64_t>(p.tiles) * p.steps;
  std::int64_t n = most_pairs;
  if (p.tiles <= most_pairs && most_pairs / p.tiles * p.tiles * 10 >= most_pairs * 9)
    n = most_pairs / p.tiles * p.tiles;
  const std::int64_t most = (total + 3) / 4 > p.tiles ? (total + 3) / 4 : p.tiles;
  if (n > most) n = most;
  p.pairs = static_cast<int>(n);
  p.cut = kCut << (a.dwt == Type::f32 ? 0 : a.dwt == Type::f16 ? 3 : 5);
  p.slots = p.cut < p.span ? 3 : 2;
  return p;
}

std::int64_t slots_bytes(const Plan& p) {
  return static_cast<std::int64_t>(p.slots) * p.pairs * kSlot * static_cast<std::int64_t>(sizeof(float));
}
std::int64_t terms_ld(const Wgrad8& a) { return (a.outs + 7) / 8 * 8; }

}  // namespace

std::int64_t wgrad8_work(const Wgrad8& a) {
  const Plan p = plan_of(a);
  return slots_bytes(p) + (as_it_is(a) ? 0 : 2ll * terms_of(a.dy.t) * a.rows * terms_ld(a));
}

cudaError_t wgrad8(const Wgrad8& a, cudaStream_t stream) {
  const auto encode = commux_ops::encode_tiled();
  if (encode == nullptr) return cudaErrorNotSupported;
  const Plan p = plan_of(a);
  const int count = terms_of(a.dy.t);
  const void* dy = a.dy.p;
  std::int64_t ld = a.dy.ld;
  if (!as_it_is(a)) {
    auto* terms = reinterpret_cast<__nv_bfloat16*>(static_cast<char*>(a.work) + slots_bytes(p));
    ld = terms_ld(a);
    const std::int64_t want = (a.rows * ld + 255) / 256, most = 32ll * sm_count();
    wgrad_terms<<<static_cast<unsigned>(want < most ? want : most), 256, 0, stream>>>(a.dy, terms, count, a.rows,
                                                                                     a.outs, ld);
    commux_ops::g_launches++;
    dy = terms;
  }
  CUtensorMap map_a, map_q;
  const cuuint32_t one[3] = {1, 1, 1};
  const cuuint64_t dim_a[3] = {static_cast<cuuint64_t>(a.outs), static_cast<cuuint64_t>(a.rows),
                               static_cast<cuuint64_t>(count)};
  const cuuint64_t stride_a[2] = {static_cast<cuuint64_t>(ld) * 2, static_cast<cuuint64_t>(ld) * 2 * a.rows};
  const cuuint32_t box_a[3] = {64, kK, 1};
  const cuuint64_t dim_q[2] = {static_cast<cuuint64_t>(p.groups) * kGroup, static_cast<cuuint64_t>(a.rows)};
  const cuuint64_t stride_q[1] = {static_cast<cuuint64_t>(p.groups) * kGroup};
  const cuuint32_t box_q[2] = {kOwnN, kK};
  if (encode(&map_a, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(dy), dim_a, stride_a, box_a, one,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS ||
      encode(&map_q, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<std::int8_t*>(a.q), dim_q, stride_q, box_q, one,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
    return cudaErrorInvalidValue;
  const cudaError_t set = allow_shared<wgrad_tiles>(kSmem);
  if (set != cudaSuccess) return set;
  const Out out{a.dw, a.db, a.dwt, a.dbt, a.w, a.b, a.wt, static_cast<float*>(a.work)};
  unsigned* status = nullptr;
  commux_ops::status_word(&status);
  wgrad_tiles<<<2 * p.pairs, kThreads, kSmem, stream>>>(map_a, map_q, p, out, a.scale, status,
                                                        commux_ops::wait_limit_ns());
  commux_ops::g_launches++;
  bool joined = false;
  for (int c = 1; c < p.pairs && !joined; ++c) joined = p.begin(c) % p.steps != 0;
  if (joined) {
    wgrad_join<<<dim3(p.tiles, kM / kJoinRows), kJoinThreads, 0, stream>>>(p, out);
    commux_ops::g_launches++;
  }
  return cudaGetLastError();
}

}  // namespace train
