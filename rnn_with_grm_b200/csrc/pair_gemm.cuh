// Matrix product of CTA pairs (tcgen05 cta_group::2) with a fused epilogue, for the vocabulary loss.
//
//   C[m, n] = sum over planes and k of A[m, k] B[n, k]        256 x 256 per pair of CTAs, fp32 in TMEM
//
// Each CTA of a pair holds 128 rows of A and 128 of the 256 columns of B in shared memory (32 KiB per
// 64-wide k block), and its own 128 rows of the result in TMEM: a pair reads (256 + 256) * 64 values per
// 2 * 256 * 256 * 64 FLOP, half of what a single CTA with a 128 x 256 tile would ask of L2 for its share,
// which is what decides whether the tensor cores are fed.  Persistent pairs; one warp loads (TMA ring of
// kStages blocks), one warp of the first CTA issues for both, the others are the epilogue in groups of four.  Two
// accumulators of 256 columns: the epilogue of a tile runs under the products of the next one.
//
// Measured and dropped: B resident in shared memory while a pair walks down its rows (contractions of at most 512: no
// gain once the card is at its power limit); an epilogue that stores by TMA from a buffer per group (594 us where a
// staging box per warp and plain stores take 536).
//
// The gradient of the scores goes out, and comes back as A of the products that follow, in panels of 64 columns
// [rows][64]: a tile's part is then whole kilobytes in a row, where lines of a wide row-major matrix would be 64 KiB
// apart (16384 x 32768, back to back: 640 -> 584 us for writing it, 2 % off each product).
//
// Operands are bf16 matrices [planes][rows][cols] read through tensor maps; either may be K-major (k is the
// contiguous index) or MN-major.  Full-precision callers pass their matrices as three bf16 planes whose sum
// is the fp32 value to 24 bits and ask for six plane products (all that matter above 2^-24); the accumulator
// is then drained into registers every kSegmentSteps blocks, so that long sums are rounded by fp32 additions
// and not by the tensor core's accumulation.
//
// Every wait is bounded; a wait that gives up raises the CTA's and its peer's abort flag, and the error word.
#pragma once

#include <cfloat>

#include "common.cuh"
#include "tc_ptx.cuh"

namespace grmx {
namespace pair {

using namespace tc;

constexpr int kTileM = 256;              // rows per pair
constexpr int kTileN = 256;              // columns per pair
constexpr int kHalf = 128;               // rows of A, columns of B and rows of the result per CTA
constexpr int kBlockK = 64;
constexpr int kOperandBytes = kHalf * kBlockK * 2;       // 16 KiB
constexpr int kGroupThreads = 128;       // an epilogue group: one warp per TMEM lane quadrant
constexpr int kStoreBytes = 16384;       // staging buffer of a TMA store: 128 rows x 128 bytes
constexpr int kBiasBytes = 2048;         // float[512] among the epilogue groups
constexpr int kSmemAlloc = 232448;

constexpr int kStages = 5;
constexpr int kStageBytes = 2 * kOperandBytes;           // [A | B]
constexpr int kOffStore = kStages * kStageBytes;         // staging of the epilogue groups
constexpr int kOffBias = kOffStore + 4 * kStoreBytes;
constexpr int kOffBars = kOffBias + kBiasBytes;
constexpr int kNumBars = 2 * kStages + 4;
constexpr int kOffMisc = kOffBars + kNumBars * 8;
constexpr int kSmemTotal = kOffMisc + 32;
static_assert(kSmemTotal <= kSmemAlloc, "shared memory plan exceeds 227 KiB");
static_assert(kOffBars % 8 == 0, "barriers are 8-byte aligned");
// k blocks between two drains of the accumulator in full precision: 8 blocks are 32 accumulations (the tensor core's
// additions drop what falls off: with 128 between drains dW of 2048 tokens was 1.6e-6 off, twice what fp32 sums are)
constexpr int kSegmentSteps = 8;

enum Epilogue { kEpiLse = 0, kEpiGrad = 1, kEpiStore = 2 };

// Epilogue groups of four warps: four where the epilogue has an exponential per score (two on each accumulator, 128
// columns each; with two groups the epilogue of a tile took longer than its products, 414 against 385 us for 16384 x
// 32768 scores of 512 terms, and with three 737 against 594 us where it also writes the gradient), two for plain
// results (one per accumulator).  In full precision four, each on 64 columns of every accumulator, because the drained
// accumulator has to fit in a thread's registers (with two groups and 128 columns it spilled).
__host__ __device__ constexpr int groups_of(int epilogue, bool seg) { return !seg && epilogue == kEpiStore ? 2 : 4; }
__host__ __device__ constexpr int threads_of(int epilogue, bool seg) { return groups_of(epilogue, seg) * kGroupThreads + 64; }
// column parts of a tile that different groups work on
__host__ __device__ constexpr int parts_of(int epilogue, bool seg) { return seg ? 4 : groups_of(epilogue, seg) / 2; }

constexpr float kLog2e = 1.4426950408889634f;

struct Params {
  int m_tiles, n_tiles, splits;
  int k_blocks;                // 64-wide blocks of the contraction
  int blocks_per_split;
  int64_t rows, cols;          // true size of the result
  // loss epilogues: columns are words v0 + n of the vocabulary
  int64_t v0, vocab;
  const void* bias;            // [vocab] or NULL
  int bias_dtype;
  const int64_t* targets;      // (kEpiStore: of the rows, or NULL)
  int64_t ignore_index;
  // kEpiLse: per row and parts_of() column parts of a tile (two; four in full precision) the maximum and the sum, base 2
  float2* partials;            // [parts][rows]
  float* target_score;         // [rows], base 2
  uint32_t* ticket;            // zeroed for the kernel that follows (or NULL)
  // kEpiGrad
  const float* row_max;        // [rows], base 2
  const float* row_sum;
  const float* grad;           // factor per row of the column sums (kEpiGrad) or of the result (kEpiStore); NULL: 1
  float* bias_partials;        // [row blocks of 32][n_tiles * 256] or NULL
  __nv_bfloat16* d_out;        // [planes][panels of 64 columns][rows][64]
  int panels;                  // kEpiGrad: of d_out; kEpiStore: of A, which is such a matrix
  // kEpiStore
  int store_f32;               // the store map is fp32 (32-column boxes) instead of bf16 (64)
  int store_add;               // add to what is there (fp32 only)
  const float* scale;          // [1] each, factors of the result (NULL: 1)
  const float* scale2;
};

struct Maps {
  CUtensorMap a, b, c;
};

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t map_to_rank(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Arrival on a barrier of either CTA.  What it hands over is an accumulator, which the tcgen05 fences order; a release at
// cluster scope would also wait for this thread's stores to memory (a fence per arrival).
__device__ __forceinline__ void arrive_cluster(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
// bounded wait; giving up raises the abort flag of both CTAs
__device__ __forceinline__ bool wait_pair(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  for (uint32_t it = 0; it < kWaitLimit; ++it) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((it & 63u) == 63u && *abort_flag) return false;
  }
  *abort_flag = 1;
  const uint32_t peer = map_to_rank(smem_u32(const_cast<int*>(abort_flag)), cluster_rank() ^ 1u);
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(peer), "r"(1) : "memory");
  return false;
}
// the same for a whole warp, which then agrees
__device__ __forceinline__ bool wait_pair_warp(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  return __all_sync(0xffffffffu, wait_pair(bar, parity, abort_flag)) != 0;
}
// barrier of the 128 threads of an epilogue group
__device__ __forceinline__ void group_sync(int id) { asm volatile("barrier.cta.sync %0, 128;" ::"r"(id) : "memory"); }
__device__ __forceinline__ bool group_all(int id, bool ok) {
  uint32_t r;
  asm volatile(
      "{\n\t"
      ".reg .pred p, q;\n\t"
      "setp.ne.u32 p, %2, 0;\n\t"
      "barrier.cta.red.and.pred q, %1, 128, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t"
      "}"
      : "=r"(r)
      : "r"(id), "r"(static_cast<uint32_t>(ok))
      : "memory");
  return r != 0;
}

// tile load whose bytes are counted on the barrier of the pair's first CTA
__device__ __forceinline__ void load_box_if(uint32_t leader, void* dst, const CUtensorMap* map, uint32_t bar_cluster,
                                            int x, int y, int z) {
  asm volatile(
      "{\n\t"
      ".reg .pred q;\n\t"
      "setp.ne.b32 q, %6, 0;\n\t"
      "@q cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%3, %4, %5}], [%2];\n\t"
      "}" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar_cluster), "r"(x), "r"(y), "r"(z), "r"(leader)
      : "memory");
}
__device__ __forceinline__ void mma_pair_if(uint32_t leader, uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc,
                                            uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t"
      "}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(leader)
      : "memory");
}
// arrives on the barrier at the same place in both CTAs once the products issued so far have retired
__device__ __forceinline__ void commit_pair_if(uint32_t leader, uint64_t* bar) {
  asm volatile(
      "{\n\t"
      ".reg .pred q;\n\t"
      "setp.ne.b32 q, %2, 0;\n\t"
      "@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n\t"
      "}" ::"r"(smem_u32(bar)),
      "h"(static_cast<uint16_t>(3)), "r"(leader)
      : "memory");
}
__device__ __forceinline__ void store_box(const void* src, const CUtensorMap* map, int x, int y, int z, bool add) {
  if (add) {
    asm volatile(
        "cp.reduce.async.bulk.tensor.3d.global.shared::cta.add.tile.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(
            reinterpret_cast<uint64_t>(map)),
        "r"(smem_u32(src)), "r"(x), "r"(y), "r"(z)
        : "memory");
  } else {
    tma_store_3d(src, map, x, y, z);
  }
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// two fp32 operations per instruction
__device__ __forceinline__ uint64_t pack2(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// y = score * log2 e + bias * log2 e for 32 columns (bias already scaled, 16-byte aligned)
__device__ __forceinline__ void scores_base2(float (&y)[32], const float* bias) {
  const uint64_t k = pack2(kLog2e, kLog2e);
#pragma unroll
  for (int j = 0; j < 32; j += 4) {
    const float4 b = *reinterpret_cast<const float4*>(bias + j);
    unpack2(fma2(pack2(y[j], y[j + 1]), k, pack2(b.x, b.y)), y[j], y[j + 1]);
    unpack2(fma2(pack2(y[j + 2], y[j + 3]), k, pack2(b.z, b.w)), y[j + 2], y[j + 3]);
  }
}

// 32 rows x 32 bf16 that a warp stages for itself: 64 bytes per row, 16-byte pieces swizzled by the row so that neither
// the rows' writes nor the reads below collide.
__device__ __forceinline__ uint8_t* box_piece(uint8_t* box, int row, int piece) {
  return box + row * 64 + ((piece ^ ((row >> 1) & 3)) << 4);
}
// The box to memory, eight rows at a time, its columns added up in fp32 on the way (a lane moves four rows of eight
// columns, each row times its lane's `factor` if WEIGHTED; the eight lanes of a column then share out the sums).  `out` is the box's
// first value; rows at and beyond `rows` are not stored.  Returns the sums of columns box_column(lane) and the next, in both lanes of a pair 4 apart.
// (A TMA store needs the whole group's barriers and a wait of 0.8 us until its buffer is free again.)
__device__ __forceinline__ int box_column(int lane) { return (lane & 3) * 8 + ((lane >> 4) & 1) * 4 + ((lane >> 3) & 1) * 2; }
template <bool SUMS, bool WEIGHTED = false>
__device__ __forceinline__ float2 box_out(uint8_t* box, __nv_bfloat16* out, int ld, int rows, int lane, float factor) {
  const int q = lane & 3, sub = lane >> 2;
  uint64_t acc[4] = {0ull, 0ull, 0ull, 0ull};
  __nv_bfloat16* dst = out + sub * ld + q * 8;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const uint4 v = *reinterpret_cast<const uint4*>(box_piece(box, 8 * r + sub, q));
    if (8 * r + sub < rows) *reinterpret_cast<uint4*>(dst) = v;
    dst += 8 * ld;
    if (SUMS) {
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
      const float f = WEIGHTED ? __shfl_sync(0xffffffffu, factor, 8 * r + sub) : 1.0f;
      const uint64_t f2 = pack2(f, f);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint64_t pair = pack2(__uint_as_float(w[e] << 16), __uint_as_float(w[e] & 0xffff0000u));
        acc[e] = WEIGHTED ? fma2(pair, f2, acc[e]) : add2(acc[e], pair);
      }
    }
  }
  float2 sums = make_float2(0.0f, 0.0f);
  if (SUMS) {
    // lanes 16 apart, then 8 apart, give away the half they do not return; lanes 4 apart return the same
    const bool upper = (lane & 16) != 0, odd = (lane & 8) != 0;
    uint64_t half[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const uint64_t keep = upper ? acc[2 + e] : acc[e], give = upper ? acc[e] : acc[2 + e];
      half[e] = add2(keep, __shfl_xor_sync(0xffffffffu, give, 16));
    }
    uint64_t one = odd ? half[1] : half[0];
    const uint64_t give = odd ? half[0] : half[1];
    one = add2(one, __shfl_xor_sync(0xffffffffu, give, 8));
    one = add2(one, __shfl_xor_sync(0xffffffffu, one, 4));
    unpack2(one, sums.x, sums.y);
  }
  return sums;
}

// The units of work of one pair and what each of them is.
template <int EPI>
struct Units {
  int begin, end, step;
  __device__ __forceinline__ Units(const Params& p) {
    const int total = p.m_tiles * p.n_tiles * p.splits, pairs = gridDim.x >> 1, pair = blockIdx.x >> 1;
    begin = pair;
    end = total;
    step = pairs;
  }
  // row tile, column tile, split
  __device__ __forceinline__ void tile(const Params& p, int u, int& m, int& n, int& s) const {
    s = 0;
    if (EPI == kEpiStore) {
      // column tiles of a row tile next to each other: they read the same A
      n = u % p.n_tiles;
      m = (u / p.n_tiles) % p.m_tiles;
      s = u / (p.n_tiles * p.m_tiles);
    } else {
      // bands of eight row tiles, column by column: the tiles that run at one time share rows and columns in L2
      const int per_band = 8 * p.n_tiles;
      const int band = u / per_band, r = u % per_band;
      const int height = min(8, p.m_tiles - 8 * band);
      m = 8 * band + r % height;
      n = r / height;
    }
  }
};

// Sums over the 32 lanes of a warp of 32 values each; lane j returns the sum of v[j].
__device__ __forceinline__ float transpose_sum(float (&v)[32], int lane) {
#pragma unroll
  for (int half = 16; half >= 1; half >>= 1) {
    const bool upper = (lane & half) != 0;
#pragma unroll
    for (int j = 0; j < half; ++j) {
      const float keep = upper ? v[j + half] : v[j];
      const float give = upper ? v[j] : v[j + half];
      v[j] = keep + __shfl_xor_sync(0xffffffffu, give, half);
    }
  }
  return v[0];
}

// A bias in base 2.  A mask of the type's lowest value overflows there; it stays finite (only -inf masks a word for good),
// so that a row in which nothing else is left has a distribution, equal over its words.
__device__ __forceinline__ float bias_base2(float b) {
  const float y = b * kLog2e;
  return y == -INFINITY && b != -INFINITY ? -FLT_MAX : y;
}
// biases of `count` words from word v, base 2, into shared memory; words beyond the vocabulary get -inf
__device__ __forceinline__ void load_bias(const Params& p, float* dst, int64_t v, int count, int thread, int threads) {
  for (int j = thread; j < count; j += threads) {
    float b = -INFINITY;
    if (v + j < p.vocab) {
      b = 0.0f;
      if (p.bias != nullptr) {
        b = p.bias_dtype == GRMX_F32 ? __ldg(static_cast<const float*>(p.bias) + v + j)
                                     : __bfloat162float(__ldg(static_cast<const __nv_bfloat16*>(p.bias) + v + j));
      }
    }
    dst[j] = bias_base2(b);
  }
}

// d = 2^(y - top) / sum - [target]; a row that does not count is all zero
struct RowTerms {
  int64_t target;              // word of the target relative to the first column, or -1
  float top, coef, g;          // coef = 1 / sum; g: the row's factor in the column sums
  bool counts;
};
template <bool WEIGHTED>
__device__ __forceinline__ RowTerms row_terms(const Params& p, int64_t row, int64_t first_word) {
  RowTerms r{-1, 0.0f, 0.0f, 0.0f, false};
  if (row < p.rows) {
    const int64_t t = __ldg(p.targets + row);
    if (t != p.ignore_index && t >= 0 && t < p.vocab) {
      if (t >= first_word) r.target = t - first_word;
      if (WEIGHTED) r.g = __ldg(p.grad + row);
      r.top = __ldg(p.row_max + row);
      r.coef = 1.0f / __ldg(p.row_sum + row);
      r.counts = true;
    }
  }
  return r;
}
// 32 scores to their gradients; `first` is the columns' place relative to the one r.target counts from
__device__ __forceinline__ void score_gradient(float (&y)[32], const float* bias, const RowTerms& r, int first) {
  scores_base2(y, bias);
  const uint64_t shift = pack2(-r.top, -r.top), factor = pack2(r.coef, r.coef);
#pragma unroll
  for (int j = 0; j < 32; j += 2) {
    float lo, hi;
    unpack2(add2(pack2(y[j], y[j + 1]), shift), lo, hi);
    unpack2(mul2(pack2(exp2_fast(lo), exp2_fast(hi)), factor), y[j], y[j + 1]);
  }
  if (!__all_sync(0xffffffffu, r.counts)) {
#pragma unroll
    for (int j = 0; j < 32; ++j) y[j] = r.counts ? y[j] : 0.0f;
  }
  const bool hit = r.target >= first && r.target < first + 32;
  if (__any_sync(0xffffffffu, hit)) {
    const int at = hit ? static_cast<int>(r.target) - first : -1;
#pragma unroll
    for (int j = 0; j < 32; ++j) {
      if (at == j) y[j] -= 1.0f;
    }
  }
}

// SEG: full precision (six plane products, accumulator drained into registers; all four epilogue groups work on
// every tile, 64 columns each).  Otherwise half of the groups work on each accumulator, so on every other tile.
// (Registers: the score gradient in full precision spills 196 bytes a thread at the 96 that 18 warps leave, 328 with WEIGHTED;
// the bf16 forms do not spill.)
// WEIGHTED (kEpiGrad): the column sums have a factor per row; a kernel of its own, since the plain one is slower by 25 us of
// 525 with both in it.
template <int EPI, bool A_MN, bool B_MN, bool SEG, bool WEIGHTED>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(threads_of(EPI, SEG), 1)
pair_gemm_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Params p, uint32_t* error_word) {
  constexpr int kGroups = groups_of(EPI, SEG);
  constexpr int kParts = parts_of(EPI, SEG);
  constexpr int kLoaderWarp = 4 * kGroups;
  constexpr int kIssuerWarp = kLoaderWarp + 1;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kOffBars);
  uint64_t* bar_full = bars;                     // [kStages] first CTA only: both CTAs' blocks landed   (1 + tx)
  uint64_t* bar_empty = bars + kStages;          // [kStages] the products that read the stage retired   (commit)
  uint64_t* bar_acc_ready = bars + 2 * kStages;  // [2] products of the accumulator retired               (commit)
  uint64_t* bar_acc_free = bar_acc_ready + 2;    // [2] first CTA only: epilogue warps of both CTAs
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(smem + kOffMisc);
  volatile int* s_abort = reinterpret_cast<volatile int*>(smem + kOffMisc + 8);

  const int tid = threadIdx.x;
  const int warp = tid >> 5;
  const int lane = tid & 31;
  const uint32_t rank = cluster_rank();
  // (the dynamic shared memory starts on a 1 KiB boundary in practice; both CTAs of a pair take the same offset)
  const bool fits = static_cast<int>(smem - smem_raw) + kSmemTotal <= kSmemAlloc;
  if (!fits) {
    if (tid == 0 && error_word != nullptr) atomicOr(error_word, kErrBoundedWait);
    return;
  }
  if (tid == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&bar_full[i], 1);
      mbar_init(&bar_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bar_acc_ready[i], 1);
      mbar_init(&bar_acc_free[i], 8 * kParts);
    }
    *s_abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kIssuerWarp) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(s_tmem)), "r"(512u)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  fence_proxy_async();
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem_base = *s_tmem;
  wait_for_previous();                  // nothing above touches memory
  if (EPI == kEpiLse && blockIdx.x == 0 && tid == 0 && p.ticket != nullptr) *p.ticket = 0u;

  const Units<EPI> units(p);
  auto split_range = [&](int s, int& k0, int& k1) {
    k0 = s * p.blocks_per_split;
    k1 = min(p.k_blocks, k0 + p.blocks_per_split);
  };

  if (warp == kLoaderWarp) {
    // ===================================================================== loader (both CTAs)
    const uint32_t leader = elect_one();
    int step = 0;
    bool ok = true;
    // plane products, smallest first: (low, high) (high, low) (mid, mid) (mid, high) (high, mid) (high, high)
    constexpr uint32_t kPlaneA = 2u | (0u << 2) | (1u << 4) | (1u << 6) | (0u << 8) | (0u << 10);
    constexpr uint32_t kPlaneB = 0u | (2u << 2) | (1u << 4) | (0u << 6) | (1u << 8) | (0u << 10);
    for (int u = units.begin; u < units.end && ok; u += units.step) {
      int m, n, s, k0, k1;
      units.tile(p, u, m, n, s);
      split_range(s, k0, k1);
      const int row = m * kTileM + static_cast<int>(rank) * kHalf;
      const int col = n * kTileN + static_cast<int>(rank) * kHalf;
      for (int kb = k0; kb < k1 && ok; ++kb) {
        const int k = kb * kBlockK;
        for (int pr = 0; pr < (SEG ? 6 : 1); ++pr, ++step) {
          const int st = step % kStages;
          if (step >= kStages && !wait_pair_warp(&bar_empty[st], (step / kStages - 1) & 1u, s_abort)) {
            ok = false;
            break;
          }
          if (rank == 0) mbar_expect_tx_if(leader, &bar_full[st], 2 * kStageBytes);
          uint8_t* a = smem + st * kStageBytes;
          const uint32_t bar = map_to_rank(smem_u32(&bar_full[st]), 0);
          const int pa = SEG ? static_cast<int>((kPlaneA >> (2 * pr)) & 3u) : 0;
          if (EPI == kEpiStore && A_MN) {                      // A in panels of 64 columns: its columns are the rows here
            load_box_if(leader, a, &maps.a, bar, 0, k, pa * p.panels + row / 64);
            load_box_if(leader, a + kOperandBytes / 2, &maps.a, bar, 0, k, pa * p.panels + row / 64 + 1);
          } else if (EPI == kEpiStore) {
            load_box_if(leader, a, &maps.a, bar, 0, row, pa * p.panels + kb);
          } else {
            load_box_if(leader, a, &maps.a, bar, k, row, pa);
          }
          uint8_t* b = a + kOperandBytes;
          const int pb = SEG ? static_cast<int>((kPlaneB >> (2 * pr)) & 3u) : 0;
          if (B_MN) {
            load_box_if(leader, b, &maps.b, bar, col, k, pb);
            load_box_if(leader, b + kOperandBytes / 2, &maps.b, bar, col + 64, k, pb);
          } else {
            load_box_if(leader, b, &maps.b, bar, k, col, pb);
          }
        }
      }
    }
    if (*s_abort) {
      // let the copies still in flight land before the shared memory is released: the first CTA's barriers
      // count the bytes of both, the second CTA can only give its copies time
      if (rank == 0) {
        for (int j = step > kStages ? step - kStages : 0; j < step; ++j) mbar_wait_quiet(&bar_full[j % kStages], (j / kStages) & 1u);
      }
      for (int i = 0; i < 2000; ++i) __nanosleep(1000);
    }
  } else if (warp == kIssuerWarp) {
    // ===================================================================== issuer (first CTA, for both)
    if (rank == 0) {
      const uint32_t leader = elect_one();
      constexpr uint32_t idesc = make_idesc(kTileM, kTileN, A_MN, B_MN);
      constexpr uint32_t kStepA = A_MN ? 2048u : 32u;      // bytes of 16 k in the operand's tile
      constexpr uint32_t kStepB = B_MN ? 2048u : 32u;
      int step = 0, it = 0;                                 // blocks and accumulators so far
      bool ok = true;
      for (int u = units.begin; u < units.end && ok; u += units.step) {
        int m, n, s, k0, k1;
        units.tile(p, u, m, n, s);
        split_range(s, k0, k1);
        const int total = (k1 - k0) * (SEG ? 6 : 1);
        const int per_segment = SEG ? kSegmentSteps : total;
        for (int done = 0; done < total && ok; done += per_segment, ++it) {
          if (it >= 2 && !wait_pair_warp(&bar_acc_free[it & 1], (it / 2 - 1) & 1u, s_abort)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t acc = tmem_base + static_cast<uint32_t>(kTileN) * (it & 1);
          const int count = min(per_segment, total - done);
          for (int i = 0; i < count; ++i, ++step) {
            const int st = step % kStages;
            if (!wait_pair_warp(&bar_full[st], (step / kStages) & 1u, s_abort)) {
              ok = false;
              break;
            }
            tc_fence_after();
            const uint32_t a = smem_u32(smem + st * kStageBytes);
            const uint32_t b = a + kOperandBytes;
            const uint64_t da = smem_desc(a, A_MN ? kOperandBytes / 2 : 16, 1024);
            const uint64_t db = smem_desc(b, B_MN ? kOperandBytes / 2 : 16, 1024);
#pragma unroll
            for (int kk = 0; kk < kBlockK / 16; ++kk) {
              mma_pair_if(leader, acc, desc_add(da, kk * kStepA), desc_add(db, kk * kStepB), idesc, (i > 0 || kk > 0) ? 1u : 0u);
            }
            commit_pair_if(leader, &bar_empty[st]);
          }
          if (ok) commit_pair_if(leader, &bar_acc_ready[it & 1]);
        }
      }
    }
  } else {
    // ===================================================================== epilogue (thread = row)
    const int group = warp >> 2;
    const int gt = tid & (kGroupThreads - 1);
    const uint32_t lane_addr = tmem_base + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    constexpr int kCols = kTileN / kParts;                  // columns of a tile this group works on
    constexpr int kBuffers = 4 / kGroups;                   // staging buffers of a group that stores by TMA
    const int part = group % kParts;
    const int c0 = part * kCols;
    static_assert(kGroups * kCols * 4 <= kBiasBytes, "biases exceed their place");
    float* s_bias = reinterpret_cast<float*>(smem + kOffBias) + group * kCols;
    uint8_t* stage = smem + kOffStore + group * kBuffers * kStoreBytes;
    static_assert(EPI != kEpiStore || kGroups * kBuffers * kStoreBytes <= 4 * kStoreBytes, "staging exceeds its place");
    static_assert(EPI != kEpiGrad || 4 * kGroups * 2048 <= 4 * kStoreBytes, "staging exceeds its place");
    const int bar_id = 1 + group;
    const uint32_t free_addr[2] = {map_to_rank(smem_u32(&bar_acc_free[0]), 0), map_to_rank(smem_u32(&bar_acc_free[1]), 0)};
    int it = 0, boxes = 0;
    bool ok = true;
    auto release = [&](int b) {
      tc_fence_before();
      __syncwarp();
      if (lane == 0) arrive_cluster(free_addr[b]);
    };
    // one 128-byte wide box of 128 rows leaves through the staging buffers: begin (the buffer is free for all
    // threads of the group) -> 16-byte pieces -> end (the store is on its way)
    auto box_begin = [&]() -> uint8_t* {
      if (gt == 0) asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(kBuffers - 1) : "memory");
      group_sync(bar_id);
      return stage + (boxes % kBuffers) * kStoreBytes + gt * 128;
    };
    auto put16 = [&](uint8_t* row_ptr, int piece, uint4 v) {
      *reinterpret_cast<uint4*>(row_ptr + ((piece ^ (gt & 7)) << 4)) = v;
    };
    auto box_end = [&](int x, int y, int z, bool add) {
      fence_proxy_async();
      group_sync(bar_id);
      if (gt == 0) {
        if (y < p.rows) store_box(stage + (boxes % kBuffers) * kStoreBytes, &maps.c, x, y, z, add);
        bulk_commit();       // a box wholly below the matrix is an empty group: box_begin counts groups as boxes
      }
      ++boxes;
    };

    for (int u = units.begin, tile_no = 0; u < units.end && ok; u += units.step, ++tile_no) {
      int m, n, s, k0, k1;
      units.tile(p, u, m, n, s);
      split_range(s, k0, k1);
      const int segments = SEG ? ((k1 - k0) * 6 + kSegmentSteps - 1) / kSegmentSteps : 1;
      if (!SEG && (tile_no & 1) != group / kParts) {
        ++it;
        continue;
      }
      const int row0 = m * kTileM + static_cast<int>(rank) * kHalf;
      const int64_t row = static_cast<int64_t>(row0) + (warp & 3) * 32 + lane;
      const bool live = row < p.rows;
      // what the tile needs beside the scores, requested before the wait
      float scale = 1.0f;
      if (EPI == kEpiStore) {
        if (p.scale != nullptr) scale = *p.scale;
        if (p.scale2 != nullptr) scale *= *p.scale2;
        if (p.grad != nullptr && live) scale = __ldg(p.grad + row);
        if (p.targets != nullptr && live && !isfinite(scale)) {
          // a row that does not count has d = 0 whatever its factor is; 0 x inf must not come of it
          const int64_t t = __ldg(p.targets + row);
          if (t == p.ignore_index || t < 0 || t >= p.vocab) scale = 0.0f;
        }
      }
      int target_col = -1;                                   // kEpiLse: the target's column among this group's
      RowTerms terms{};
      if (EPI != kEpiStore) {
        group_sync(bar_id);                                  // everyone is done with the previous tile's s_bias
        const int64_t first_word = p.v0 + static_cast<int64_t>(n) * kTileN + c0;
        load_bias(p, s_bias, first_word, kCols, gt, kGroupThreads);
        if (EPI == kEpiGrad) terms = row_terms<WEIGHTED>(p, row, first_word);
        if (EPI == kEpiLse && live) {
          const int64_t rel = __ldg(p.targets + row) - first_word;
          if (rel >= 0 && rel < kCols && __ldg(p.targets + row) != p.ignore_index) target_col = static_cast<int>(rel);
        }
      }
      // ---- the accumulator: streamed from TMEM, or drained segment by segment into registers
      float acc[SEG ? kCols : 1];
      if (SEG) {
#pragma unroll
        for (int j = 0; j < kCols; ++j) acc[SEG ? j : 0] = 0.0f;
        for (int sg = 0; sg < segments; ++sg, ++it) {
          ok = group_all(bar_id, wait_pair(&bar_acc_ready[it & 1], (it / 2) & 1u, s_abort));
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int c = 0; c < kCols; c += 16) {              // 16 at a time: the accumulators take most of the registers
            uint32_t v[16];
            tc_ld16_async(lane_addr + kTileN * (it & 1) + c0 + c, v);
            tc_wait_ld();
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              float& a = acc[SEG ? c + j : 0];
              a += __uint_as_float(v[j]);
            }
          }
          release(it & 1);
        }
      } else {
        ok = group_all(bar_id, wait_pair(&bar_acc_ready[it & 1], (it / 2) & 1u, s_abort));
        tc_fence_after();
      }
      if (!ok) break;
      // (group_all above also made s_bias visible to the group)
      const uint32_t acc_addr = lane_addr + kTileN * (it & 1) + c0;
      auto fetch = [&](int c, float (&v)[32]) {              // columns [c, c + 32) of this group's part
        if (SEG) {
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = acc[SEG ? c + j : 0];
        } else {
          uint32_t raw[32];
          tc_ld32_async(acc_addr + c, raw);
          tc_wait_ld();
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(raw[j]);
        }
      };

      if (EPI == kEpiLse) {
        // running maximum and sum over the columns, base 2
        float mx = -INFINITY, sum = 0.0f;
#pragma unroll
        for (int c = 0; c < kCols; c += 32) {
          float y[32];
          fetch(c, y);
          scores_base2(y, s_bias + c);
          float best[4] = {y[0], y[1], y[2], y[3]};
#pragma unroll
          for (int j = 4; j < 32; ++j) best[j & 3] = fmaxf(best[j & 3], y[j]);
          const int hit = target_col - c;
          if (__any_sync(0xffffffffu, hit >= 0 && hit < 32)) {
#pragma unroll
            for (int j = 0; j < 32; ++j) {
              if (hit == j) p.target_score[row] = y[j];
            }
          }
          const float next = fmaxf(fmaxf(mx, fmaxf(best[0], best[1])), fmaxf(best[2], best[3]));
          const float base = next == -INFINITY ? 0.0f : next;   // nothing finite so far: every term is 2^-inf = 0
          const uint64_t shift = pack2(-base, -base);
          uint64_t part[2] = {0ull, 0ull};
#pragma unroll
          for (int j = 0; j < 32; j += 2) {
            float lo, hi;
            unpack2(add2(pack2(y[j], y[j + 1]), shift), lo, hi);
            part[(j >> 1) & 1] = add2(part[(j >> 1) & 1], pack2(exp2_fast(lo), exp2_fast(hi)));
          }
          float lo, hi;
          unpack2(add2(part[0], part[1]), lo, hi);
          sum = fmaf(sum, exp2_fast(mx - base), lo + hi);
          mx = next;
        }
        if (!SEG) release(it & 1);
        if (live) {
          p.partials[(static_cast<int64_t>(n) * kParts + part) * p.rows + row] = make_float2(mx, sum);
        }
      } else if constexpr (EPI == kEpiGrad) {
        // Every warp stages and sends its own 32 rows, 32 columns at a time; no barrier between warps.
        uint8_t* box = smem + kOffStore + warp * 2048;
        const int64_t first_col = static_cast<int64_t>(n) * kTileN + c0;
        const int rows_here = static_cast<int>(max(int64_t(0), min(int64_t(32), p.rows - row + lane)));
        const int64_t panel = p.rows * 64;
        __nv_bfloat16* out = p.d_out + (first_col / 64) * panel + (row - lane) * 64;
        // column sums: one row of them per 32 token rows, added up by a kernel of its own
        float* col_sums = p.bias_partials + (static_cast<int64_t>(m) * 8 + rank * 4 + (warp & 3)) * (static_cast<int64_t>(p.n_tiles) * kTileN) + first_col;
#pragma unroll
        for (int c = 0; c < kCols; c += 32) {
          float d[32];
          fetch(c, d);
          if (!SEG && c + 32 == kCols) release(it & 1);
          score_gradient(d, s_bias + c, terms, c);
          if (SEG && p.bias_partials != nullptr) {
            float v[32];
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = WEIGHTED ? d[j] * terms.g : d[j];
            col_sums[c + lane] = transpose_sum(v, lane);
          }
#pragma unroll
          for (int pl = 0; pl < (SEG ? 3 : 1); ++pl) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              uint32_t w[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                float& lo = d[8 * q + 2 * e];
                float& hi = d[8 * q + 2 * e + 1];
                w[e] = pack_bf16(lo, hi);
                if (SEG) {
                  const __nv_bfloat162 b = *reinterpret_cast<const __nv_bfloat162*>(&w[e]);
                  lo -= __low2float(b);
                  hi -= __high2float(b);
                }
              }
              *reinterpret_cast<uint4*>(box_piece(box, lane, q)) = make_uint4(w[0], w[1], w[2], w[3]);
            }
            __syncwarp();
            __nv_bfloat16* dst = out + (c / 64) * panel + c % 64 + pl * (p.panels * panel);
            if (!SEG && p.bias_partials != nullptr) {
              // Sums of the values as they are stored: they are in the warp's hands there, while sums of the fp32
              // values take a transposition through 31 shuffles.  The roundings (half a bf16 step of each value, either way)
              // are those that dW is made of as well, and average out: db is 1.2e-4 off at 2048 ... 16384 tokens.
              const float2 sums = box_out<true, WEIGHTED>(box, dst, 64, rows_here, lane, terms.g);
              if ((lane & 4) == 0) *reinterpret_cast<float2*>(col_sums + c + box_column(lane)) = sums;
            } else {
              box_out<false>(box, dst, 64, rows_here, lane, 0.0f);
            }
            __syncwarp();
          }
        }
      } else {
        // plain result: fp32 boxes of 32 columns or bf16 boxes of 64; rows and columns beyond the matrix are
        // clipped by the store, boxes wholly beyond it are not sent
        const int limit = static_cast<int>(min(p.cols - static_cast<int64_t>(n) * kTileN, static_cast<int64_t>(kTileN)));
        if (p.store_f32) {
#pragma unroll
          for (int c = 0; c < kCols; c += 32) {
            float d[32];
            fetch(c, d);
            if (!SEG && c + 32 == kCols) release(it & 1);
            if (c0 + c >= limit) continue;
            uint8_t* dst = box_begin();
#pragma unroll
            for (int q = 0; q < 8; ++q) {
              put16(dst, q, make_uint4(__float_as_uint(d[4 * q] * scale), __float_as_uint(d[4 * q + 1] * scale),
                                       __float_as_uint(d[4 * q + 2] * scale), __float_as_uint(d[4 * q + 3] * scale)));
            }
            box_end(n * kTileN + c0 + c, row0, s, p.store_add != 0);
          }
        } else if constexpr (!SEG) {                         // full precision has no bf16 results
#pragma unroll
          for (int c = 0; c < kCols; c += 64) {
            uint32_t w[32];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              float d[32];
              fetch(c + 32 * h, d);
#pragma unroll
              for (int j = 0; j < 16; ++j) w[16 * h + j] = pack_bf16(d[2 * j] * scale, d[2 * j + 1] * scale);
            }
            if (c + 64 == kCols) release(it & 1);
            if (c0 + c >= limit) continue;
            uint8_t* dst = box_begin();
#pragma unroll
            for (int q = 0; q < 8; ++q) put16(dst, q, make_uint4(w[4 * q], w[4 * q + 1], w[4 * q + 2], w[4 * q + 3]));
            box_end(n * kTileN + c0 + c, row0, s, false);
          }
        }
      }
      if (!SEG) ++it;
    }
    if (gt == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }

  let_next_start();                     // (at the start it costs the products 2 %)
  tc_fence_before();
  __syncthreads();
  if (tid == 0 && *s_abort && error_word != nullptr) atomicOr(error_word, kErrBoundedWait);
  cluster_sync();       // neither CTA leaves while the other may still arrive on its barriers or read its tiles
  if (warp == kIssuerWarp) {
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512u) : "memory");
  }
}

}  // namespace pair
}  // namespace grmx
