// Matrix product of CTA pairs (tcgen05 cta_group::2) with a fused epilogue, for the vocabulary loss.
//
//   C[m, n] = sum over planes and k of A[m, k] B[n, k]        256 x 256 per pair of CTAs, fp32 in TMEM
//
// Each CTA of a pair holds 128 rows of A and 128 of the 256 columns of B in shared memory (32 KiB per
// 64-wide k block), and its own 128 rows of the result in TMEM: a pair reads (256 + 256) * 64 values per
// 2 * 256 * 256 * 64 FLOP, half of what a single CTA with a 128 x 256 tile would ask of L2 for its share,
// which is what decides whether the tensor cores are fed.  Persistent pairs; warp 8 loads (TMA ring of
// kStages blocks), warp 9 of the first CTA issues for both, warps 0-7 are the epilogue.  Two accumulators
// of 256 columns: the epilogue of a tile runs under the products of the next one.
//
// Operands are bf16 matrices [planes][rows][cols] read through tensor maps; either may be K-major (k is the
// contiguous index) or MN-major.  Full-precision callers pass their matrices as three bf16 planes whose sum
// is the fp32 value to 24 bits and ask for six plane products (all that matter above 2^-24); the accumulator
// is then drained into registers every kSegmentSteps blocks, so that long sums are rounded by fp32 additions
// and not by the tensor core's accumulation.
//
// Every wait is bounded; a wait that gives up raises the CTA's and its peer's abort flag, and the error word.
#pragma once

#include "common.cuh"
#include "tc_ptx.cuh"

namespace grmx {
namespace pair {

using namespace tc;

constexpr int kTileM = 256;              // rows per pair
constexpr int kTileN = 256;              // columns per pair
constexpr int kHalf = 128;               // rows of A, columns of B and rows of the result per CTA
constexpr int kBlockK = 64;
constexpr int kStages = 5;
constexpr int kOperandBytes = kHalf * kBlockK * 2;       // 16 KiB
constexpr int kStageBytes = 2 * kOperandBytes;
constexpr int kThreads = 320;
constexpr int kLoaderWarp = 8;
constexpr int kIssuerWarp = 9;
constexpr int kGroupThreads = 128;       // an epilogue group: one warp per TMEM lane quadrant
constexpr int kStoreBytes = 16384;       // staging buffer: 128 rows x 128 bytes
constexpr int kOffStore = kStages * kStageBytes;         // [group][2]
constexpr int kOffBias = kOffStore + 4 * kStoreBytes;    // float[2][256]
constexpr int kOffBars = kOffBias + 2 * kTileN * 4;
constexpr int kNumBars = 2 * kStages + 4;
constexpr int kOffMisc = kOffBars + kNumBars * 8;
constexpr int kSmemTotal = kOffMisc + 32;
constexpr int kSmemAlloc = 232448;
static_assert(kSmemTotal <= kSmemAlloc, "shared memory plan exceeds 227 KiB");
static_assert(kOffBars % 8 == 0, "barriers are 8-byte aligned");
// k blocks between two drains of the accumulator in full precision: 32 blocks are 128 accumulations
constexpr int kSegmentSteps = 32;

enum Epilogue { kEpiLse = 0, kEpiGrad = 1, kEpiStore = 2 };

constexpr float kLog2e = 1.4426950408889634f;

struct Params {
  int m_tiles, n_tiles, splits;
  int k_blocks;                // 64-wide blocks of the contraction
  int blocks_per_split;
  int products;                // 1, or 6 plane products per block
  int64_t rows, cols;          // true size of the result
  // loss epilogues: columns are words v0 + n of the vocabulary
  int64_t v0, vocab;
  const void* bias;            // [vocab] or NULL
  int bias_dtype;
  const int64_t* targets;
  int64_t ignore_index;
  // kEpiLse: per row and column tile (times column half in full precision) the maximum and the sum, base 2
  float2* partials;            // [parts][rows]
  float* target_score;         // [rows], base 2
  uint32_t* ticket;            // zeroed for the kernel that follows (or NULL)
  // kEpiGrad
  const float* row_max;        // [rows], base 2
  const float* row_sum;
  const float* grad;           // [rows], or NULL: 1 (a factor that all rows share is applied to the results)
  float* bias_partials;        // [row blocks of 128][n_tiles * 256] or NULL
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
__device__ __forceinline__ void arrive_cluster(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
__device__ __forceinline__ uint32_t try_wait_cluster(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t"
      "}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok;
}
// bounded wait; giving up raises the abort flag of both CTAs
__device__ __forceinline__ bool wait_pair(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  for (uint32_t it = 0; it < kWaitLimit; ++it) {
    if (try_wait_cluster(bar, parity)) return true;
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

// unit of work -> (row tile, column tile, split)
template <int EPI>
__device__ __forceinline__ void unit_to_tile(const Params& p, int u, int& m, int& n, int& s) {
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
    s = 0;
  }
}

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

// SEG: full precision (six plane products, accumulator drained into registers; both epilogue groups work on
// every tile, 128 columns each).  Otherwise the groups take alternate tiles, one accumulator each.
template <int EPI, bool A_MN, bool B_MN, bool SEG>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
pair_gemm_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Params p, uint32_t* error_word) {
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
      mbar_init(&bar_acc_free[i], SEG ? 16 : 8);
    }
    *s_abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (EPI == kEpiLse && blockIdx.x == 0 && tid == 0 && p.ticket != nullptr) *p.ticket = 0u;
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

  const int units = p.m_tiles * p.n_tiles * p.splits;
  const int n_pairs = gridDim.x >> 1;
  const int pair_id = blockIdx.x >> 1;
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
    for (int u = pair_id; u < units && ok; u += n_pairs) {
      int m, n, s, k0, k1;
      unit_to_tile<EPI>(p, u, m, n, s);
      split_range(s, k0, k1);
      const int row = m * kTileM + static_cast<int>(rank) * kHalf;
      const int col = n * kTileN + static_cast<int>(rank) * kHalf;
      for (int kb = k0; kb < k1 && ok; ++kb) {
        for (int pr = 0; pr < (SEG ? 6 : 1); ++pr, ++step) {
          const int st = step % kStages;
          if (step >= kStages && !wait_pair_warp(&bar_empty[st], (step / kStages - 1) & 1u, s_abort)) {
            ok = false;
            break;
          }
          const uint32_t bar = map_to_rank(smem_u32(&bar_full[st]), 0);
          if (rank == 0) mbar_expect_tx_if(leader, &bar_full[st], 2 * kStageBytes);
          uint8_t* a = smem + st * kStageBytes;
          uint8_t* b = a + kOperandBytes;
          const int pa = SEG ? static_cast<int>((kPlaneA >> (2 * pr)) & 3u) : 0;
          const int pb = SEG ? static_cast<int>((kPlaneB >> (2 * pr)) & 3u) : 0;
          const int k = kb * kBlockK;
          if (A_MN) {
            load_box_if(leader, a, &maps.a, bar, row, k, pa);
            load_box_if(leader, a + kOperandBytes / 2, &maps.a, bar, row + 64, k, pa);
          } else {
            load_box_if(leader, a, &maps.a, bar, k, row, pa);
          }
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
      for (int u = pair_id; u < units && ok; u += n_pairs) {
        int m, n, s, k0, k1;
        unit_to_tile<EPI>(p, u, m, n, s);
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
            const uint64_t da = smem_desc(a, A_MN ? kOperandBytes / 2 : 16, 1024);
            const uint64_t db = smem_desc(a + kOperandBytes, B_MN ? kOperandBytes / 2 : 16, 1024);
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
    constexpr int kCols = SEG ? 128 : 256;                  // columns of a tile this group works on
    const int c0 = SEG ? group * kCols : 0;
    float* s_bias = reinterpret_cast<float*>(smem + kOffBias) + group * kTileN;
    uint8_t* stage = smem + kOffStore + group * 2 * kStoreBytes;
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
      if (gt == 0) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
      group_sync(bar_id);
      return stage + (boxes & 1) * kStoreBytes + gt * 128;
    };
    auto put16 = [&](uint8_t* row_ptr, int piece, uint4 v) {
      *reinterpret_cast<uint4*>(row_ptr + ((piece ^ (gt & 7)) << 4)) = v;
    };
    auto box_end = [&](int x, int y, int z, bool add) {
      fence_proxy_async();
      group_sync(bar_id);
      if (gt == 0 && y < p.rows) {                           // a box wholly below the matrix is not sent
        store_box(stage + (boxes & 1) * kStoreBytes, &maps.c, x, y, z, add);
        bulk_commit();
      }
      ++boxes;
    };

    for (int u = pair_id, tile_no = 0; u < units && ok; u += n_pairs, ++tile_no) {
      int m, n, s, k0, k1;
      unit_to_tile<EPI>(p, u, m, n, s);
      split_range(s, k0, k1);
      const int segments = SEG ? ((k1 - k0) * 6 + kSegmentSteps - 1) / kSegmentSteps : 1;
      if (!SEG && (tile_no & 1) != group) {
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
      }
      int target_col = -1;                                   // the target's column in this tile
      float top = 0.0f, coef = 0.0f, g = 0.0f;
      if (EPI != kEpiStore) {
        group_sync(bar_id);                                  // everyone is done with the previous tile's s_bias
        for (int j = gt; j < kTileN; j += kGroupThreads) {
          const int64_t v = p.v0 + static_cast<int64_t>(n) * kTileN + j;
          float b = -INFINITY;                               // no such word
          if (v < p.vocab) {
            b = 0.0f;
            if (p.bias != nullptr) {
              b = p.bias_dtype == GRMX_F32 ? static_cast<const float*>(p.bias)[v]
                                           : __bfloat162float(static_cast<const __nv_bfloat16*>(p.bias)[v]);
            }
          }
          s_bias[j] = b * kLog2e;
        }
        if (live) {
          const int64_t t = p.targets[row];
          const bool counts = t != p.ignore_index && t >= 0 && t < p.vocab;
          const int64_t rel = t - p.v0 - static_cast<int64_t>(n) * kTileN;
          if (counts && rel >= 0 && rel < kTileN) target_col = static_cast<int>(rel);
          if (EPI == kEpiGrad && counts) {
            g = p.grad != nullptr ? p.grad[row] : 1.0f;
            top = p.row_max[row];
            coef = g / p.row_sum[row];
          }
        }
      }
      // ---- the accumulator: streamed from TMEM, or drained segment by segment into registers
      float acc[SEG ? kCols : 1];
      if (SEG) {
        for (int sg = 0; sg < segments; ++sg, ++it) {
          ok = group_all(bar_id, wait_pair(&bar_acc_ready[it & 1], (it / 2) & 1u, s_abort));
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int c = 0; c < kCols; c += 32) {
            uint32_t v[32];
            tc_ld32_async(lane_addr + kTileN * (it & 1) + c0 + c, v);
            tc_wait_ld();
#pragma unroll
            for (int j = 0; j < 32; ++j) acc[(SEG ? c : 0) + (SEG ? j : 0)] = (sg == 0 ? 0.0f : acc[(SEG ? c : 0) + (SEG ? j : 0)]) + __uint_as_float(v[j]);
          }
          release(it & 1);
        }
      } else {
        ok = group_all(bar_id, wait_pair(&bar_acc_ready[it & 1], (it / 2) & 1u, s_abort));
        tc_fence_after();
      }
      if (!ok) break;
      // (group_all above also made s_bias visible to the group)
      const uint32_t acc_addr = lane_addr + kTileN * (it & 1);
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
        // running maximum and sum over the columns, base 2: y = score * log2 e + bias * log2 e
        float mx = -INFINITY, sum = 0.0f;
#pragma unroll
        for (int c = 0; c < kCols; c += 32) {
          float y[32];
          fetch(c, y);
          float best = -INFINITY;
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            y[j] = fmaf(y[j], kLog2e, s_bias[c0 + c + j]);
            best = fmaxf(best, y[j]);
          }
          const int hit = target_col - c0 - c;
          if (__any_sync(0xffffffffu, hit >= 0 && hit < 32)) {
#pragma unroll
            for (int j = 0; j < 32; ++j) {
              if (hit == j) p.target_score[row] = y[j];
            }
          }
          const float next = fmaxf(mx, best);
          const float base = next == -INFINITY ? 0.0f : next;   // nothing finite so far: every term is 2^-inf = 0
          float part = 0.0f;
#pragma unroll
          for (int j = 0; j < 32; ++j) part += exp2_fast(y[j] - base);
          sum = sum * exp2_fast(mx - base) + part;
          mx = next;
        }
        if (!SEG) release(it & 1);
        if (live) {
          const int64_t part = SEG ? 2 * static_cast<int64_t>(n) + group : n;
          p.partials[part * p.rows + row] = make_float2(mx, sum);
        }
      } else if (EPI == kEpiGrad) {
        // d = g * (2^(y - top) / sum - [target]); ignored rows have g = coef = 0 and are written as zeros
        const bool counts = coef != 0.0f || g != 0.0f;
        constexpr int nplanes = SEG ? 3 : 1;
#pragma unroll
        for (int c = 0; c < kCols; c += 64) {
          float d[64];
#pragma unroll
          for (int h = 0; h < 64; h += 32) {
            float y[32];
            fetch(c + h, y);
#pragma unroll
            for (int j = 0; j < 32; ++j) {
              const float e = exp2_fast(fmaf(y[j], kLog2e, s_bias[c0 + c + h + j]) - top);
              d[h + j] = counts ? e * coef : 0.0f;
            }
            const int hit = target_col - c0 - c - h;
            if (__any_sync(0xffffffffu, hit >= 0 && hit < 32)) {
#pragma unroll
              for (int j = 0; j < 32; ++j) {
                if (hit == j) d[h + j] -= g;
              }
            }
            if (p.bias_partials != nullptr) {
              float v[32];
#pragma unroll
              for (int j = 0; j < 32; ++j) v[j] = d[h + j];
              const float total = transpose_sum(v, lane);
              // one row of sums per 32 token rows; the reduction over them follows in a kernel of its own
              const int64_t block = static_cast<int64_t>(m) * 8 + rank * 4 + (warp & 3);
              p.bias_partials[block * (static_cast<int64_t>(p.n_tiles) * kTileN) + static_cast<int64_t>(n) * kTileN + c0 + c + h + lane] = total;
            }
          }
          if (!SEG && c + 64 == kCols) release(it & 1);
#pragma unroll
          for (int pl = 0; pl < nplanes; ++pl) {
            uint8_t* dst = box_begin();
#pragma unroll
            for (int q = 0; q < 8; ++q) {
              uint32_t w[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const int j = 8 * q + 2 * e;
                w[e] = pack_bf16(d[j], d[j + 1]);
                if (SEG) {
                  const __nv_bfloat162 b = *reinterpret_cast<const __nv_bfloat162*>(&w[e]);
                  d[j] -= __low2float(b);
                  d[j + 1] -= __high2float(b);
                }
              }
              put16(dst, q, make_uint4(w[0], w[1], w[2], w[3]));
            }
            box_end(n * kTileN + c0 + c, row0, pl, false);
          }
        }
      } else {
        // plain result: fp32 boxes of 32 columns or bf16 boxes of 64; rows and columns beyond the matrix are
        // clipped by the store, boxes wholly beyond it are not sent
        const int limit = static_cast<int>(min(p.cols - static_cast<int64_t>(n) * kTileN, static_cast<int64_t>(kTileN)));
#pragma unroll
        for (int c = 0; c < kCols; c += 64) {
          float d[64];
#pragma unroll
          for (int h = 0; h < 64; h += 32) {
            float y[32];
            fetch(c + h, y);
#pragma unroll
            for (int j = 0; j < 32; ++j) d[h + j] = y[j] * scale;
          }
          if (!SEG && c + 64 == kCols) release(it & 1);
          if (c0 + c >= limit) continue;
          if (p.store_f32) {
#pragma unroll
            for (int h = 0; h < 64; h += 32) {
              if (c0 + c + h >= limit) continue;
              uint8_t* dst = box_begin();
#pragma unroll
              for (int q = 0; q < 8; ++q) {
                put16(dst, q, make_uint4(__float_as_uint(d[h + 4 * q]), __float_as_uint(d[h + 4 * q + 1]),
                                         __float_as_uint(d[h + 4 * q + 2]), __float_as_uint(d[h + 4 * q + 3])));
              }
              box_end(n * kTileN + c0 + c + h, row0, s, p.store_add != 0);
            }
          } else {
            uint8_t* dst = box_begin();
#pragma unroll
            for (int q = 0; q < 8; ++q) {
              put16(dst, q, make_uint4(pack_bf16(d[8 * q], d[8 * q + 1]), pack_bf16(d[8 * q + 2], d[8 * q + 3]),
                                       pack_bf16(d[8 * q + 4], d[8 * q + 5]), pack_bf16(d[8 * q + 6], d[8 * q + 7])));
            }
            box_end(n * kTileN + c0 + c, row0, s, false);
          }
        }
      }
      if (!SEG) ++it;
    }
    if (gt == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }

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
