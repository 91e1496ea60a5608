// Softmax cross entropy of a vocabulary projection, with its gradient, without keeping the scores.
//
//   y_ij = x_i . W_j + b_j     lse_i = log sum_j exp(y_ij)     loss_i = lse_i - y_{i,t_i}
//   d_ij = g_i (exp(y_ij - lse_i) - [j = t_i])     dx = d W     dW = d^T x     db_j = sum_i d_ij
//
// Forward: one product x W^T whose epilogue reduces every 256-column tile of scores to a maximum and a sum
// per row (base 2), and one small kernel that joins the tiles' pairs and adds the rows up.  Backward: the
// vocabulary in pieces; for each piece the scores once more, their epilogue writing d (bf16, or three bf16
// planes in full precision) to a workspace, then the two products that read it.  8 N V D FLOP in all, of
// which 2 N V D are the scores computed a second time because they are not kept.
//
// Bound by the tensor cores at training sizes, by the stream of W where a few tokens are scored.  16384 tokens x 512
// x 32768 words, bf16, cool / back to back (then the card is at its power limit): scores and their maxima 350 / 400 us
// (1.57 PFLOP/s cool, 0.95 of cuBLAS's burst), gradient of the scores 519 / 595, dx 355 / 450, dW 375 / 475.  The gradient
// kernel is bound by its epilogue: 110 us of it go when nothing is stored (1 GB), 30 each for exponentials and column sums.
// The maximum and the sum are kept apart (never as one log-sum-exp): exp(y - max) / sum then carries no
// rounding of a sum that is as large as the scores, and a target that is the maximum itself leaves exactly
// log(sum) as its loss.
//
// Roundings below fp32, all of them of bf16 inputs (full precision has none): d is held in bf16, half a step (2^-8 of itself
// or less) each, because it is an operand of two bf16 products and a gigabyte as it is; with a factor per token, x times its
// factor is rounded once more for dW, because d (p - [target], whose -1 is exact) must not carry the factor.  Against 64
// bits dx and dW are then 1.66e-3 off where fp32 scores' gradients give 1.65e-3 (16384 x 512 x 32768; most of both is
// the rounding of the result to bf16), dW with a factor per token 2.1e-3 to 2.4e-3.  bf16 sums over the whole contraction stay in the
// tensor core's fp32 accumulator; full precision drains it (kSegmentSteps).
#include <cuda.h>

#include <cstring>
#include <mutex>

#include "pair_gemm.cuh"

namespace grmx {
namespace {

using namespace pair;

constexpr float kLn2 = 0.6931471805599453f;

inline int64_t round_up(int64_t a, int64_t b) { return (a + b - 1) / b * b; }
inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// ------------------------------------------------------------------ operands as bf16 planes

// [rows, cols] fp32 or bf16 -> planes of bf16 whose sum is the value (one plane for bf16: a copy with a pitch
// that a tensor map can take).  x = h + m + l with h = bf16(x), m = bf16(x - h), l = bf16(x - h - m): 24 bits.
// Values that are not finite stay whole in the first plane.  With targets the rows are tokens: one that does not
// count becomes zeros (whatever it holds), the others are multiplied by grad[row] if there is such a factor.
struct TokenRows {
  const int64_t* targets;      // NULL: plain rows
  int64_t ignore_index, vocab;
  const float* grad;           // [rows] or NULL
};
template <typename T, int PLANES>
__global__ void __launch_bounds__(256) planes_kernel(const T* __restrict__ src, __nv_bfloat16* __restrict__ dst, int64_t rows,
                                                     int cols, int ld, int64_t plane_stride, TokenRows tokens) {
  let_next_start();
  wait_for_previous();
  const int64_t pairs = ld / 2;
  const int64_t total = rows * pairs;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < total; i += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t r = i / pairs;
    const int c = static_cast<int>(i - r * pairs) * 2;
    float v[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) v[e] = c + e < cols ? to_float<T>(src[r * cols + c + e]) : 0.0f;
    if (tokens.targets != nullptr) {
      const int64_t t = __ldg(tokens.targets + r);
      const bool counts = t != tokens.ignore_index && t >= 0 && t < tokens.vocab;
      const float factor = tokens.grad != nullptr ? __ldg(tokens.grad + r) : 1.0f;
#pragma unroll
      for (int e = 0; e < 2; ++e) v[e] = counts ? v[e] * factor : 0.0f;
    }
#pragma unroll
    for (int pl = 0; pl < PLANES; ++pl) {
      __nv_bfloat162 b;
      b.x = __float2bfloat16_rn(v[0]);
      b.y = __float2bfloat16_rn(v[1]);
      *reinterpret_cast<__nv_bfloat162*>(dst + pl * plane_stride + r * ld + c) = b;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float rest = v[e] - __bfloat162float(e == 0 ? b.x : b.y);
        v[e] = isfinite(rest) ? rest : 0.0f;
      }
    }
  }
}

struct Operand {
  const void* ptr;
  int64_t ld, plane_stride;
  int planes;
};

bool readable_in_place(const void* ptr, int64_t cols, int dtype) {
  return dtype == GRMX_BF16 && cols % 8 == 0 && (reinterpret_cast<uintptr_t>(ptr) & 15u) == 0;
}
// By the width alone: a workspace is sized before the pointers are known, and has room for the copy of a
// misaligned matrix too.
int64_t operand_bytes(int64_t rows, int64_t cols, int dtype) {
  return (dtype == GRMX_F32 ? 3 : 1) * round_up(rows * round_up(cols, 8) * 2, 256);
}

// Always a copy, in planes, at dst (operand_bytes of it).
int copy_operand(Operand* out, const void* src, int64_t rows, int64_t cols, int dtype, uint8_t* dst, const TokenRows& tokens,
                 cudaStream_t s) {
  const int64_t ld = round_up(cols, 8);
  const int planes = dtype == GRMX_F32 ? 3 : 1;
  const int64_t stride = operand_bytes(rows, cols, dtype) / planes / 2;
  const int64_t blocks = ceil_div(rows * (ld / 2), 256);
  const unsigned grid = static_cast<unsigned>(blocks < 148 * 16 ? blocks : 148 * 16);
  __nv_bfloat16* d = reinterpret_cast<__nv_bfloat16*>(dst);
  if (dtype == GRMX_F32) {
    launch_after(planes_kernel<float, 3>, grid, 1, 256, 0, s, static_cast<const float*>(src), d, rows, static_cast<int>(cols),
                                                  static_cast<int>(ld), stride, tokens);
  } else {
    launch_after(planes_kernel<__nv_bfloat16, 1>, grid, 1, 256, 0, s, static_cast<const __nv_bfloat16*>(src), d, rows,
                                                          static_cast<int>(cols), static_cast<int>(ld), stride, tokens);
  }
  *out = Operand{dst, ld, stride, planes};
  return check_launch("loss operand planes");
}
// The matrix as it is where a tensor map can read it, otherwise a copy.
int make_operand(Operand* out, const void* src, int64_t rows, int64_t cols, int dtype, uint8_t* dst, cudaStream_t s) {
  if (readable_in_place(src, cols, dtype)) {
    *out = Operand{src, cols, rows * cols, 1};
    return GRMX_OK;
  }
  return copy_operand(out, src, rows, cols, dtype, dst, TokenRows{nullptr, 0, 0, nullptr}, s);
}

// ------------------------------------------------------------------ a few tokens

__device__ __forceinline__ float bias_of(const void* bias, int dtype, int64_t word) {
  return dtype == GRMX_F32 ? static_cast<const float*>(bias)[word] : __bfloat162float(static_cast<const __nv_bfloat16*>(bias)[word]);
}

// two (maximum, sum of 2^(score - maximum)) pairs into one
__device__ __forceinline__ float2 join(float2 a, float2 b) {
  const float next = fmaxf(a.x, b.x);
  const float base = next == -INFINITY ? 0.0f : next;       // neither has a finite score
  return make_float2(next, a.y * exp2_fast(a.x - base) + b.y * exp2_fast(b.x - base));
}

// Up to eight tokens (a decoding step): bound by the stream of W, one pass over it with plain fused multiply-adds.
// A warp takes ROWS words at a time, a lane 32 bytes of each; the tokens' features wait in shared memory.  The lanes' sums
// are exchanged so that every lane ends up with the score of one (word, token) and keeps that pair's running maximum and
// sum; lanes, warps and (in loss_join_kernel) CTAs are joined at the end.
// One token, 512 x 32768 bf16: 21 us as a padded tile of the product, 11.5 us so (2.9 TB/s).  Bound by latency: at 100 registers
// two CTAs fit an SM, so the 512 CTAs come in two rounds and nothing is in flight between them; with four or eight bf16
// tokens (201 and 156 registers) one fits.  Calls of 1, 2, 4 and 8 tokens: 13, 13, 18 and 29 us in bf16; of 1 and 8 in fp32
// 17 and 24 us.
constexpr int kFewTokens = 8;
constexpr int kFewThreads = 256;
constexpr int kFewShared = 160 * 1024;       // most shared memory for the tokens' features

// sum of each of M values over the lanes; lane l returns that of value l / (32 / M)
template <int M>
__device__ __forceinline__ float spread_sums(float (&v)[M], int lane) {
  int width = M;
#pragma unroll
  for (int half = 16; half >= 1; half >>= 1) {
    if (width > 1) {
      const bool upper = (lane & half) != 0;
      width >>= 1;
#pragma unroll
      for (int j = 0; j < M / 2; ++j) {
        if (j < width) {
          const float keep = upper ? v[j + width] : v[j];
          const float give = upper ? v[j] : v[j + width];
          v[j] = keep + __shfl_xor_sync(0xffffffffu, give, half);
        }
      }
    } else {
      v[0] += __shfl_xor_sync(0xffffffffu, v[0], half);
    }
  }
  return v[0];
}

// 16 bytes of features: whole where they are all there, value by value at a row's end or off a 16-byte boundary
template <typename T>
__device__ __forceinline__ uint4 load_features(const T* row, int d, int D, bool aligned) {
  constexpr int G = 16 / sizeof(T);
  if (aligned && d + G <= D) return __ldcs(reinterpret_cast<const uint4*>(row + d));
  union { T v[G]; uint4 q; } u;
#pragma unroll
  for (int e = 0; e < G; ++e) u.v[e] = d + e < D ? row[d + e] : from_float<T>(0.0f);
  return u.q;
}
template <typename T>
__device__ __forceinline__ void widen(uint4 q, float (&x)[16 / sizeof(T)]) {
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if constexpr (sizeof(T) == 2) {
      x[2 * e] = __uint_as_float(w[e] << 16);
      x[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
    } else {
      x[e] = __uint_as_float(w[e]);
    }
  }
}

template <typename T, int TOKENS, int ROWS>
__global__ void __launch_bounds__(kFewThreads)
few_tokens_kernel(const T* __restrict__ hidden, const T* __restrict__ weight, const void* __restrict__ bias, int bias_dtype,
                  const int64_t* __restrict__ targets, int64_t ignore_index, int tokens, int D, int64_t V, int aligned,
                  float2* __restrict__ partials, float* __restrict__ target_score, uint32_t* ticket) {
  constexpr int G = 16 / static_cast<int>(sizeof(T)), kChunk = 64 * G;       // features per piece, and per chunk of two pieces
  constexpr int M = TOKENS * ROWS, kLanesPer = 32 / M;
  static_assert(M <= 32, "a lane holds one (word, token)");
  extern __shared__ float s_x[];                           // [TOKENS][D rounded up to whole chunks], zero beyond D
  __shared__ float2 s_part[kFewThreads / 32][TOKENS];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int pitch = (D + kChunk - 1) / kChunk * kChunk;
  const int64_t step = static_cast<int64_t>(gridDim.x) * (kFewThreads / 32) * ROWS;
  int64_t v0 = (static_cast<int64_t>(blockIdx.x) * (kFewThreads / 32) + warp) * ROWS;
  uint4 raw[ROWS][2];
  auto load = [&](int64_t first, int d0) {
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const T* row = weight + (first + r < V ? first + r : V - 1) * D;       // words beyond the last are not counted below
#pragma unroll
      for (int h = 0; h < 2; ++h) raw[r][h] = load_features(row, d0 + (h * 32 + lane) * G, D, aligned != 0);
    }
  };
  let_next_start();
  wait_for_previous();
  load(v0, 0);                                             // on its way while the tokens are staged
  if (blockIdx.x == 0 && threadIdx.x == 0) *ticket = 0u;
  for (int i = threadIdx.x; i < TOKENS * pitch; i += kFewThreads) {
    const int t = i / pitch, d = i - t * pitch;
    s_x[i] = t < tokens && d < D ? to_float<T>(hidden[static_cast<int64_t>(t) * D + d]) : 0.0f;
  }
  const int mine = lane / kLanesPer, my_row = mine / TOKENS, my_token = mine % TOKENS;
  int64_t my_target = -1;
  if (my_token < tokens) {
    const int64_t t = targets[my_token];
    if (t != ignore_index) my_target = t;
  }
  __syncthreads();
  float2 all = make_float2(-INFINITY, 0.0f);
  for (bool loaded = true; v0 < V; v0 += step) {
    const int64_t v = v0 + my_row;
    const float b = bias != nullptr && v < V ? bias_of(bias, bias_dtype, v) : 0.0f;
    float acc[M];
#pragma unroll
    for (int i = 0; i < M; ++i) acc[i] = 0.0f;
    for (int d0 = 0; d0 < D; d0 += kChunk) {
      if (!loaded) load(v0, d0);
      loaded = false;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float w[ROWS][G];
#pragma unroll
        for (int r = 0; r < ROWS; ++r) widen<T>(raw[r][h], w[r]);
#pragma unroll
        for (int t = 0; t < TOKENS; ++t) {
#pragma unroll
          for (int e = 0; e < G; e += 4) {
            const float4 x = *reinterpret_cast<const float4*>(s_x + t * pitch + d0 + (h * 32 + lane) * G + e);
#pragma unroll
            for (int r = 0; r < ROWS; ++r) {
              float& a = acc[r * TOKENS + t];
              a = fmaf(x.x, w[r][e], a);
              a = fmaf(x.y, w[r][e + 1], a);
              a = fmaf(x.z, w[r][e + 2], a);
              a = fmaf(x.w, w[r][e + 3], a);
            }
          }
        }
      }
    }
    const float y = fmaf(spread_sums<M>(acc, lane), kLog2e, bias_base2(b));
    if (v < V) {
      if (v == my_target && lane % kLanesPer == 0) target_score[my_token] = y;
      const float next = fmaxf(all.x, y);
      const float base = next == -INFINITY ? 0.0f : next;
      all = make_float2(next, fmaf(all.y, exp2_fast(all.x - base), exp2_fast(y - base)));
    }
  }
  // lanes with the same token (other words), then warps
#pragma unroll
  for (int o = kLanesPer * TOKENS; o < 32; o <<= 1) {
    all = join(all, make_float2(__shfl_xor_sync(0xffffffffu, all.x, o), __shfl_xor_sync(0xffffffffu, all.y, o)));
  }
  if (my_row == 0 && lane % kLanesPer == 0) s_part[warp][my_token] = all;
  __syncthreads();
  if (threadIdx.x < tokens) {
    float2 sum = s_part[0][threadIdx.x];
    for (int i = 1; i < kFewThreads / 32; ++i) sum = join(sum, s_part[i][threadIdx.x]);
    partials[static_cast<int64_t>(blockIdx.x) * tokens + threadIdx.x] = sum;
  }
}

constexpr int kFewRows = 8;                                // words at a time per warp (4 with eight tokens)
// (more than are resident: what is left over starts where a CTA ends)
int few_tokens_blocks(int64_t V) {
  const int64_t need = (V + kFewThreads / 32 * kFewRows - 1) / (kFewThreads / 32 * kFewRows);
  return static_cast<int>(need < 4 * 148 ? need : 4 * 148);
}

template <typename T>
int launch_few_tokens(const void* hidden, const void* weight, const void* bias, int bias_dtype, const int64_t* targets,
                      int64_t ignore_index, int tokens, int D, int64_t V, float2* partials, float* target_score,
                      uint32_t* ticket, cudaStream_t s) {
  constexpr int kChunk = 1024 / static_cast<int>(sizeof(T));
  const int padded = tokens <= 1 ? 1 : tokens <= 2 ? 2 : tokens <= 4 ? 4 : 8;
  const int smem = padded * ((D + kChunk - 1) / kChunk * kChunk) * 4;
  const int aligned = D % (16 / static_cast<int>(sizeof(T))) == 0 && (reinterpret_cast<uintptr_t>(weight) & 15u) == 0;
  auto kernel = padded == 1   ? few_tokens_kernel<T, 1, kFewRows>
                : padded == 2 ? few_tokens_kernel<T, 2, kFewRows>
                : padded == 4 ? few_tokens_kernel<T, 4, kFewRows>
                              : few_tokens_kernel<T, 8, 4>;
  // always the same size: a limit of this call's own could be lowered by another thread's call before the launch below
  if (smem > 40 * 1024 && cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kFewShared) != cudaSuccess) {
    return fail(GRMX_ERR_LAUNCH, "loss of a few tokens: cannot reserve %d bytes of shared memory: %s", kFewShared, cudaGetErrorString(cudaGetLastError()));
  }
  launch_after(kernel, few_tokens_blocks(V), 1, kFewThreads, smem, s, static_cast<const T*>(hidden), static_cast<const T*>(weight), bias, bias_dtype,
                                                         targets, ignore_index, tokens, D, V, aligned, partials, target_score, ticket);
  return check_launch("loss of a few tokens");
}

// few enough tokens, and their features fit in shared memory
bool takes_few_tokens(int64_t N, int64_t D) { return N <= kFewTokens && (D + 511) / 512 * 512 * kFewTokens * 4 <= kFewShared; }

// ------------------------------------------------------------------ joining the tiles' maxima and sums

constexpr int kJoinThreads = 256;

// partials [parts][rows] -> maximum, sum and loss per row, ROWS rows per block; with a reduction, the blocks' sums are
// added up by the block that finishes last, always in the same order.
template <int ROWS>
__global__ void __launch_bounds__(kJoinThreads)
loss_join_kernel(const float2* __restrict__ partials, const float* __restrict__ target_score, const void* bias, int bias_dtype,
                 const int64_t* __restrict__ targets, int64_t ignore_index, int64_t vocab, int64_t rows, int parts,
                 int reduction, float* __restrict__ row_max, float* __restrict__ row_sum, float* __restrict__ loss,
                 float* __restrict__ inv_count, double* __restrict__ block_loss, int* __restrict__ block_count,
                 uint32_t* ticket, uint32_t* error_word) {
  constexpr int kSlices = kJoinThreads / ROWS;
  __shared__ float2 s_part[kSlices][ROWS];
  __shared__ double s_loss[kJoinThreads];
  __shared__ int s_count[kJoinThreads];
  __shared__ bool s_last;
  let_next_start();
  wait_for_previous();
  const int r = threadIdx.x % ROWS, slice = threadIdx.x / ROWS;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * ROWS + r;
  float2 all = make_float2(-INFINITY, 0.0f);
  if (row < rows) {
    const float2* src = partials + row;
    int i = slice;
    for (; i + 3 * kSlices < parts; i += 4 * kSlices) {
      float2 q[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) q[e] = src[static_cast<int64_t>(i + e * kSlices) * rows];
#pragma unroll
      for (int e = 0; e < 4; ++e) all = join(all, q[e]);
    }
    for (; i < parts; i += kSlices) all = join(all, src[static_cast<int64_t>(i) * rows]);
  }
  s_part[slice][r] = all;
  __syncthreads();
#pragma unroll
  for (int o = kSlices / 2; o > 0; o >>= 1) {
    if (slice < o) s_part[slice][r] = join(s_part[slice][r], s_part[slice + o][r]);
    __syncthreads();
  }
  float value = 0.0f;
  int counted = 0;
  if (slice == 0 && row < rows) {
    const float mx = s_part[0][r].x;
    float sum = s_part[0][r].y;
    if (mx == -INFINITY) sum = __int_as_float(0x7fc00000);    // every word masked: no distribution
    row_max[row] = mx;
    row_sum[row] = sum;
    const int64_t t = targets[row];
    if (t != ignore_index) {
      if (t >= 0 && t < vocab) {
        const float below = mx - target_score[row];
        value = (below + log2f(sum)) * kLn2;
        // a target masked with the type's lowest value, whose score in base 2 is not the whole of it: beside the mask the
        // score itself vanishes
        if (below > 1e38f && bias != nullptr) value = (mx + log2f(sum)) * kLn2 - bias_of(bias, bias_dtype, t);
        counted = 1;
      } else if (error_word != nullptr) {
        atomicOr(error_word, kErrTarget);
      }
    }
    if (reduction == GRMX_REDUCE_NONE) loss[row] = value;
  }
  if (reduction == GRMX_REDUCE_NONE) return;
  s_loss[threadIdx.x] = value;
  s_count[threadIdx.x] = counted;
  __syncthreads();
  if (threadIdx.x == 0) {
    double v = 0.0;
    int n = 0;
    for (int i = 0; i < ROWS; ++i) {
      v += s_loss[i];
      n += s_count[i];
    }
    block_loss[blockIdx.x] = v;
    block_count[blockIdx.x] = n;
    __threadfence();
    s_last = atomicAdd(ticket, 1u) == gridDim.x - 1;
  }
  __syncthreads();
  if (!s_last) return;
  __threadfence();
  double v = 0.0;
  int n = 0;
  for (unsigned i = threadIdx.x; i < gridDim.x; i += kJoinThreads) {
    v += __ldcg(block_loss + i);
    n += __ldcg(block_count + i);
  }
  s_loss[threadIdx.x] = v;
  s_count[threadIdx.x] = n;
  __syncthreads();
  for (int o = kJoinThreads / 2; o > 0; o >>= 1) {
    if (threadIdx.x < o) {
      s_loss[threadIdx.x] += s_loss[threadIdx.x + o];
      s_count[threadIdx.x] += s_count[threadIdx.x + o];
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    const double count = s_count[0];
    // no token counts: the mean is 0 / 0, as of an empty list, and no row has a gradient
    *loss = static_cast<float>(reduction == GRMX_REDUCE_MEAN ? s_loss[0] / count : s_loss[0]);
    *inv_count = reduction == GRMX_REDUCE_MEAN ? (count > 0.0 ? static_cast<float>(1.0 / count) : 0.0f) : 1.0f;
  }
}

// rows per block: whole lines of the partials where there are rows enough for all SMs, more slices where not
int join_rows(int64_t N) { return N >= 16384 ? 32 : N >= 512 ? 8 : 1; }

// ------------------------------------------------------------------ sums of partial results

// out[r, c] = sum over s of part[s][r][c]   (part pitch ld, out dense), VEC columns per thread
template <typename T, int VEC>
__global__ void __launch_bounds__(256) sum_splits_kernel(const float* __restrict__ part, T* __restrict__ out, int64_t rows,
                                                         int cols, int ld, int64_t split_stride, int splits) {
  let_next_start();
  wait_for_previous();
  const int per_row = cols / VEC;
  const int64_t total = rows * per_row;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < total; i += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t r = i / per_row;
    const int c = static_cast<int>(i - r * per_row) * VEC;
    const float* src = part + r * ld + c;
    float v[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = 0.0f;
    for (int s = 0; s < splits; ++s) {
      if (VEC == 4) {
        const float4 q = __ldcs(reinterpret_cast<const float4*>(src + s * split_stride));
        v[0] += q.x;
        if (VEC > 1) { v[1 % VEC] += q.y; v[2 % VEC] += q.z; v[3 % VEC] += q.w; }
      } else {
        v[0] += src[s * split_stride];
      }
    }
    if (VEC == 4 && sizeof(T) == 2) {
      *reinterpret_cast<uint2*>(out + r * cols + c) = make_uint2(pack_bf16(v[0], v[1 % VEC]), pack_bf16(v[2 % VEC], v[3 % VEC]));
    } else if (VEC == 4) {
      *reinterpret_cast<float4*>(out + r * cols + c) = make_float4(v[0], v[1 % VEC], v[2 % VEC], v[3 % VEC]);
    } else {
      out[r * cols + c] = from_float<T>(v[0]);
    }
  }
}

int launch_sum_splits(const float* part, void* out, int64_t rows, int64_t cols, int64_t ld, int64_t split_stride, int splits,
                      int dtype, cudaStream_t s) {
  const bool vec = cols % 4 == 0 && (reinterpret_cast<uintptr_t>(out) & 15u) == 0;
  const int64_t blocks = ceil_div(rows * cols, vec ? 1024 : 256);
  const unsigned grid = static_cast<unsigned>(blocks < 148 * 16 ? blocks : 148 * 16);
  const int c = static_cast<int>(cols), l = static_cast<int>(ld);
  if (dtype == GRMX_F32) {
    if (vec) launch_after(sum_splits_kernel<float, 4>, grid, 1, 256, 0, s, part, static_cast<float*>(out), rows, c, l, split_stride, splits);
    else launch_after(sum_splits_kernel<float, 1>, grid, 1, 256, 0, s, part, static_cast<float*>(out), rows, c, l, split_stride, splits);
  } else {
    __nv_bfloat16* o = static_cast<__nv_bfloat16*>(out);
    if (vec) launch_after(sum_splits_kernel<__nv_bfloat16, 4>, grid, 1, 256, 0, s, part, o, rows, c, l, split_stride, splits);
    else launch_after(sum_splits_kernel<__nv_bfloat16, 1>, grid, 1, 256, 0, s, part, o, rows, c, l, split_stride, splits);
  }
  return check_launch("loss split sums");
}

// db[v0 + c] = sum over the blocks of 32 token rows; 32 columns x 8 slices per block, slices joined in order
template <typename T>
__global__ void __launch_bounds__(256) bias_sum_kernel(const float* __restrict__ partials, int64_t blocks, int64_t pitch,
                                                       int64_t cols, const float* scale, const float* scale2,
                                                       T* __restrict__ out) {
  __shared__ float s_sum[8][32];
  let_next_start();
  wait_for_previous();
  const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + lane;
  float sum = 0.0f;
  for (int64_t b = slice; b < blocks; b += 8) sum += partials[b * pitch + c];   // the pitch covers whole tiles
  s_sum[slice][lane] = sum;
  __syncthreads();
  if (slice == 0 && c < cols) {
    for (int i = 1; i < 8; ++i) sum += s_sum[i][lane];
    if (scale != nullptr) sum *= *scale;
    if (scale2 != nullptr) sum *= *scale2;
    out[c] = from_float<T>(sum);
  }
}

// ------------------------------------------------------------------ launches

int pairs_on_device() {
  static std::mutex mutex;
  static int cached[64] = {0};
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess || device < 0 || device >= 64) return 74;
  std::lock_guard<std::mutex> lock(mutex);
  if (cached[device] == 0) {
    int sms = 0;
    if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device) != cudaSuccess || sms < 2) sms = 148;
    cached[device] = sms / 2;
  }
  return cached[device];
}

template <int EPI, bool A_MN, bool B_MN, bool SEG, bool WEIGHTED = false>
int launch_pair(const Maps& maps, const Params& p, const char* what, cudaStream_t s) {
  auto kernel = pair_gemm_kernel<EPI, A_MN, B_MN, SEG, WEIGHTED>;
  static std::mutex mutex;
  static bool configured[64] = {false};
  int device = 0;
  cudaGetDevice(&device);
  {
    std::lock_guard<std::mutex> lock(mutex);
    if (device < 0 || device >= 64 || !configured[device]) {
      const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemAlloc);
      if (e != cudaSuccess) {
        cudaGetLastError();
        return fail(GRMX_ERR_LAUNCH, "%s: cannot reserve %d bytes of shared memory: %s", what, kSmemAlloc, cudaGetErrorString(e));
      }
      if (device >= 0 && device < 64) configured[device] = true;
    }
  }
  const int64_t units = static_cast<int64_t>(p.m_tiles) * p.n_tiles * p.splits;
  const int pairs = pairs_on_device();
  const unsigned grid = 2u * static_cast<unsigned>(units < pairs ? units : pairs);
  launch_after(kernel, grid, 1, threads_of(EPI, SEG), kSmemAlloc, s, maps, p, device_error_word_ptr());
  return check_launch(what);
}

// the products whose epilogue works on scores
template <int EPI>
int launch_scores(const Maps& maps, const Params& p, int dtype, const char* what, cudaStream_t s) {
  if (EPI == kEpiGrad && p.grad != nullptr) {
    return dtype == GRMX_F32 ? launch_pair<EPI, false, false, true, EPI == kEpiGrad>(maps, p, what, s)
                             : launch_pair<EPI, false, false, false, EPI == kEpiGrad>(maps, p, what, s);
  }
  if (dtype == GRMX_F32) return launch_pair<EPI, false, false, true>(maps, p, what, s);
  return launch_pair<EPI, false, false, false>(maps, p, what, s);
}

// A K-major operand tile is one box of 64 k x 128 rows; an MN-major one is two boxes of 64 columns x 64 k.
bool operand_map(CUtensorMap* map, const Operand& o, int64_t rows, int64_t cols, bool mn_major) {
  return make_matrix_map(map, o.ptr, false, o.planes, rows, cols, o.ld, o.plane_stride, 64, mn_major ? 64 : 128);
}

constexpr int64_t kMostSplits = 64;
// How many parts the contraction of an [m_tiles x n_tiles] result is cut into so that the pairs are busy to the
// end: waves of blocks (0.29 us per 256 x 256 x 64 block and plane product, measured) against writing and
// reading one more fp32 copy of the result (about 5 TB/s).
int choose_splits(int64_t tiles, int64_t k_blocks, int64_t result_elems, int products, int pairs) {
  int best = 1;
  double best_cost = 1e30;
  const int64_t most = k_blocks < kMostSplits ? k_blocks : kMostSplits;
  for (int64_t s = 1; s <= most; ++s) {
    const int64_t per = ceil_div(k_blocks, s);
    if (ceil_div(k_blocks, per) != s) continue;
    const double cost = ceil_div(tiles * s, pairs) * (per * products * 0.29 + 2.0) + (s > 1 ? s * result_elems * 8.0 / 5e6 + 3.0 : 0.0);
    if (cost < best_cost * 0.97) {
      best_cost = cost;
      best = static_cast<int>(s);
    }
  }
  return best;
}

// The plan of a backward pass and the layout of its workspace: a function of the sizes alone.
struct BackwardPlan {
  int64_t piece;               // words per piece, a multiple of 256
  int pieces;
  int splits_x, splits_w;
  int64_t pitch;               // of the fp32 partial results
  int64_t off_x, off_w, off_xc, off_d, off_dx, off_dw, off_bias, bytes;
};

constexpr int64_t kPieceBytes = int64_t(1) << 30;            // most of the gradient of the scores that is held at a time

BackwardPlan plan_backward(int64_t N, int64_t D, int64_t V, int dtype, int pairs) {
  BackwardPlan b;
  const int planes = dtype == GRMX_F32 ? 3 : 1;
  const int products = dtype == GRMX_F32 ? 6 : 1;
  const int64_t whole = round_up(V, kTileN);
  int64_t most = kPieceBytes / (2 * planes * N) / kTileN * kTileN;
  if (most < kTileN) most = kTileN;
  if (most > whole) most = whole;
  b.pieces = static_cast<int>(ceil_div(whole, most));
  b.piece = round_up(ceil_div(whole, b.pieces), kTileN);
  b.pieces = static_cast<int>(ceil_div(whole, b.piece));
  b.pitch = round_up(D, 8);
  const int64_t nt = ceil_div(D, kTileN);
  b.splits_x = choose_splits(ceil_div(N, kTileM) * nt, b.piece / kBlockK, N * D, products, pairs);
  b.splits_w = choose_splits(b.piece / kTileM * nt, ceil_div(N, kBlockK), b.piece * D, products, pairs);
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += round_up(bytes, 1024);
    return here;
  };
  b.off_x = take(operand_bytes(N, D, dtype));
  b.off_w = take(operand_bytes(V, D, dtype));
  b.off_xc = take(operand_bytes(N, D, dtype));
  b.off_d = take(planes * N * b.piece * 2);
  b.off_dx = take(b.splits_x * N * b.pitch * 4);
  b.off_dw = take(b.splits_w * b.piece * b.pitch * 4);
  b.off_bias = take(ceil_div(N, kTileM) * 8 * b.piece * 4);
  b.bytes = at;
  return b;
}

struct ForwardPlan {
  bool few;
  int parts;
  int64_t join_blocks;
  int64_t off_x, off_w, off_part, off_target, off_loss, off_count, off_ticket, bytes;
};

ForwardPlan plan_forward(int64_t N, int64_t D, int64_t V, int dtype) {
  ForwardPlan f;
  f.few = takes_few_tokens(N, D);
  f.parts = f.few ? few_tokens_blocks(V) : static_cast<int>(ceil_div(V, kTileN)) * parts_of(kEpiLse, dtype == GRMX_F32);
  f.join_blocks = ceil_div(N, join_rows(N));
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += round_up(bytes, 1024);
    return here;
  };
  f.off_x = take(f.few ? 0 : operand_bytes(N, D, dtype));
  f.off_w = take(f.few ? 0 : operand_bytes(V, D, dtype));
  f.off_part = take(f.parts * N * 8);
  f.off_target = take(N * 4);
  f.off_loss = take(f.join_blocks * 8);
  f.off_count = take(f.join_blocks * 4);
  f.off_ticket = take(4);
  f.bytes = at;
  return f;
}

int check_sizes(const char* who, int64_t N, int64_t D, int64_t V, int dtype) {
  GRMX_REQUIRE(dtype == GRMX_F32 || dtype == GRMX_BF16, "%s: dtype must be f32 or bf16", who);
  GRMX_REQUIRE(N >= 0 && D > 0 && V > 0, "%s: bad sizes", who);
  // tile coordinates and unit numbers are 32-bit
  GRMX_REQUIRE(N <= (int64_t(1) << 28) && V <= (int64_t(1) << 28) && D <= (int64_t(1) << 20), "%s: sizes exceed the tile coordinates", who);
  const int64_t nt = ceil_div(N, kTileM), vt = ceil_div(V, kTileN), dt = ceil_div(D, kTileN);
  GRMX_REQUIRE(nt * vt <= 0x3fffffffLL && (nt + vt) * dt <= 0x3fffffffLL / kMostSplits, "%s: too many tiles", who);
  return GRMX_OK;
}

int check_device(const char* who) {
  if (!tc::device_is_sm100() || tc::encode_tiled_fn() == nullptr) {
    return fail(GRMX_ERR_DEVICE, "%s: needs an sm_100 device with tensor-map support", who);
  }
  return GRMX_OK;
}

#define GRMX_TRY(call)                 \
  do {                                 \
    const int rc_ = (call);            \
    if (rc_ != GRMX_OK) return rc_;    \
  } while (0)

}  // namespace
}  // namespace grmx

extern "C" int64_t grmx_linear_xent_workspace(int64_t N, int64_t D, int64_t V, int dtype, int backward) {
  using namespace grmx;
  if (check_sizes("grmx_linear_xent_workspace", N, D, V, dtype) != GRMX_OK) return -1;
  if (N == 0) return 0;
  return backward ? plan_backward(N, D, V, dtype, pairs_on_device()).bytes : plan_forward(N, D, V, dtype).bytes;
}

extern "C" int grmx_linear_xent_fwd(const void* hidden, const void* weight, const void* bias, const int64_t* targets,
                                    int64_t ignore_index, float* loss, float* row_stats, float* inv_count, int64_t N,
                                    int64_t D, int64_t V, int dtype, int bias_dtype, int reduction, void* workspace,
                                    int64_t workspace_bytes, void* stream) {
  using namespace grmx;
  const char* who = "grmx_linear_xent_fwd";
  GRMX_TRY(check_sizes(who, N, D, V, dtype));
  GRMX_REQUIRE(reduction == GRMX_REDUCE_NONE || reduction == GRMX_REDUCE_SUM || reduction == GRMX_REDUCE_MEAN, "%s: bad reduction", who);
  GRMX_REQUIRE(bias == nullptr || bias_dtype == GRMX_F32 || bias_dtype == GRMX_BF16, "%s: bias must be f32 or bf16", who);
  GRMX_REQUIRE(N > 0, "%s: needs at least one token", who);
  GRMX_REQUIRE(hidden && weight && targets && loss && row_stats && inv_count, "%s: NULL tensor pointer", who);
  const ForwardPlan f = plan_forward(N, D, V, dtype);
  GRMX_REQUIRE(workspace != nullptr && workspace_bytes >= f.bytes, "%s: workspace of %lld bytes, needs %lld", who,
               (long long)workspace_bytes, (long long)f.bytes);
  GRMX_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 255u) == 0, "%s: workspace must be 256-byte aligned", who);
  GRMX_TRY(check_device(who));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  float2* partials = reinterpret_cast<float2*>(ws + f.off_part);
  float* target_score = reinterpret_cast<float*>(ws + f.off_target);
  uint32_t* ticket = reinterpret_cast<uint32_t*>(ws + f.off_ticket);
  if (f.few) {
    const int n = static_cast<int>(N), d = static_cast<int>(D);
    GRMX_TRY(dtype == GRMX_F32 ? launch_few_tokens<float>(hidden, weight, bias, bias_dtype, targets, ignore_index, n, d, V, partials, target_score, ticket, s)
                               : launch_few_tokens<__nv_bfloat16>(hidden, weight, bias, bias_dtype, targets, ignore_index, n, d, V, partials, target_score, ticket, s));
  } else {
    Operand x, w;
    GRMX_TRY(make_operand(&x, hidden, N, D, dtype, ws + f.off_x, s));
    GRMX_TRY(make_operand(&w, weight, V, D, dtype, ws + f.off_w, s));
    Maps maps;
    if (!operand_map(&maps.a, x, N, D, false) || !operand_map(&maps.b, w, V, D, false)) {
      return fail(GRMX_ERR_LAUNCH, "%s: cuTensorMapEncodeTiled failed", who);
    }
    maps.c = maps.a;
    Params p;
    memset(&p, 0, sizeof(p));
    p.m_tiles = static_cast<int>(ceil_div(N, kTileM));
    p.n_tiles = static_cast<int>(ceil_div(V, kTileN));
    p.splits = 1;
    p.k_blocks = p.blocks_per_split = static_cast<int>(ceil_div(D, kBlockK));
    p.rows = N;
    p.cols = V;
    p.vocab = V;
    p.bias = bias;
    p.bias_dtype = bias_dtype;
    p.targets = targets;
    p.ignore_index = ignore_index;
    p.partials = partials;
    p.target_score = target_score;
    p.ticket = ticket;
    GRMX_TRY(launch_scores<kEpiLse>(maps, p, dtype, "loss scores", s));
  }
  auto join_kernel = join_rows(N) == 32 ? loss_join_kernel<32> : join_rows(N) == 8 ? loss_join_kernel<8> : loss_join_kernel<1>;
  launch_after(
      join_kernel, static_cast<unsigned>(f.join_blocks), 1, kJoinThreads, 0, s, partials, target_score, bias, bias_dtype, targets, ignore_index, V, N, f.parts, reduction, row_stats, row_stats + N, loss, inv_count,
      reinterpret_cast<double*>(ws + f.off_loss), reinterpret_cast<int*>(ws + f.off_count), ticket, device_error_word_ptr());
  return check_launch("loss join");
}

extern "C" int grmx_linear_xent_bwd(const float* grad_loss, const void* hidden, const void* weight, const void* bias,
                                    const int64_t* targets, int64_t ignore_index, const float* row_stats,
                                    const float* inv_count, void* grad_hidden, void* grad_weight, void* grad_bias, int64_t N,
                                    int64_t D, int64_t V, int dtype, int bias_dtype, int reduction, void* workspace,
                                    int64_t workspace_bytes, void* stream) {
  using namespace grmx;
  const char* who = "grmx_linear_xent_bwd";
  GRMX_TRY(check_sizes(who, N, D, V, dtype));
  GRMX_REQUIRE(reduction == GRMX_REDUCE_NONE || reduction == GRMX_REDUCE_SUM || reduction == GRMX_REDUCE_MEAN, "%s: bad reduction", who);
  GRMX_REQUIRE((bias == nullptr && grad_bias == nullptr) || bias_dtype == GRMX_F32 || bias_dtype == GRMX_BF16,
               "%s: bias must be f32 or bf16", who);
  GRMX_REQUIRE(N > 0, "%s: needs at least one token", who);
  if (!grad_hidden && !grad_weight && !grad_bias) return GRMX_OK;
  GRMX_REQUIRE(grad_loss && hidden && weight && targets && row_stats && inv_count, "%s: NULL tensor pointer", who);
  const int pairs = pairs_on_device();
  const BackwardPlan b = plan_backward(N, D, V, dtype, pairs);
  GRMX_REQUIRE(workspace != nullptr && workspace_bytes >= b.bytes, "%s: workspace of %lld bytes, needs %lld", who,
               (long long)workspace_bytes, (long long)b.bytes);
  GRMX_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 255u) == 0, "%s: workspace must be 256-byte aligned", who);
  GRMX_TRY(check_device(who));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const bool f32 = dtype == GRMX_F32;
  const int planes = f32 ? 3 : 1;
  const int64_t elem = f32 ? 4 : 2;
  Operand x, w;
  GRMX_TRY(make_operand(&w, weight, V, D, dtype, ws + b.off_w, s));
  const int n_tiles_d = static_cast<int>(ceil_div(D, kTileN));
  float* part_x = reinterpret_cast<float*>(ws + b.off_dx);
  float* part_w = reinterpret_cast<float*>(ws + b.off_dw);
  float* part_b = reinterpret_cast<float*>(ws + b.off_bias);
  // d is held as p - [target] without its factor: the -1 of a target, which carries most of the gradient, is then exact
  // in bf16 where p is small.  A factor that all tokens share (the upstream gradient of a sum or a mean, 1 / count)
  // multiplies the finished sums.  A factor per token multiplies the finished rows of dx, goes into the sums of db, and
  // for dW into a copy of the tokens, in which tokens that do not count are zeros: nothing that they hold reaches dW.
  const bool per_row = reduction == GRMX_REDUCE_NONE;
  const float* scale = per_row ? nullptr : grad_loss;
  const float* scale2 = reduction == GRMX_REDUCE_MEAN ? inv_count : nullptr;
  Operand x_counted;
  if (grad_weight != nullptr) {
    GRMX_TRY(copy_operand(&x_counted, hidden, N, D, dtype, ws + b.off_xc, TokenRows{targets, ignore_index, V, per_row ? grad_loss : nullptr}, s));
  }
  if (grad_weight != nullptr && !per_row && !readable_in_place(hidden, D, dtype)) {
    x = x_counted;             // the scores of tokens that do not count are not looked at
  } else {
    GRMX_TRY(make_operand(&x, hidden, N, D, dtype, ws + b.off_x, s));
  }
  // a result that is complete after one product leaves its epilogue in the caller's type
  auto storable = [&](const void* out) { return D * elem % 16 == 0 && (reinterpret_cast<uintptr_t>(out) & 15u) == 0; };
  const bool direct_x = b.pieces == 1 && b.splits_x == 1 && storable(grad_hidden);
  const bool direct_w = b.splits_w == 1 && storable(grad_weight);

  for (int piece = 0; piece < b.pieces; ++piece) {
    const int64_t v0 = piece * b.piece;
    const int64_t words = V - v0 < b.piece ? V - v0 : b.piece;       // of the vocabulary in this piece
    const int64_t width = round_up(words, kTileN);
    const int panels = static_cast<int>(width / 64);
    const void* d = ws + b.off_d;
    // boxes of 64 columns x 128 rows (d as it is) or x 64 rows (d transposed)
    auto d_map = [&](CUtensorMap* map, int rows) {
      return make_matrix_map(map, d, false, static_cast<int64_t>(planes) * panels, N, 64, 64, N * 64, 64, rows);
    };
    const Operand w_piece{static_cast<const uint8_t*>(w.ptr) + v0 * w.ld * 2, w.ld, w.plane_stride, w.planes};
    {
      Maps maps;
      if (!operand_map(&maps.a, x, N, D, false) || !operand_map(&maps.b, w_piece, words, D, false)) {
        return fail(GRMX_ERR_LAUNCH, "%s: cuTensorMapEncodeTiled failed", who);
      }
      maps.c = maps.a;
      Params p;
      memset(&p, 0, sizeof(p));
      p.d_out = reinterpret_cast<__nv_bfloat16*>(ws + b.off_d);
      p.panels = panels;
      p.m_tiles = static_cast<int>(ceil_div(N, kTileM));
      p.n_tiles = static_cast<int>(width / kTileN);
      p.splits = 1;
      p.k_blocks = p.blocks_per_split = static_cast<int>(ceil_div(D, kBlockK));
      p.rows = N;
      p.cols = width;
      p.v0 = v0;
      p.vocab = V;
      p.bias = bias;
      p.bias_dtype = bias_dtype;
      p.targets = targets;
      p.ignore_index = ignore_index;
      p.row_max = row_stats;
      p.row_sum = row_stats + N;
      p.grad = per_row ? grad_loss : nullptr;
      p.bias_partials = grad_bias != nullptr ? part_b : nullptr;
      GRMX_TRY(launch_scores<kEpiGrad>(maps, p, dtype, "loss score gradient", s));
    }
    if (grad_bias != nullptr) {
      const int64_t blocks = ceil_div(N, kTileM) * 8;
      const unsigned grid = static_cast<unsigned>(ceil_div(words, 32));
      if (bias_dtype == GRMX_F32) {
        launch_after(bias_sum_kernel<float>, grid, 1, 256, 0, s, part_b, blocks, width, words, scale, scale2, static_cast<float*>(grad_bias) + v0);
      } else {
        launch_after(bias_sum_kernel<__nv_bfloat16>, grid, 1, 256, 0, s, part_b, blocks, width, words, scale, scale2,
                                                             static_cast<__nv_bfloat16*>(grad_bias) + v0);
      }
      GRMX_TRY(check_launch("loss bias gradient"));
    }
    if (grad_hidden != nullptr) {
      // dx = d W: the words of the piece are the contraction; later pieces add to the first one's result
      Maps maps;
      const bool to_f32 = f32 || !direct_x;
      const int64_t ld = direct_x ? D : b.pitch;
      if (!d_map(&maps.a, 128) || !operand_map(&maps.b, w_piece, words, D, true) ||
          !make_matrix_map(&maps.c, direct_x ? grad_hidden : part_x, to_f32, b.splits_x, N, D, ld, N * ld, to_f32 ? 32 : 64, 128)) {
        return fail(GRMX_ERR_LAUNCH, "%s: cuTensorMapEncodeTiled failed", who);
      }
      Params p;
      memset(&p, 0, sizeof(p));
      p.m_tiles = static_cast<int>(ceil_div(N, kTileM));
      p.n_tiles = n_tiles_d;
      p.k_blocks = static_cast<int>(width / kBlockK);
      p.blocks_per_split = static_cast<int>(ceil_div(b.piece / kBlockK, b.splits_x));
      // a last piece that is narrower than the others has fewer parts; the ones that it leaves out keep their sums
      p.splits = static_cast<int>(ceil_div(p.k_blocks, p.blocks_per_split));
      p.rows = N;
      p.cols = D;
      p.panels = panels;
      p.store_f32 = to_f32;
      p.store_add = piece > 0;
      p.grad = per_row ? grad_loss : nullptr;
      p.targets = targets;
      p.ignore_index = ignore_index;
      p.vocab = V;
      p.scale = scale;
      p.scale2 = scale2;
      GRMX_TRY(f32 ? (launch_pair<kEpiStore, false, true, true>(maps, p, "loss hidden gradient", s))
                   : (launch_pair<kEpiStore, false, true, false>(maps, p, "loss hidden gradient", s)));
    }
    if (grad_weight != nullptr) {
      // dW = d^T x: the tokens are the contraction
      Maps maps;
      const bool to_f32 = f32 || !direct_w;
      const int64_t ld = direct_w ? D : b.pitch;
      void* out = static_cast<uint8_t*>(grad_weight) + v0 * D * elem;
      if (!d_map(&maps.a, 64) || !operand_map(&maps.b, x_counted, N, D, true) ||
          !make_matrix_map(&maps.c, direct_w ? out : part_w, to_f32, b.splits_w, words, D, ld, b.piece * ld, to_f32 ? 32 : 64, 128)) {
        return fail(GRMX_ERR_LAUNCH, "%s: cuTensorMapEncodeTiled failed", who);
      }
      Params p;
      memset(&p, 0, sizeof(p));
      p.m_tiles = static_cast<int>(width / kTileM);
      p.n_tiles = n_tiles_d;
      p.k_blocks = static_cast<int>(ceil_div(N, kBlockK));
      p.blocks_per_split = static_cast<int>(ceil_div(p.k_blocks, b.splits_w));
      p.splits = b.splits_w;
      p.rows = words;
      p.cols = D;
      p.panels = panels;
      p.store_f32 = to_f32;
      p.scale = scale;
      p.scale2 = scale2;
      GRMX_TRY(f32 ? (launch_pair<kEpiStore, true, true, true>(maps, p, "loss weight gradient", s))
                   : (launch_pair<kEpiStore, true, true, false>(maps, p, "loss weight gradient", s)));
      if (!direct_w) {
        GRMX_TRY(launch_sum_splits(part_w, out, words, D, b.pitch, b.piece * b.pitch, b.splits_w, dtype, s));
      }
    }
  }
  if (grad_hidden != nullptr && !direct_x) {
    GRMX_TRY(launch_sum_splits(part_x, grad_hidden, N, D, b.pitch, N * b.pitch, b.splits_x, dtype, s));
  }
  return GRMX_OK;
}
