// The mixing rule after a block, its LayerNorm and the gradient of both, one pass each way:
//
//   u = scale * update        s = online + u                          (residual rule, scale optional)
//                             s = G online + (1 - G) u,  G = sigmoid(gate)        (gate rule)
//   y = (s - mean) * rstd * weight + bias,   rstd = 1 / sqrt(var + eps)
//
// backward, with xh = (s - mean) rstd and a = dy * weight:
//   ds = rstd (a - mean(a) - xh mean(a xh)) + d(sum)
//   residual: d_online = d_u = ds      gate: d_online = G ds, d_u = (1 - G) ds, d_gate = ds (online - u) G (1 - G)
//   d_update = scale d_u;   d_scale = sum_rows d_u update,  d_weight = sum_rows dy xh,  d_bias = sum_rows dy
//
// (the reference runs these as separate ATen calls: grm/core/aggregator.py:116-145 for the rules,
// grm/core/multilayer_grm.py:93,96 for the residual block between layers.)
//
// Bound by memory: every row tensor crosses once.  A row belongs to 32 ... 1024 threads, at most 16 values each forward
// and 8 backward, so that a row, and in the backward pass the column sums of all rows a thread has seen, stay in registers
// with enough warps resident to cover the loads (backward with 16 values: one CTA per SM, 157 us for 65536 x 512 bf16 against
// 121 with 8); mean and variance are two passes over those registers.  Three CTAs per SM leave 80 registers a thread,
// and the backward pass spills (bytes stored per thread, whole pieces / shifted ones): with gate and scale up to 200 / 336, with
// one of them 16 / 112 in bf16 and 104 / 104 in fp32; the fp32 forward pass with a gate up to 140.  Row sums are fp32; column sums are fp32 per
// thread, then joined in a fixed order (groups of a CTA in shared memory, CTAs by a second kernel).
#include "common.cuh"

namespace grmx {
namespace {

// values of a row per thread
constexpr int kForward = 16, kBackward = 8;
constexpr int kMaxWidth = 1024 * kBackward;

struct RowArgs {
  const void *online, *update, *gate;     // [rows, H]; gate may be NULL
  const void *scale, *weight, *bias;      // [H] or NULL
  float eps;
  void *out, *sum_out;                    // [rows, H]; sum_out may be NULL
  float2* stats;                          // [rows] mean and rstd; may be NULL in the forward pass
  const void *grad_out, *grad_sum;        // backward: either may be NULL
  void *grad_online, *grad_update, *grad_gate;      // NULL: not wanted
  float* col_partials;                    // backward: [kinds][CTAs][H]
  int64_t rows;
  int H;
  int param_bf16;                         // scale, weight and bias are bf16, not fp32
  int want_scale, want_weight, want_bias;
};

template <typename T, int VEC>
struct Raw;
template <typename T>
struct Raw<T, 1> {
  T v;
  __device__ __forceinline__ void load(const T* p) { v = __ldg(p); }
  __device__ __forceinline__ void set(const T (&x)[1]) { v = x[0]; }
  __device__ __forceinline__ void unpack(float (&x)[1]) const { x[0] = to_float<T>(v); }
};
template <>
struct Raw<float, 4> {
  float4 v;
  __device__ __forceinline__ void load(const float* p) { v = __ldg(reinterpret_cast<const float4*>(p)); }
  __device__ __forceinline__ void set(const float (&x)[4]) { v = make_float4(x[0], x[1], x[2], x[3]); }
  __device__ __forceinline__ void unpack(float (&x)[4]) const { x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w; }
};
template <>
struct Raw<__nv_bfloat16, 8> {
  uint4 v;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { v = __ldg(reinterpret_cast<const uint4*>(p)); }
  __device__ __forceinline__ void set(const __nv_bfloat16 (&x)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = static_cast<uint32_t>(__bfloat16_as_ushort(x[2 * i])) | (static_cast<uint32_t>(__bfloat16_as_ushort(x[2 * i + 1])) << 16);
    v = make_uint4(w[0], w[1], w[2], w[3]);
  }
  __device__ __forceinline__ void unpack(float (&x)[8]) const {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
};
template <typename T>
__device__ __forceinline__ void store_vec(T* p, const float (&x)[1]) { *p = from_float<T>(x[0]); }
__device__ __forceinline__ void store_vec(float* p, const float (&x)[4]) {
  *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
}
__device__ __forceinline__ void store_vec(__nv_bfloat16* p, const float (&x)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 b = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&b);
  }
  *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}

// sigmoid(g) and 1 - sigmoid(g), both to full relative precision: with t = exp(-|g|) they are 1 / (1 + t) and t / (1 + t)
__device__ __forceinline__ void sigmoid_pair(float g, float& yes, float& no) {
  float t, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(t) : "f"(fabsf(g) * -1.4426950408889634f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + t));
  const float small = t * r;
  yes = g >= 0.0f ? r : small;
  no = g >= 0.0f ? small : r;
}

// ---- arithmetic on a piece: two values per instruction for the eight of a bf16 piece; fp32 pieces keep to single ones,
// where pairs cost registers (backward 16384 x 1024 with scale and sum: 92 us single, 103 paired) ----
__device__ __forceinline__ uint64_t pack2(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
// x = x * m + a, x = x * m, x = x + a over VEC values
template <int VEC>
__device__ __forceinline__ void fma_all(float (&x)[VEC], const float (&m)[VEC], const float (&a)[VEC]) {
  if constexpr (VEC < 8) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) x[j] = fmaf(x[j], m[j], a[j]);
  } else {
#pragma unroll
    for (int j = 0; j < VEC; j += 2) {
      uint64_t r;
      asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(pack2(x[j], x[j + 1])), "l"(pack2(m[j], m[j + 1])), "l"(pack2(a[j], a[j + 1])));
      unpack2(r, x[j], x[j + 1]);
    }
  }
}
template <int VEC>
__device__ __forceinline__ void mul_all(float (&x)[VEC], const float (&m)[VEC]) {
  if constexpr (VEC < 8) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) x[j] *= m[j];
  } else {
#pragma unroll
    for (int j = 0; j < VEC; j += 2) {
      uint64_t r;
      asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(pack2(x[j], x[j + 1])), "l"(pack2(m[j], m[j + 1])));
      unpack2(r, x[j], x[j + 1]);
    }
  }
}
template <int VEC>
__device__ __forceinline__ void add_all(float (&x)[VEC], const float (&a)[VEC]) {
  if constexpr (VEC < 8) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) x[j] += a[j];
  } else {
#pragma unroll
    for (int j = 0; j < VEC; j += 2) {
      uint64_t r;
      asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(pack2(x[j], x[j + 1])), "l"(pack2(a[j], a[j + 1])));
      unpack2(r, x[j], x[j + 1]);
    }
  }
}
// sums += x * y
template <int VEC>
__device__ __forceinline__ void add_products(float (&sums)[VEC], const float (&x)[VEC], const float (&y)[VEC]) {
  if constexpr (VEC < 8) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) sums[j] = fmaf(x[j], y[j], sums[j]);
  } else {
#pragma unroll
    for (int j = 0; j < VEC; j += 2) {
      uint64_t r;
      asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(pack2(x[j], x[j + 1])), "l"(pack2(y[j], y[j + 1])), "l"(pack2(sums[j], sums[j + 1])));
      unpack2(r, sums[j], sums[j + 1]);
    }
  }
}
// sums += x * x
template <int VEC>
__device__ __forceinline__ void add_squares(float (&sums)[VEC], const float (&x)[VEC]) {
  if constexpr (VEC < 8) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) sums[j] = fmaf(x[j], x[j], sums[j]);
  } else {
#pragma unroll
    for (int j = 0; j < VEC; j += 2) {
      const uint64_t v = pack2(x[j], x[j + 1]);
      uint64_t r;
      asm("fma.rn.f32x2 %0, %1, %1, %2;" : "=l"(r) : "l"(v), "l"(pack2(sums[j], sums[j + 1])));
      unpack2(r, sums[j], sums[j + 1]);
    }
  }
}
template <int VEC>
__device__ __forceinline__ void fill_all(float (&x)[VEC], float v) {
#pragma unroll
  for (int j = 0; j < VEC; ++j) x[j] = v;
}

// Sums over the G threads of a row; all of them get the result.  `turn` alternates between two places for the warps'
// parts: whoever writes to one of them has passed the barrier that followed the last read of it.
template <int G>
__device__ __forceinline__ float2 row_sum2(float2 v, float2 (*scratch)[G / 32], int& turn) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
    v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
  }
  if (G > 32) {
    float2* parts = scratch[turn];
    turn ^= 1;
    if ((threadIdx.x & 31) == 0) parts[(threadIdx.x % G) >> 5] = v;
    asm volatile("barrier.cta.sync %0, %1;" ::"r"(1 + static_cast<int>(threadIdx.x) / G), "n"(G) : "memory");
    v = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < G / 32; ++i) {
      v.x += parts[i].x;
      v.y += parts[i].y;
    }
  }
  return v;
}

template <int G>
__device__ __forceinline__ float row_sum(float v, float2 (*scratch)[G / 32], int& turn) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (G > 32) {
    float2* parts = scratch[turn];
    turn ^= 1;
    if ((threadIdx.x & 31) == 0) parts[(threadIdx.x % G) >> 5].x = v;
    asm volatile("barrier.cta.sync %0, %1;" ::"r"(1 + static_cast<int>(threadIdx.x) / G), "n"(G) : "memory");
    v = 0.0f;
#pragma unroll
    for (int i = 0; i < G / 32; ++i) v += parts[i].x;
  }
  return v;
}

__host__ __device__ constexpr int threads_of(int G) { return G > 256 ? G : 256; }

// How a thread sees the rows it works on.
//
//   kWhole   rows start on 16-byte boundaries: pieces of VEC values (16 bytes)
//   kShifted rows of any width in tensors that start on a 16-byte boundary: the same 16-byte pieces of memory, so a row begins
//            `off` values into its first piece and its pieces' columns are shifted by that.  off = row * H mod VEC is the
//            same for all rows of a thread because the number of row groups of a launch is a multiple of VEC.  Pieces that
//            stick out of the row are stored value by value, the one that sticks out of the tensor is read so.
//   kSingle  tensors that start anywhere: value by value (VEC = 1)
//
// Piece i < count (the same for all threads of the row) starts at column at(i).  With whole pieces and single values the
// last piece of a thread may lie behind the row: it reads the row's last columns instead and does not count.
enum Access { kWhole, kShifted, kSingle };

template <int VEC, int G, int ACCESS>
struct Columns {
  int H, off, count, first;
  __device__ __forceinline__ Columns(int width, int64_t first_row, int lane) : H(width) {
    off = ACCESS == kShifted ? static_cast<int>((first_row * H) % VEC) : 0;
    count = (H + off + G * VEC - 1) / (G * VEC);
    first = lane * VEC - off;
  }
  __device__ __forceinline__ int start(int i) const { return first + G * VEC * i; }
  // any of the piece's values belongs to the row
  __device__ __forceinline__ bool live(int i) const { return start(i) < H; }
  __device__ __forceinline__ int at(int i) const { return ACCESS == kShifted ? start(i) : min(start(i), H - VEC); }
  __device__ __forceinline__ bool holds(int c) const { return ACCESS != kShifted || (c >= 0 && c < H); }
  __device__ __forceinline__ bool inside(int i) const { return ACCESS != kShifted || (start(i) >= 0 && start(i) + VEC <= H); }
};

template <typename T, int VEC, int ACCESS>
__device__ __forceinline__ void load_piece(Raw<T, VEC>& raw, const void* tensor, int64_t base, int c, bool live, int64_t total) {
  const T* p = static_cast<const T*>(tensor) + base + c;
  if (ACCESS != kShifted) {
    raw.load(p);
  } else if (live && base + c + VEC <= total) {
    raw.load(p);
  } else {
    T v[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[j] = live && base + c + j < total ? __ldg(p + j) : from_float<T>(0.0f);
    raw.set(v);
  }
}
template <typename T, int VEC, int ACCESS, int G>
__device__ __forceinline__ void store_piece(void* tensor, int64_t base, const Columns<VEC, G, ACCESS>& col, int i, const float (&x)[VEC]) {
  if (!col.live(i)) return;
  T* p = static_cast<T*>(tensor) + base + col.at(i);
  if (col.inside(i)) {
    store_vec(p, x);
  } else {
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      if (col.holds(col.at(i) + j)) p[j] = from_float<T>(x[j]);
    }
  }
}

// Parameters of a piece's columns.  Shifted rows take them from shared memory (fp32, one word of padding after every
// eight, so that the 32 lanes' reads at a distance of a piece do not collide).
__device__ __forceinline__ int padded(int c) { return c + (c >> 3); }
// (Volatile reads: the values are the same for all rows of a thread, and a compiler that keeps them in registers from row
// to row spills others.)
__device__ __forceinline__ uint4 load_again(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
template <int VEC, int ACCESS>
__device__ __forceinline__ void load_param(const RowArgs& a, const void* base, const float* staged, int c, float fill, float (&x)[VEC]) {
  if (base == nullptr) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) x[j] = fill;
  } else if (ACCESS == kShifted) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) x[j] = static_cast<const volatile float*>(staged)[padded(max(0, min(c + j, a.H - 1)))];
  } else if (a.param_bf16) {
    const __nv_bfloat16* p = static_cast<const __nv_bfloat16*>(base) + c;
    if constexpr (VEC == 8) {
      Raw<__nv_bfloat16, 8> raw;
      raw.v = load_again(p);
      raw.unpack(x);
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j) x[j] = __bfloat162float(__ldg(p + j));
    }
  } else {
    const float* p = static_cast<const float*>(base) + c;
    if constexpr (VEC % 4 == 0) {
#pragma unroll
      for (int j = 0; j < VEC; j += 4) {
        const uint4 q = load_again(p + j);
        x[j] = __uint_as_float(q.x); x[j + 1] = __uint_as_float(q.y); x[j + 2] = __uint_as_float(q.z); x[j + 3] = __uint_as_float(q.w);
      }
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j) x[j] = __ldg(p + j);
    }
  }
}
__device__ __forceinline__ void stage_params(const RowArgs& a, float* dst, const void* base, int threads) {
  if (base == nullptr) return;
  for (int c = threadIdx.x; c < a.H; c += threads) {
    dst[padded(c)] = a.param_bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(base)[c]) : static_cast<const float*>(base)[c];
  }
}
__host__ __device__ constexpr int staged_words(int H) { return H + H / 8 + 1; }
constexpr int kMostShared = 3 * staged_words(kMaxWidth) * 4;      // of any launch below: the forward pass of the widest row

template <typename T, int VEC, int G, int ACCESS, bool GATE>
__global__ void __launch_bounds__(threads_of(G), G > 256 ? 1 : 3)
fuse_norm_fwd_kernel(const __grid_constant__ RowArgs a) {
  constexpr int kPieces = kForward / VEC;
  constexpr int kGroups = threads_of(G) / G;
  __shared__ float2 s_scratch[kGroups][2][G / 32];
  int turn = 0;
  let_next_start();
  wait_for_previous();
  extern __shared__ float s_params[];                    // shifted rows: weight, bias, scale
  const int group = threadIdx.x / G, lane = threadIdx.x % G;
  const int H = a.H;
  const float *p_weight = s_params, *p_bias = s_params + staged_words(H), *p_scale = s_params + 2 * staged_words(H);
  if (ACCESS == kShifted) {
    stage_params(a, s_params, a.weight, threads_of(G));
    stage_params(a, s_params + staged_words(H), a.bias, threads_of(G));
    stage_params(a, s_params + 2 * staged_words(H), a.scale, threads_of(G));
    __syncthreads();
  }
  const int64_t first_row = static_cast<int64_t>(blockIdx.x) * kGroups + group, total = a.rows * H;
  const Columns<VEC, G, ACCESS> col(H, first_row, lane);
  const float inv = 1.0f / static_cast<float>(H);
#pragma unroll 1
  for (int64_t row = first_row; row < a.rows; row += static_cast<int64_t>(gridDim.x) * kGroups) {
    const int64_t base = row * H;
    Raw<T, VEC> ro[kPieces], ru[kPieces], rg[kPieces];
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      if (i < col.count) {
        load_piece<T, VEC, ACCESS>(ro[i], a.online, base, col.at(i), col.live(i), total);
        load_piece<T, VEC, ACCESS>(ru[i], a.update, base, col.at(i), col.live(i), total);
        if (GATE) load_piece<T, VEC, ACCESS>(rg[i], a.gate, base, col.at(i), col.live(i), total);
      }
    }
    float s[kPieces][VEC], part[VEC];
    fill_all(part, 0.0f);
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      if (i < col.count) {
        const bool live = col.live(i);
        float o[VEC], u[VEC], k[VEC];
        ro[i].unpack(o);
        ru[i].unpack(u);
        if (a.scale != nullptr) {
          load_param<VEC, ACCESS>(a, a.scale, p_scale, col.at(i), 1.0f, k);
          mul_all(u, k);
        }
        if (GATE) {
          float yes[VEC];
          rg[i].unpack(k);
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            float no;
            sigmoid_pair(k[j], yes[j], no);
            k[j] = no;
          }
          mul_all(u, k);
          fma_all(o, yes, u);
        } else {
          add_all(o, u);
        }
#pragma unroll
        for (int j = 0; j < VEC; ++j) s[i][j] = live && col.holds(col.at(i) + j) ? o[j] : 0.0f;
        add_all(part, s[i]);
        if (a.sum_out != nullptr) store_piece<T>(a.sum_out, base, col, i, s[i]);
      }
    }
    float sum = 0.0f;
#pragma unroll
    for (int j = 0; j < VEC; ++j) sum += part[j];
    const float mean = row_sum<G>(sum, s_scratch[group], turn) * inv;
    float minus[VEC];
    fill_all(minus, -mean);
    fill_all(part, 0.0f);
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      if (i < col.count) {
        add_all(s[i], minus);
        if (ACCESS == kShifted || !col.live(i)) {            // what is not of the row does not count
#pragma unroll
          for (int j = 0; j < VEC; ++j) s[i][j] = col.live(i) && col.holds(col.at(i) + j) ? s[i][j] : 0.0f;
        }
        add_squares(part, s[i]);
      }
    }
    sum = 0.0f;
#pragma unroll
    for (int j = 0; j < VEC; ++j) sum += part[j];
    const float rstd = rsqrtf(row_sum<G>(sum, s_scratch[group], turn) * inv + a.eps);
    float scale_by[VEC];
    fill_all(scale_by, rstd);
    if (lane == 0 && a.stats != nullptr) a.stats[row] = make_float2(mean, rstd);
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      if (i < col.count) {
        float w[VEC], b[VEC];
        load_param<VEC, ACCESS>(a, a.weight, p_weight, col.at(i), 1.0f, w);
        load_param<VEC, ACCESS>(a, a.bias, p_bias, col.at(i), 0.0f, b);
        mul_all(s[i], scale_by);
        fma_all(s[i], w, b);
        store_piece<T>(a.out, base, col, i, s[i]);
      }
    }
  }
}

template <typename T, int VEC, int G, int ACCESS, bool GATE, bool SCALE>
__global__ void __launch_bounds__(threads_of(G), G > 256 ? 1 : 3)
fuse_norm_bwd_kernel(const __grid_constant__ RowArgs a) {
  constexpr int kPieces = kBackward / VEC;
  constexpr int kGroups = threads_of(G) / G;
  __shared__ float2 s_scratch[kGroups][2][G / 32];
  int turn = 0;
  let_next_start();
  wait_for_previous();
  extern __shared__ float s_dynamic[];                   // shifted rows: weight, scale; then, at the end, the column sums
  const int group = threadIdx.x / G, lane = threadIdx.x % G;
  const int H = a.H;
  const float *p_weight = s_dynamic, *p_scale = s_dynamic + staged_words(H);
  if (ACCESS == kShifted) {
    stage_params(a, s_dynamic, a.weight, threads_of(G));
    stage_params(a, s_dynamic + staged_words(H), a.scale, threads_of(G));
    __syncthreads();
  }
  const int64_t first_row = static_cast<int64_t>(blockIdx.x) * kGroups + group, total = a.rows * H;
  const Columns<VEC, G, ACCESS> col(H, first_row, lane);
  const float inv = 1.0f / static_cast<float>(H);
  float cw[kPieces][VEC], cb[kPieces][VEC], cs[SCALE ? kPieces : 1][VEC];
#pragma unroll
  for (int i = 0; i < kPieces; ++i) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) cw[i][j] = cb[i][j] = cs[SCALE ? i : 0][j] = 0.0f;
  }
#pragma unroll 1
  for (int64_t row = first_row; row < a.rows; row += static_cast<int64_t>(gridDim.x) * kGroups) {
    const int64_t base = row * H;
    Raw<T, VEC> rd[kPieces], ro[kPieces], ru[kPieces], rg[kPieces];
    const float2 st = __ldg(a.stats + row);
    const bool have_dy = a.grad_out != nullptr;
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      if (i < col.count) {
        if (have_dy) load_piece<T, VEC, ACCESS>(rd[i], a.grad_out, base, col.at(i), col.live(i), total);
        load_piece<T, VEC, ACCESS>(ro[i], a.online, base, col.at(i), col.live(i), total);
        load_piece<T, VEC, ACCESS>(ru[i], a.update, base, col.at(i), col.live(i), total);
        if (GATE) load_piece<T, VEC, ACCESS>(rg[i], a.gate, base, col.at(i), col.live(i), total);
      }
    }
    float xh[kPieces][VEC], da[kPieces][VEC], part[VEC], part_xh[VEC], minus[VEC], by[VEC];
    float2 sum = make_float2(0.0f, 0.0f);
    fill_all(part, 0.0f);
    fill_all(part_xh, 0.0f);
    fill_all(minus, -st.x);
    fill_all(by, st.y);
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      if (i < col.count) {
        float u[VEC], k[VEC];
        ro[i].unpack(xh[i]);
        ru[i].unpack(u);
        if (SCALE) {
          load_param<VEC, ACCESS>(a, a.scale, p_scale, col.at(i), 1.0f, k);
          mul_all(u, k);
        }
        if (GATE) {
          float yes[VEC];
          rg[i].unpack(k);
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            float no;
            sigmoid_pair(k[j], yes[j], no);
            k[j] = no;
          }
          mul_all(u, k);
          fma_all(xh[i], yes, u);
        } else {
          add_all(xh[i], u);
        }
        add_all(xh[i], minus);
        mul_all(xh[i], by);
        if (have_dy) {
          rd[i].unpack(da[i]);
        } else {
          fill_all(da[i], 0.0f);
        }
        if (ACCESS == kShifted || !col.live(i)) {              // what is not of the row does not count
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            const bool counts = col.live(i) && col.holds(col.at(i) + j);
            xh[i][j] = counts ? xh[i][j] : 0.0f;
            da[i][j] = counts ? da[i][j] : 0.0f;
          }
        }
        add_products(cw[i], da[i], xh[i]);
        add_all(cb[i], da[i]);
        load_param<VEC, ACCESS>(a, a.weight, p_weight, col.at(i), 1.0f, k);
        mul_all(da[i], k);
        if constexpr (VEC == 8) {
          add_all(part, da[i]);
          add_products(part_xh, da[i], xh[i]);
        } else {
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            sum.x += da[i][j];
            sum.y = fmaf(da[i][j], xh[i][j], sum.y);
          }
        }
      }
    }
    if constexpr (VEC == 8) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        sum.x += part[j];
        sum.y += part_xh[j];
      }
    }
    sum = row_sum2<G>(sum, s_scratch[group], turn);
    float minus_xh[VEC];
    fill_all(minus, -sum.x * inv);
    fill_all(minus_xh, -sum.y * inv);
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      if (i < col.count) {
        float dv[VEC], u[VEC], k[VEC];
        float (&ds)[VEC] = da[i];
        add_products(ds, xh[i], minus_xh);
        add_all(ds, minus);
        mul_all(ds, by);
        if (a.grad_sum != nullptr) {
          Raw<T, VEC> raw;
          load_piece<T, VEC, ACCESS>(raw, a.grad_sum, base, col.at(i), col.live(i), total);
          raw.unpack(dv);
          add_all(ds, dv);
        }
        ru[i].unpack(u);
        if (SCALE) load_param<VEC, ACCESS>(a, a.scale, p_scale, col.at(i), 1.0f, k);
        if (GATE) {
          float dg[VEC], g[VEC], yes[VEC], other[VEC];
          // online - scale update
          ro[i].unpack(dg);
#pragma unroll
          for (int j = 0; j < VEC; ++j) other[j] = SCALE ? -k[j] : -1.0f;
          add_products(dg, u, other);
          rg[i].unpack(g);
#pragma unroll
          for (int j = 0; j < VEC; ++j) sigmoid_pair(g[j], yes[j], dv[j]);
          mul_all(dg, ds);
#pragma unroll
          for (int j = 0; j < VEC; ++j) other[j] = yes[j];
          mul_all(other, dv);
          mul_all(dg, other);
          mul_all(dv, ds);
          mul_all(ds, yes);
          if (a.grad_gate != nullptr) store_piece<T>(a.grad_gate, base, col, i, dg);
        } else {
#pragma unroll
          for (int j = 0; j < VEC; ++j) dv[j] = ds[j];
        }
        if (a.grad_online != nullptr) store_piece<T>(a.grad_online, base, col, i, ds);
        if constexpr (SCALE) {
          if (ACCESS == kShifted || !col.live(i)) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) u[j] = col.live(i) && col.holds(col.at(i) + j) ? u[j] : 0.0f;
          }
          add_products(cs[i], dv, u);
          mul_all(dv, k);
        }
        if (a.grad_update != nullptr) store_piece<T>(a.grad_update, base, col, i, dv);
      }
    }
  }
  // column sums of this CTA: its groups in order, then one row of partials per kind
  if (a.col_partials == nullptr) return;
  int kind = 0;
  auto emit = [&](float (&c)[kPieces][VEC]) {
    float* dst = a.col_partials + (static_cast<int64_t>(kind++) * gridDim.x + blockIdx.x) * H;
    if (kGroups > 1) __syncthreads();                    // the parameters, or the last kind's sums, have been read
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      if (i < col.count && col.live(i)) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const int h = col.at(i) + j;
          if (col.holds(h)) (kGroups > 1 ? s_dynamic + group * H : dst)[h] = c[i][j];
        }
      }
    }
    if (kGroups > 1) {
      __syncthreads();
      for (int h = threadIdx.x; h < H; h += threads_of(G)) {
        float sum = 0.0f;
#pragma unroll
        for (int g = 0; g < kGroups; ++g) sum += s_dynamic[g * H + h];
        dst[h] = sum;
      }
    }
  };
  if (a.want_weight) emit(cw);
  if (a.want_bias) emit(cb);
  if constexpr (SCALE) {
    if (a.want_scale) emit(cs);
  }
}

// out_k[h] = sum over the CTAs' partials, in order: 32 columns x 32 slices per block
template <typename P>
__global__ void __launch_bounds__(1024) fuse_norm_cols_kernel(const float* __restrict__ partials, int ctas, int H, P* out0, P* out1,
                                                              P* out2) {
  __shared__ float s_sum[32][33];
  let_next_start();
  wait_for_previous();
  const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5;
  const int h = blockIdx.x * 32 + lane;
  const float* src = partials + static_cast<int64_t>(blockIdx.y) * ctas * H;
  float sum = 0.0f;
  if (h < H) {
#pragma unroll 4
    for (int i = slice; i < ctas; i += 32) sum += src[static_cast<int64_t>(i) * H + h];
  }
  s_sum[slice][lane] = sum;
  __syncthreads();
  sum = s_sum[lane][slice];            // column `slice` of the block, one slice per lane
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  const int col = blockIdx.x * 32 + slice;
  if (lane == 0 && col < H) {
    P* out = blockIdx.y == 0 ? out0 : blockIdx.y == 1 ? out1 : out2;
    out[col] = from_float<P>(sum);
  }
}

int sm_count() {
  static std::atomic<int> cached[64];
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess || device < 0 || device >= 64) return 148;
  int n = cached[device].load();
  if (n == 0) {
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device) != cudaSuccess || n < 1) n = 148;
    cached[device].store(n);
  }
  return n;
}

// `width`: a row's values, and for shifted rows what a piece may stick out by
int threads_per_row(int64_t width, int values) {
  for (int G : {32, 64, 128, 256, 512}) {
    if (width <= G * values) return G;
  }
  return 1024;
}
enum { kSlack = 7 };           // values of a 16-byte piece that may lie before a shifted row

// CTAs of a backward pass: three per SM (two of 512 threads, one of 1024), or as many as there are rows; a multiple of eight row
// groups, so that a thread's rows all start at the same place of a 16-byte piece
int64_t backward_ctas(int64_t rows, int G) {
  const int64_t per = threads_of(G) / G, unit = per >= 8 ? 1 : 8 / per;
  const int64_t need = (rows + per - 1) / per;
  const int64_t most = (G > 512 ? 1 : G > 256 ? 2 : 3) * static_cast<int64_t>(sm_count()) / unit * unit;
  return need < most ? (need + unit - 1) / unit * unit : most;
}
// of either way to see the rows: the workspace is sized before the pointers are known
int64_t most_backward_ctas(int64_t rows, int64_t H) {
  const int64_t a = backward_ctas(rows, threads_per_row(H, kBackward)), b = backward_ctas(rows, threads_per_row(H + kSlack, kBackward));
  return a > b ? a : b;
}

template <typename Kernel>
int launch_rows(Kernel kernel, const RowArgs& a, int64_t grid, int threads, int smem, const char* what, cudaStream_t s) {
  // (48 KiB without being asked for, less what the kernel holds itself: up to 512 bytes)  Always the same size: a limit of
  // this call's own could be lowered by another thread's call before the launch below.
  if (smem > 40 * 1024 && cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostShared) != cudaSuccess) {
    return fail(GRMX_ERR_LAUNCH, "%s: cannot reserve %d bytes of shared memory: %s", what, kMostShared, cudaGetErrorString(cudaGetLastError()));
  }
  launch_after(kernel, static_cast<unsigned>(grid), 1, threads, smem, s, a);
  return check_launch(what);
}

template <typename T, int VEC, int G, int ACCESS>
int launch_forward(const RowArgs& a, cudaStream_t s) {
  constexpr int kGroups = threads_of(G) / G;
  constexpr int64_t kUnit = kGroups >= 8 ? 1 : 8 / kGroups;
  int64_t grid = ((a.rows + kGroups - 1) / kGroups + kUnit - 1) / kUnit * kUnit;
  // a CTA lives for several rows (its set-up costs a fifth of a row of 512)
  const int64_t most = (G > 256 ? 2 : 6) * static_cast<int64_t>(sm_count()) / kUnit * kUnit;
  if (grid > most) grid = most;
  const int smem = ACCESS == kShifted ? 3 * staged_words(a.H) * 4 : 0;
  return a.gate != nullptr ? launch_rows(fuse_norm_fwd_kernel<T, VEC, G, ACCESS, true>, a, grid, threads_of(G), smem, "fuse_norm", s)
                           : launch_rows(fuse_norm_fwd_kernel<T, VEC, G, ACCESS, false>, a, grid, threads_of(G), smem, "fuse_norm", s);
}

template <typename T, int VEC, int G, int ACCESS>
int launch_group(const RowArgs& a, bool backward, cudaStream_t s) {
  constexpr int kGroups = threads_of(G) / G;
  if constexpr (G * kForward <= kMaxWidth) {      // more threads than that no forward pass asks for
    if (!backward) return launch_forward<T, VEC, G, ACCESS>(a, s);
  }
  const int64_t grid = backward_ctas(a.rows, G);
  const int staged = ACCESS == kShifted ? 2 * staged_words(a.H) * 4 : 0, sums = kGroups > 1 ? kGroups * a.H * 4 : 0;
  const int smem = staged > sums ? staged : sums;
  const char* what = "fuse_norm gradient";
  auto kernel = a.gate != nullptr ? (a.scale != nullptr ? fuse_norm_bwd_kernel<T, VEC, G, ACCESS, true, true> : fuse_norm_bwd_kernel<T, VEC, G, ACCESS, true, false>)
                                  : (a.scale != nullptr ? fuse_norm_bwd_kernel<T, VEC, G, ACCESS, false, true> : fuse_norm_bwd_kernel<T, VEC, G, ACCESS, false, false>);
  return launch_rows(kernel, a, grid, threads_of(G), smem, what, s);
}

template <typename T, int VEC, int ACCESS>
int launch_width(const RowArgs& a, bool backward, cudaStream_t s) {
  switch (threads_per_row(a.H + (ACCESS == kShifted ? kSlack : 0), backward ? kBackward : kForward)) {
    case 32: return launch_group<T, VEC, 32, ACCESS>(a, backward, s);
    case 64: return launch_group<T, VEC, 64, ACCESS>(a, backward, s);
    case 128: return launch_group<T, VEC, 128, ACCESS>(a, backward, s);
    case 256: return launch_group<T, VEC, 256, ACCESS>(a, backward, s);
    case 512: return launch_group<T, VEC, 512, ACCESS>(a, backward, s);
    default: return launch_group<T, VEC, 1024, ACCESS>(a, backward, s);
  }
}

template <typename T>
int launch_access(const RowArgs& a, int access, bool backward, cudaStream_t s) {
  constexpr int kVec = 16 / static_cast<int>(sizeof(T));
  if (access == kWhole) return launch_width<T, kVec, kWhole>(a, backward, s);
  if (access == kShifted) return launch_width<T, kVec, kShifted>(a, backward, s);
  return launch_width<T, 1, kSingle>(a, backward, s);
}

int launch_types(RowArgs& a, int dtype, int param_dtype, int access, bool backward, cudaStream_t s) {
  a.param_bf16 = param_dtype == GRMX_BF16;
  return dtype == GRMX_F32 ? launch_access<float>(a, access, backward, s) : launch_access<__nv_bfloat16>(a, access, backward, s);
}

int check_common(const char* who, int64_t rows, int64_t H, int dtype, int param_dtype) {
  GRMX_REQUIRE(rows >= 0 && H > 0, "%s: bad sizes", who);
  GRMX_REQUIRE(dtype == GRMX_F32 || dtype == GRMX_BF16, "%s: dtype must be f32 or bf16", who);
  GRMX_REQUIRE(param_dtype == GRMX_F32 || param_dtype == dtype, "%s: parameters must be f32 or of the rows' dtype", who);
  if (H > kMaxWidth) return fail(GRMX_ERR_UNSUPPORTED, "%s: rows of at most %d values", who, kMaxWidth);
  return GRMX_OK;
}

// 16-byte pieces where every tensor starts on a 16-byte boundary, shifted where the rows do not
int access_of(int64_t H, int dtype, const void* const* rows, int n_rows, const void* const* params, int n_params) {
  uintptr_t row_bits = 0, param_bits = 0;
  for (int i = 0; i < n_rows; ++i) row_bits |= reinterpret_cast<uintptr_t>(rows[i]);
  for (int i = 0; i < n_params; ++i) param_bits |= reinterpret_cast<uintptr_t>(params[i]);
  if ((row_bits & 15u) != 0) return kSingle;
  if (H % (dtype == GRMX_F32 ? 4 : 8) == 0 && (param_bits & 15u) == 0) return kWhole;
  return H + kSlack <= kMaxWidth ? kShifted : kSingle;
}

}  // namespace
}  // namespace grmx

extern "C" int grmx_fuse_norm_fwd(const void* online, const void* update, const void* gate, const void* scale,
                                  const void* ln_weight, const void* ln_bias, float eps, void* out, void* sum_out,
                                  float* row_stats, int64_t rows, int64_t H, int dtype, int param_dtype, void* stream) {
  using namespace grmx;
  const char* who = "grmx_fuse_norm_fwd";
  const int rc = check_common(who, rows, H, dtype, param_dtype);
  if (rc != GRMX_OK) return rc;
  if (rows == 0) return GRMX_OK;
  GRMX_REQUIRE(online && update && out, "%s: NULL tensor pointer", who);
  GRMX_REQUIRE((reinterpret_cast<uintptr_t>(row_stats) & 7u) == 0, "%s: row_stats must be 8-byte aligned", who);
  RowArgs a = {};
  a.online = online;
  a.update = update;
  a.gate = gate;
  a.scale = scale;
  a.weight = ln_weight;
  a.bias = ln_bias;
  a.eps = eps;
  a.out = out;
  a.sum_out = sum_out;
  a.stats = reinterpret_cast<float2*>(row_stats);
  a.rows = rows;
  a.H = static_cast<int>(H);
  const void* row_ptrs[] = {online, update, gate, out, sum_out};
  const void* param_ptrs[] = {scale, ln_weight, ln_bias};
  return launch_types(a, dtype, param_dtype, access_of(H, dtype, row_ptrs, 5, param_ptrs, 3), false, static_cast<cudaStream_t>(stream));
}

extern "C" int64_t grmx_fuse_norm_workspace(int64_t rows, int64_t H) {
  using namespace grmx;
  if (check_common("grmx_fuse_norm_workspace", rows, H, GRMX_F32, GRMX_F32) != GRMX_OK) return -1;
  return rows == 0 ? 0 : 3 * most_backward_ctas(rows, H) * H * 4;
}

extern "C" int grmx_fuse_norm_bwd(const void* grad_out, const void* grad_sum, const void* online, const void* update,
                                  const void* gate, const void* scale, const void* ln_weight, const float* row_stats,
                                  void* grad_online, void* grad_update, void* grad_gate, void* grad_scale, void* grad_weight,
                                  void* grad_bias, int64_t rows, int64_t H, int dtype, int param_dtype, void* workspace,
                                  int64_t workspace_bytes, void* stream) {
  using namespace grmx;
  const char* who = "grmx_fuse_norm_bwd";
  const int rc = check_common(who, rows, H, dtype, param_dtype);
  if (rc != GRMX_OK) return rc;
  GRMX_REQUIRE(grad_scale == nullptr || scale != nullptr, "%s: there is no scale to differentiate", who);
  GRMX_REQUIRE(grad_gate == nullptr || gate != nullptr, "%s: there is no gate to differentiate", who);
  const size_t param_bytes = param_dtype == GRMX_F32 ? 4 : 2;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (rows == 0) {
    for (void* out : {grad_scale, grad_weight, grad_bias}) {
      if (out != nullptr && cudaMemsetAsync(out, 0, H * param_bytes, s) != cudaSuccess) {
        return fail(GRMX_ERR_LAUNCH, "%s: %s", who, cudaGetErrorString(cudaGetLastError()));
      }
    }
    return GRMX_OK;
  }
  GRMX_REQUIRE(online && update && row_stats, "%s: NULL tensor pointer", who);
  GRMX_REQUIRE((reinterpret_cast<uintptr_t>(row_stats) & 7u) == 0, "%s: row_stats must be 8-byte aligned", who);
  GRMX_REQUIRE(grad_out || grad_sum, "%s: neither output has a gradient", who);
  const int kinds = (grad_weight != nullptr) + (grad_bias != nullptr) + (grad_scale != nullptr);
  RowArgs a = {};
  a.online = online;
  a.update = update;
  a.gate = gate;
  a.scale = scale;
  a.weight = ln_weight;
  a.stats = reinterpret_cast<float2*>(const_cast<float*>(row_stats));
  a.grad_out = grad_out;
  a.grad_sum = grad_sum;
  a.grad_online = grad_online;
  a.grad_update = grad_update;
  a.grad_gate = grad_gate;
  a.rows = rows;
  a.H = static_cast<int>(H);
  a.want_scale = grad_scale != nullptr;
  a.want_weight = grad_weight != nullptr;
  a.want_bias = grad_bias != nullptr;
  const void* row_ptrs[] = {online, update, gate, grad_out, grad_sum, grad_online, grad_update, grad_gate};
  const void* param_ptrs[] = {scale, ln_weight};
  const int access = access_of(H, dtype, row_ptrs, 8, param_ptrs, 2);
  const int64_t ctas = backward_ctas(rows, threads_per_row(H + (access == kShifted ? kSlack : 0), kBackward));
  if (kinds > 0) {
    GRMX_REQUIRE(workspace != nullptr && workspace_bytes >= 3 * most_backward_ctas(rows, H) * H * 4, "%s: workspace of %lld bytes, needs %lld", who,
                 (long long)workspace_bytes, (long long)(3 * most_backward_ctas(rows, H) * H * 4));
    GRMX_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 15u) == 0, "%s: workspace must be 16-byte aligned", who);
    a.col_partials = static_cast<float*>(workspace);
  }
  const int status = launch_types(a, dtype, param_dtype, access, true, s);
  if (status != GRMX_OK || kinds == 0) return status;
  void* outs[3] = {nullptr, nullptr, nullptr};
  int n = 0;
  for (void* out : {grad_weight, grad_bias, grad_scale}) {
    if (out != nullptr) outs[n++] = out;
  }
  const dim3 grid(static_cast<unsigned>((H + 31) / 32), static_cast<unsigned>(kinds));
  if (param_dtype == GRMX_F32) {
    launch_after(fuse_norm_cols_kernel<float>, grid.x, grid.y, 1024, 0, s, a.col_partials, static_cast<int>(ctas), a.H, static_cast<float*>(outs[0]),
                                                       static_cast<float*>(outs[1]), static_cast<float*>(outs[2]));
  } else {
    launch_after(fuse_norm_cols_kernel<__nv_bfloat16>, grid.x, grid.y, 1024, 0, s, 
        a.col_partials, static_cast<int>(ctas), a.H, static_cast<__nv_bfloat16*>(outs[0]), static_cast<__nv_bfloat16*>(outs[1]),
        static_cast<__nv_bfloat16*>(outs[2]));
  }
  return check_launch("fuse_norm column sums");
}
