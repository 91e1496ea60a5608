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
// Bound by memory: every row tensor crosses once.  A row belongs to 32, 128 or 512 threads, at most 16 values
// each, so that a row, and in the backward pass the column sums of all rows a thread has seen, stay in
// registers; mean and variance are two passes over those registers.  Row sums are fp32; column sums are fp32
// per thread, then joined in a fixed order (groups of a CTA in shared memory, CTAs by a second kernel).
#include "common.cuh"

namespace grmx {
namespace {

constexpr int kPerThread = 16;
constexpr int kMaxWidth = 512 * kPerThread;

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
  int want_scale, want_weight, want_bias;
};

template <typename T, int VEC>
struct Raw;
template <typename T>
struct Raw<T, 1> {
  T v;
  __device__ __forceinline__ void load(const T* p) { v = __ldg(p); }
  __device__ __forceinline__ void unpack(float (&x)[1]) const { x[0] = to_float<T>(v); }
};
template <>
struct Raw<float, 4> {
  float4 v;
  __device__ __forceinline__ void load(const float* p) { v = __ldg(reinterpret_cast<const float4*>(p)); }
  __device__ __forceinline__ void unpack(float (&x)[4]) const { x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w; }
};
template <>
struct Raw<__nv_bfloat16, 8> {
  uint4 v;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { v = __ldg(reinterpret_cast<const uint4*>(p)); }
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

// sigmoid(g) and 1 - sigmoid(g), both to full relative precision
__device__ __forceinline__ void sigmoid_pair(float g, float& yes, float& no) {
  const float t = __expf(-fabsf(g));
  const float r = __fdividef(1.0f, 1.0f + t);
  const float small = t * r;
  yes = g >= 0.0f ? r : small;
  no = g >= 0.0f ? small : r;
  if (isnan(g)) yes = no = g;
}

// sums over the G threads of a row; all of them get the result
template <int G>
__device__ __forceinline__ float2 row_sum2(float2 v, float2* scratch) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
    v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
  }
  if (G > 32) {
    constexpr int kWarps = G / 32;
    const int warp = (threadIdx.x % G) >> 5;
    const int id = 1 + threadIdx.x / G;
    asm volatile("barrier.cta.sync %0, %1;" ::"r"(id), "n"(G) : "memory");       // the scratch of the last sum has been read
    if ((threadIdx.x & 31) == 0) scratch[warp] = v;
    asm volatile("barrier.cta.sync %0, %1;" ::"r"(id), "n"(G) : "memory");
    v = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < kWarps; ++i) {
      v.x += scratch[i].x;
      v.y += scratch[i].y;
    }
  }
  return v;
}

template <typename P, int VEC>
__device__ __forceinline__ void load_param(const void* base, int h, float fill, float (&x)[VEC]) {
  if (base == nullptr) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) x[j] = fill;
    return;
  }
  const P* p = static_cast<const P*>(base) + h;
  if constexpr (VEC == 1) {
    x[0] = to_float<P>(__ldg(p));
  } else if constexpr (sizeof(P) == 4) {
#pragma unroll
    for (int j = 0; j < VEC; j += 4) {
      const float4 q = __ldg(reinterpret_cast<const float4*>(p + j));
      x[j] = q.x; x[j + 1] = q.y; x[j + 2] = q.z; x[j + 3] = q.w;
    }
  } else {
    Raw<P, VEC> raw;
    raw.load(p);
    raw.unpack(x);
  }
}

__host__ __device__ constexpr int threads_of(int G) { return G == 512 ? 512 : 256; }

// The columns of a row that a thread holds: pieces i < count (the same count for all threads), piece i at column
// (lane + G i) VEC.  The last piece may lie behind the row: its loads go to the row's last columns instead (always
// in bounds), its values count as zero and are not stored.
template <int VEC, int G>
struct Columns {
  int count, first, last;      // last: the largest column a piece can start at
  __device__ __forceinline__ Columns(int H, int lane) : count((H + G * VEC - 1) / (G * VEC)), first(lane * VEC), last(H - VEC) {}
  __device__ __forceinline__ int at(int i) const { return min(first + G * VEC * i, last); }
  __device__ __forceinline__ bool live(int i) const { return first + G * VEC * i <= last; }
};

template <typename T, typename P, int VEC, int G, bool GATE>
__global__ void __launch_bounds__(threads_of(G))
fuse_norm_fwd_kernel(const __grid_constant__ RowArgs a) {
  constexpr int kPieces = kPerThread / VEC;
  constexpr int kGroups = threads_of(G) / G;
  __shared__ float2 s_scratch[kGroups][G / 32];
  const int group = threadIdx.x / G, lane = threadIdx.x % G;
  const int H = a.H;
  const Columns<VEC, G> col(H, lane);
  const float inv = 1.0f / static_cast<float>(H);
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * kGroups + group; row < a.rows; row += static_cast<int64_t>(gridDim.x) * kGroups) {
    const int64_t base = row * H;
    Raw<T, VEC> ro[kPieces], ru[kPieces], rg[kPieces];
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      if (i < col.count) {
        ro[i].load(static_cast<const T*>(a.online) + base + col.at(i));
        ru[i].load(static_cast<const T*>(a.update) + base + col.at(i));
        if (GATE) rg[i].load(static_cast<const T*>(a.gate) + base + col.at(i));
      }
    }
    float s[kPieces][VEC];
    float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      if (i < col.count) {
        const int h = col.at(i);
        const bool live = col.live(i);
        float o[VEC], u[VEC], k[VEC];
        ro[i].unpack(o);
        ru[i].unpack(u);
        if (a.scale != nullptr) {
          load_param<P, VEC>(a.scale, h, 1.0f, k);
#pragma unroll
          for (int j = 0; j < VEC; ++j) u[j] *= k[j];
        }
        if (GATE) rg[i].unpack(k);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          if (GATE) {
            float yes, no;
            sigmoid_pair(k[j], yes, no);
            s[i][j] = fmaf(yes, o[j], no * u[j]);
          } else {
            s[i][j] = o[j] + u[j];
          }
          if (live) sum.x += s[i][j];
        }
        if (a.sum_out != nullptr && live) store_vec(static_cast<T*>(a.sum_out) + base + h, s[i]);
      }
    }
    const float mean = row_sum2<G>(sum, s_scratch[group]).x * inv;
    sum = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      if (i < col.count && col.live(i)) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float d = s[i][j] - mean;
          sum.x = fmaf(d, d, sum.x);
        }
      }
    }
    const float rstd = rsqrtf(row_sum2<G>(sum, s_scratch[group]).x * inv + a.eps);
    if (lane == 0 && a.stats != nullptr) a.stats[row] = make_float2(mean, rstd);
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      if (i < col.count) {
        const int h = col.at(i);
        float w[VEC], b[VEC], y[VEC];
        load_param<P, VEC>(a.weight, h, 1.0f, w);
        load_param<P, VEC>(a.bias, h, 0.0f, b);
#pragma unroll
        for (int j = 0; j < VEC; ++j) y[j] = fmaf((s[i][j] - mean) * rstd, w[j], b[j]);
        if (col.live(i)) store_vec(static_cast<T*>(a.out) + base + h, y);
      }
    }
  }
}

template <typename T, typename P, int VEC, int G, bool GATE, bool SCALE>
__global__ void __launch_bounds__(threads_of(G))
fuse_norm_bwd_kernel(const __grid_constant__ RowArgs a) {
  constexpr int kPieces = kPerThread / VEC;
  constexpr int kGroups = threads_of(G) / G;
  __shared__ float2 s_scratch[kGroups][G / 32];
  __shared__ float s_cols[kGroups > 1 ? kGroups * G * kPerThread : 1];
  const int group = threadIdx.x / G, lane = threadIdx.x % G;
  const int H = a.H;
  const Columns<VEC, G> col(H, lane);
  const float inv = 1.0f / static_cast<float>(H);
  float cw[kPieces][VEC], cb[kPieces][VEC], cs[SCALE ? kPieces : 1][VEC];
#pragma unroll
  for (int i = 0; i < kPieces; ++i) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) cw[i][j] = cb[i][j] = cs[SCALE ? i : 0][j] = 0.0f;
  }
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * kGroups + group; row < a.rows; row += static_cast<int64_t>(gridDim.x) * kGroups) {
    const int64_t base = row * H;
    Raw<T, VEC> rd[kPieces], ro[kPieces], ru[kPieces], rg[kPieces];
    const float2 st = __ldg(a.stats + row);
    const bool have_dy = a.grad_out != nullptr;
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      if (i < col.count) {
        if (have_dy) rd[i].load(static_cast<const T*>(a.grad_out) + base + col.at(i));
        ro[i].load(static_cast<const T*>(a.online) + base + col.at(i));
        ru[i].load(static_cast<const T*>(a.update) + base + col.at(i));
        if (GATE) rg[i].load(static_cast<const T*>(a.gate) + base + col.at(i));
      }
    }
    float xh[kPieces][VEC], da[kPieces][VEC];
    float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      if (i < col.count) {
        const int h = col.at(i);
        const bool live = col.live(i);
        float o[VEC], u[VEC], k[VEC], w[VEC];
        ro[i].unpack(o);
        ru[i].unpack(u);
        if (SCALE) {
          load_param<P, VEC>(a.scale, h, 1.0f, k);
#pragma unroll
          for (int j = 0; j < VEC; ++j) u[j] *= k[j];
        }
        if (GATE) rg[i].unpack(k);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          float s;
          if (GATE) {
            float yes, no;
            sigmoid_pair(k[j], yes, no);
            s = fmaf(yes, o[j], no * u[j]);
          } else {
            s = o[j] + u[j];
          }
          xh[i][j] = (s - st.x) * st.y;
        }
        load_param<P, VEC>(a.weight, h, 1.0f, w);
        if (have_dy) {
          rd[i].unpack(o);
        } else {
#pragma unroll
          for (int j = 0; j < VEC; ++j) o[j] = 0.0f;
        }
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          da[i][j] = o[j] * w[j];
          if (live) {
            cw[i][j] = fmaf(o[j], xh[i][j], cw[i][j]);
            cb[i][j] += o[j];
            sum.x += da[i][j];
            sum.y = fmaf(da[i][j], xh[i][j], sum.y);
          }
        }
      }
    }
    sum = row_sum2<G>(sum, s_scratch[group]);
    const float m1 = sum.x * inv, m2 = sum.y * inv;
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      if (i < col.count) {
        const int h = col.at(i);
        const bool live = col.live(i);
        float ds[VEC], dv[VEC], u[VEC], k[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) ds[j] = st.y * (da[i][j] - m1 - xh[i][j] * m2);
        if (a.grad_sum != nullptr) {
          Raw<T, VEC> raw;
          raw.load(static_cast<const T*>(a.grad_sum) + base + h);
          raw.unpack(dv);
#pragma unroll
          for (int j = 0; j < VEC; ++j) ds[j] += dv[j];
        }
        if (SCALE) load_param<P, VEC>(a.scale, h, 1.0f, k);
        ru[i].unpack(u);
        if (GATE) {
          float o[VEC], g[VEC], dg[VEC];
          ro[i].unpack(o);
          rg[i].unpack(g);
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            float yes, no;
            sigmoid_pair(g[j], yes, no);
            dg[j] = ds[j] * (o[j] - (SCALE ? u[j] * k[j] : u[j])) * (yes * no);
            dv[j] = ds[j] * no;
            ds[j] *= yes;
          }
          if (a.grad_gate != nullptr && live) store_vec(static_cast<T*>(a.grad_gate) + base + h, dg);
        } else {
#pragma unroll
          for (int j = 0; j < VEC; ++j) dv[j] = ds[j];
        }
        if (a.grad_online != nullptr && live) store_vec(static_cast<T*>(a.grad_online) + base + h, ds);
        if (SCALE) {
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            if (live) cs[SCALE ? i : 0][j] = fmaf(dv[j], u[j], cs[SCALE ? i : 0][j]);
            dv[j] *= k[j];
          }
        }
        if (a.grad_update != nullptr && live) store_vec(static_cast<T*>(a.grad_update) + base + h, dv);
      }
    }
  }
  // column sums of this CTA: its groups in order, then one row of partials per kind
  if (a.col_partials == nullptr) return;
  int kind = 0;
  auto emit = [&](float (&c)[kPieces][VEC]) {
    float* dst = a.col_partials + (static_cast<int64_t>(kind++) * gridDim.x + blockIdx.x) * H;
    if (kGroups == 1) {
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        const int h = (lane + G * i) * VEC;
        if (h < H) {
#pragma unroll
          for (int j = 0; j < VEC; ++j) dst[h + j] = c[i][j];
        }
      }
      return;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) s_cols[group * (G * kPerThread) + (lane + G * i) * VEC + j] = c[i][j];
    }
    __syncthreads();
    for (int h = threadIdx.x; h < H; h += threads_of(G)) {
      float sum = 0.0f;
#pragma unroll
      for (int g = 0; g < kGroups; ++g) sum += s_cols[g * (G * kPerThread) + h];
      dst[h] = sum;
    }
  };
  if (a.want_weight) emit(cw);
  if (a.want_bias) emit(cb);
  if constexpr (SCALE) {
    if (a.want_scale) emit(cs);
  }
}

// out_k[h] = sum over the CTAs' partials, in order: 32 columns x 8 slices per block
template <typename P>
__global__ void __launch_bounds__(256) fuse_norm_cols_kernel(const float* __restrict__ partials, int ctas, int H, P* out0, P* out1,
                                                             P* out2) {
  __shared__ float s_sum[8][32];
  const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5;
  const int h = blockIdx.x * 32 + lane;
  const float* src = partials + static_cast<int64_t>(blockIdx.y) * ctas * H;
  float sum = 0.0f;
  if (h < H) {
    for (int i = slice; i < ctas; i += 8) sum += src[static_cast<int64_t>(i) * H + h];
  }
  s_sum[slice][lane] = sum;
  __syncthreads();
  if (slice == 0 && h < H) {
    for (int i = 1; i < 8; ++i) sum += s_sum[i][lane];
    P* out = blockIdx.y == 0 ? out0 : blockIdx.y == 1 ? out1 : out2;
    out[h] = from_float<P>(sum);
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

int threads_per_row(int64_t H) { return H <= 32 * kPerThread ? 32 : H <= 128 * kPerThread ? 128 : 512; }

// CTAs of a backward pass: two per SM, or as many as there are rows
int64_t backward_ctas(int64_t rows, int64_t H) {
  const int G = threads_per_row(H);
  const int64_t per = threads_of(G) / G;
  const int64_t need = (rows + per - 1) / per;
  const int64_t most = 2 * static_cast<int64_t>(sm_count());
  return need < most ? need : most;
}

template <typename T, typename P, int VEC, int G>
void launch_fwd(const RowArgs& a, cudaStream_t s) {
  constexpr int kGroups = threads_of(G) / G;
  const int64_t need = (a.rows + kGroups - 1) / kGroups;
  const unsigned grid = static_cast<unsigned>(need < 0x7fffffffLL ? need : 0x7fffffffLL);
  if (a.gate != nullptr) fuse_norm_fwd_kernel<T, P, VEC, G, true><<<grid, threads_of(G), 0, s>>>(a);
  else fuse_norm_fwd_kernel<T, P, VEC, G, false><<<grid, threads_of(G), 0, s>>>(a);
}

template <typename T, typename P, int VEC, int G>
void launch_bwd(const RowArgs& a, cudaStream_t s) {
  const unsigned grid = static_cast<unsigned>(backward_ctas(a.rows, a.H));
  const int threads = threads_of(G);
  if (a.gate != nullptr) {
    if (a.scale != nullptr) fuse_norm_bwd_kernel<T, P, VEC, G, true, true><<<grid, threads, 0, s>>>(a);
    else fuse_norm_bwd_kernel<T, P, VEC, G, true, false><<<grid, threads, 0, s>>>(a);
  } else {
    if (a.scale != nullptr) fuse_norm_bwd_kernel<T, P, VEC, G, false, true><<<grid, threads, 0, s>>>(a);
    else fuse_norm_bwd_kernel<T, P, VEC, G, false, false><<<grid, threads, 0, s>>>(a);
  }
}

template <typename T, typename P, int VEC>
void launch_width(const RowArgs& a, bool backward, cudaStream_t s) {
  const int G = threads_per_row(a.H);
  if (!backward) {
    if (G == 32) launch_fwd<T, P, VEC, 32>(a, s);
    else if (G == 128) launch_fwd<T, P, VEC, 128>(a, s);
    else launch_fwd<T, P, VEC, 512>(a, s);
  } else {
    if (G == 32) launch_bwd<T, P, VEC, 32>(a, s);
    else if (G == 128) launch_bwd<T, P, VEC, 128>(a, s);
    else launch_bwd<T, P, VEC, 512>(a, s);
  }
}

void launch_types(const RowArgs& a, int dtype, int param_dtype, bool vec, bool backward, cudaStream_t s) {
  if (dtype == GRMX_F32) {
    if (vec) launch_width<float, float, 4>(a, backward, s);
    else launch_width<float, float, 1>(a, backward, s);
  } else if (param_dtype == GRMX_F32) {
    if (vec) launch_width<__nv_bfloat16, float, 8>(a, backward, s);
    else launch_width<__nv_bfloat16, float, 1>(a, backward, s);
  } else {
    if (vec) launch_width<__nv_bfloat16, __nv_bfloat16, 8>(a, backward, s);
    else launch_width<__nv_bfloat16, __nv_bfloat16, 1>(a, backward, s);
  }
}

int check_common(const char* who, int64_t rows, int64_t H, int dtype, int param_dtype) {
  GRMX_REQUIRE(rows >= 0 && H > 0, "%s: bad sizes", who);
  GRMX_REQUIRE(dtype == GRMX_F32 || dtype == GRMX_BF16, "%s: dtype must be f32 or bf16", who);
  GRMX_REQUIRE(param_dtype == GRMX_F32 || param_dtype == dtype, "%s: parameters must be f32 or of the rows' dtype", who);
  if (H > kMaxWidth) return fail(GRMX_ERR_UNSUPPORTED, "%s: rows of at most %d values", who, kMaxWidth);
  return GRMX_OK;
}

// 16-byte pieces where every row and every parameter starts on a 16-byte boundary
bool whole_pieces(int64_t H, int dtype, const void* const* ptrs, int n) {
  uintptr_t all = 0;
  for (int i = 0; i < n; ++i) all |= reinterpret_cast<uintptr_t>(ptrs[i]);
  return (all & 15u) == 0 && H % (dtype == GRMX_F32 ? 4 : 8) == 0;
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
  const void* ptrs[] = {online, update, gate, scale, ln_weight, ln_bias, out, sum_out};
  launch_types(a, dtype, param_dtype, whole_pieces(H, dtype, ptrs, 8), false, static_cast<cudaStream_t>(stream));
  return check_launch("fuse_norm");
}

extern "C" int64_t grmx_fuse_norm_workspace(int64_t rows, int64_t H) {
  using namespace grmx;
  if (check_common("grmx_fuse_norm_workspace", rows, H, GRMX_F32, GRMX_F32) != GRMX_OK) return -1;
  return rows == 0 ? 0 : 3 * backward_ctas(rows, H) * H * 4;
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
  const int64_t ctas = backward_ctas(rows, H);
  if (kinds > 0) {
    GRMX_REQUIRE(workspace != nullptr && workspace_bytes >= 3 * ctas * H * 4, "%s: workspace of %lld bytes, needs %lld", who,
                 (long long)workspace_bytes, (long long)(3 * ctas * H * 4));
    GRMX_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 15u) == 0, "%s: workspace must be 16-byte aligned", who);
    a.col_partials = static_cast<float*>(workspace);
  }
  const void* ptrs[] = {online, update, gate, scale, ln_weight, grad_out, grad_sum, grad_online, grad_update, grad_gate};
  launch_types(a, dtype, param_dtype, whole_pieces(H, dtype, ptrs, 10), true, s);
  int status = check_launch("fuse_norm gradient");
  if (status != GRMX_OK || kinds == 0) return status;
  void* outs[3] = {nullptr, nullptr, nullptr};
  int n = 0;
  for (void* out : {grad_weight, grad_bias, grad_scale}) {
    if (out != nullptr) outs[n++] = out;
  }
  const dim3 grid(static_cast<unsigned>((H + 31) / 32), static_cast<unsigned>(kinds));
  if (param_dtype == GRMX_F32) {
    fuse_norm_cols_kernel<float><<<grid, 256, 0, s>>>(a.col_partials, static_cast<int>(ctas), a.H, static_cast<float*>(outs[0]),
                                                       static_cast<float*>(outs[1]), static_cast<float*>(outs[2]));
  } else {
    fuse_norm_cols_kernel<__nv_bfloat16><<<grid, 256, 0, s>>>(
        a.col_partials, static_cast<int>(ctas), a.H, static_cast<__nv_bfloat16*>(outs[0]), static_cast<__nv_bfloat16*>(outs[1]),
        static_cast<__nv_bfloat16*>(outs[2]));
  }
  return check_launch("fuse_norm column sums");
}
