// PyTorch face of the engine: registers torch.ops.grm_cuda.* with the schemas
// of the reference extension (grm/csrc/bindings.cpp:5-11) for the CUDA
// dispatch key, plus torch.ops.grmx.* for the calls the reference has no op
// for.  Every kernel is reached through the C ABI of grmx.h; this file only
// checks shapes, allocates outputs from the caching allocator and passes the
// current stream.  There is no CPU registration: a CPU tensor fails loudly in
// the dispatcher.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <torch/csrc/autograd/functions/basic_ops.h>

#include <array>
#include <atomic>
#include <cmath>
#include <initializer_list>
#include <tuple>

#include "grmx.h"

namespace {

std::atomic<int> g_scan_path{GRMX_PATH_AUTO};

int dtype_code(at::ScalarType t, const char* what) {
  switch (t) {
    case at::kFloat: return GRMX_F32;
    case at::kBFloat16: return GRMX_BF16;
    case at::kHalf: return GRMX_F16;
    default: TORCH_CHECK(false, "grm_cuda: ", what, " has unsupported dtype ", t, " (float32, bfloat16, float16)");
  }
  return -1;
}

void check_status(int rc) { TORCH_CHECK(rc == GRMX_OK, "grm_cuda: ", grmx_last_error()); }

void* current_stream() { return static_cast<void*>(at::cuda::getCurrentCUDAStream().stream()); }

void require_cuda(const at::Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda(), "grm_cuda: ", name, " must be a CUDA tensor (this engine has no CPU path)");
}

// shape contract of the reference: grm/csrc/grm_cuda.cpp:13-27
void check_chunk_inputs(const at::Tensor& keys, const at::Tensor& values, const at::Tensor& queries,
                        const at::Tensor& memory) {
  TORCH_CHECK(keys.dim() == 3, "keys must have shape [B, T, K]");
  TORCH_CHECK(values.dim() == 3, "values must have shape [B, T, H]");
  TORCH_CHECK(queries.dim() == 3, "queries must have shape [B, T, K]");
  TORCH_CHECK(memory.dim() == 3, "memory must have shape [B, H, K]");
  TORCH_CHECK(keys.sizes().slice(0, 2) == values.sizes().slice(0, 2), "keys and values batch/time dims must match");
  TORCH_CHECK(keys.sizes() == queries.sizes(), "keys and queries must have the same shape");
  TORCH_CHECK(values.size(0) == memory.size(0), "memory batch dim must match values batch dim");
  TORCH_CHECK(values.size(2) == memory.size(1), "memory hidden dim must match values hidden dim");
  TORCH_CHECK(keys.size(2) == memory.size(2), "memory key dim must match keys key dim");
  require_cuda(keys, "keys");
  require_cuda(values, "values");
  require_cuda(queries, "queries");
  require_cuda(memory, "memory");
  TORCH_CHECK(keys.scalar_type() == values.scalar_type() && keys.scalar_type() == queries.scalar_type(),
              "grm_cuda: keys, values and queries must share one dtype");
  TORCH_CHECK(memory.scalar_type() == at::kFloat || memory.scalar_type() == keys.scalar_type(),
              "grm_cuda: memory must be float32 or have the dtype of keys");
}

// grm/csrc/grm_cuda.cpp:29-42
void check_apply_query_inputs(const at::Tensor& memories, const at::Tensor& queries) {
  TORCH_CHECK(memories.dim() == 4 || memories.dim() == 5, "memories must have shape [B, R, H, K] or [B, Q, R, H, K]");
  if (memories.dim() == 4) {
    TORCH_CHECK(queries.dim() == 2, "queries must have shape [B, K] when memories rank is 4");
    TORCH_CHECK(memories.size(0) == queries.size(0), "batch dim mismatch between memories and queries");
    TORCH_CHECK(memories.size(3) == queries.size(1), "key dim mismatch between memories and queries");
  } else {
    TORCH_CHECK(queries.dim() == 3, "queries must have shape [B, Q, K] when memories rank is 5");
    TORCH_CHECK(memories.size(0) == queries.size(0), "batch dim mismatch between memories and queries");
    TORCH_CHECK(memories.size(1) == queries.size(1), "query dim mismatch between memories and queries");
    TORCH_CHECK(memories.size(4) == queries.size(2), "key dim mismatch between memories and queries");
  }
  require_cuda(memories, "memories");
  require_cuda(queries, "queries");
  TORCH_CHECK(memories.scalar_type() == queries.scalar_type(), "grm_cuda: memories and queries must share one dtype");
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> chunk_update_forward_cuda(
    const at::Tensor& keys, const at::Tensor& values, const at::Tensor& queries,
    const at::Tensor& memory, double memory_decay) {
  check_chunk_inputs(keys, values, queries, memory);
  c10::cuda::CUDAGuard guard(keys.device());
  auto k = keys.contiguous();
  auto v = values.contiguous();
  auto q = queries.contiguous();
  auto m = memory.contiguous();
  const int64_t B = k.size(0), T = k.size(1), K = k.size(2), H = v.size(2);
  auto aux = at::empty({0}, m.options());
  if (T == 0) {
    return {at::zeros({B, 0, H}, v.options()), m, aux};
  }
  auto hidden = at::empty({B, T, H}, v.options());
  auto memory_out = at::empty_like(m);
  const int io = dtype_code(k.scalar_type(), "keys");
  const int st = dtype_code(m.scalar_type(), "memory");
  // few rows, many tokens: give the kernel a workspace so it can cut the rows along T
  // Few rows and many tokens: the scan is cut along T.  Up to four pieces the library does that in one
  // launch without a workspace; the two-kernel form over a workspace pays when the call allows more
  // pieces than that, i.e. when the workspace holds five or more piece states per row.
  int64_t scratch_bytes = g_scan_path.load() == GRMX_PATH_FFMA ? 0 : grmx_chunk_scan_scratch_bytes(B, T, K, H, io, st);
  if (scratch_bytes < 5 * B * H * K * static_cast<int64_t>(sizeof(float))) scratch_bytes = 0;
  at::Tensor scratch;
  if (scratch_bytes > 0) scratch = at::empty({scratch_bytes}, k.options().dtype(at::kByte));
  check_status(grmx_chunk_scan_fwd_ws(k.data_ptr(), v.data_ptr(), q.data_ptr(), m.data_ptr(),
                                      hidden.data_ptr(), memory_out.data_ptr(), B, T, K, H,
                                      static_cast<float>(memory_decay), io, st, g_scan_path.load(),
                                      scratch_bytes > 0 ? scratch.data_ptr() : nullptr, scratch_bytes,
                                      current_stream()));
  return {hidden, memory_out, aux};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> chunk_update_backward_cuda(
    const at::Tensor& grad_hidden, const at::Tensor& grad_memory_out, const at::Tensor& keys,
    const at::Tensor& values, const at::Tensor& queries, const at::Tensor& memory,
    const at::Tensor& aux, double memory_decay) {
  (void)aux;
  check_chunk_inputs(keys, values, queries, memory);
  require_cuda(grad_hidden, "grad_hidden");
  require_cuda(grad_memory_out, "grad_memory_out");
  TORCH_CHECK(grad_hidden.sizes() == values.sizes(), "grad_hidden must have the shape of values");
  TORCH_CHECK(grad_memory_out.sizes() == memory.sizes(), "grad_memory_out must have the shape of memory");
  c10::cuda::CUDAGuard guard(keys.device());
  auto k = keys.contiguous();
  auto v = values.contiguous();
  auto q = queries.contiguous();
  auto m = memory.contiguous();
  auto gh = grad_hidden.to(v.scalar_type()).contiguous();
  auto gm = grad_memory_out.to(m.scalar_type()).contiguous();
  const int64_t B = k.size(0), T = k.size(1), K = k.size(2), H = v.size(2);
  auto grad_k = at::empty_like(k);
  auto grad_v = at::empty_like(v);
  auto grad_q = at::empty_like(q);
  auto grad_m = at::empty_like(m);
  check_status(grmx_chunk_scan_bwd(gh.data_ptr(), gm.data_ptr(), k.data_ptr(), v.data_ptr(), q.data_ptr(),
                                   m.data_ptr(), grad_k.data_ptr(), grad_v.data_ptr(), grad_q.data_ptr(),
                                   grad_m.data_ptr(), B, T, K, H, static_cast<float>(memory_decay),
                                   dtype_code(k.scalar_type(), "keys"), dtype_code(m.scalar_type(), "memory"),
                                   g_scan_path.load(), current_stream()));
  return {grad_k, grad_v, grad_q, grad_m};
}

at::Tensor apply_query_forward_cuda(const at::Tensor& memories, const at::Tensor& queries) {
  check_apply_query_inputs(memories, queries);
  c10::cuda::CUDAGuard guard(memories.device());
  auto mem = memories.contiguous();
  auto q = queries.contiguous();
  const bool rank5 = mem.dim() == 5;
  const int64_t N = rank5 ? mem.size(0) * mem.size(1) : mem.size(0);
  const int64_t R = mem.size(rank5 ? 2 : 1), H = mem.size(rank5 ? 3 : 2), K = mem.size(rank5 ? 4 : 3);
  at::Tensor hidden = rank5 ? at::empty({mem.size(0), mem.size(1), R, H}, mem.options())
                            : at::empty({mem.size(0), R, H}, mem.options());
  if (K == 0) hidden.zero_();
  check_status(grmx_apply_query_fwd(mem.data_ptr(), q.data_ptr(), hidden.data_ptr(), N, R, H, K,
                                    dtype_code(mem.scalar_type(), "memories"), current_stream()));
  return hidden;
}

std::tuple<at::Tensor, at::Tensor> apply_query_backward_cuda(const at::Tensor& grad_hidden,
                                                             const at::Tensor& memories,
                                                             const at::Tensor& queries) {
  check_apply_query_inputs(memories, queries);
  require_cuda(grad_hidden, "grad_hidden");
  c10::cuda::CUDAGuard guard(memories.device());
  auto mem = memories.contiguous();
  auto q = queries.contiguous();
  auto gh = grad_hidden.to(mem.scalar_type()).contiguous();
  const bool rank5 = mem.dim() == 5;
  const int64_t N = rank5 ? mem.size(0) * mem.size(1) : mem.size(0);
  const int64_t R = mem.size(rank5 ? 2 : 1), H = mem.size(rank5 ? 3 : 2), K = mem.size(rank5 ? 4 : 3);
  TORCH_CHECK(gh.numel() == N * R * H, "grad_hidden has the wrong number of elements");
  auto grad_mem = at::empty_like(mem);
  auto grad_q = at::empty_like(q);
  check_status(grmx_apply_query_bwd(gh.data_ptr(), mem.data_ptr(), q.data_ptr(), grad_mem.data_ptr(),
                                    grad_q.data_ptr(), N, R, H, K, dtype_code(mem.scalar_type(), "memories"),
                                    current_stream()));
  return {grad_mem, grad_q};
}

// grm/csrc/grm_cuda.cpp:156-161
at::Tensor batched_memory_gather_cuda(const at::Tensor& memories_per_batch, const at::Tensor& topk_indices) {
  TORCH_CHECK(memories_per_batch.dim() == 4, "memories_per_batch must have shape [B, S, H, K]");
  TORCH_CHECK(topk_indices.dim() == 2 || topk_indices.dim() == 3, "topk_indices must have shape [B, R] or [B, Q, R]");
  TORCH_CHECK(memories_per_batch.size(0) == topk_indices.size(0),
              "batch dim mismatch between memories_per_batch and topk_indices");
  require_cuda(memories_per_batch, "memories_per_batch");
  require_cuda(topk_indices, "topk_indices");
  c10::cuda::CUDAGuard guard(memories_per_batch.device());
  auto mem = memories_per_batch.contiguous();
  auto idx = topk_indices.toType(at::kLong).contiguous();
  const int64_t B = mem.size(0), S = mem.size(1), H = mem.size(2), K = mem.size(3);
  dtype_code(mem.scalar_type(), "memories_per_batch");
  std::vector<int64_t> shape(idx.sizes().begin(), idx.sizes().end());
  shape.push_back(H);
  shape.push_back(K);
  auto out = at::empty(shape, mem.options());
  const int64_t J = B > 0 ? idx.numel() / B : 0;
  check_status(grmx_batched_gather(mem.data_ptr(), idx.data_ptr<int64_t>(), out.data_ptr(), B, S, J, H * K,
                                   static_cast<int>(mem.element_size()), current_stream()));
  return out;
}

// ---- calls with no counterpart op in the reference (namespace grmx) ----

std::tuple<at::Tensor, at::Tensor> linear_scan_cuda(const at::Tensor& keys, const at::Tensor& values,
                                                    const at::Tensor& queries, const at::Tensor& memory,
                                                    double decay, double update_coeff, double hidden_scale,
                                                    double memory_out_scale, bool reverse,
                                                    bool first_step_no_decay, int64_t path) {
  check_chunk_inputs(keys, values, queries, memory);
  c10::cuda::CUDAGuard guard(keys.device());
  auto k = keys.contiguous();
  auto v = values.contiguous();
  auto q = queries.contiguous();
  auto m = memory.contiguous();
  const int64_t B = k.size(0), T = k.size(1), K = k.size(2), H = v.size(2);
  auto hidden = at::empty({B, T, H}, v.options());
  auto memory_out = at::empty_like(m);
  check_status(grmx_linear_scan(k.data_ptr(), v.data_ptr(), q.data_ptr(), m.data_ptr(), K, 1,
                                hidden.data_ptr(), memory_out.data_ptr(), B, T, K, H,
                                static_cast<float>(decay), static_cast<float>(update_coeff),
                                static_cast<float>(hidden_scale), static_cast<float>(memory_out_scale),
                                reverse ? 1 : 0, first_step_no_decay ? 1 : 0,
                                dtype_code(k.scalar_type(), "keys"), dtype_code(m.scalar_type(), "memory"),
                                static_cast<int>(path), current_stream()));
  return {hidden, memory_out};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> topk_route_cuda(const at::Tensor& queries,
                                                               const at::Tensor& keys,
                                                               const c10::optional<at::Tensor>& visible,
                                                               int64_t top_k, double scale,
                                                               double temperature, bool return_scores) {
  TORCH_CHECK(queries.dim() == 3, "queries must have shape [B, Q, D]");
  TORCH_CHECK(keys.dim() == 3, "keys must have shape [B, S, D]");
  TORCH_CHECK(queries.size(0) == keys.size(0), "batch dim mismatch between queries and keys");
  TORCH_CHECK(queries.size(2) == keys.size(2), "feature dim mismatch between queries and keys");
  require_cuda(queries, "queries");
  require_cuda(keys, "keys");
  c10::cuda::CUDAGuard guard(queries.device());
  auto k = keys.to(at::kFloat).contiguous();
  const int64_t B = queries.size(0), Q = queries.size(1), D = queries.size(2), S = k.size(1);
  // bf16 queries of the per-token shapes are read as they are (grmx_topk_route_bf16q); everything else
  // is widened to fp32 first
  at::Tensor q = queries.contiguous();
  const bool lowp = q.scalar_type() == at::kBFloat16 && S >= 1 && S <= 16 && Q >= 64 && D >= 8 && D % 8 == 0 &&
                    D <= 1024 && B <= 65535 && (reinterpret_cast<uintptr_t>(q.data_ptr()) & 15u) == 0 &&
                    (reinterpret_cast<uintptr_t>(k.data_ptr()) & 15u) == 0;
  if (!lowp) q = q.to(at::kFloat);
  at::Tensor vis;
  const int32_t* vis_ptr = nullptr;
  if (visible.has_value() && visible->defined()) {
    require_cuda(*visible, "visible");
    TORCH_CHECK(visible->numel() == Q, "visible must hold one count per query");
    vis = visible->to(at::kInt).contiguous();
    vis_ptr = vis.data_ptr<int32_t>();
  }
  auto idx = at::empty({B, Q, top_k}, k.options().dtype(at::kLong));
  auto gates = at::empty({B, Q, top_k}, k.options());
  at::Tensor scores = return_scores ? at::empty({B, Q, S}, k.options()) : at::empty({0}, k.options());
  if (lowp) {
    check_status(grmx_topk_route_bf16q(q.data_ptr(), k.data_ptr<float>(), vis_ptr, B, Q, S, D,
                                       static_cast<int>(top_k), static_cast<float>(scale),
                                       static_cast<float>(temperature), idx.data_ptr<int64_t>(),
                                       gates.data_ptr<float>(), return_scores ? scores.data_ptr<float>() : nullptr,
                                       current_stream()));
    return {gates, idx, scores};
  }
  check_status(grmx_topk_route(q.data_ptr<float>(), k.data_ptr<float>(), vis_ptr, B, Q, S, D,
                               static_cast<int>(top_k), static_cast<float>(scale),
                               static_cast<float>(temperature), idx.data_ptr<int64_t>(),
                               gates.data_ptr<float>(), return_scores ? scores.data_ptr<float>() : nullptr,
                               current_stream()));
  return {gates, idx, scores};
}

// selection and gates on scores the caller holds (after masking with -inf, say): [B,Q,S] -> gates, indices [B,Q,top_k]
std::tuple<at::Tensor, at::Tensor> topk_select_cuda(const at::Tensor& scores, const c10::optional<at::Tensor>& visible,
                                                    int64_t top_k, double temperature) {
  TORCH_CHECK(scores.dim() == 3, "scores must have shape [B, Q, S]");
  require_cuda(scores, "scores");
  c10::cuda::CUDAGuard guard(scores.device());
  auto sc = scores.to(at::kFloat).contiguous();
  const int64_t B = sc.size(0), Q = sc.size(1), S = sc.size(2);
  at::Tensor vis;
  const int32_t* vis_ptr = nullptr;
  if (visible.has_value() && visible->defined()) {
    require_cuda(*visible, "visible");
    TORCH_CHECK(visible->numel() == Q, "visible must hold one count per query");
    vis = visible->to(at::kInt).contiguous();
    vis_ptr = vis.data_ptr<int32_t>();
  }
  auto idx = at::empty({B, Q, top_k}, sc.options().dtype(at::kLong));
  auto gates = at::empty({B, Q, top_k}, sc.options());
  check_status(grmx_topk_select(sc.data_ptr<float>(), vis_ptr, B, Q, S, static_cast<int>(top_k),
                                static_cast<float>(temperature), idx.data_ptr<int64_t>(), gates.data_ptr<float>(),
                                current_stream()));
  return {gates, idx};
}

// states [B,Q,S,H] (fp32 or bf16), indices [B,Q,R], gates [B,Q,R] -> [B,Q,H] in the dtype of states
at::Tensor select_fuse_cuda(const at::Tensor& states, const at::Tensor& indices, const at::Tensor& gates,
                            const c10::optional<at::Tensor>& online, const c10::optional<at::Tensor>& ln_weight,
                            const c10::optional<at::Tensor>& ln_bias, double ln_eps, int64_t mode) {
  TORCH_CHECK(states.dim() == 4, "states must have shape [B, Q, S, H]");
  TORCH_CHECK(indices.dim() == 3 && gates.dim() == 3, "indices and gates must have shape [B, Q, R]");
  TORCH_CHECK(indices.sizes() == gates.sizes(), "indices and gates differ in shape");
  TORCH_CHECK(states.size(0) == indices.size(0) && states.size(1) == indices.size(1), "batch/query dim mismatch");
  require_cuda(states, "states");
  require_cuda(indices, "indices");
  require_cuda(gates, "gates");
  TORCH_CHECK(states.scalar_type() == at::kFloat || states.scalar_type() == at::kBFloat16,
              "states must be float32 or bfloat16");
  c10::cuda::CUDAGuard guard(states.device());
  auto st = states.contiguous();
  auto idx = indices.toType(at::kLong).contiguous();
  auto g = gates.to(at::kFloat).contiguous();
  const int64_t B = st.size(0), Q = st.size(1), S = st.size(2), H = st.size(3), R = idx.size(2);
  at::Tensor o_keep, w_keep, b_keep;
  const void* o_ptr = nullptr;
  if (online.has_value() && online->defined()) {
    require_cuda(*online, "online");
    o_keep = online->to(st.scalar_type()).contiguous();
    TORCH_CHECK(o_keep.sizes() == at::IntArrayRef({B, Q, H}), "online has the wrong shape");
    o_ptr = o_keep.data_ptr();
  }
  auto opt = [&](const c10::optional<at::Tensor>& t, const char* name, at::Tensor& keep) -> const float* {
    if (!t.has_value() || !t->defined()) return nullptr;
    require_cuda(*t, name);
    keep = t->to(at::kFloat).contiguous();
    TORCH_CHECK(keep.numel() == H, name, " has the wrong shape");
    return keep.data_ptr<float>();
  };
  const float* w_ptr = opt(ln_weight, "ln_weight", w_keep);
  const float* b_ptr = opt(ln_bias, "ln_bias", b_keep);
  at::Tensor out = at::empty({B, Q, H}, st.options());
  check_status(grmx_select_fuse(st.data_ptr(), idx.data_ptr<int64_t>(), g.data_ptr<float>(), o_ptr, w_ptr, b_ptr,
                                static_cast<float>(ln_eps), out.data_ptr(), B, Q, S, R, H,
                                st.scalar_type() == at::kFloat ? GRMX_F32 : GRMX_BF16, static_cast<int>(mode),
                                current_stream()));
  return out;
}

// LayerNorm(a + b) over the last dimension (fp32 or bf16 rows of whole 16-byte pieces, H <= 1024)
at::Tensor add_layer_norm_cuda(const at::Tensor& a, const at::Tensor& b, const c10::optional<at::Tensor>& ln_weight,
                               const c10::optional<at::Tensor>& ln_bias, double ln_eps) {
  TORCH_CHECK(a.sizes() == b.sizes() && a.dim() >= 1, "a and b must have the same shape");
  TORCH_CHECK(a.scalar_type() == b.scalar_type() && (a.scalar_type() == at::kFloat || a.scalar_type() == at::kBFloat16),
              "a and b must both be float32 or bfloat16");
  require_cuda(a, "a");
  require_cuda(b, "b");
  c10::cuda::CUDAGuard guard(a.device());
  auto ca = a.contiguous(), cb = b.contiguous();
  const int64_t H = ca.size(-1);
  const int64_t rows = H > 0 ? ca.numel() / H : 0;
  at::Tensor w_keep, b_keep;
  auto opt = [&](const c10::optional<at::Tensor>& t, const char* name, at::Tensor& keep) -> const float* {
    if (!t.has_value() || !t->defined()) return nullptr;
    require_cuda(*t, name);
    keep = t->to(at::kFloat).contiguous();
    TORCH_CHECK(keep.numel() == H, name, " has the wrong shape");
    return keep.data_ptr<float>();
  };
  const float* w_ptr = opt(ln_weight, "ln_weight", w_keep);
  const float* b_ptr = opt(ln_bias, "ln_bias", b_keep);
  at::Tensor out = at::empty_like(ca);
  check_status(grmx_add_layer_norm(ca.data_ptr(), cb.data_ptr(), w_ptr, b_ptr, static_cast<float>(ln_eps), out.data_ptr(),
                                   rows, H, ca.scalar_type() == at::kFloat ? GRMX_F32 : GRMX_BF16, current_stream()));
  return out;
}

std::tuple<at::Tensor, at::Tensor> chunk_scan_segments_cuda(const at::Tensor& keys, const at::Tensor& values,
                                                            const at::Tensor& queries, const at::Tensor& memory,
                                                            double memory_decay, at::Tensor archive, int64_t first_slot,
                                                            int64_t segment_tokens) {
  check_chunk_inputs(keys, values, queries, memory);
  TORCH_CHECK(archive.is_cuda() && archive.dim() == 4 && archive.scalar_type() == at::kFloat && archive.is_contiguous(),
              "archive must be a contiguous float32 CUDA tensor [B, capacity, H, K]");
  c10::cuda::CUDAGuard guard(keys.device());
  auto k = keys.contiguous();
  auto v = values.contiguous();
  auto q = queries.contiguous();
  auto m = memory.contiguous();
  const int64_t B = k.size(0), T = k.size(1), K = k.size(2), H = v.size(2);
  TORCH_CHECK(archive.size(0) == B && archive.size(2) == H && archive.size(3) == K, "archive does not match the scan");
  auto hidden = at::empty({B, T, H}, v.options());
  auto memory_out = at::empty_like(m);
  check_status(grmx_chunk_scan_fwd_segments(k.data_ptr(), v.data_ptr(), q.data_ptr(), m.data_ptr(), hidden.data_ptr(),
                                            memory_out.data_ptr(), archive.data_ptr<float>(), archive.size(1),
                                            first_slot, segment_tokens, B, T, K, H, static_cast<float>(memory_decay),
                                            dtype_code(k.scalar_type(), "keys"), dtype_code(m.scalar_type(), "memory"),
                                            current_stream()));
  return {hidden, memory_out};
}

at::Tensor l2_normalize_cuda(const at::Tensor& x, double eps, bool to_bfloat16) {
  TORCH_CHECK(x.is_cuda(), "l2_normalize needs a CUDA tensor");
  TORCH_CHECK(x.dim() >= 1, "l2_normalize needs at least one dimension");
  TORCH_CHECK(x.scalar_type() == at::kFloat || x.scalar_type() == at::kBFloat16, "l2_normalize takes float32 or bfloat16");
  c10::cuda::CUDAGuard guard(x.device());
  auto in = x.contiguous();
  const bool cast = to_bfloat16 && in.scalar_type() == at::kFloat;
  auto out = at::empty_like(in, cast ? in.options().dtype(at::kBFloat16) : in.options());
  const int64_t K = in.size(-1);
  const int64_t N = K == 0 ? 0 : in.numel() / K;
  check_status(grmx_normalize_rows(in.data_ptr(), out.data_ptr(), N, K, static_cast<float>(eps),
                                   in.scalar_type() == at::kFloat ? GRMX_F32 : GRMX_BF16,
                                   out.scalar_type() == at::kFloat ? GRMX_F32 : GRMX_BF16, current_stream()));
  return out;
}

// x bf16 [..., D], weights bf16 [128, D] (two stacked 64-row matrices), bias fp32 [128]? -> two bf16 [..., 64]
std::tuple<at::Tensor, at::Tensor> project_normalize_cuda(const at::Tensor& x, const at::Tensor& weights,
                                                          const c10::optional<at::Tensor>& bias, double eps) {
  TORCH_CHECK(x.is_cuda() && weights.is_cuda(), "project_normalize needs CUDA tensors");
  TORCH_CHECK(x.scalar_type() == at::kBFloat16 && weights.scalar_type() == at::kBFloat16, "x and weights must be bfloat16");
  TORCH_CHECK(x.dim() >= 2 && weights.dim() == 2 && weights.size(1) == x.size(-1) && weights.size(0) % 2 == 0,
              "weights must be [2K, D] for x [..., D]");
  c10::cuda::CUDAGuard guard(x.device());
  auto in = x.contiguous();
  auto w = weights.contiguous();
  const int64_t D = in.size(-1), K = w.size(0) / 2;
  const int64_t rows = in.numel() / D;
  at::Tensor b_keep;
  const float* b_ptr = nullptr;
  if (bias.has_value() && bias->defined()) {
    b_keep = bias->to(at::kFloat).contiguous();
    TORCH_CHECK(b_keep.numel() == 2 * K, "bias must hold 2K values");
    b_ptr = b_keep.data_ptr<float>();
  }
  std::vector<int64_t> shape(in.sizes().begin(), in.sizes().end());
  shape.back() = K;
  auto a = at::empty(shape, in.options());
  auto b = at::empty(shape, in.options());
  check_status(grmx_project_normalize(in.data_ptr(), w.data_ptr(), b_ptr, a.data_ptr(), b.data_ptr(), rows, D, K,
                                      static_cast<float>(eps), current_stream()));
  return {a, b};
}

void archive_push_cuda(const at::Tensor& memory, at::Tensor archive, c10::optional<at::Tensor> shadow, int64_t slot) {
  TORCH_CHECK(archive.dim() == 4 && memory.dim() == 3, "memory [B, H, K] goes into archive [B, S, H, K]");
  TORCH_CHECK(memory.is_cuda() && archive.is_cuda(), "archive_push needs CUDA tensors");
  TORCH_CHECK(memory.scalar_type() == at::kFloat && archive.scalar_type() == at::kFloat, "memory and archive are float32");
  TORCH_CHECK(archive.is_contiguous(), "archive must be contiguous: it is written in place");
  const int64_t B = archive.size(0), S = archive.size(1), H = archive.size(2), K = archive.size(3);
  TORCH_CHECK(memory.size(0) == B && memory.size(1) == H && memory.size(2) == K, "memory does not match the archive");
  void* shadow_ptr = nullptr;
  if (shadow.has_value() && shadow->defined()) {
    TORCH_CHECK(shadow->scalar_type() == at::kBFloat16 && shadow->is_contiguous() && shadow->sizes() == archive.sizes() &&
                    shadow->is_cuda(), "the bf16 ring must be a contiguous bfloat16 CUDA tensor shaped like the archive");
    shadow_ptr = shadow->data_ptr();
  }
  c10::cuda::CUDAGuard guard(archive.device());
  auto mem = memory.contiguous();
  check_status(grmx_archive_push(mem.data_ptr<float>(), archive.data_ptr<float>(), shadow_ptr, B, S, slot, H * K,
                                 current_stream()));
}

at::Tensor retrieve_fuse_cuda(const at::Tensor& archive, const at::Tensor& indices,
                              const c10::optional<at::Tensor>& gates, const at::Tensor& queries,
                              const c10::optional<at::Tensor>& online,
                              const c10::optional<at::Tensor>& ln_weight,
                              const c10::optional<at::Tensor>& ln_bias, double ln_eps, int64_t mode) {
  TORCH_CHECK(archive.dim() == 4, "archive must have shape [B, S, H, K]");
  TORCH_CHECK(indices.dim() == 3, "indices must have shape [B, Q, R]");
  TORCH_CHECK(queries.dim() == 3, "queries must have shape [B, Q, K]");
  TORCH_CHECK(archive.size(0) == indices.size(0) && archive.size(0) == queries.size(0), "batch dim mismatch");
  TORCH_CHECK(indices.size(1) == queries.size(1), "query dim mismatch between indices and queries");
  TORCH_CHECK(archive.size(3) == queries.size(2), "key dim mismatch between archive and queries");
  require_cuda(archive, "archive");
  require_cuda(indices, "indices");
  require_cuda(queries, "queries");
  TORCH_CHECK(archive.scalar_type() == at::kFloat, "archive must be float32");
  c10::cuda::CUDAGuard guard(archive.device());
  auto arch = archive.contiguous();
  auto idx = indices.toType(at::kLong).contiguous();
  auto q = queries.to(at::kFloat).contiguous();
  const int64_t B = arch.size(0), S = arch.size(1), H = arch.size(2), K = arch.size(3);
  const int64_t Q = idx.size(1), R = idx.size(2);
  auto opt = [&](const c10::optional<at::Tensor>& t, std::vector<int64_t> shape, const char* name,
                 at::Tensor& keep) -> const float* {
    if (!t.has_value() || !t->defined()) return nullptr;
    require_cuda(*t, name);
    keep = t->to(at::kFloat).contiguous();
    TORCH_CHECK(keep.sizes() == at::IntArrayRef(shape), name, " has the wrong shape");
    return keep.data_ptr<float>();
  };
  at::Tensor g_keep, o_keep, w_keep, b_keep;
  const float* g_ptr = opt(gates, {B, Q, R}, "gates", g_keep);
  const float* o_ptr = opt(online, {B, Q, H}, "online", o_keep);
  const float* w_ptr = opt(ln_weight, {H}, "ln_weight", w_keep);
  const float* b_ptr = opt(ln_bias, {H}, "ln_bias", b_keep);
  at::Tensor out = mode == GRMX_FUSE_RETRIEVED ? at::empty({B, Q, R, H}, arch.options())
                                               : at::empty({B, Q, H}, arch.options());
  check_status(grmx_retrieve_fuse(arch.data_ptr<float>(), idx.data_ptr<int64_t>(), g_ptr,
                                  q.data_ptr<float>(), o_ptr, w_ptr, b_ptr, static_cast<float>(ln_eps),
                                  out.data_ptr(), B, S, Q, R, H, K, static_cast<int>(mode),
                                  current_stream()));
  return out;
}

// bf16 archive ring [B,S,H,K], bf16 queries [B,Q,K], bf16 online [B,Q,H] -> bf16 [B,Q,H] (tensor-core retrieval)
at::Tensor retrieve_fuse_tc_cuda(const at::Tensor& archive, const at::Tensor& indices, const at::Tensor& gates,
                                 const at::Tensor& queries, const c10::optional<at::Tensor>& online,
                                 const c10::optional<at::Tensor>& ln_weight, const c10::optional<at::Tensor>& ln_bias,
                                 double ln_eps, int64_t mode) {
  TORCH_CHECK(archive.dim() == 4, "archive must have shape [B, S, H, K]");
  TORCH_CHECK(indices.dim() == 3 && gates.dim() == 3 && indices.sizes() == gates.sizes(),
              "indices and gates must have shape [B, Q, R]");
  TORCH_CHECK(queries.dim() == 3, "queries must have shape [B, Q, K]");
  TORCH_CHECK(archive.size(0) == indices.size(0) && archive.size(0) == queries.size(0), "batch dim mismatch");
  TORCH_CHECK(indices.size(1) == queries.size(1), "query dim mismatch between indices and queries");
  TORCH_CHECK(archive.size(3) == queries.size(2), "key dim mismatch between archive and queries");
  require_cuda(archive, "archive");
  require_cuda(indices, "indices");
  require_cuda(gates, "gates");
  require_cuda(queries, "queries");
  TORCH_CHECK(archive.scalar_type() == at::kBFloat16 && queries.scalar_type() == at::kBFloat16,
              "archive and queries must be bfloat16");
  c10::cuda::CUDAGuard guard(archive.device());
  auto arch = archive.contiguous();
  auto idx = indices.toType(at::kLong).contiguous();
  auto g = gates.to(at::kFloat).contiguous();
  auto q = queries.contiguous();
  const int64_t B = arch.size(0), S = arch.size(1), H = arch.size(2), K = arch.size(3);
  const int64_t Q = idx.size(1), R = idx.size(2);
  at::Tensor o_keep, w_keep, b_keep;
  const void* o_ptr = nullptr;
  if (online.has_value() && online->defined()) {
    require_cuda(*online, "online");
    o_keep = online->to(at::kBFloat16).contiguous();
    TORCH_CHECK(o_keep.sizes() == at::IntArrayRef({B, Q, H}), "online has the wrong shape");
    o_ptr = o_keep.data_ptr();
  }
  auto opt = [&](const c10::optional<at::Tensor>& t, const char* name, at::Tensor& keep) -> const float* {
    if (!t.has_value() || !t->defined()) return nullptr;
    require_cuda(*t, name);
    keep = t->to(at::kFloat).contiguous();
    TORCH_CHECK(keep.numel() == H, name, " has the wrong shape");
    return keep.data_ptr<float>();
  };
  const float* w_ptr = opt(ln_weight, "ln_weight", w_keep);
  const float* b_ptr = opt(ln_bias, "ln_bias", b_keep);
  at::Tensor out = at::empty({B, Q, H}, arch.options());
  check_status(grmx_retrieve_fuse_tc(arch.data_ptr(), idx.data_ptr<int64_t>(), g.data_ptr<float>(), q.data_ptr(), o_ptr,
                                     w_ptr, b_ptr, static_cast<float>(ln_eps), out.data_ptr(), B, S, Q, R, H, K,
                                     static_cast<int>(mode), current_stream()));
  return out;
}

// ---- vocabulary loss: hidden [...,D] and weight [V,D] (bf16 or fp32), targets int64 [...], bias [V]? ----

struct LossArgs {
  at::Tensor hidden, weight, targets, bias;
  int64_t N, D, V;
  int dtype, bias_dtype;
};

LossArgs check_loss_inputs(const at::Tensor& hidden, const at::Tensor& weight, const at::Tensor& targets,
                           const c10::optional<at::Tensor>& bias, int64_t reduction) {
  TORCH_CHECK(hidden.dim() >= 1, "hidden must have shape [..., D]");
  TORCH_CHECK(weight.dim() == 2, "weight must have shape [V, D]");
  TORCH_CHECK(hidden.size(-1) == weight.size(1), "feature dim mismatch between hidden and weight");
  TORCH_CHECK(targets.sizes() == hidden.sizes().slice(0, hidden.dim() - 1), "targets must have the shape of hidden without its features");
  TORCH_CHECK(weight.size(0) > 0 && weight.size(1) > 0, "weight must not be empty");
  require_cuda(hidden, "hidden");
  require_cuda(weight, "weight");
  require_cuda(targets, "targets");
  TORCH_CHECK(weight.device() == hidden.device() && targets.device() == hidden.device(),
              "hidden, weight and targets must be on one device");
  TORCH_CHECK(hidden.scalar_type() == at::kFloat || hidden.scalar_type() == at::kBFloat16,
              "hidden must be float32 or bfloat16");
  TORCH_CHECK(weight.scalar_type() == hidden.scalar_type(), "hidden and weight must share one dtype");
  TORCH_CHECK(targets.scalar_type() == at::kLong || targets.scalar_type() == at::kInt, "targets must be int64 or int32");
  TORCH_CHECK(reduction >= GRMX_REDUCE_NONE && reduction <= GRMX_REDUCE_MEAN, "reduction must be 0 (none), 1 (sum) or 2 (mean)");
  LossArgs a;
  a.hidden = hidden.contiguous();
  a.weight = weight.contiguous();
  a.targets = targets.to(at::kLong).contiguous();
  a.N = targets.numel();
  a.D = weight.size(1);
  a.V = weight.size(0);
  a.dtype = a.bias_dtype = dtype_code(hidden.scalar_type(), "hidden");
  if (bias.has_value() && bias->defined()) {
    require_cuda(*bias, "bias");
    TORCH_CHECK(bias->device() == hidden.device(), "bias must be on the device of hidden");
    TORCH_CHECK(bias->dim() == 1 && bias->size(0) == a.V, "bias must have shape [V]");
    TORCH_CHECK(bias->scalar_type() == at::kFloat || bias->scalar_type() == hidden.scalar_type(),
                "bias must be float32 or have the dtype of hidden");
    a.bias = bias->contiguous();
    a.bias_dtype = dtype_code(a.bias.scalar_type(), "bias");
  }
  return a;
}

at::Tensor loss_workspace(const LossArgs& a, int backward) {
  const int64_t bytes = grmx_linear_xent_workspace(a.N, a.D, a.V, a.dtype, backward);
  TORCH_CHECK(bytes >= 0, "grm_cuda: ", grmx_last_error());
  return at::empty({bytes}, a.hidden.options().dtype(at::kByte));
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> linear_xent_fwd_cuda(const at::Tensor& hidden, const at::Tensor& weight,
                                                                    const at::Tensor& targets,
                                                                    const c10::optional<at::Tensor>& bias,
                                                                    int64_t ignore_index, int64_t reduction) {
  LossArgs a = check_loss_inputs(hidden, weight, targets, bias, reduction);
  c10::cuda::CUDAGuard guard(a.hidden.device());
  const auto f32 = a.hidden.options().dtype(at::kFloat);
  auto loss = reduction == GRMX_REDUCE_NONE ? at::empty(targets.sizes(), f32) : at::empty({}, f32);
  auto stats = at::empty({2, a.N}, f32);
  auto inv_count = at::empty({1}, f32);
  if (a.N == 0) {      // no token: an empty list, a sum of 0, a mean of 0 / 0
    if (reduction != GRMX_REDUCE_NONE) loss.fill_(reduction == GRMX_REDUCE_SUM ? 0.0 : std::nan(""));
    inv_count.zero_();
    return {loss, stats, inv_count};
  }
  auto ws = loss_workspace(a, 0);
  check_status(grmx_linear_xent_fwd(a.hidden.data_ptr(), a.weight.data_ptr(), a.bias.defined() ? a.bias.data_ptr() : nullptr,
                                    a.targets.data_ptr<int64_t>(), ignore_index, loss.data_ptr<float>(),
                                    stats.data_ptr<float>(), inv_count.data_ptr<float>(), a.N, a.D, a.V, a.dtype,
                                    a.bias_dtype, static_cast<int>(reduction), ws.data_ptr(), ws.numel(), current_stream()));
  return {loss, stats, inv_count};
}

// the gradients that are asked for; the others come back empty
std::tuple<at::Tensor, at::Tensor, at::Tensor> linear_xent_bwd_cuda(
    const at::Tensor& grad_loss, const at::Tensor& hidden, const at::Tensor& weight, const at::Tensor& targets,
    const c10::optional<at::Tensor>& bias, const at::Tensor& row_stats, const at::Tensor& inv_count, int64_t ignore_index,
    int64_t reduction, bool want_hidden, bool want_weight, bool want_bias) {
  LossArgs a = check_loss_inputs(hidden, weight, targets, bias, reduction);
  require_cuda(grad_loss, "grad_loss");
  TORCH_CHECK(grad_loss.numel() == (reduction == GRMX_REDUCE_NONE ? a.N : 1), "grad_loss has the wrong number of elements");
  TORCH_CHECK(row_stats.is_cuda() && row_stats.scalar_type() == at::kFloat && row_stats.is_contiguous() &&
                  row_stats.numel() == 2 * a.N, "row_stats must be the float32 [2, N] of the forward call");
  TORCH_CHECK(inv_count.is_cuda() && inv_count.scalar_type() == at::kFloat && inv_count.numel() == 1,
              "inv_count must be the float32 [1] of the forward call");
  TORCH_CHECK(grad_loss.device() == hidden.device() && row_stats.device() == hidden.device() &&
                  inv_count.device() == hidden.device(), "the tensors of a backward call must be on one device");
  TORCH_CHECK(!want_bias || a.bias.defined(), "there is no bias to differentiate");
  c10::cuda::CUDAGuard guard(a.hidden.device());
  auto g = grad_loss.to(at::kFloat).contiguous();
  auto dh = want_hidden ? at::empty_like(a.hidden) : at::empty({0}, a.hidden.options());
  auto dw = want_weight ? at::empty_like(a.weight) : at::empty({0}, a.weight.options());
  auto db = want_bias ? at::empty_like(a.bias) : at::empty({0}, a.hidden.options());
  if (a.N == 0) {
    dw.zero_();
    db.zero_();
    return {dh, dw, db};
  }
  if (!want_hidden && !want_weight && !want_bias) return {dh, dw, db};
  auto ws = loss_workspace(a, 1);
  check_status(grmx_linear_xent_bwd(g.data_ptr<float>(), a.hidden.data_ptr(), a.weight.data_ptr(),
                                    a.bias.defined() ? a.bias.data_ptr() : nullptr, a.targets.data_ptr<int64_t>(),
                                    ignore_index, row_stats.data_ptr<float>(), inv_count.data_ptr<float>(),
                                    want_hidden ? dh.data_ptr() : nullptr, want_weight ? dw.data_ptr() : nullptr,
                                    want_bias ? db.data_ptr() : nullptr, a.N, a.D, a.V, a.dtype, a.bias_dtype,
                                    static_cast<int>(reduction), ws.data_ptr(), ws.numel(), current_stream()));
  return {dh, dw, db};
}

// ---- mixing rule + LayerNorm: rows [..., H] in one dtype, parameters [H] in float32 or that dtype ----

struct FuseNormArgs {
  at::Tensor online, update, gate, scale, weight, bias;
  int64_t rows, H;
  int dtype, param_dtype;
};

FuseNormArgs check_fuse_norm_inputs(const at::Tensor& online, const at::Tensor& update, const c10::optional<at::Tensor>& gate,
                                    const c10::optional<at::Tensor>& scale, const c10::optional<at::Tensor>& ln_weight,
                                    const c10::optional<at::Tensor>& ln_bias) {
  TORCH_CHECK(online.dim() >= 1 && online.size(-1) > 0, "online must have shape [..., H]");
  require_cuda(online, "online");
  TORCH_CHECK(online.scalar_type() == at::kFloat || online.scalar_type() == at::kBFloat16,
              "online must be float32 or bfloat16");
  FuseNormArgs a;
  a.H = online.size(-1);
  a.rows = online.numel() / a.H;
  a.dtype = dtype_code(online.scalar_type(), "online");
  a.param_dtype = GRMX_F32;
  auto row_tensor = [&](const at::Tensor& t, const char* name) {
    require_cuda(t, name);
    TORCH_CHECK(t.sizes() == online.sizes(), name, " must have the shape of online");
    TORCH_CHECK(t.scalar_type() == online.scalar_type(), name, " must have the dtype of online");
    TORCH_CHECK(t.device() == online.device(), name, " must be on the device of online");
    return t.contiguous();
  };
  bool first = true;
  auto param = [&](const c10::optional<at::Tensor>& t, const char* name) {
    if (!t.has_value() || !t->defined()) return at::Tensor();
    require_cuda(*t, name);
    TORCH_CHECK(t->dim() == 1 && t->size(0) == a.H, name, " must have shape [H]");
    TORCH_CHECK(t->device() == online.device(), name, " must be on the device of online");
    TORCH_CHECK(t->scalar_type() == at::kFloat || t->scalar_type() == online.scalar_type(),
                name, " must be float32 or have the dtype of online");
    const int code = dtype_code(t->scalar_type(), name);
    TORCH_CHECK(first || code == a.param_dtype, "scale, ln_weight and ln_bias must share one dtype");
    first = false;
    a.param_dtype = code;
    return t->contiguous();
  };
  a.online = online.contiguous();
  a.update = row_tensor(update, "update");
  if (gate.has_value() && gate->defined()) a.gate = row_tensor(*gate, "gate");
  a.scale = param(scale, "scale");
  a.weight = param(ln_weight, "ln_weight");
  a.bias = param(ln_bias, "ln_bias");
  return a;
}

void* ptr_or_null(const at::Tensor& t) { return t.defined() && t.numel() > 0 ? t.data_ptr() : nullptr; }

// out, sum (empty unless asked for), row statistics [rows, 2] (empty unless asked for)
std::tuple<at::Tensor, at::Tensor, at::Tensor> fuse_norm_fwd_cuda(
    const at::Tensor& online, const at::Tensor& update, const c10::optional<at::Tensor>& gate,
    const c10::optional<at::Tensor>& scale, const c10::optional<at::Tensor>& ln_weight,
    const c10::optional<at::Tensor>& ln_bias, double eps, bool want_sum, bool want_stats) {
  FuseNormArgs a = check_fuse_norm_inputs(online, update, gate, scale, ln_weight, ln_bias);
  c10::cuda::CUDAGuard guard(a.online.device());
  auto out = at::empty_like(a.online);
  auto sum = want_sum ? at::empty_like(a.online) : at::empty({0}, a.online.options());
  const auto f32 = a.online.options().dtype(at::kFloat);
  auto stats = want_stats ? at::empty({a.rows, 2}, f32) : at::empty({0}, f32);
  check_status(grmx_fuse_norm_fwd(a.online.data_ptr(), a.update.data_ptr(), ptr_or_null(a.gate), ptr_or_null(a.scale),
                                  ptr_or_null(a.weight), ptr_or_null(a.bias), static_cast<float>(eps), out.data_ptr(),
                                  ptr_or_null(sum), static_cast<float*>(ptr_or_null(stats)), a.rows, a.H, a.dtype,
                                  a.param_dtype, current_stream()));
  return {out, sum, stats};
}

// gradients of online, update, gate, scale, ln_weight, ln_bias; those that are not asked for come back empty
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor> fuse_norm_bwd_cuda(
    const c10::optional<at::Tensor>& grad_out, const c10::optional<at::Tensor>& grad_sum, const at::Tensor& online,
    const at::Tensor& update, const c10::optional<at::Tensor>& gate, const c10::optional<at::Tensor>& scale,
    const c10::optional<at::Tensor>& ln_weight, const c10::optional<at::Tensor>& ln_bias, const at::Tensor& row_stats,
    std::array<bool, 6> want) {
  FuseNormArgs a = check_fuse_norm_inputs(online, update, gate, scale, ln_weight, ln_bias);
  TORCH_CHECK(row_stats.is_cuda() && row_stats.device() == a.online.device() && row_stats.scalar_type() == at::kFloat &&
                  row_stats.is_contiguous() && row_stats.numel() == 2 * a.rows,
              "row_stats must be the float32 [rows, 2] of the forward call");
  TORCH_CHECK(!want[2] || a.gate.defined(), "there is no gate to differentiate");
  TORCH_CHECK(!want[3] || a.scale.defined(), "there is no scale to differentiate");
  TORCH_CHECK((!want[4] || a.weight.defined()) && (!want[5] || a.bias.defined()), "there is no ln_weight or ln_bias to differentiate");
  c10::cuda::CUDAGuard guard(a.online.device());
  auto grad = [&](const c10::optional<at::Tensor>& t, const char* name) {
    if (!t.has_value() || !t->defined()) return at::Tensor();
    require_cuda(*t, name);
    TORCH_CHECK(t->numel() == a.online.numel() && t->device() == a.online.device(), name, " does not fit online");
    return t->to(a.online.scalar_type()).contiguous();
  };
  at::Tensor dy = grad(grad_out, "grad_out"), dsum = grad(grad_sum, "grad_sum");
  TORCH_CHECK(dy.defined() || dsum.defined(), "neither output has a gradient");
  auto like = [&](const at::Tensor& t, bool wanted) {
    return wanted ? at::empty_like(t) : at::empty({0}, a.online.options());
  };
  auto d_online = like(a.online, want[0]), d_update = like(a.update, want[1]), d_gate = like(a.gate, want[2]);
  auto d_scale = like(a.scale, want[3]), d_weight = like(a.weight, want[4]), d_bias = like(a.bias, want[5]);
  const int64_t bytes = grmx_fuse_norm_workspace(a.rows, a.H);
  TORCH_CHECK(bytes >= 0, "grm_cuda: ", grmx_last_error());
  const bool columns = want[3] || want[4] || want[5];
  auto ws = at::empty({columns ? bytes : 0}, a.online.options().dtype(at::kByte));
  check_status(grmx_fuse_norm_bwd(ptr_or_null(dy), ptr_or_null(dsum), a.online.data_ptr(), a.update.data_ptr(),
                                  ptr_or_null(a.gate), ptr_or_null(a.scale), ptr_or_null(a.weight),
                                  row_stats.data_ptr<float>(), ptr_or_null(d_online), ptr_or_null(d_update),
                                  ptr_or_null(d_gate), ptr_or_null(d_scale), ptr_or_null(d_weight), ptr_or_null(d_bias),
                                  a.rows, a.H, a.dtype, a.param_dtype, ptr_or_null(ws), ws.numel(), current_stream()));
  return {d_online, d_update, d_gate, d_scale, d_weight, d_bias};
}

// ---- the same with autograd: in C++, so that a training step spends its host time on launches ----

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

c10::optional<at::Tensor> maybe(const at::Tensor& t) { return t.defined() ? c10::optional<at::Tensor>(t) : c10::nullopt; }
at::Tensor or_undefined(const c10::optional<at::Tensor>& t) { return t.has_value() ? *t : at::Tensor(); }
at::Tensor if_wanted(const at::Tensor& t, bool wanted) { return wanted ? t : at::Tensor(); }
using MaybeTensor = c10::optional<at::Tensor>;

// neither operator has a forward-mode derivative: a tangent would be lost without a word where no input requires a gradient
void refuse_tangents(std::initializer_list<const at::Tensor*> inputs, const char* what) {
  for (const at::Tensor* t : inputs) {
    TORCH_CHECK(!t->defined() || !t->_fw_grad(0).defined(), what, " has no forward-mode derivative; use reverse mode");
  }
}

// gradients with a gradient of their own are asked for (create_graph): they get one that reports its absence
variable_list no_second_derivative(variable_list grads, const char* what) {
  if (!at::GradMode::is_enabled()) return grads;
  std::vector<size_t> at_index;
  variable_list defined;
  for (size_t i = 0; i < grads.size(); ++i) {
    if (grads[i].defined()) {
      at_index.push_back(i);
      defined.push_back(grads[i].requires_grad() ? grads[i] : grads[i].detach().requires_grad_());
    }
  }
  auto node = std::make_shared<torch::autograd::DelayedError>(std::string(what) + " is differentiable once only",
                                                              static_cast<int64_t>(defined.size()));
  variable_list marked = (*node)(std::move(defined));
  for (size_t i = 0; i < at_index.size(); ++i) grads[at_index[i]] = marked[i];
  return grads;
}

struct LinearCrossEntropyFn : public torch::autograd::Function<LinearCrossEntropyFn> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& hidden, const at::Tensor& weight, const MaybeTensor& bias,
                            const at::Tensor& targets, int64_t ignore_index, int64_t reduction) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [loss, stats, inv_count] = linear_xent_fwd_cuda(hidden, weight, targets, bias, ignore_index, reduction);
    ctx->save_for_backward({hidden, weight, or_undefined(bias), targets, stats, inv_count});
    ctx->saved_data["ignore_index"] = ignore_index;
    ctx->saved_data["reduction"] = reduction;
    return loss;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const bool wh = ctx->needs_input_grad(0), ww = ctx->needs_input_grad(1), wb = saved[2].defined() && ctx->needs_input_grad(2);
    variable_list out(6);
    {
      at::AutoDispatchBelowADInplaceOrView below;
      auto [dh, dw, db] = linear_xent_bwd_cuda(grads[0], saved[0], saved[1], saved[3], maybe(saved[2]), saved[4], saved[5],
                                               ctx->saved_data["ignore_index"].toInt(), ctx->saved_data["reduction"].toInt(), wh, ww, wb);
      out[0] = if_wanted(dh, wh);
      out[1] = if_wanted(dw, ww);
      out[2] = if_wanted(db, wb);
    }
    return no_second_derivative(std::move(out), "linear_cross_entropy");
  }
};

at::Tensor linear_cross_entropy(const at::Tensor& hidden, const at::Tensor& weight, const at::Tensor& targets,
                                const c10::optional<at::Tensor>& bias, int64_t ignore_index, int64_t reduction) {
  const at::Tensor b = or_undefined(bias);
  refuse_tangents({&hidden, &weight, &b}, "linear_cross_entropy");
  if (at::GradMode::is_enabled() && (hidden.requires_grad() || weight.requires_grad() || (b.defined() && b.requires_grad()))) {
    return LinearCrossEntropyFn::apply(hidden, weight, maybe(b), targets, ignore_index, reduction);
  }
  at::AutoDispatchBelowADInplaceOrView below;
  return std::get<0>(linear_xent_fwd_cuda(hidden, weight, targets, bias, ignore_index, reduction));
}

struct FuseLayerNormFn : public torch::autograd::Function<FuseLayerNormFn> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& online, const at::Tensor& update, const MaybeTensor& gate,
                               const MaybeTensor& scale, const MaybeTensor& weight, const MaybeTensor& bias, double eps, bool want_sum) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [out, sum, stats] = fuse_norm_fwd_cuda(online, update, gate, scale, weight, bias, eps, want_sum, true);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({online, update, or_undefined(gate), or_undefined(scale), or_undefined(weight), or_undefined(bias), stats});
    return want_sum ? variable_list{out, sum} : variable_list{out};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(8);
    const at::Tensor dy = grads[0], dsum = grads.size() > 1 ? grads[1] : at::Tensor();
    if (!dy.defined() && !dsum.defined()) return out;
    const auto saved = ctx->get_saved_variables();
    bool want[6];
    // inputs are numbered without the ones that were not given
    for (size_t i = 0, given = 0; i < 6; ++i) want[i] = saved[i].defined() && ctx->needs_input_grad(given++);
    // without gate and scale both row tensors have the same gradient: one is written
    const bool shared = !saved[2].defined() && !saved[3].defined() && want[0] && want[1];
    {
      at::AutoDispatchBelowADInplaceOrView below;
      auto [d0, d1, d2, d3, d4, d5] = fuse_norm_bwd_cuda(maybe(dy), maybe(dsum), saved[0], saved[1], maybe(saved[2]), maybe(saved[3]),
                                                         maybe(saved[4]), maybe(saved[5]), saved[6],
                                                         {want[0], want[1] && !shared, want[2], want[3], want[4], want[5]});
      out[0] = if_wanted(d0, want[0]);
      out[1] = if_wanted(shared ? d0 : d1, want[1]);
      out[2] = if_wanted(d2, want[2]);
      out[3] = if_wanted(d3, want[3]);
      out[4] = if_wanted(d4, want[4]);
      out[5] = if_wanted(d5, want[5]);
    }
    return no_second_derivative(std::move(out), "fuse_layer_norm");
  }
};

// (out,) or (out, sum)
variable_list fuse_layer_norm(const at::Tensor& online, const at::Tensor& update, const c10::optional<at::Tensor>& weight,
                              const c10::optional<at::Tensor>& bias, const c10::optional<at::Tensor>& gate,
                              const c10::optional<at::Tensor>& scale, double eps, bool want_sum) {
  const at::Tensor g = or_undefined(gate), k = or_undefined(scale), w = or_undefined(weight), b = or_undefined(bias);
  refuse_tangents({&online, &update, &w, &b, &g, &k}, "fuse_layer_norm");
  auto needs = [](const at::Tensor& t) { return t.defined() && t.requires_grad(); };
  if (at::GradMode::is_enabled() && (needs(online) || needs(update) || needs(g) || needs(k) || needs(w) || needs(b))) {
    return FuseLayerNormFn::apply(online, update, maybe(g), maybe(k), maybe(w), maybe(b), eps, want_sum);
  }
  at::AutoDispatchBelowADInplaceOrView below;
  auto [out, sum, stats] = fuse_norm_fwd_cuda(online, update, gate, scale, weight, bias, eps, want_sum, false);
  return want_sum ? variable_list{out, sum} : variable_list{out};
}

}  // namespace

TORCH_LIBRARY(grm_cuda, m) {
  m.def("chunk_update_forward(Tensor keys, Tensor values, Tensor queries, Tensor memory, float memory_decay) -> (Tensor hidden, Tensor memory_out, Tensor aux)");
  m.def("chunk_update_backward(Tensor grad_hidden, Tensor grad_memory_out, Tensor keys, Tensor values, Tensor queries, Tensor memory, Tensor aux, float memory_decay) -> (Tensor grad_keys, Tensor grad_values, Tensor grad_queries, Tensor grad_memory)");
  m.def("apply_query_forward(Tensor memories, Tensor queries) -> Tensor");
  m.def("apply_query_backward(Tensor grad_hidden, Tensor memories, Tensor queries) -> (Tensor grad_memories, Tensor grad_queries)");
  m.def("batched_memory_gather(Tensor memories_per_batch, Tensor topk_indices) -> Tensor");
}

TORCH_LIBRARY_IMPL(grm_cuda, CUDA, m) {
  m.impl("chunk_update_forward", chunk_update_forward_cuda);
  m.impl("chunk_update_backward", chunk_update_backward_cuda);
  m.impl("apply_query_forward", apply_query_forward_cuda);
  m.impl("apply_query_backward", apply_query_backward_cuda);
  m.impl("batched_memory_gather", batched_memory_gather_cuda);
}

TORCH_LIBRARY(grmx, m) {
  m.def("linear_scan(Tensor keys, Tensor values, Tensor queries, Tensor memory, float decay, float update_coeff, float hidden_scale, float memory_out_scale, bool reverse, bool first_step_no_decay, int path) -> (Tensor hidden, Tensor memory_out)");
  m.def("topk_route(Tensor queries, Tensor keys, Tensor? visible, int top_k, float scale, float temperature, bool return_scores) -> (Tensor gates, Tensor indices, Tensor scores)");
  m.def("topk_select(Tensor scores, Tensor? visible, int top_k, float temperature) -> (Tensor gates, Tensor indices)");
  m.def("retrieve_fuse(Tensor archive, Tensor indices, Tensor? gates, Tensor queries, Tensor? online, Tensor? ln_weight, Tensor? ln_bias, float ln_eps, int mode) -> Tensor");
  m.def("retrieve_fuse_tc(Tensor archive, Tensor indices, Tensor gates, Tensor queries, Tensor? online, Tensor? ln_weight, Tensor? ln_bias, float ln_eps, int mode) -> Tensor");
  m.def("chunk_scan_segments(Tensor keys, Tensor values, Tensor queries, Tensor memory, float decay, Tensor(a!) archive, int first_slot, int segment_tokens) -> (Tensor hidden, Tensor memory_out)");
  m.def("l2_normalize(Tensor x, float eps, bool to_bfloat16) -> Tensor");
  m.def("project_normalize(Tensor x, Tensor weights, Tensor? bias, float eps) -> (Tensor a, Tensor b)");
  m.def("archive_push(Tensor memory, Tensor(a!) archive, Tensor(b!)? shadow, int slot) -> ()");
  m.def("add_layer_norm(Tensor a, Tensor b, Tensor? ln_weight, Tensor? ln_bias, float ln_eps) -> Tensor");
  m.def("linear_xent_fwd(Tensor hidden, Tensor weight, Tensor targets, Tensor? bias, int ignore_index, int reduction) -> (Tensor loss, Tensor row_stats, Tensor inv_count)");
  m.def("linear_xent_bwd(Tensor grad_loss, Tensor hidden, Tensor weight, Tensor targets, Tensor? bias, Tensor row_stats, Tensor inv_count, int ignore_index, int reduction, bool want_hidden, bool want_weight, bool want_bias) -> (Tensor grad_hidden, Tensor grad_weight, Tensor grad_bias)");
  m.def("fuse_norm_fwd(Tensor online, Tensor update, Tensor? gate, Tensor? scale, Tensor? ln_weight, Tensor? ln_bias, float eps, bool want_sum, bool want_stats) -> (Tensor out, Tensor sum, Tensor row_stats)");
  m.def("fuse_norm_bwd(Tensor? grad_out, Tensor? grad_sum, Tensor online, Tensor update, Tensor? gate, Tensor? scale, Tensor? ln_weight, Tensor? ln_bias, Tensor row_stats, bool[6] want) -> (Tensor grad_online, Tensor grad_update, Tensor grad_gate, Tensor grad_scale, Tensor grad_weight, Tensor grad_bias)");
  m.def("select_fuse(Tensor states, Tensor indices, Tensor gates, Tensor? online, Tensor? ln_weight, Tensor? ln_bias, float ln_eps, int mode) -> Tensor");
}

TORCH_LIBRARY_IMPL(grmx, CUDA, m) {
  m.impl("linear_scan", linear_scan_cuda);
  m.impl("topk_route", topk_route_cuda);
  m.impl("topk_select", topk_select_cuda);
  m.impl("retrieve_fuse", retrieve_fuse_cuda);
  m.impl("retrieve_fuse_tc", retrieve_fuse_tc_cuda);
  m.impl("linear_xent_fwd", linear_xent_fwd_cuda);
  m.impl("linear_xent_bwd", linear_xent_bwd_cuda);
  m.impl("fuse_norm_fwd", fuse_norm_fwd_cuda);
  m.impl("fuse_norm_bwd", fuse_norm_bwd_cuda);
  m.impl("select_fuse", select_fuse_cuda);
  m.impl("add_layer_norm", add_layer_norm_cuda);
  m.impl("archive_push", archive_push_cuda);
  m.impl("project_normalize", project_normalize_cuda);
  m.impl("l2_normalize", l2_normalize_cuda);
  m.impl("chunk_scan_segments", chunk_scan_segments_cuda);
}

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.doc() = "GRM segment-memory engine for B200 (sm_100a): torch.ops.grm_cuda.* over the grmx C ABI";
  m.attr("__grm_cuda_with_kernels__") = pybind11::bool_(true);
  m.def("grmx_version", []() { return grmx_version(); });
  m.def("launch_count", []() { return grmx_launch_count(); });
  m.def("set_scan_path", [](int path) {
    TORCH_CHECK(path == GRMX_PATH_AUTO || path == GRMX_PATH_FFMA || path == GRMX_PATH_TCGEN05,
                "scan path must be 0 (auto), 1 (ffma) or 2 (tcgen05)");
    g_scan_path.store(path);
  });
  m.def("get_scan_path", []() { return g_scan_path.load(); });
  // The device error word of the current device: kernels report a bounded wait that gave up or an
  // out-of-range routing index there instead of trapping.  Reading it waits for the current stream.
  m.def("device_error_word", []() {
    uint32_t word = 0;
    check_status(grmx_device_error_word(&word, current_stream()));
    return word;
  });
  // the training operators with autograd (Python: loss.linear_cross_entropy, fusion.fuse_layer_norm)
  m.def("linear_cross_entropy", linear_cross_entropy, pybind11::call_guard<pybind11::gil_scoped_release>());
  m.def("fuse_layer_norm", fuse_layer_norm, pybind11::call_guard<pybind11::gil_scoped_release>());
  m.def("device_error_reset", []() { check_status(grmx_device_error_reset(current_stream())); });
}
