// PyTorch operator library torch.ops.mrun_b200.* over the C ABI of libmrun_b200.so.
//
// A thin layer: each operator takes tensors, checks that they are CUDA tensors of the
// expected dtype and layout, and calls the matching mrb_* entry point on the current CUDA
// stream of the first tensor's device. Outputs are caller-allocated (`Tensor(a!)` in the
// schemas), so the operators allocate nothing and can be captured in CUDA graphs. The
// Python mirror (mrun_b200/dense_qstore_cuda.py, moe.py, qstore_build.py, paged_kv4.py) validates
// arguments with the reference's messages and then calls these operators. A failed C call
// raises ValueError for a bad argument (MRB_ERR_ARG) and RuntimeError otherwise, with the
// library's message.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/library.h>

#include <algorithm>
#include <optional>
#include <utility>

#include "../../include/mrun_b200.h"

namespace {

void check_status(int rc, const char* what) {
  if (rc == MRB_OK) return;
  const char* msg = mrb_last_error();
  if (rc == MRB_ERR_ARG) TORCH_CHECK_VALUE(false, what, ": ", msg);
  TORCH_CHECK(false, what, ": ", msg);
}

void* stream_of(const at::Tensor& t) { return at::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

void need(const at::Tensor& t, at::ScalarType dtype, const char* what) {
  TORCH_CHECK_VALUE(t.is_cuda(), what, " must be a CUDA tensor");
  TORCH_CHECK_VALUE(t.scalar_type() == dtype, what, " has dtype ", t.scalar_type(), ", expected ", dtype);
  TORCH_CHECK_VALUE(t.is_contiguous(), what, " must be contiguous");
}

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return MRB_F32;
    case at::kBFloat16: return MRB_BF16;
    case at::kHalf: return MRB_F16;
    default: TORCH_CHECK_VALUE(false, "unsupported activation dtype ", t);
  }
  return -1;
}

template <typename T>
T* opt_ptr(const std::optional<at::Tensor>& t) {
  return t.has_value() && t->defined() ? static_cast<T*>(t->data_ptr()) : nullptr;
}

// y = x @ (codes * scales[:, None]).T (+ bias): mrb_qrow_matmul
void qrow_linear(const at::Tensor& x, const at::Tensor& codes, const at::Tensor& scales,
                 const std::optional<at::Tensor>& bias, at::Tensor& out, const std::optional<at::Tensor>& workspace) {
  TORCH_CHECK_VALUE(x.dim() == 2 && codes.dim() == 2 && out.dim() == 2, "qrow_linear: 2-D tensors expected");
  need(x, x.scalar_type(), "activations");
  need(codes, at::kChar, "codes");
  need(scales, at::kFloat, "scales");
  need(out, x.scalar_type(), "out");
  const int64_t m = x.size(0), k = x.size(1), n = codes.size(0);
  TORCH_CHECK_VALUE(codes.size(1) == k && scales.numel() == n && out.size(0) == m && out.size(1) == n,
                    "qrow_linear: shapes do not match");
  if (bias.has_value() && bias->defined()) need(*bias, at::kFloat, "bias");
  if (workspace.has_value() && workspace->defined()) need(*workspace, at::kByte, "workspace");
  const int code = dtype_code(x.scalar_type());
  check_status(mrb_qrow_matmul(x.data_ptr(), code, m, k, codes.data_ptr<int8_t>(), scales.data_ptr<float>(), n,
                               opt_ptr<float>(bias), out.data_ptr(), code, opt_ptr<void>(workspace),
                               workspace.has_value() && workspace->defined() ? (size_t)workspace->numel() : 0,
                               stream_of(x)),
               "qrow_linear");
}

// y = bf16(silu(bf16(x.Wg)) * bf16(x.Wu)): mrb_qrow_swiglu
void qrow_swiglu(const at::Tensor& x, const at::Tensor& gate_codes, const at::Tensor& gate_scales,
                 const at::Tensor& up_codes, const at::Tensor& up_scales, at::Tensor& out,
                 const std::optional<at::Tensor>& workspace) {
  need(x, at::kBFloat16, "activations");
  need(gate_codes, at::kChar, "gate codes");
  need(up_codes, at::kChar, "up codes");
  need(gate_scales, at::kFloat, "gate scales");
  need(up_scales, at::kFloat, "up scales");
  need(out, at::kBFloat16, "out");
  const int64_t m = x.size(0), k = x.size(1), n = gate_codes.size(0);
  TORCH_CHECK_VALUE(gate_codes.sizes() == up_codes.sizes() && gate_codes.size(1) == k && out.size(0) == m &&
                        out.size(1) == n,
                    "qrow_swiglu: shapes do not match");
  if (workspace.has_value() && workspace->defined()) need(*workspace, at::kByte, "workspace");
  check_status(mrb_qrow_swiglu(x.data_ptr(), m, k, gate_codes.data_ptr<int8_t>(), gate_scales.data_ptr<float>(),
                               up_codes.data_ptr<int8_t>(), up_scales.data_ptr<float>(), n, out.data_ptr(),
                               opt_ptr<void>(workspace),
                               workspace.has_value() && workspace->defined() ? (size_t)workspace->numel() : 0,
                               stream_of(x)),
               "qrow_swiglu");
}

// per-output-channel symmetric int8: mrb_quant_row_int8
void quant_row_int8(const at::Tensor& weight, at::Tensor& codes, at::Tensor& scales) {
  need(weight, at::kFloat, "weight");
  need(codes, at::kChar, "codes");
  need(scales, at::kFloat, "scales");
  TORCH_CHECK_VALUE(weight.dim() == 2 && codes.sizes() == weight.sizes() && scales.numel() == weight.size(0),
                    "quant_row_int8: shapes do not match");
  check_status(mrb_quant_row_int8(weight.data_ptr<float>(), weight.size(0), weight.size(1), codes.data_ptr<int8_t>(),
                                  scales.data_ptr<float>(), stream_of(weight)),
               "quant_row_int8");
}

// softmax / top-k / renorm: mrb_router_topk
void router_topk(const at::Tensor& logits, int64_t k, bool renorm, at::Tensor& top_idx, at::Tensor& top_w_f32,
                 at::Tensor& top_w_bf16) {
  need(logits, logits.scalar_type(), "logits");
  TORCH_CHECK_VALUE(logits.dim() == 2, "router_topk: logits must be [tokens, experts]");
  need(top_idx, at::kLong, "top_idx");
  need(top_w_f32, at::kFloat, "top_w_f32");
  need(top_w_bf16, at::kBFloat16, "top_w_bf16");
  const int64_t t = logits.size(0), e = logits.size(1);
  TORCH_CHECK_VALUE(top_idx.numel() == t * k && top_w_f32.numel() == t * k && top_w_bf16.numel() == t * k,
                    "router_topk: outputs must hold tokens * k entries");
  check_status(mrb_router_topk(logits.data_ptr(), dtype_code(logits.scalar_type()), t, e, k, renorm ? 1 : 0,
                               top_idx.data_ptr<int64_t>(), top_w_f32.data_ptr<float>(), top_w_bf16.data_ptr(),
                               stream_of(logits)),
               "router_topk");
}

// stable expert-major route plan: mrb_route_compile
void route_compile(const at::Tensor& top_idx, const at::Tensor& top_w, int64_t experts, at::Tensor& counts,
                   at::Tensor& starts, at::Tensor& token_ids, at::Tensor& coef, at::Tensor& inverse) {
  need(top_idx, at::kLong, "top_idx");
  need(top_w, at::kFloat, "top_w");
  TORCH_CHECK_VALUE(top_idx.dim() == 2, "route_compile: top_idx must be [tokens, k]");
  need(counts, at::kInt, "counts");
  need(starts, at::kInt, "starts");
  need(token_ids, at::kLong, "token_ids");
  need(coef, at::kFloat, "coef");
  need(inverse, at::kLong, "inverse");
  const int64_t t = top_idx.size(0), k = top_idx.size(1), a = t * k;
  TORCH_CHECK_VALUE(top_w.numel() == a && counts.numel() == experts && starts.numel() == experts &&
                        token_ids.numel() == a && coef.numel() == a && inverse.numel() == a,
                    "route_compile: shapes do not match");
  check_status(mrb_route_compile(top_idx.data_ptr<int64_t>(), top_w.data_ptr<float>(), t, k, experts,
                                 counts.data_ptr<int32_t>(), starts.data_ptr<int32_t>(), token_ids.data_ptr<int64_t>(),
                                 coef.data_ptr<float>(), inverse.data_ptr<int64_t>(), nullptr, stream_of(top_idx)),
               "route_compile");
}

// fixed-rank combine: mrb_stable_route_reduce
void stable_route_reduce(const at::Tensor& expert_out, const at::Tensor& coef, const at::Tensor& inverse,
                         int64_t tokens, int64_t k, const std::optional<at::Tensor>& out_f32,
                         const std::optional<at::Tensor>& out_bf16) {
  need(expert_out, at::kBFloat16, "expert_out");
  need(coef, at::kFloat, "coef");
  need(inverse, at::kLong, "inverse");
  TORCH_CHECK_VALUE(expert_out.dim() == 2, "stable_route_reduce: expert_out must be [tokens * k, hidden]");
  const int64_t hidden = expert_out.size(1);
  TORCH_CHECK_VALUE(expert_out.size(0) == tokens * k && coef.numel() == tokens * k && inverse.numel() == tokens * k,
                    "stable_route_reduce: shapes do not match");
  const bool f32 = out_f32.has_value() && out_f32->defined(), bf16 = out_bf16.has_value() && out_bf16->defined();
  TORCH_CHECK_VALUE(f32 || bf16, "stable_route_reduce: give out_f32, out_bf16 or both");
  if (f32) {
    need(*out_f32, at::kFloat, "out_f32");
    TORCH_CHECK_VALUE(out_f32->numel() == tokens * hidden, "stable_route_reduce: out_f32 must be [tokens, hidden]");
  }
  if (bf16) {
    need(*out_bf16, at::kBFloat16, "out_bf16");
    TORCH_CHECK_VALUE(out_bf16->numel() == tokens * hidden, "stable_route_reduce: out_bf16 must be [tokens, hidden]");
  }
  check_status(mrb_stable_route_reduce(expert_out.data_ptr(), coef.data_ptr<float>(), inverse.data_ptr<int64_t>(),
                                       tokens, k, hidden, opt_ptr<float>(out_f32), opt_ptr<void>(out_bf16),
                                       stream_of(expert_out)),
               "stable_route_reduce");
}

// gate/up (SwiGLU) then down over expert pages, the down launch overlapping: mrb_grouped_expert_mlp
void grouped_expert_mlp(const at::Tensor& x, const at::Tensor& token_ids, const at::Tensor& starts,
                        const at::Tensor& counts, const at::Tensor& pages, int64_t page_stride,
                        int64_t gate_up_codes_offset, int64_t gate_up_scales_offset, int64_t down_codes_offset,
                        int64_t down_scales_offset, const std::optional<at::Tensor>& slot_of, at::Tensor& act,
                        at::Tensor& y, at::Tensor& sync) {
  need(x, at::kBFloat16, "activations");
  need(token_ids, at::kLong, "token_ids");
  need(starts, at::kInt, "starts");
  need(counts, at::kInt, "counts");
  need(pages, at::kByte, "pages");
  need(act, at::kBFloat16, "act");
  need(y, at::kBFloat16, "y");
  need(sync, at::kInt, "sync");
  if (slot_of.has_value() && slot_of->defined()) need(*slot_of, at::kInt, "slot_of");
  const int64_t experts = counts.numel(), a = token_ids.numel();
  TORCH_CHECK_VALUE(act.dim() == 2 && y.dim() == 2 && act.size(0) == a && y.size(0) == a,
                    "grouped_expert_mlp: act and y must be [assignments, ...]");
  TORCH_CHECK_VALUE(sync.numel() >= 2 * experts + 1, "grouped_expert_mlp: sync must be int32 [2 * experts + 1]");
  check_status(mrb_grouped_expert_mlp(x.data_ptr(), token_ids.data_ptr<int64_t>(), starts.data_ptr<int32_t>(),
                                      counts.data_ptr<int32_t>(), experts, pages.data_ptr(), page_stride,
                                      gate_up_codes_offset, gate_up_scales_offset, down_codes_offset,
                                      down_scales_offset, opt_ptr<int32_t>(slot_of), y.size(1), act.size(1), a,
                                      act.data_ptr(), y.data_ptr(), reinterpret_cast<uint32_t*>(sync.data_ptr<int32_t>()),
                                      stream_of(x)),
               "grouped_expert_mlp");
}

// ---- 4-bit paged K/V cache

struct Pool {
  int64_t pages, hkv, page_size, stride_page, stride_head, head_dim;
};

// a pool view [pages, kv_heads, page_size / 16, block_bytes] whose blocks of one head are contiguous
Pool pool_of(const at::Tensor& pool, int64_t group) {
  TORCH_CHECK_VALUE(pool.is_cuda() && pool.scalar_type() == at::kByte && pool.dim() == 4,
                    "the pool must be a CUDA uint8 tensor [pages, kv_heads, page_size / 16, block_bytes]");
  const int64_t bytes = pool.size(3);
  TORCH_CHECK_VALUE(group == 32 || group == 64 || group == 128, "group must be 32, 64 or 128, not ", group);
  const int64_t per_dim = 16 * group + 128;  // block bytes of `group` dimensions
  TORCH_CHECK_VALUE(bytes * group % per_dim == 0, "blocks of ", bytes, " bytes do not hold groups of ", group);
  TORCH_CHECK_VALUE(pool.stride(3) == 1 && (pool.size(2) == 1 || pool.stride(2) == bytes),
                    "the blocks of a page and head must be contiguous");
  return {pool.size(0), pool.size(1), pool.size(2) * 16, pool.stride(0), pool.stride(1), bytes * group / per_dim};
}

void need_same_device(const at::Tensor& a, const at::Tensor& b, const char* what) {
  TORCH_CHECK_VALUE(a.device() == b.device(), what, ": tensors must share one device");
}

int32_t* flag_ptr(const std::optional<at::Tensor>& flag, const at::Tensor& like, const char* what) {
  if (!flag.has_value() || !flag->defined()) return nullptr;
  need(*flag, at::kInt, "error_flag");
  TORCH_CHECK_VALUE(flag->numel() >= 1, "error_flag must hold one int32");
  need_same_device(*flag, like, what);
  return flag->data_ptr<int32_t>();
}

const int32_t* opt_i32(const std::optional<at::Tensor>& t, const at::Tensor& like, int64_t numel, const char* name,
                       const char* what) {
  if (!t.has_value() || !t->defined()) return nullptr;
  need(*t, at::kInt, name);
  TORCH_CHECK_VALUE(t->numel() == numel, what, ": ", name, " must hold ", numel, " entries");
  need_same_device(*t, like, what);
  return t->data_ptr<int32_t>();
}

void need_table(const at::Tensor& t, const at::Tensor& like, const char* what) {
  TORCH_CHECK_VALUE(t.is_cuda() && t.scalar_type() == at::kInt && t.dim() == 2 && t.stride(1) == 1 && t.size(1) > 0,
                    what, ": the block table must be a CUDA int32 tensor [sequences, pages] with contiguous rows");
  need_same_device(t, like, what);
}

// a table's row stride: what a one-row view says of it is not used by the kernels
int64_t table_stride(const at::Tensor& t) { return std::max(t.stride(0), t.size(1)); }

void kv_plan_step(const at::Tensor& new_tokens, const std::optional<at::Tensor>& row_seq, const at::Tensor& lengths,
                  at::Tensor& lengths_out, at::Tensor& block_table, const at::Tensor& free_pages,
                  const at::Tensor& free_count, at::Tensor& free_count_out, int64_t page_size, at::Tensor& q_starts,
                  at::Tensor& row_len, at::Tensor& positions, at::Tensor& token_rows, at::Tensor& slots,
                  const std::optional<at::Tensor>& error_flag) {
  const char* what = "kv_plan_step";
  const c10::cuda::CUDAGuard guard(new_tokens.device());
  need(new_tokens, at::kInt, "new_tokens");
  for (const auto& [t, name] : {std::pair<const at::Tensor&, const char*>{lengths, "lengths"},
                                {lengths_out, "lengths_out"},
                                {free_pages, "free_pages"},
                                {free_count, "free_count"},
                                {free_count_out, "free_count_out"},
                                {q_starts, "q_starts"},
                                {row_len, "row_len"},
                                {positions, "positions"},
                                {token_rows, "token_rows"},
                                {slots, "slots"}}) {
    need(t, at::kInt, name);
    need_same_device(t, new_tokens, what);
  }
  need_table(block_table, new_tokens, what);
  const int64_t rows = new_tokens.numel(), seqs = lengths.numel(), tokens = slots.numel();
  TORCH_CHECK_VALUE(row_seq.has_value() || rows <= seqs, what, ": more requests than sequences");
  TORCH_CHECK_VALUE(block_table.size(0) == seqs && lengths_out.numel() == seqs, what,
                    ": lengths, lengths_out and the block table must have one row a sequence");
  TORCH_CHECK_VALUE(free_count.numel() == 1 && free_count_out.numel() == 1, what, ": free_count must hold one int32");
  TORCH_CHECK_VALUE(q_starts.numel() == rows + 1 && row_len.numel() == rows && positions.numel() == tokens &&
                        token_rows.numel() == tokens,
                    what, ": outputs do not match the requests and max_tokens");
  check_status(
      mrb_kv_plan_step(new_tokens.data_ptr<int32_t>(), opt_i32(row_seq, new_tokens, rows, "row_seq", what), rows,
                       lengths.data_ptr<int32_t>(), lengths_out.data_ptr<int32_t>(), seqs,
                       block_table.data_ptr<int32_t>(), table_stride(block_table), block_table.size(1),
                       free_pages.data_ptr<int32_t>(), free_pages.numel(), free_count.data_ptr<int32_t>(),
                       free_count_out.data_ptr<int32_t>(), page_size, tokens, q_starts.data_ptr<int32_t>(),
                       row_len.data_ptr<int32_t>(), positions.data_ptr<int32_t>(), token_rows.data_ptr<int32_t>(),
                       slots.data_ptr<int32_t>(), flag_ptr(error_flag, new_tokens, what), stream_of(new_tokens)),
      what);
}

void kv_release(const at::Tensor& seqs, at::Tensor& lengths, at::Tensor& block_table, at::Tensor& free_pages,
                at::Tensor& free_count, int64_t page_size, const std::optional<at::Tensor>& error_flag) {
  const char* what = "kv_release";
  const c10::cuda::CUDAGuard guard(seqs.device());
  need(seqs, at::kInt, "seqs");
  for (const auto& [t, name] : {std::pair<const at::Tensor&, const char*>{lengths, "lengths"},
                                {free_pages, "free_pages"},
                                {free_count, "free_count"}}) {
    need(t, at::kInt, name);
    need_same_device(t, seqs, what);
  }
  need_table(block_table, seqs, what);
  TORCH_CHECK_VALUE(block_table.size(0) == lengths.numel() && free_count.numel() == 1, what, ": shapes do not match");
  check_status(mrb_kv_release(seqs.data_ptr<int32_t>(), seqs.numel(), lengths.data_ptr<int32_t>(), lengths.numel(),
                              block_table.data_ptr<int32_t>(), table_stride(block_table), block_table.size(1),
                              free_pages.data_ptr<int32_t>(), free_pages.numel(), free_count.data_ptr<int32_t>(),
                              page_size, flag_ptr(error_flag, seqs, what), stream_of(seqs)),
               what);
}

// bf16 rows [tokens, width] whose elements are contiguous
void need_rows(const at::Tensor& t, const at::Tensor& like, int64_t tokens, int64_t width, const char* name,
               const char* what) {
  TORCH_CHECK_VALUE(t.is_cuda() && t.scalar_type() == at::kBFloat16 && t.dim() == 2 && t.size(0) == tokens &&
                        t.size(1) == width && (t.stride(1) == 1 || width == 1),
                    what, ": ", name, " must be CUDA bf16 rows [", tokens, ", ", width, "] with contiguous elements");
  need_same_device(t, like, what);
}

void rope_kv4_append(const std::optional<at::Tensor>& q_in, const at::Tensor& k_in, const at::Tensor& v_in,
                     at::Tensor& pool, int64_t group, const at::Tensor& slots,
                     const std::optional<at::Tensor>& positions, const std::optional<at::Tensor>& rope_cos,
                     const std::optional<at::Tensor>& rope_sin, bool interleaved,
                     const std::optional<at::Tensor>& q_norm, const std::optional<at::Tensor>& k_norm,
                     double norm_eps, const std::optional<at::Tensor>& q_out,
                     const std::optional<at::Tensor>& error_flag) {
  const char* what = "rope_kv4_append";
  const c10::cuda::CUDAGuard guard(pool.device());
  const Pool p = pool_of(pool, group);
  need(slots, at::kInt, "slots");
  need_same_device(slots, pool, what);
  const int64_t t = slots.numel(), kw = p.hkv * p.head_dim;
  need_rows(k_in, pool, t, kw, "k_in", what);
  need_rows(v_in, pool, t, kw, "v_in", what);
  int64_t hq = 0;
  const bool has_q = q_in.has_value() && q_in->defined();
  TORCH_CHECK_VALUE(has_q == (q_out.has_value() && q_out->defined()), what, ": q_in and q_out come together");
  if (has_q) {
    TORCH_CHECK_VALUE(q_in->dim() == 2 && q_in->size(1) % p.head_dim == 0, what,
                      ": q_in must hold whole heads of ", p.head_dim);
    hq = q_in->size(1) / p.head_dim;
    need_rows(*q_in, pool, t, hq * p.head_dim, "q_in", what);
    need(*q_out, at::kBFloat16, "q_out");
    need_same_device(*q_out, pool, what);
    TORCH_CHECK_VALUE(q_out->numel() == t * hq * p.head_dim, what, ": q_out must be [tokens, heads, head_dim]");
  }
  const bool rope = rope_cos.has_value() && rope_cos->defined();
  TORCH_CHECK_VALUE(rope == (rope_sin.has_value() && rope_sin->defined()), what,
                    ": give both rotary tables or neither");
  if (rope) {
    need(*rope_cos, at::kFloat, "rope cos");
    need(*rope_sin, at::kFloat, "rope sin");
    need_same_device(*rope_cos, pool, what);
    need_same_device(*rope_sin, pool, what);
    TORCH_CHECK_VALUE(rope_cos->dim() == 2 && rope_cos->sizes() == rope_sin->sizes(), what,
                      ": rotary tables must be [positions, rotary_dim / 2]");
    TORCH_CHECK_VALUE(positions.has_value() && positions->defined(), what, ": a rotation needs positions");
  }
  for (const auto* w : {&q_norm, &k_norm})
    if (w->has_value() && (*w)->defined()) {
      need(**w, at::kBFloat16, "norm weight");
      need_same_device(**w, pool, what);
      TORCH_CHECK_VALUE((*w)->numel() == p.head_dim, what, ": norm weights must be [head_dim]");
    }
  const auto stride = [t](const at::Tensor& x) { return t > 1 ? x.stride(0) : 0; };  // of one row: not used
  check_status(
      mrb_rope_kv4_append_strided(
                          has_q ? q_in->data_ptr() : nullptr, k_in.data_ptr(), v_in.data_ptr(),
                          has_q ? stride(*q_in) : 0, stride(k_in), stride(v_in), t, hq, p.hkv, p.head_dim, group, opt_i32(positions, pool, t, "positions", what),
                          slots.data_ptr<int32_t>(), opt_ptr<float>(rope_cos), opt_ptr<float>(rope_sin),
                          rope ? rope_cos->size(0) : 0, rope ? 2 * rope_cos->size(1) : 0, interleaved ? 1 : 0,
                          opt_ptr<void>(q_norm), opt_ptr<void>(k_norm), (float)norm_eps, opt_ptr<void>(q_out),
                          pool.data_ptr(), p.pages, p.page_size, p.stride_page, p.stride_head,
                          flag_ptr(error_flag, pool, what), stream_of(pool)),
      what);
}

void kv4_read(const at::Tensor& pool, int64_t group, const at::Tensor& slots, at::Tensor& k_out, at::Tensor& v_out,
              const std::optional<at::Tensor>& error_flag) {
  const char* what = "kv4_read";
  const c10::cuda::CUDAGuard guard(pool.device());
  const Pool p = pool_of(pool, group);
  need(slots, at::kInt, "slots");
  need(k_out, k_out.scalar_type(), "k_out");
  need(v_out, k_out.scalar_type(), "v_out");
  for (const auto* t : {&slots, (const at::Tensor*)&k_out, (const at::Tensor*)&v_out}) need_same_device(*t, pool, what);
  const int64_t n = slots.numel() * p.hkv * p.head_dim;
  TORCH_CHECK_VALUE(k_out.numel() == n && v_out.numel() == n, what, ": outputs must be [tokens, kv_heads, head_dim]");
  check_status(mrb_kv4_read(pool.data_ptr(), p.pages, p.hkv, p.head_dim, group, p.page_size, p.stride_page,
                            p.stride_head, slots.data_ptr<int32_t>(), slots.numel(), k_out.data_ptr(),
                            v_out.data_ptr(), dtype_code(k_out.scalar_type()), flag_ptr(error_flag, pool, what),
                            stream_of(pool)),
               what);
}

// the shapes that the two attention operators share; returns the query heads
int64_t need_queries(const at::Tensor& q, const at::Tensor& out, const at::Tensor& pool, const Pool& p,
                     const char* what) {
  need(q, at::kBFloat16, "query");
  need(out, at::kBFloat16, "out");
  need_same_device(q, pool, what);
  need_same_device(out, pool, what);
  TORCH_CHECK_VALUE(q.dim() == 3 && q.size(2) == p.head_dim, what, ": query must be [tokens, heads, ", p.head_dim, "]");
  TORCH_CHECK_VALUE(out.sizes() == q.sizes(), what, ": out must have the query's shape");
  TORCH_CHECK_VALUE(q.size(1) > 0 && q.size(1) % p.hkv == 0, what,
                    ": query heads must be an exact multiple of K/V heads");
  return q.size(1);
}

void kv4_paged_attention(const at::Tensor& q, const at::Tensor& pool, int64_t group, const at::Tensor& block_table,
                         const at::Tensor& row_len, const std::optional<at::Tensor>& row_seq, double scale,
                         int64_t max_total_tokens, at::Tensor& out, const std::optional<at::Tensor>& workspace,
                         const std::optional<at::Tensor>& error_flag) {
  const char* what = "kv4_paged_attention";
  const c10::cuda::CUDAGuard guard(pool.device());
  const Pool p = pool_of(pool, group);
  const int64_t hq = need_queries(q, out, pool, p, what), rows = q.size(0);
  need_table(block_table, pool, what);
  need(row_len, at::kInt, "row_len");
  need_same_device(row_len, pool, what);
  TORCH_CHECK_VALUE(row_len.numel() == rows, what, ": row_len must hold one length a row");
  TORCH_CHECK_VALUE((row_seq.has_value() && row_seq->defined()) || rows <= block_table.size(0), what,
                    ": more rows than sequences");
  const bool ws = workspace.has_value() && workspace->defined();
  if (ws) {
    need(*workspace, at::kByte, "workspace");
    need_same_device(*workspace, pool, what);
  }
  check_status(mrb_kv4_paged_attention(
                   q.data_ptr(), rows, hq, p.hkv, p.head_dim, group, pool.data_ptr(), p.pages, p.page_size,
                   p.stride_page, p.stride_head, block_table.data_ptr<int32_t>(), block_table.size(0),
                   table_stride(block_table), block_table.size(1), opt_i32(row_seq, pool, rows, "row_seq", what), row_len.data_ptr<int32_t>(),
                   (float)scale, max_total_tokens, out.data_ptr(), ws ? workspace->data_ptr() : nullptr,
                   ws ? (size_t)workspace->numel() : 0, flag_ptr(error_flag, pool, what), stream_of(pool)),
               what);
}

void kv4_prefill_attention(const at::Tensor& q, const at::Tensor& pool, int64_t group, const at::Tensor& block_table,
                           const at::Tensor& q_starts, const at::Tensor& row_len,
                           const std::optional<at::Tensor>& row_seq, double scale, at::Tensor& out,
                           const at::Tensor& workspace, const std::optional<at::Tensor>& error_flag, bool zero_rest) {
  const char* what = "kv4_prefill_attention";
  const c10::cuda::CUDAGuard guard(pool.device());
  const Pool p = pool_of(pool, group);
  const int64_t hq = need_queries(q, out, pool, p, what), rows = row_len.numel();
  need_table(block_table, pool, what);
  need(row_len, at::kInt, "row_len");
  need(q_starts, at::kInt, "q_starts");
  need_same_device(row_len, pool, what);
  need_same_device(q_starts, pool, what);
  need(workspace, at::kByte, "workspace");
  need_same_device(workspace, pool, what);
  TORCH_CHECK_VALUE(q_starts.numel() == rows + 1, what, ": q_starts must hold one entry a row and the end");
  TORCH_CHECK_VALUE((row_seq.has_value() && row_seq->defined()) || rows <= block_table.size(0), what,
                    ": more rows than sequences");
  const auto run = zero_rest ? &mrb_kv4_prefill_attention_all : &mrb_kv4_prefill_attention;
  check_status(run(
                   q.data_ptr(), q.size(0), rows, hq, p.hkv, p.head_dim, group, pool.data_ptr(), p.pages, p.page_size,
                   p.stride_page, p.stride_head, block_table.data_ptr<int32_t>(), block_table.size(0),
                   table_stride(block_table), block_table.size(1), q_starts.data_ptr<int32_t>(), opt_i32(row_seq, pool, rows, "row_seq", what),
                   row_len.data_ptr<int32_t>(), (float)scale, out.data_ptr(), workspace.data_ptr(),
                   (size_t)workspace.numel(), flag_ptr(error_flag, pool, what), stream_of(pool)),
               what);
}

}  // namespace

TORCH_LIBRARY(mrun_b200, m) {
  m.def("qrow_linear(Tensor x, Tensor codes, Tensor scales, Tensor? bias, Tensor(a!) out, Tensor? workspace) -> ()");
  m.def("qrow_swiglu(Tensor x, Tensor gate_codes, Tensor gate_scales, Tensor up_codes, Tensor up_scales, "
        "Tensor(a!) out, Tensor? workspace) -> ()");
  m.def("quant_row_int8(Tensor weight, Tensor(a!) codes, Tensor(b!) scales) -> ()");
  m.def("router_topk(Tensor logits, int k, bool renorm, Tensor(a!) top_idx, Tensor(b!) top_w_f32, "
        "Tensor(c!) top_w_bf16) -> ()");
  m.def("route_compile(Tensor top_idx, Tensor top_w, int experts, Tensor(a!) counts, Tensor(b!) starts, "
        "Tensor(c!) token_ids, Tensor(d!) coef, Tensor(e!) inverse) -> ()");
  m.def("stable_route_reduce(Tensor expert_out, Tensor coef, Tensor inverse, int tokens, int k, "
        "Tensor(a!)? out_f32, Tensor(b!)? out_bf16) -> ()");
  m.def("grouped_expert_mlp(Tensor x, Tensor token_ids, Tensor starts, Tensor counts, Tensor pages, int page_stride, "
        "int gate_up_codes_offset, int gate_up_scales_offset, int down_codes_offset, int down_scales_offset, "
        "Tensor? slot_of, Tensor(a!) act, Tensor(b!) y, Tensor(c!) sync) -> ()");
  m.def("kv_plan_step(Tensor new_tokens, Tensor? row_seq, Tensor lengths, Tensor(a!) lengths_out, "
        "Tensor(b!) block_table, Tensor free_pages, Tensor free_count, Tensor(c!) free_count_out, int page_size, "
        "Tensor(d!) q_starts, Tensor(e!) row_len, Tensor(f!) positions, Tensor(g!) token_rows, Tensor(h!) slots, "
        "Tensor(i!)? error_flag) -> ()");
  m.def("kv_release(Tensor seqs, Tensor(a!) lengths, Tensor(b!) block_table, Tensor(c!) free_pages, "
        "Tensor(d!) free_count, int page_size, Tensor(e!)? error_flag) -> ()");
  m.def("rope_kv4_append(Tensor? q_in, Tensor k_in, Tensor v_in, Tensor(a!) pool, int group, Tensor slots, "
        "Tensor? positions, Tensor? rope_cos, Tensor? rope_sin, bool interleaved, Tensor? q_norm, Tensor? k_norm, "
        "float norm_eps, Tensor(b!)? q_out, Tensor(c!)? error_flag) -> ()");
  m.def("kv4_read(Tensor pool, int group, Tensor slots, Tensor(a!) k_out, Tensor(b!) v_out, "
        "Tensor(c!)? error_flag) -> ()");
  m.def("kv4_paged_attention(Tensor q, Tensor pool, int group, Tensor block_table, Tensor row_len, Tensor? row_seq, "
        "float scale, int max_total_tokens, Tensor(a!) out, Tensor(b!)? workspace, Tensor(c!)? error_flag) -> ()");
  m.def("kv4_prefill_attention(Tensor q, Tensor pool, int group, Tensor block_table, Tensor q_starts, "
        "Tensor row_len, Tensor? row_seq, float scale, Tensor(a!) out, Tensor(c!) workspace, Tensor(b!)? error_flag, "
        "bool zero_rest=False) -> ()");
}

TORCH_LIBRARY_IMPL(mrun_b200, CUDA, m) {
  m.impl("qrow_linear", &qrow_linear);
  m.impl("qrow_swiglu", &qrow_swiglu);
  m.impl("quant_row_int8", &quant_row_int8);
  m.impl("router_topk", &router_topk);
  m.impl("route_compile", &route_compile);
  m.impl("stable_route_reduce", &stable_route_reduce);
  m.impl("grouped_expert_mlp", &grouped_expert_mlp);
  m.impl("kv_plan_step", &kv_plan_step);
  m.impl("kv_release", &kv_release);
  m.impl("rope_kv4_append", &rope_kv4_append);
  m.impl("kv4_read", &kv4_read);
  m.impl("kv4_paged_attention", &kv4_paged_attention);
  m.impl("kv4_prefill_attention", &kv4_prefill_attention);
}
