// sv_torch.cpp -- the thin PyTorch C++ extension over the C ABI
// (include/starvector_sampling.h).
//
// Each function takes torch tensors, checks them (device, dtype, sizes) with
// TORCH_CHECK, calls the C entry point on the tensors' current CUDA stream and
// returns its code (0 or a negative SV_E_*; ops.py turns codes into the same
// exceptions as before).  Shapes and the history form are decided by the Python
// wrappers (ops.py), which pass the same sizes and strides as the C signatures;
// nothing here synchronises or allocates.  The cache operators (window_attention,
// prefix_attention, quantized_attention, kv_quantize, kv_dequantize, kv_evict) are called
// once per layer or token, where each tensor attribute read from Python counts: they look at the shapes here (ValueError where
// ops.py would raise one) and allocate their outputs, the attention functions also a
// workspace kept per device, stream and size.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <cmath>
#include <cstdint>
#include <map>
#include <optional>
#include <tuple>

#include "../../include/starvector_sampling.h"

namespace {

using OptT = std::optional<at::Tensor>;

void on_device(const at::Tensor& t, const at::Device& dev, const char* name) {
  TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor (the B200 sampling kernels have no CPU path)");
  TORCH_CHECK(t.device() == dev, name, " must be on ", dev, ", not ", t.device());
}

template <typename T>
T* ptr(const at::Tensor& t, const at::Device& dev, const char* name, at::ScalarType st, int64_t min_numel = 1) {
  on_device(t, dev, name);
  TORCH_CHECK(t.scalar_type() == st, name, " must be ", st, ", not ", t.scalar_type());
  TORCH_CHECK(t.numel() >= min_numel, name, " holds ", t.numel(), " elements, needs ", min_numel);
  return reinterpret_cast<T*>(t.data_ptr());
}

template <typename T>
T* optptr(const OptT& t, const at::Device& dev, const char* name, at::ScalarType st, int64_t min_numel = 1) {
  return t.has_value() ? ptr<T>(*t, dev, name, st, min_numel) : nullptr;
}

void* raw(const OptT& t, const at::Device& dev, const char* name) {
  if (!t.has_value()) return nullptr;
  on_device(*t, dev, name);
  return t->data_ptr();
}

int32_t logit_code(const at::Tensor& x) {
  switch (x.scalar_type()) {
    case at::kFloat: return SV_F32;
    case at::kHalf: return SV_F16;
    case at::kBFloat16: return SV_BF16;
    default: TORCH_CHECK(false, "logits must be float32, float16 or bfloat16, not ", x.scalar_type());
  }
  return -1;
}

void* stream_of(const at::Tensor& t) { return at::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

// sv_sample_step (runtime_shared.py:194-202).
int sample_step(const at::Tensor& logits, int64_t rows, int64_t vocab, int64_t row_stride, const OptT& history,
                 int64_t history_kind, int64_t history_row_stride, const OptT& history_len, int64_t history_cols,
                 const at::Tensor& uniforms, double temperature, double top_p, int64_t top_k, int64_t keep,
                 double repetition_penalty, const at::Tensor& out_token, const OptT& out_count, const OptT& out_idx,
                 const OptT& out_prob, const OptT& out_score, int64_t out_capacity, const OptT& out_dense,
                 int64_t dense_mode, int64_t dense_row_stride, const at::Tensor& out_status, const OptT& seen_update,
                 int64_t seen_update_row_stride, int64_t flags) {
  const at::Device dev = logits.device();
  on_device(logits, dev, "logits");
  const c10::cuda::CUDAGuard guard(dev);
  const int rc = sv_sample_step(
      logits.data_ptr(), logit_code(logits), (int32_t)rows, (int32_t)vocab, row_stride, raw(history, dev, "history"),
      (int32_t)history_kind, history_row_stride, optptr<int32_t>(history_len, dev, "history_len", at::kInt, rows),
      (int32_t)history_cols, ptr<float>(uniforms, dev, "uniforms", at::kFloat, rows), temperature, top_p,
      (int32_t)top_k, (int32_t)keep, repetition_penalty, ptr<int64_t>(out_token, dev, "token", at::kLong, rows),
      optptr<int32_t>(out_count, dev, "count", at::kInt, rows),
      optptr<int32_t>(out_idx, dev, "idx", at::kInt, rows * out_capacity),
      optptr<float>(out_prob, dev, "prob", at::kFloat, rows * out_capacity),
      optptr<float>(out_score, dev, "score", at::kFloat, rows * out_capacity), (int32_t)out_capacity,
      optptr<float>(out_dense, dev, "dense", at::kFloat, rows * vocab), (int32_t)dense_mode, dense_row_stride,
      ptr<int32_t>(out_status, dev, "status", at::kInt, rows),
      optptr<uint32_t>(seen_update, dev, "update_seen_bits", at::kInt), seen_update_row_stride, (int32_t)flags,
      stream_of(logits));
  return rc;
}

// sv_beam_step (runtime_shared.py:230-237).
int beam_step(const at::Tensor& logits, int64_t beams, int64_t vocab, int64_t row_stride, const OptT& history,
               int64_t history_kind, int64_t history_row_stride, const OptT& history_len, int64_t history_cols,
               const at::Tensor& running_scores, const at::Tensor& uniforms, int64_t num_picks, double temperature,
               double top_p, int64_t top_k, int64_t keep, double repetition_penalty, const at::Tensor& out_picks,
               const at::Tensor& out_pick_scores, const at::Tensor& out_num_picks, const at::Tensor& out_status,
               const OptT& out_kept_count, const OptT& out_kept_idx, const OptT& out_kept_logprob,
               const OptT& out_kept_prob, int64_t out_capacity, const OptT& out_dense_logprob,
               int64_t dense_row_stride, const at::Tensor& workspace, int64_t flags) {
  const at::Device dev = logits.device();
  on_device(logits, dev, "logits");
  const c10::cuda::CUDAGuard guard(dev);
  const int rc = sv_beam_step(
      logits.data_ptr(), logit_code(logits), (int32_t)beams, (int32_t)vocab, row_stride,
      raw(history, dev, "history"), (int32_t)history_kind, history_row_stride,
      optptr<int32_t>(history_len, dev, "history_len", at::kInt, beams), (int32_t)history_cols,
      ptr<float>(running_scores, dev, "running_scores", at::kFloat, beams),
      ptr<float>(uniforms, dev, "uniforms", at::kFloat, num_picks), (int32_t)num_picks, temperature, top_p,
      (int32_t)top_k, (int32_t)keep, repetition_penalty, ptr<int64_t>(out_picks, dev, "picks", at::kLong, num_picks),
      ptr<float>(out_pick_scores, dev, "scores", at::kFloat, num_picks),
      ptr<int32_t>(out_num_picks, dev, "n", at::kInt), ptr<int32_t>(out_status, dev, "status", at::kInt),
      optptr<int32_t>(out_kept_count, dev, "kept_count", at::kInt, beams),
      optptr<int32_t>(out_kept_idx, dev, "kept_idx", at::kInt, beams * out_capacity),
      optptr<float>(out_kept_logprob, dev, "kept_logprob", at::kFloat, beams * out_capacity),
      optptr<float>(out_kept_prob, dev, "kept_prob", at::kFloat, beams * out_capacity), (int32_t)out_capacity,
      optptr<float>(out_dense_logprob, dev, "dense_logprob", at::kFloat, beams * vocab), dense_row_stride,
      ptr<uint8_t>(workspace, dev, "workspace", at::kByte), (size_t)workspace.numel(), (int32_t)flags,
      stream_of(logits));
  return rc;
}

// sv_beam_advance (runtime_shared.py:237-259).
int beam_advance(const at::Tensor& picks, const at::Tensor& pick_scores, const at::Tensor& n_picks,
                  const at::Tensor& status, int64_t beams, int64_t vocab, int64_t step, bool last,
                  const OptT& stop_ids, int64_t eos_id, const OptT& tails_in, const OptT& tails_out,
                  const at::Tensor& running_out, const at::Tensor& parents_out, const at::Tensor& tokens_out,
                  const OptT& seen_in, const OptT& seen_out, int64_t seen_stride_words, const OptT& hist_in,
                  const OptT& hist_out, int64_t hist_stride, const OptT& whash_in, const OptT& whash_out,
                  const OptT& guard_table, int64_t window) {
  const at::Device dev = picks.device();
  const c10::cuda::CUDAGuard guard(dev);
  const int64_t num_picks = picks.numel();
  const int64_t n_stop = stop_ids.has_value() ? stop_ids->numel() : 0;
  const int rc = sv_beam_advance(
      ptr<int64_t>(picks, dev, "picks", at::kLong), ptr<float>(pick_scores, dev, "scores", at::kFloat, num_picks),
      ptr<int32_t>(n_picks, dev, "n", at::kInt), ptr<int32_t>(status, dev, "status", at::kInt), (int32_t)beams,
      (int32_t)vocab, (int32_t)num_picks, (int32_t)step, last ? 1 : 0,
      n_stop ? optptr<int64_t>(stop_ids, dev, "stop_ids", at::kLong) : nullptr, (int32_t)n_stop, eos_id,
      n_stop ? optptr<int64_t>(tails_in, dev, "tails_in", at::kLong, beams * n_stop) : nullptr,
      n_stop ? optptr<int64_t>(tails_out, dev, "tails_out", at::kLong, beams * n_stop) : nullptr,
      ptr<float>(running_out, dev, "running_out", at::kFloat, beams),
      ptr<int64_t>(parents_out, dev, "parents_out", at::kLong, beams),
      ptr<int64_t>(tokens_out, dev, "tokens_out", at::kLong, beams),
      optptr<uint32_t>(seen_in, dev, "seen_in", at::kInt), optptr<uint32_t>(seen_out, dev, "seen_out", at::kInt),
      seen_stride_words, optptr<int32_t>(hist_in, dev, "hist_in", at::kInt),
      optptr<int32_t>(hist_out, dev, "hist_out", at::kInt), hist_stride,
      optptr<uint32_t>(whash_in, dev, "whash_in", at::kInt, beams),
      optptr<uint32_t>(whash_out, dev, "whash_out", at::kInt, beams),
      optptr<unsigned long long>(guard_table, dev, "guard_table", at::kLong),
      guard_table.has_value() ? guard_table->numel() : 0, (int32_t)window, stream_of(picks));
  return rc;
}

// sv_kv_reorder (runtime_shared.py:388-394).
int kv_reorder(const at::Tensor& keys, const OptT& values, int64_t layers, int64_t beams, int64_t heads,
                int64_t length, int64_t head_dim, int64_t stride_layer, int64_t stride_beam, int64_t stride_head,
                int64_t stride_slot, const at::Tensor& parents, const OptT& out_status) {
  const at::Device dev = keys.device();
  on_device(keys, dev, "keys");
  const c10::cuda::CUDAGuard guard(dev);
  const int rc = sv_kv_reorder(keys.data_ptr(), raw(values, dev, "values"), (int32_t)keys.element_size(),
                               (int32_t)layers, (int32_t)beams, (int32_t)heads, length, (int32_t)head_dim,
                               stride_layer, stride_beam, stride_head, stride_slot,
                               ptr<int64_t>(parents, dev, "parents", at::kLong, beams),
                               optptr<int32_t>(out_status, dev, "status", at::kInt), stream_of(keys));
  return rc;
}

// sv_loop_guard (runtime_shared.py:156-167).
int loop_guard(const at::Tensor& tokens, int64_t rows, int64_t row_stride, const at::Tensor& lengths, int64_t window,
                int64_t repeats, const at::Tensor& out_verdict) {
  const at::Device dev = tokens.device();
  on_device(tokens, dev, "tokens");
  const c10::cuda::CUDAGuard guard(dev);
  const int rc = sv_loop_guard(tokens.data_ptr(), (int32_t)tokens.element_size(), (int32_t)rows, row_stride,
                               ptr<int32_t>(lengths, dev, "lengths", at::kInt, rows), (int32_t)window,
                               (int32_t)repeats, ptr<uint8_t>(out_verdict, dev, "verdict", at::kByte, rows),
                               stream_of(tokens));
  return rc;
}

// sv_loop_guard_incremental (runtime_shared.py:156-167, :207, :254).
int loop_guard_incremental(const at::Tensor& table, const at::Tensor& tokens, int64_t insert_from, int64_t length,
                            int64_t window, int64_t repeats, const at::Tensor& out_verdict, const OptT& out_status) {
  const at::Device dev = tokens.device();
  on_device(tokens, dev, "tokens");
  const c10::cuda::CUDAGuard guard(dev);
  const int rc = sv_loop_guard_incremental(
      ptr<unsigned long long>(table, dev, "table", at::kLong), table.numel(), tokens.data_ptr(),
      (int32_t)tokens.element_size(), insert_from, length, (int32_t)window, (int32_t)repeats,
      ptr<uint8_t>(out_verdict, dev, "verdict", at::kByte), optptr<int32_t>(out_status, dev, "status", at::kInt),
      stream_of(tokens));
  return rc;
}

// A workspace of at least `bytes` whose first `zeroed` bytes were zero before its
// first use, kept per device, stream and power of two for the life of the process
// (calls on different streams may overlap).  Under a stream capture it comes from the
// graph's own pool instead, cleared by a node of the graph: a kept one would be
// cleared only when the graph runs, and eager calls could overlap the graph's.
at::Tensor workspace_for(const at::Device& dev, c10::cuda::CUDAStream stream, size_t bytes, size_t zeroed) {
  const auto opts = at::TensorOptions().dtype(at::kByte).device(dev);
  if (bytes == 0) return at::Tensor();
  if (c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None) {
    at::Tensor t = at::empty({(int64_t)bytes}, opts);
    t.narrow(0, 0, (int64_t)std::min(bytes, zeroed)).zero_();
    return t;
  }
  static auto* kept = new std::map<std::tuple<int, void*, size_t>, at::Tensor>;
  size_t size = 1 << 16;
  while (size < bytes) size *= 2;
  at::Tensor& t = (*kept)[std::make_tuple((int)dev.index(), (void*)stream.stream(), size)];
  if (!t.defined()) t = at::zeros({(int64_t)size}, opts);
  return t;
}

// Strides of a dimension of one entry mean nothing: 0 stands for them.
int64_t stride_of(const at::Tensor& t, int64_t d) { return t.size(d) > 1 ? t.stride(d) : 0; }

// Whether b is laid out as a.
bool same_layout(const at::Tensor& a, const at::Tensor& b) {
  if (a.sizes() != b.sizes()) return false;
  for (int64_t d = 0; d < a.dim(); ++d)
    if (stride_of(a, d) != stride_of(b, d)) return false;
  return true;
}

// Whether dimension d lies contiguously (a broadcast one, of stride 0, does not).
bool contiguous_along(const at::Tensor& t, int64_t d) { return t.size(d) <= 1 || t.stride(d) == 1; }

// A size as the C interface takes it.
int32_t size32(const at::Tensor& t, int64_t d) {
  TORCH_CHECK_VALUE(t.size(d) <= INT32_MAX, "a dimension of ", t.size(d), " entries is too large");
  return (int32_t)t.size(d);
}

bool aligned(const at::Tensor& t, int64_t dims) {
  if (reinterpret_cast<uintptr_t>(t.data_ptr()) % 16) return false;
  const int64_t e = t.element_size();
  for (int64_t d = 0; d < dims; ++d)
    if (stride_of(t, d) * e % 16) return false;
  return true;
}

// q as [rows, tokens, heads, head_dim] with 16-byte aligned rows; [rows, heads,
// head_dim] stands for one token.
at::Tensor queries(const at::Tensor& q) {
  TORCH_CHECK(q.is_cuda(), "q must be a CUDA tensor (the B200 sampling kernels have no CPU path)");
  TORCH_CHECK_VALUE(q.dim() == 3 || q.dim() == 4,
                    "q must be [rows, tokens, heads, head_dim] or [rows, heads, head_dim]");
  const auto st = q.scalar_type();
  TORCH_CHECK_VALUE(st == at::kFloat || st == at::kHalf || st == at::kBFloat16, "unsupported dtype ", st);
  at::Tensor x = q.dim() == 3 ? q.unsqueeze(1) : q;
  if (!contiguous_along(x, 3) || !aligned(x, 3)) x = x.clone(at::MemoryFormat::Contiguous);
  return x;
}

// One layer's keys or values as [rows, kv_heads, capacity, head_dim].
at::Tensor layer_cache(const at::Tensor& t) { return t.dim() == 3 ? t.unsqueeze(1) : t; }

void check_cache(const at::Tensor& k, const at::Tensor& v, const at::Tensor& q) {
  const at::Device dev = q.device();
  on_device(k, dev, "keys");
  on_device(v, dev, "values");
  TORCH_CHECK_VALUE(k.dim() == 4 && same_layout(k, v),
                    "keys must be [rows, capacity, head_dim] or [rows, kv_heads, capacity, head_dim], and values "
                    "have their shape and strides");
  TORCH_CHECK_VALUE(k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(),
                    "keys and values must have q's dtype");
  TORCH_CHECK_VALUE(k.size(0) == q.size(0) && k.size(3) == q.size(3) && k.size(1) > 0 && q.size(2) % k.size(1) == 0,
                    "keys must have q's rows and head_dim, and kv_heads must divide heads");
  TORCH_CHECK_VALUE(contiguous_along(k, 3), "head_dim must be contiguous");
}

// A per-row int32 tensor from a tensor of whole numbers (none stays none).
OptT row_ints(const OptT& t, int64_t rows, const at::Device& dev, const char* name) {
  if (!t.has_value()) return t;
  const auto st = t->scalar_type();
  TORCH_CHECK_VALUE((st == at::kInt || st == at::kLong) && t->numel() == rows, name,
                    " must be an int32 or int64 tensor with one value per row");
  if (st == at::kInt && t->device() == dev && t->is_contiguous()) return t;
  return t->reshape({-1}).to(dev, at::kInt).contiguous();
}

// A status per row, or none.
int32_t* status_ptr(const OptT& t, int64_t rows, const at::Device& dev) {
  TORCH_CHECK(!t.has_value() || t->is_contiguous(), "status must be contiguous");
  return optptr<int32_t>(t, dev, "status", at::kInt, rows);
}

// The statuses of a call that has no queries or no slots, and launches nothing.
void fill_status(const OptT& status, const OptT& lengths, const OptT& starts, int64_t rows, int64_t capacity,
                 const at::Device& dev) {
  if (status_ptr(status, rows, dev) == nullptr || rows == 0) return;
  const auto ints = at::TensorOptions().dtype(at::kInt).device(dev);
  const at::Tensor end = lengths.has_value() ? lengths->reshape({-1}) : at::full({rows}, capacity, ints);
  at::Tensor bad = end.lt(0).logical_or(end.gt(capacity));
  if (starts.has_value()) {
    const at::Tensor start = starts->reshape({-1});
    bad = bad.logical_or(start.lt(0)).logical_or(start.gt(end.clamp_min(0)));
  }
  status->view({-1}).narrow(0, 0, rows).copy_(bad.to(at::kInt).mul(SV_ST_LENGTH));
}

at::Tensor attention_out(const OptT& out, const at::Tensor& q) {
  if (!out.has_value()) return at::empty(q.sizes(), q.options());
  on_device(*out, q.device(), "out");
  TORCH_CHECK(out->scalar_type() == q.scalar_type() && out->sizes() == q.sizes() && out->is_contiguous(),
              "out must be a contiguous tensor of the queries' shape and dtype");
  return *out;
}

void check_window(int64_t window, int64_t sinks, std::optional<double> scale) {
  TORCH_CHECK_VALUE(window >= 0 && sinks >= 0, "window and sinks must not be negative");
  TORCH_CHECK_VALUE(!scale.has_value() || std::isfinite(*scale), "scale must be finite");
}

// The accumulator of an attention's weights as [rows, kv_heads, slots], or none.
OptT check_weights(const OptT& given, int64_t rows, int64_t kv, int64_t capacity) {
  OptT weights = given;
  if (!weights.has_value()) return weights;
  if (weights->dim() == 2) weights = weights->unsqueeze(1);
  TORCH_CHECK_VALUE(weights->scalar_type() == at::kFloat && weights->dim() == 3 && weights->size(0) == rows &&
                        weights->size(1) == kv && weights->size(2) >= capacity && contiguous_along(*weights, 2),
                    "weights must be float32 [rows, kv_heads, capacity], contiguous along the slots");
  TORCH_CHECK_VALUE((rows <= 1 || weights->stride(0) > 0) && (kv <= 1 || weights->stride(1) > 0),
                    "weights are added to in place: rows and heads must not be broadcast");
  return weights;
}

// sv_window_attention.
std::tuple<int, at::Tensor> window_attention(const at::Tensor& q_in, const at::Tensor& keys_in,
                                             const at::Tensor& values_in, const OptT& lengths_in,
                                             const OptT& starts_in, int64_t window, int64_t sinks,
                                             std::optional<double> scale, const OptT& weights_in, const OptT& out,
                                             const OptT& out_status) {
  const at::Tensor q = queries(q_in), keys = layer_cache(keys_in), values = layer_cache(values_in);
  check_cache(keys, values, q);
  const at::Device dev = q.device();
  const c10::cuda::CUDAGuard guard(dev);
  const auto stream = at::cuda::getCurrentCUDAStream(dev.index());
  const int32_t rows = size32(q, 0), n = size32(q, 1), heads = size32(q, 2), dim = size32(q, 3);
  const int32_t kv = size32(keys, 1), capacity = size32(keys, 2), code = logit_code(q);
  check_window(window, sinks, scale);
  const OptT weights = check_weights(weights_in, rows, kv, capacity);
  const OptT lengths = row_ints(lengths_in, rows, dev, "lengths"), starts = row_ints(starts_in, rows, dev, "starts");
  const int32_t w = (int32_t)std::min<int64_t>(window, 1 << 30), s = (int32_t)std::min<int64_t>(sinks, 1 << 30);
  at::Tensor o = attention_out(out, q_in);
  if (o.numel() == 0 || capacity == 0) {  // no slots: every query sees nothing
    fill_status(out_status, lengths, starts, rows, capacity, dev);
    return {0, o.zero_()};
  }
  const size_t bytes =
      sv_window_attention_workspace_bytes(code, rows, n, heads, kv, dim, capacity, w, s, weights.has_value());
  at::Tensor ws = workspace_for(dev, stream, bytes, 4 * ((size_t)rows * kv + 1024));
  const int rc = sv_window_attention(
      q.data_ptr(), code, rows, n, heads, kv, dim, stride_of(q, 0), stride_of(q, 1), stride_of(q, 2), keys.data_ptr(),
      values.data_ptr(), capacity, stride_of(keys, 0), stride_of(keys, 1), stride_of(keys, 2),
      optptr<int32_t>(lengths, dev, "lengths", at::kInt, rows), optptr<int32_t>(starts, dev, "starts", at::kInt, rows),
      w, s, scale.has_value() ? *scale : 1.0 / std::sqrt((double)dim),
      optptr<float>(weights, dev, "weights", at::kFloat), weights.has_value() ? stride_of(*weights, 0) : 0,
      weights.has_value() ? stride_of(*weights, 1) : 0, o.data_ptr(), ws.defined() ? ws.data_ptr() : nullptr,
      ws.defined() ? (size_t)ws.numel() : 0, status_ptr(out_status, rows, dev),
      stream.stream());
  return {rc, o};
}

// One layer of a cache held in 4 bits as [rows, kv_heads, capacity, record].
void check_records(const at::Tensor& k, const OptT& v, int64_t rows, int64_t dim, const at::Device& dev) {
  on_device(k, dev, "cache_keys");
  if (v.has_value()) on_device(*v, dev, "cache_values");
  const int64_t bytes = dim >= 0 && dim <= INT32_MAX ? sv_kv_record_bytes((int32_t)dim) : 0;
  TORCH_CHECK_VALUE(bytes > 0, "head_dim must be a multiple of 8 in [8, 128]");
  TORCH_CHECK_VALUE(k.scalar_type() == at::kByte && (!v.has_value() || v->scalar_type() == at::kByte),
                    "caches held in 4 bits must be uint8");
  TORCH_CHECK_VALUE(k.dim() == 4 && k.size(3) == bytes && k.size(0) == rows && k.size(1) > 0,
                    "cache_keys must be [rows, capacity, record] or [rows, kv_heads, capacity, record], of ", bytes,
                    " bytes a record for this head_dim");
  TORCH_CHECK_VALUE(!v.has_value() || same_layout(k, *v), "cache_values must have the shape and strides of cache_keys");
  TORCH_CHECK_VALUE(contiguous_along(k, 3), "records must be contiguous");
}

OptT layer_cache(const OptT& t) { return t.has_value() ? OptT(layer_cache(*t)) : t; }

// sv_kv_quantize.
int kv_quantize(const at::Tensor& keys_in, const OptT& values_in, const at::Tensor& cache_keys_in,
                const OptT& cache_values_in, const OptT& lengths_in, const OptT& out_status) {
  at::Tensor keys = layer_cache(keys_in);
  OptT values = layer_cache(values_in);
  const at::Tensor ck = layer_cache(cache_keys_in);
  const OptT cv = layer_cache(cache_values_in);
  const at::Device dev = keys.device();
  on_device(keys, dev, "keys");
  const auto st = keys.scalar_type();
  TORCH_CHECK_VALUE(st == at::kFloat || st == at::kHalf || st == at::kBFloat16, "unsupported dtype ", st);
  TORCH_CHECK_VALUE(keys.dim() == 4, "keys must be [rows, tokens, head_dim] or [rows, kv_heads, tokens, head_dim]");
  TORCH_CHECK_VALUE(values.has_value() == cv.has_value(), "values and cache_values go together");
  if (values.has_value()) {
    on_device(*values, dev, "values");
    TORCH_CHECK_VALUE(values->scalar_type() == st && values->sizes() == keys.sizes(),
                      "values must have the keys' shape and dtype");
  }
  check_records(ck, cv, keys.size(0), keys.size(3), dev);
  TORCH_CHECK_VALUE(ck.size(1) == keys.size(1), "the cache must have the keys' heads");
  const c10::cuda::CUDAGuard guard(dev);
  const OptT lengths = row_ints(lengths_in, keys.size(0), dev, "lengths");
  if (keys.numel() == 0 || ck.numel() == 0) {
    fill_status(out_status, lengths, std::nullopt, keys.size(0), ck.size(2), dev);
    return 0;
  }
  // Other layouts are copied first (values at strides of their own among them).
  if (!contiguous_along(keys, 3) || !aligned(keys, 3) ||
      (values.has_value() && (!same_layout(keys, *values) || !aligned(*values, 3)))) {
    keys = keys.clone(at::MemoryFormat::Contiguous);
    if (values.has_value()) values = values->clone(at::MemoryFormat::Contiguous);
  }
  return sv_kv_quantize(keys.data_ptr(), raw(values, dev, "values"), logit_code(keys), size32(keys, 0), size32(keys, 1),
                        size32(keys, 2), size32(keys, 3), stride_of(keys, 0), stride_of(keys, 1), stride_of(keys, 2),
                        ck.data_ptr(), raw(cv, dev, "cache_values"), size32(ck, 2), stride_of(ck, 0), stride_of(ck, 1),
                        stride_of(ck, 2), optptr<int32_t>(lengths, dev, "lengths", at::kInt, keys.size(0)),
                        status_ptr(out_status, keys.size(0), dev), stream_of(keys));
}

// sv_kv_dequantize.
std::tuple<int, at::Tensor, OptT> kv_dequantize(const at::Tensor& cache_keys_in, const OptT& cache_values_in,
                                                int64_t head_dim, const OptT& lengths_in, std::optional<int64_t> tokens,
                                                at::ScalarType dtype, const OptT& keys_out, const OptT& values_out,
                                                const OptT& out_status) {
  const at::Tensor ck = layer_cache(cache_keys_in);
  const OptT cv = layer_cache(cache_values_in);
  const at::Device dev = ck.device();
  TORCH_CHECK_VALUE(ck.dim() == 4, "cache_keys must be [rows, capacity, record] or [rows, kv_heads, capacity, record]");
  check_records(ck, cv, ck.size(0), head_dim, dev);
  TORCH_CHECK_VALUE(dtype == at::kFloat || dtype == at::kHalf || dtype == at::kBFloat16, "unsupported dtype ", dtype);
  TORCH_CHECK_VALUE(!tokens.has_value() || (*tokens >= 0 && *tokens <= 1 << 29), "tokens must be in [0, 2^29]");
  const int64_t places = tokens.has_value() ? *tokens : ck.size(2);
  auto shape = cache_keys_in.sizes().vec();
  shape[shape.size() - 2] = places;
  shape[shape.size() - 1] = head_dim;
  const c10::cuda::CUDAGuard guard(dev);
  const auto make = [&](const OptT& given, const char* name) {
    if (!given.has_value()) return at::empty(shape, ck.options().dtype(dtype));
    on_device(*given, dev, name);
    TORCH_CHECK(given->scalar_type() == dtype && given->sizes() == at::IntArrayRef(shape) && given->is_contiguous(),
                "out must be contiguous tensors of the outputs' shape and dtype");
    return *given;
  };
  at::Tensor keys = make(keys_out, "out");
  OptT values;
  if (cv.has_value()) values = make(values_out, "out");
  const OptT lengths = row_ints(lengths_in, ck.size(0), dev, "lengths");
  if (keys.numel() == 0 || ck.numel() == 0) {
    fill_status(out_status, lengths, std::nullopt, ck.size(0), ck.size(2), dev);
    keys.zero_();
    if (values.has_value()) values->zero_();
    return {0, keys, values};
  }
  const int rc = sv_kv_dequantize(
      ck.data_ptr(), raw(cv, dev, "cache_values"), size32(ck, 0), size32(ck, 1), (int32_t)head_dim, size32(ck, 2),
      stride_of(ck, 0), stride_of(ck, 1), stride_of(ck, 2),
      optptr<int32_t>(lengths, dev, "lengths", at::kInt, ck.size(0)), tokens.has_value() ? (int32_t)places : 0,
      keys.data_ptr(), values.has_value() ? values->data_ptr() : nullptr, logit_code(keys),
      status_ptr(out_status, ck.size(0), dev), stream_of(ck));
  return {rc, keys, values};
}

// sv_quantized_attention.
std::tuple<int, at::Tensor> quantized_attention(const at::Tensor& q_in, const at::Tensor& cache_keys_in,
                                                const at::Tensor& cache_values_in, const OptT& lengths_in,
                                                const OptT& starts_in, int64_t window, int64_t sinks,
                                                std::optional<double> scale, const OptT& weights_in, const OptT& out,
                                                const OptT& out_status) {
  const at::Tensor q = queries(q_in), ck = layer_cache(cache_keys_in), cv = layer_cache(cache_values_in);
  const at::Device dev = q.device();
  check_records(ck, cv, q.size(0), q.size(3), dev);
  TORCH_CHECK_VALUE(q.size(2) % ck.size(1) == 0, "kv_heads must divide heads");
  const c10::cuda::CUDAGuard guard(dev);
  const auto stream = at::cuda::getCurrentCUDAStream(dev.index());
  const int32_t rows = size32(q, 0), n = size32(q, 1), heads = size32(q, 2), dim = size32(q, 3);
  const int32_t kv = size32(ck, 1), capacity = size32(ck, 2), code = logit_code(q);
  check_window(window, sinks, scale);
  const OptT weights = check_weights(weights_in, rows, kv, capacity);
  const OptT lengths = row_ints(lengths_in, rows, dev, "lengths"), starts = row_ints(starts_in, rows, dev, "starts");
  const int32_t w = (int32_t)std::min<int64_t>(window, 1 << 30), s = (int32_t)std::min<int64_t>(sinks, 1 << 30);
  at::Tensor o = attention_out(out, q_in);
  if (o.numel() == 0 || capacity == 0) {  // no slots: every query sees nothing
    fill_status(out_status, lengths, starts, rows, capacity, dev);
    return {0, o.zero_()};
  }
  const size_t bytes =
      sv_quantized_attention_workspace_bytes(code, rows, n, heads, kv, dim, capacity, w, s, weights.has_value());
  at::Tensor ws = workspace_for(dev, stream, bytes, 4 * ((size_t)rows * kv * 4 + 1024));
  const int rc = sv_quantized_attention(
      q.data_ptr(), code, rows, n, heads, kv, dim, stride_of(q, 0), stride_of(q, 1), stride_of(q, 2), ck.data_ptr(),
      cv.data_ptr(), capacity, stride_of(ck, 0), stride_of(ck, 1), stride_of(ck, 2),
      optptr<int32_t>(lengths, dev, "lengths", at::kInt, rows), optptr<int32_t>(starts, dev, "starts", at::kInt, rows),
      w, s, scale.has_value() ? *scale : 1.0 / std::sqrt((double)dim),
      optptr<float>(weights, dev, "weights", at::kFloat), weights.has_value() ? stride_of(*weights, 0) : 0,
      weights.has_value() ? stride_of(*weights, 1) : 0, o.data_ptr(), ws.defined() ? ws.data_ptr() : nullptr,
      ws.defined() ? (size_t)ws.numel() : 0, status_ptr(out_status, rows, dev), stream.stream());
  return {rc, o};
}

// sv_prefix_attention.
std::tuple<int, at::Tensor> prefix_attention(const at::Tensor& q_in, const at::Tensor& prefix_keys_in,
                                             const at::Tensor& prefix_values_in, const at::Tensor& keys_in,
                                             const at::Tensor& values_in, const OptT& lengths_in,
                                             std::optional<int64_t> prefix_length, std::optional<double> scale,
                                             const OptT& out, const OptT& out_status) {
  const at::Tensor q = queries(q_in), keys = layer_cache(keys_in), values = layer_cache(values_in);
  check_cache(keys, values, q);
  const at::Tensor pk = prefix_keys_in.dim() == 2 ? prefix_keys_in.unsqueeze(0) : prefix_keys_in;
  const at::Tensor pv = prefix_values_in.dim() == 2 ? prefix_values_in.unsqueeze(0) : prefix_values_in;
  const at::Device dev = q.device();
  on_device(pk, dev, "prefix_keys");
  on_device(pv, dev, "prefix_values");
  TORCH_CHECK_VALUE(pk.dim() == 3 && same_layout(pk, pv) &&
                        pk.scalar_type() == q.scalar_type() && pv.scalar_type() == q.scalar_type() &&
                        pk.size(0) == keys.size(1) && pk.size(2) == q.size(3) && contiguous_along(pk, 2),
                    "prefix_keys and prefix_values must be [kv_heads, prefix, head_dim] of q's dtype with the same "
                    "strides");
  TORCH_CHECK_VALUE(!prefix_length.has_value() || (*prefix_length >= 0 && *prefix_length <= pk.size(1)),
                    "prefix_length must be in [0, the prefix's slots]");
  TORCH_CHECK_VALUE(!scale.has_value() || std::isfinite(*scale), "scale must be finite");
  const c10::cuda::CUDAGuard guard(dev);
  const auto stream = at::cuda::getCurrentCUDAStream(dev.index());
  const int32_t rows = size32(q, 0), n = size32(q, 1), heads = size32(q, 2), dim = size32(q, 3);
  const int32_t kv = size32(keys, 1), capacity = size32(keys, 2), code = logit_code(q);
  const int32_t prefix = prefix_length.has_value() ? (int32_t)std::min<int64_t>(*prefix_length, INT32_MAX) : size32(pk, 1);
  const OptT lengths = row_ints(lengths_in, rows, dev, "lengths");
  at::Tensor o = attention_out(out, q_in);
  if (o.numel() == 0 || capacity == 0) {
    fill_status(out_status, lengths, std::nullopt, rows, capacity, dev);
    if (o.numel() == 0) return {0, o};
    // No own slots: as a cache of one that no row has filled.
    const at::Tensor none = at::zeros({rows, kv, 1, dim}, q.options());
    const at::Tensor zero = at::zeros({rows}, at::TensorOptions().dtype(at::kInt).device(dev));
    const int rc = std::get<0>(
        prefix_attention(q, pk, pv, none, none, zero, prefix, scale, o.view(q.sizes()), std::nullopt));
    return {rc, o};
  }
  const size_t bytes = sv_prefix_attention_workspace_bytes(code, rows, n, heads, kv, dim, prefix, capacity);
  at::Tensor ws = workspace_for(dev, stream, bytes, 4 * ((size_t)rows * kv + 1024));
  const int rc = sv_prefix_attention(
      q.data_ptr(), code, rows, n, heads, kv, dim, stride_of(q, 0), stride_of(q, 1), stride_of(q, 2), pk.data_ptr(),
      pv.data_ptr(), prefix, stride_of(pk, 0), stride_of(pk, 1), keys.data_ptr(), values.data_ptr(), capacity,
      stride_of(keys, 0), stride_of(keys, 1), stride_of(keys, 2),
      optptr<int32_t>(lengths, dev, "lengths", at::kInt, rows),
      scale.has_value() ? *scale : 1.0 / std::sqrt((double)dim), o.data_ptr(),
      ws.defined() ? ws.data_ptr() : nullptr, ws.defined() ? (size_t)ws.numel() : 0,
      status_ptr(out_status, rows, dev), stream.stream());
  return {rc, o};
}

// sv_kv_evict.  keys / values [layers, rows, (heads,) capacity, head_dim], weights /
// positions the same without head_dim.  lengths_in: a tensor, a number or none.
std::tuple<int, at::Tensor, at::Tensor, at::Tensor> kv_evict(
    const at::Tensor& keys, const OptT& values, const at::Tensor& weights, const at::Tensor& positions,
    const OptT& lengths_in, std::optional<int64_t> length, int64_t budget, int64_t sinks, int64_t recent,
    const OptT& weights_out, const OptT& positions_out, const OptT& lengths_out, const OptT& out_status) {
  const at::Device dev = keys.device();
  on_device(keys, dev, "keys");
  TORCH_CHECK_VALUE(keys.dim() == 4 || keys.dim() == 5,
                    "keys must be [layers, rows, capacity, head_dim] or [layers, rows, heads, capacity, head_dim]");
  const int64_t last = keys.dim() - 1;
  const bool heads_dim = keys.dim() == 5;
  TORCH_CHECK_VALUE(contiguous_along(keys, last), "head_dim must be contiguous");
  TORCH_CHECK_VALUE(!values.has_value() || (same_layout(keys, *values) && values->scalar_type() == keys.scalar_type()),
                    "values must have the keys' shape, strides and dtype");
  TORCH_CHECK_VALUE(weights.scalar_type() == at::kFloat && positions.scalar_type() == at::kInt &&
                        weights.sizes() == keys.sizes().slice(0, last) && positions.sizes() == weights.sizes(),
                    "weights (float32) and positions (int32) must have the keys' shape without head_dim");
  const int64_t layers = size32(keys, 0), rows = size32(keys, 1), heads = heads_dim ? size32(keys, 2) : 1;
  const int64_t capacity = size32(keys, last - 1), all = layers * rows * heads * capacity;
  TORCH_CHECK_VALUE(budget >= 1 && budget <= capacity, "budget must be in [1, capacity]");
  TORCH_CHECK_VALUE(sinks >= 0 && recent >= 0 && sinks + recent <= budget,
                    "sinks and recent must not be negative and must fit in the budget");
  TORCH_CHECK_VALUE(!length.has_value() || (*length >= 0 && *length <= capacity), "lengths must be in [0, capacity]");
  const c10::cuda::CUDAGuard guard(dev);
  const auto ints = at::TensorOptions().dtype(at::kInt).device(dev);
  OptT lengths = row_ints(lengths_in, rows, dev, "lengths");
  if (length.has_value()) lengths = at::full({rows}, *length, ints);
  at::Tensor wo = weights_out.has_value() ? *weights_out : at::empty(weights.sizes(), weights.options());
  at::Tensor po = positions_out.has_value() ? *positions_out : at::empty(positions.sizes(), positions.options());
  at::Tensor lo = lengths_out.has_value() ? *lengths_out : at::empty({rows}, ints);
  TORCH_CHECK(weights.is_contiguous() && positions.is_contiguous() && wo.is_contiguous() && po.is_contiguous() &&
                  lo.is_contiguous(),
              "weights and positions must be contiguous");
  const int rc = sv_kv_evict(
      keys.data_ptr(), raw(values, dev, "values"), (int32_t)keys.element_size(), (int32_t)layers, (int32_t)rows,
      (int32_t)heads, (int32_t)capacity, size32(keys, last), stride_of(keys, 0), stride_of(keys, 1),
      heads_dim ? stride_of(keys, 2) : 0, stride_of(keys, last - 1),
      ptr<float>(weights, dev, "weights", at::kFloat, all), ptr<int32_t>(positions, dev, "positions", at::kInt, all),
      optptr<int32_t>(lengths, dev, "lengths", at::kInt, rows), (int32_t)budget, (int32_t)sinks, (int32_t)recent,
      ptr<float>(wo, dev, "weights_out", at::kFloat, all), ptr<int32_t>(po, dev, "positions_out", at::kInt, all),
      ptr<int32_t>(lo, dev, "lengths_out", at::kInt, rows), status_ptr(out_status, rows, dev),
      stream_of(keys));
  return {rc, lo, wo, po};
}

}  // namespace

PYBIND11_MODULE(sv_torch, m) {
  m.doc() = "Thin PyTorch extension over the StarVector B200 sampling C ABI (include/starvector_sampling.h)";
  m.def("abi_version", &sv_abi_version);
  m.def("sample_step", &sample_step);
  m.def("beam_step", &beam_step);
  m.def("beam_advance", &beam_advance);
  m.def("kv_reorder", &kv_reorder);
  m.def("loop_guard", &loop_guard);
  m.def("loop_guard_incremental", &loop_guard_incremental);
  m.def("window_attention", &window_attention);
  m.def("prefix_attention", &prefix_attention);
  m.def("kv_evict", &kv_evict);
  m.def("kv_quantize", &kv_quantize);
  m.def("kv_dequantize", &kv_dequantize);
  m.def("quantized_attention", &quantized_attention);
}
