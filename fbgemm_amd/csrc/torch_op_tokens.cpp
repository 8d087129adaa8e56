// torch operators of a decoding step, continued (torch_op_decode.cpp): rotary positions, cache rows read back,
// sampling. The same manner: namespace fbgemm_amd, all work through the C ABI, results from torch's allocator.
// The rotation has a gradient; where it writes into given tensors it refuses to be recorded.
#include <torch/csrc/autograd/custom_function.h>

#include <tuple>

#include "torch_op_decode.h"

namespace {

std::tuple<Tensor, Tensor> kv_cache_read(
    const Tensor& key_cache, const Tensor& value_cache, const Tensor& block_tables, const Tensor& offsets, int64_t num_tokens, int64_t dim,
    std::optional<at::ScalarType> dtype, const OptTensor& starts, const OptTensor& status, int64_t row_bits) {
  TORCH_CHECK(dim > 0 && dim <= (1 << 16), "fbgemm_amd: dim must be in 1..65536");
  const fbgemm_amd_paged_cache cache = cache_of(key_cache, value_cache, dim, row_bits);
  const int32_t bits = index_bits(offsets, "offsets");
  TORCH_CHECK(offsets.dim() == 1 && offsets.size(0) > 0, "fbgemm_amd: offsets must hold one entry more than there are requests, got ", offsets.sizes());
  const int64_t R = offsets.size(0) - 1;
  list_of(offsets, R + 1, key_cache, offsets.scalar_type(), "offsets");
  if (starts.has_value()) list_of(*starts, R, key_cache, offsets.scalar_type(), "starts");
  on_device(block_tables, key_cache, "block_tables");
  TORCH_CHECK(block_tables.scalar_type() == at::kInt && block_tables.dim() == 2 && block_tables.size(0) == R,
              "fbgemm_amd: block_tables must be int32 [", R, ", blocks], got ", block_tables.scalar_type(), " ", block_tables.sizes());
  rows_dense(block_tables, "block_tables");
  TORCH_CHECK(num_tokens >= 0 && num_tokens <= 0x7fffffff, "fbgemm_amd: num_tokens must be in 0..2^31-1");
  const bool codes = key_cache.scalar_type() == at::kByte;
  const at::ScalarType out = dtype.has_value() ? *dtype : codes ? at::kFloat : key_cache.scalar_type();
  const int32_t ty = float_type(out, "dtype");
  TORCH_CHECK(codes || out == key_cache.scalar_type(), "fbgemm_amd: rows come as they are stored, ", key_cache.scalar_type(), ": got dtype ", out);
  const c10::OptionalDeviceGuard guard(key_cache.device());
  Tensor key = at::empty({num_tokens, cache.heads, dim}, key_cache.options().dtype(out)), value = at::empty_like(key);
  CHECK_CALL(fbgemm_amd_kv_cache_read(&cache, key_cache.data_ptr(), value_cache.data_ptr(), (const int32_t*)block_tables.data_ptr(), stride_of(block_tables, 0),
                                      block_tables.size(1), offsets.data_ptr(), pointer(starts), bits, R, num_tokens, ty, key.data_ptr(), value.data_ptr(),
                                      status_pointer(status, key_cache), current_stream(key_cache)));
  return {key, value};
}

fbgemm_amd_head_rows rows_of(const Tensor& in, const Tensor& out) {
  fbgemm_amd_head_rows r;
  r.in = in.data_ptr();
  r.out = out.data_ptr();
  for (int k = 0; k < 2; ++k) {
    r.in_strides[k] = stride_of(in, k);
    r.out_strides[k] = stride_of(out, k);
  }
  r.heads = (int32_t)in.size(1);
  return r;
}

std::tuple<Tensor, Tensor> rotate(
    const Tensor& query, const Tensor& key, const Tensor& positions, const Tensor& frequencies, bool interleaved, double magnitude, bool inverse,
    Tensor query_out, Tensor key_out) {
  TORCH_CHECK(query.dim() == 3 && key.dim() == 3 && query.size(0) == key.size(0) && query.size(2) == key.size(2) && query.scalar_type() == key.scalar_type(),
              "fbgemm_amd: query and key must be [tokens, heads, dim] of one type, got ", query.sizes(), " and ", key.sizes());
  TORCH_CHECK(query_out.sizes() == query.sizes() && key_out.sizes() == key.sizes() && query_out.scalar_type() == query.scalar_type() &&
                  key_out.scalar_type() == key.scalar_type(),
              "fbgemm_amd: results must have the shapes and type of query and key");
  on_device(key, query, "key");
  on_device(query_out, query, "query_out");
  on_device(key_out, query, "key_out");
  const int32_t ty = float_type(query.scalar_type(), "query");
  const int64_t N = query.size(0), dim = query.size(2);
  TORCH_CHECK(dim > 0, "fbgemm_amd: dim must be positive");
  TORCH_CHECK(query.size(1) <= (1 << 16) && key.size(1) <= (1 << 16) && dim <= (1 << 16), "fbgemm_amd: at most 65536 heads, of at most 65536 elements");
  list_of(positions, N, query, positions.scalar_type(), "positions");
  const int32_t bits = index_bits(positions, "positions");
  list_of(frequencies, frequencies.numel(), query, at::kDouble, "frequencies");
  TORCH_CHECK(2 * frequencies.numel() <= dim, "fbgemm_amd: ", frequencies.numel(), " frequencies turn more than the ", dim, " elements of a head");
  for (const Tensor* t : {&query, &key, (const Tensor*)&query_out, (const Tensor*)&key_out}) rows_dense(*t, "query, key and results");
  const fbgemm_amd_head_rows q = rows_of(query, query_out), k = rows_of(key, key_out);
  const c10::OptionalDeviceGuard guard(query.device());
  CHECK_CALL(fbgemm_amd_rotate_positions(&q, &k, ty, N, (int32_t)dim, positions.data_ptr(), bits, (const double*)frequencies.data_ptr(),
                                         (int32_t)frequencies.numel(), interleaved, (float)magnitude, inverse, current_stream(query)));
  return {query_out, key_out};
}
std::tuple<Tensor, Tensor> rotate_new(
    const Tensor& query, const Tensor& key, const Tensor& positions, const Tensor& frequencies, bool interleaved, double magnitude, bool inverse) {
  const c10::OptionalDeviceGuard guard(query.device());
  return rotate(query, key, positions, frequencies, interleaved, magnitude, inverse, at::empty(query.sizes(), query.options()), at::empty(key.sizes(), key.options()));
}

// ---- the rotation's gradient ----

// the operators as the dispatcher has them
const auto& dispatched() {
  static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("fbgemm_amd::rotate_positions", "").typed<decltype(rotate_new)>();
  return op;
}
const auto& dispatched_out() {
  static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("fbgemm_amd::rotate_positions", "out").typed<decltype(rotate)>();
  return op;
}

// Linear in queries and keys: a gradient goes the other way round, with the same magnitude, by the operator itself (so that it has a gradient too)
struct Rotation : torch::autograd::Function<Rotation> {
  static torch::autograd::variable_list forward(
      torch::autograd::AutogradContext* ctx, const Tensor& query, const Tensor& key, const Tensor& positions, const Tensor& frequencies, bool interleaved,
      double magnitude, bool inverse) {
    const at::AutoDispatchBelowADInplaceOrView below;
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({positions, frequencies});
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["magnitude"] = magnitude;
    ctx->saved_data["inverse"] = inverse;
    const auto turned = dispatched().call(query, key, positions, frequencies, interleaved, magnitude, inverse);
    return {std::get<0>(turned), std::get<1>(turned)};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    torch::autograd::variable_list result(7);
    const bool of[2] = {grads[0].defined() && ctx->needs_input_grad(0), grads[1].defined() && ctx->needs_input_grad(1)};
    if (!of[0] && !of[1]) return result;
    Tensor in[2];
    for (int k = 0; k < 2; ++k) {
      if (of[k]) in[k] = grads[k].size(2) > 1 && grads[k].stride(2) != 1 ? grads[k].contiguous() : grads[k]; // (that of a sum is one number for all)
      else in[k] = grads[1 - k].new_empty({grads[1 - k].size(0), 0, grads[1 - k].size(2)}); // no heads
    }
    const auto saved = ctx->get_saved_variables();
    const auto back = dispatched().call(in[0], in[1], saved[0], saved[1], ctx->saved_data["interleaved"].toBool(), ctx->saved_data["magnitude"].toDouble(),
                                 !ctx->saved_data["inverse"].toBool());
    if (of[0]) result[0] = std::get<0>(back);
    if (of[1]) result[1] = std::get<1>(back);
    return result;
  }
};
// whether what is made of a tensor would be followed
bool followed(const Tensor& t) { return (at::GradMode::is_enabled() && t.requires_grad()) || t._fw_grad(0).defined(); }

std::tuple<Tensor, Tensor> rotate_new_autograd(
    c10::DispatchKeySet keys, const Tensor& query, const Tensor& key, const Tensor& positions, const Tensor& frequencies, bool interleaved, double magnitude, bool inverse) {
  TORCH_CHECK(!followed(frequencies), "fbgemm_amd: rotate_positions has no gradient for its frequencies");
  if (!followed(query) && !followed(key))
    return dispatched().redispatch(keys & c10::after_ADInplaceOrView_keyset, query, key, positions, frequencies, interleaved, magnitude, inverse);
  const auto turned = Rotation::apply(query, key, positions, frequencies, interleaved, magnitude, inverse);
  return {turned[0], turned[1]};
}
std::tuple<Tensor, Tensor> rotate_autograd(
    c10::DispatchKeySet keys, const Tensor& query, const Tensor& key, const Tensor& positions, const Tensor& frequencies, bool interleaved, double magnitude, bool inverse,
    Tensor query_out, Tensor key_out) {
  for (const Tensor* t : {&query, &key, &frequencies, (const Tensor*)&query_out, (const Tensor*)&key_out})
    TORCH_CHECK(!followed(*t), "fbgemm_amd: rotate_positions into given tensors has no gradient, and one of its tensors requires it: "
                               "take new results, or call it under torch.no_grad()");
  return dispatched_out().redispatch(keys & c10::after_autograd_keyset, query, key, positions, frequencies, interleaved, magnitude, inverse, query_out, key_out);
}
// given tensors have other contents now: a graph that holds the former ones has to know
std::tuple<Tensor, Tensor> rotate_written(
    c10::DispatchKeySet keys, const Tensor& query, const Tensor& key, const Tensor& positions, const Tensor& frequencies, bool interleaved, double magnitude, bool inverse,
    Tensor query_out, Tensor key_out) {
  dispatched_out().redispatch(keys & c10::after_ADInplaceOrView_keyset, query, key, positions, frequencies, interleaved, magnitude, inverse, query_out, key_out);
  for (const Tensor* t : {(const Tensor*)&query_out, (const Tensor*)&key_out})
    if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
  return {query_out, key_out};
}

std::tuple<Tensor, Tensor> sample_tokens(
    const Tensor& logits, const Tensor& uniform, const OptTensor& temperature, const OptTensor& top_k, const OptTensor& top_p, const OptTensor& min_p) {
  TORCH_CHECK(logits.dim() == 2, "fbgemm_amd: logits must be [rows, vocab], got ", logits.sizes());
  rows_dense(logits, "logits");
  const int32_t ty = float_type(logits.scalar_type(), "logits");
  const int64_t rows = logits.size(0), vocab = logits.size(1);
  list_of(uniform, rows, logits, at::kFloat, "uniform");
  if (temperature.has_value()) list_of(*temperature, rows, logits, at::kFloat, "temperature");
  if (top_k.has_value()) list_of(*top_k, rows, logits, at::kInt, "top_k");
  if (top_p.has_value()) list_of(*top_p, rows, logits, at::kFloat, "top_p");
  if (min_p.has_value()) list_of(*min_p, rows, logits, at::kFloat, "min_p");
  const c10::OptionalDeviceGuard guard(logits.device());
  Tensor tokens = at::empty({rows}, logits.options().dtype(at::kLong)), log_probability = at::empty({rows}, logits.options().dtype(at::kFloat));
  CHECK_CALL(fbgemm_amd_sample_tokens(logits.data_ptr(), ty, rows, vocab, stride_of(logits, 0), (const float*)uniform.data_ptr(), (const float*)pointer(temperature),
                                      (const int32_t*)pointer(top_k), (const float*)pointer(top_p), (const float*)pointer(min_p),
                                      (int64_t*)tokens.data_ptr(), (float*)log_probability.data_ptr(), current_stream(logits)));
  return {tokens, log_probability};
}

// Shape functions for tracing
std::tuple<Tensor, Tensor> kv_cache_read_meta(
    const Tensor& key_cache, const Tensor&, const Tensor&, const Tensor&, int64_t num_tokens, int64_t dim, std::optional<at::ScalarType> dtype, const OptTensor&,
    const OptTensor&, int64_t) {
  const at::ScalarType out = dtype.has_value() ? *dtype : key_cache.scalar_type() == at::kByte ? at::kFloat : key_cache.scalar_type();
  const auto like = key_cache.options().dtype(out);
  return {at::empty({num_tokens, key_cache.size(1), dim}, like), at::empty({num_tokens, key_cache.size(1), dim}, like)};
}
std::tuple<Tensor, Tensor> rotate_new_meta(const Tensor& query, const Tensor& key, const Tensor&, const Tensor&, bool, double, bool) {
  return {at::empty(query.sizes(), query.options()), at::empty(key.sizes(), key.options())};
}
std::tuple<Tensor, Tensor> rotate_out_meta(const Tensor& query, const Tensor& key, const Tensor&, const Tensor&, bool, double, bool, Tensor query_out, Tensor key_out) {
  TORCH_CHECK(query_out.sizes() == query.sizes() && key_out.sizes() == key.sizes() && query_out.scalar_type() == query.scalar_type() &&
                  key_out.scalar_type() == key.scalar_type(),
              "fbgemm_amd: results must have the shapes and type of query and key");
  return {query_out, key_out};
}
std::tuple<Tensor, Tensor> sample_tokens_meta(
    const Tensor& logits, const Tensor&, const OptTensor&, const OptTensor&, const OptTensor&, const OptTensor&) {
  return {at::empty({logits.size(0)}, logits.options().dtype(at::kLong)), at::empty({logits.size(0)}, logits.options().dtype(at::kFloat))};
}

} // namespace

TORCH_LIBRARY_FRAGMENT(fbgemm_amd, m) {
  m.def(
      "kv_cache_read(Tensor key_cache, Tensor value_cache, Tensor block_tables, Tensor offsets, int num_tokens, int dim, ScalarType? dtype=None, Tensor? starts=None, Tensor(a!)? status=None, int row_bits=8) -> (Tensor, Tensor)");
  m.def(
      "rotate_positions(Tensor query, Tensor key, Tensor positions, Tensor frequencies, bool interleaved=False, float magnitude=1.0, bool inverse=False) -> (Tensor, Tensor)");
  m.def(
      "rotate_positions.out(Tensor query, Tensor key, Tensor positions, Tensor frequencies, bool interleaved=False, float magnitude=1.0, bool inverse=False, *, Tensor(a!) query_out, Tensor(b!) key_out) -> (Tensor(a!), Tensor(b!))");
  m.def(
      "sample_tokens(Tensor logits, Tensor uniform, Tensor? temperature=None, Tensor? top_k=None, Tensor? top_p=None, Tensor? min_p=None) -> (Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(fbgemm_amd, CUDA, m) {
  m.impl("kv_cache_read", TORCH_FN(kv_cache_read));
  m.impl("rotate_positions", TORCH_FN(rotate_new));
  m.impl("rotate_positions.out", TORCH_FN(rotate));
  m.impl("sample_tokens", TORCH_FN(sample_tokens));
}
TORCH_LIBRARY_IMPL(fbgemm_amd, Meta, m) {
  m.impl("kv_cache_read", TORCH_FN(kv_cache_read_meta));
  m.impl("rotate_positions", TORCH_FN(rotate_new_meta));
  m.impl("rotate_positions.out", TORCH_FN(rotate_out_meta));
  m.impl("sample_tokens", TORCH_FN(sample_tokens_meta));
}
TORCH_LIBRARY_IMPL(fbgemm_amd, Autograd, m) {
  m.impl("rotate_positions", TORCH_FN(rotate_new_autograd));
  m.impl("rotate_positions.out", TORCH_FN(rotate_autograd));
}
TORCH_LIBRARY_IMPL(fbgemm_amd, ADInplaceOrView, m) { m.impl("rotate_positions.out", TORCH_FN(rotate_written)); }
