// torch operators of a decoding step over a paged key-value cache. They have no counterpart among
// the reference's operators of the quantized-embedding path: namespace fbgemm_amd. torch owns
// tensors and streams; all work goes through the C ABI of include/fbgemm_amd.h. What a call
// returns and its scratch come from torch's allocator, for the current stream.
#include <algorithm>
#include <cmath>
#include <limits>
#include <tuple>

#include "torch_op_decode.h"

namespace {

std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> kv_block_tables(
    const Tensor& lengths, const Tensor& new_tokens, Tensor block_tables, const Tensor& free_blocks, const Tensor& free_start,
    int64_t block_size, int64_t num_tokens, const OptTensor& status) {
  const int32_t bits = index_bits(lengths, "lengths");
  TORCH_CHECK(lengths.dim() == 1, "fbgemm_amd: lengths must have 1 dimension, got ", lengths.sizes());
  const int64_t R = lengths.size(0);
  list_of(lengths, R, lengths, lengths.scalar_type(), "lengths");
  list_of(new_tokens, R, lengths, lengths.scalar_type(), "new_tokens");
  on_device(block_tables, lengths, "block_tables");
  TORCH_CHECK(block_tables.scalar_type() == at::kInt && block_tables.dim() == 2 && block_tables.size(0) == R,
              "fbgemm_amd: block_tables must be int32 [", R, ", blocks], got ", block_tables.scalar_type(), " ", block_tables.sizes());
  rows_dense(block_tables, "block_tables");
  list_of(free_blocks, free_blocks.numel(), lengths, at::kInt, "free_blocks");
  list_of(free_start, 1, lengths, at::kInt, "free_start");
  TORCH_CHECK(block_size > 0 && block_size <= (1 << 20), "fbgemm_amd: block_size must be in 1..1048576");
  TORCH_CHECK(num_tokens >= 0 && num_tokens <= 0x7fffffff, "fbgemm_amd: num_tokens must be in 0..2^31-1");
  const c10::OptionalDeviceGuard guard(lengths.device());
  const auto wide = lengths.options().dtype(at::kLong), narrow = lengths.options().dtype(at::kInt);
  Tensor slots = at::empty({num_tokens}, wide), positions = at::empty({num_tokens}, wide);
  Tensor offsets = at::empty({R + 1}, narrow), total = at::empty({R}, lengths.options()), next = at::empty({1}, narrow);
  CHECK_CALL(fbgemm_amd_kv_block_tables(
      lengths.data_ptr(), new_tokens.data_ptr(), bits, R, (int32_t*)block_tables.data_ptr(), R > 1 ? block_tables.stride(0) : block_tables.size(1),
      block_tables.size(1), (const int32_t*)free_blocks.data_ptr(), free_blocks.numel(), (const int32_t*)free_start.data_ptr(), (int32_t)block_size,
      num_tokens, (int64_t*)slots.data_ptr(), (int64_t*)positions.data_ptr(), (int32_t*)offsets.data_ptr(), total.data_ptr(),
      (int32_t*)next.data_ptr(), status_pointer(status, lengths), current_stream(lengths)));
  return {slots, positions, offsets, total, next};
}

void kv_cache_append(const Tensor& key, const Tensor& value, Tensor key_cache, Tensor value_cache, const Tensor& slots, const OptTensor& status,
                     int64_t row_bits) {
  TORCH_CHECK(key.dim() == 3 && key.sizes() == value.sizes() && key.scalar_type() == value.scalar_type(),
              "fbgemm_amd: key and value must be [tokens, heads, dim] of one type, got ", key.sizes(), " and ", value.sizes());
  on_device(value, key, "value");
  on_device(key_cache, key, "key_cache");
  rows_dense(key, "key");
  rows_dense(value, "value");
  list_of(slots, key.size(0), key, at::kLong, "slots");
  const fbgemm_amd_paged_cache cache = cache_of(key_cache, value_cache, key.size(2), row_bits);
  TORCH_CHECK(key.size(1) == cache.heads, "fbgemm_amd: key has ", key.size(1), " heads, its cache ", cache.heads);
  const int64_t ks[2] = {stride_of(key, 0), stride_of(key, 1)}, vs[2] = {stride_of(value, 0), stride_of(value, 1)};
  const c10::OptionalDeviceGuard guard(key.device());
  CHECK_CALL(fbgemm_amd_kv_cache_append(&cache, key.data_ptr(), value.data_ptr(), float_type(key.scalar_type(), "key"), key.size(0), ks, vs,
                                        (const int64_t*)slots.data_ptr(), key_cache.data_ptr(), value_cache.data_ptr(),
                                        status_pointer(status, key), current_stream(key)));
}

std::tuple<Tensor, Tensor> paged_attention(
    const Tensor& query, const Tensor& key_cache, const Tensor& value_cache, const Tensor& block_tables, const Tensor& lengths,
    std::optional<double> scale, int64_t window, double softcap, int64_t row_bits) {
  TORCH_CHECK(query.dim() == 3, "fbgemm_amd: query must be [requests, heads, dim], got ", query.sizes());
  rows_dense(query, "query");
  const int64_t B = query.size(0), heads = query.size(1), dim = query.size(2);
  TORCH_CHECK(dim > 0, "fbgemm_amd: dim must be positive");
  on_device(key_cache, query, "key_cache");
  const fbgemm_amd_paged_cache cache = cache_of(key_cache, value_cache, dim, row_bits);
  list_of(lengths, B, query, lengths.scalar_type(), "lengths");
  on_device(block_tables, query, "block_tables");
  TORCH_CHECK(block_tables.scalar_type() == at::kInt && block_tables.dim() == 2 && block_tables.size(0) == B,
              "fbgemm_amd: block_tables must be int32 [", B, ", blocks], got ", block_tables.scalar_type(), " ", block_tables.sizes());
  rows_dense(block_tables, "block_tables");
  TORCH_CHECK(heads <= 0x7fffffff, "fbgemm_amd: too many heads");
  const c10::OptionalDeviceGuard guard(query.device()); // sizes go by the current device's compute units
  const int64_t bytes = fbgemm_amd_paged_attention_workspace(&cache, B, (int32_t)heads, block_tables.size(1));
  TORCH_CHECK(bytes >= 0, "fbgemm_amd: ", fbgemm_amd_last_error());
  // a cap below every fp32 number is one all the same: 0 would be none
  const float cap = softcap == 0.0 ? 0.0f : (float)std::copysign(std::max(std::fabs(softcap), (double)std::numeric_limits<float>::min()), softcap);
  Tensor out = at::empty({B, heads, dim}, query.options());
  Tensor lse = at::empty({B, heads}, query.options().dtype(at::kFloat));
  Tensor space = at::empty({bytes}, query.options().dtype(at::kByte));
  CHECK_CALL(fbgemm_amd_paged_attention(
      &cache, query.data_ptr(), float_type(query.scalar_type(), "query"), B, (int32_t)heads, stride_of(query, 0), stride_of(query, 1),
      key_cache.data_ptr(), value_cache.data_ptr(), (const int32_t*)block_tables.data_ptr(), stride_of(block_tables, 0), block_tables.size(1),
      lengths.data_ptr(), index_bits(lengths, "lengths"), (float)(scale.has_value() ? *scale : 1.0 / std::sqrt((double)dim)), window, cap,
      out.data_ptr(), (float*)lse.data_ptr(), space.data_ptr(), bytes, current_stream(query)));
  return {out, lse};
}

Tensor penalize_logits(
    const Tensor& logits, const OptTensor& tokens, const OptTensor& offsets, const OptTensor& prompt_lengths, const OptTensor& repetition,
    const OptTensor& frequency, const OptTensor& presence, const OptTensor& bias_ids, const OptTensor& bias_values,
    const OptTensor& bias_offsets, const OptTensor& mask, const OptTensor& out_) {
  TORCH_CHECK(logits.dim() == 2, "fbgemm_amd: logits must be [rows, vocab], got ", logits.sizes());
  rows_dense(logits, "logits");
  const int32_t ty = float_type(logits.scalar_type(), "logits");
  const int64_t rows = logits.size(0), vocab = logits.size(1);
  TORCH_CHECK(tokens.has_value() == offsets.has_value(), "fbgemm_amd: tokens and offsets go together");
  TORCH_CHECK(!prompt_lengths.has_value() || tokens.has_value(), "fbgemm_amd: prompt_lengths go with tokens");
  TORCH_CHECK(bias_ids.has_value() == bias_offsets.has_value() && bias_ids.has_value() == bias_values.has_value(),
              "fbgemm_amd: bias_ids, bias_values and bias_offsets go together");
  const at::ScalarType index = tokens.has_value() ? tokens->scalar_type() : bias_ids.has_value() ? bias_ids->scalar_type() : at::kLong;
  TORCH_CHECK(index == at::kInt || index == at::kLong, "fbgemm_amd: lists must be int32 or int64");
  if (tokens.has_value()) {
    list_of(*tokens, tokens->numel(), logits, index, "tokens");
    list_of(*offsets, rows + 1, logits, index, "offsets");
  }
  if (prompt_lengths.has_value()) list_of(*prompt_lengths, rows, logits, index, "prompt_lengths");
  if (bias_ids.has_value()) {
    list_of(*bias_ids, bias_ids->numel(), logits, index, "bias_ids");
    list_of(*bias_values, bias_ids->numel(), logits, at::kFloat, "bias_values");
    list_of(*bias_offsets, rows + 1, logits, index, "bias_offsets");
  }
  if (repetition.has_value()) list_of(*repetition, rows, logits, at::kFloat, "repetition");
  if (frequency.has_value()) list_of(*frequency, rows, logits, at::kFloat, "frequency");
  if (presence.has_value()) list_of(*presence, rows, logits, at::kFloat, "presence");
  if (mask.has_value()) {
    on_device(*mask, logits, "mask");
    TORCH_CHECK(mask->scalar_type() == at::kInt && mask->dim() == 2 && mask->size(0) == rows && mask->size(1) >= (vocab + 31) / 32,
                "fbgemm_amd: mask must be int32 [", rows, ", ", (vocab + 31) / 32, "], got ", mask->scalar_type(), " ", mask->sizes());
    rows_dense(*mask, "mask");
  }
  const c10::OptionalDeviceGuard guard(logits.device());
  Tensor out = out_.has_value() ? *out_ : at::empty({rows, vocab}, logits.options());
  on_device(out, logits, "out");
  TORCH_CHECK(out.sizes() == logits.sizes() && out.scalar_type() == logits.scalar_type(), "fbgemm_amd: out must have the logits' shape and type");
  rows_dense(out, "out");
  CHECK_CALL(fbgemm_amd_penalize_logits(
      logits.data_ptr(), ty, rows, vocab, rows > 1 ? logits.stride(0) : vocab, pointer(tokens), tokens.has_value() ? tokens->numel() : 0,
      pointer(offsets), pointer(prompt_lengths), index == at::kLong ? 64 : 32, (const float*)pointer(repetition), (const float*)pointer(frequency),
      (const float*)pointer(presence), pointer(bias_ids), (const float*)pointer(bias_values), bias_ids.has_value() ? bias_ids->numel() : 0,
      pointer(bias_offsets), (const int32_t*)pointer(mask), mask.has_value() && rows > 1 ? mask->stride(0) : (vocab + 31) / 32, out.data_ptr(),
      rows > 1 ? out.stride(0) : vocab, current_stream(logits)));
  return out;
}

// Shape functions for tracing
std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> kv_block_tables_meta(
    const Tensor& lengths, const Tensor&, Tensor, const Tensor&, const Tensor&, int64_t, int64_t num_tokens, const OptTensor&) {
  const auto wide = lengths.options().dtype(at::kLong), narrow = lengths.options().dtype(at::kInt);
  return {at::empty({num_tokens}, wide), at::empty({num_tokens}, wide), at::empty({lengths.size(0) + 1}, narrow), at::empty_like(lengths),
          at::empty({1}, narrow)};
}
void kv_cache_append_meta(const Tensor&, const Tensor&, Tensor, Tensor, const Tensor&, const OptTensor&, int64_t) {}
std::tuple<Tensor, Tensor> paged_attention_meta(
    const Tensor& query, const Tensor&, const Tensor&, const Tensor&, const Tensor&, std::optional<double>, int64_t, double, int64_t) {
  return {at::empty(query.sizes(), query.options()), at::empty({query.size(0), query.size(1)}, query.options().dtype(at::kFloat))};
}
Tensor penalize_logits_new(
    const Tensor& logits, const OptTensor& tokens, const OptTensor& offsets, const OptTensor& prompt_lengths, const OptTensor& repetition,
    const OptTensor& frequency, const OptTensor& presence, const OptTensor& bias_ids, const OptTensor& bias_values,
    const OptTensor& bias_offsets, const OptTensor& mask) {
  return penalize_logits(logits, tokens, offsets, prompt_lengths, repetition, frequency, presence, bias_ids, bias_values, bias_offsets, mask, std::nullopt);
}
Tensor penalize_logits_out(
    const Tensor& logits, const OptTensor& tokens, const OptTensor& offsets, const OptTensor& prompt_lengths, const OptTensor& repetition,
    const OptTensor& frequency, const OptTensor& presence, const OptTensor& bias_ids, const OptTensor& bias_values,
    const OptTensor& bias_offsets, const OptTensor& mask, Tensor out) {
  return penalize_logits(logits, tokens, offsets, prompt_lengths, repetition, frequency, presence, bias_ids, bias_values, bias_offsets, mask, out);
}
Tensor penalize_logits_new_meta(
    const Tensor& logits, const OptTensor&, const OptTensor&, const OptTensor&, const OptTensor&, const OptTensor&, const OptTensor&,
    const OptTensor&, const OptTensor&, const OptTensor&, const OptTensor&) {
  return at::empty(logits.sizes(), logits.options());
}
Tensor penalize_logits_out_meta(
    const Tensor& logits, const OptTensor&, const OptTensor&, const OptTensor&, const OptTensor&, const OptTensor&, const OptTensor&,
    const OptTensor&, const OptTensor&, const OptTensor&, const OptTensor&, Tensor out) {
  TORCH_CHECK(out.sizes() == logits.sizes() && out.scalar_type() == logits.scalar_type(), "fbgemm_amd: out must have the logits' shape and type");
  return out;
}

} // namespace

TORCH_LIBRARY_FRAGMENT(fbgemm_amd, m) {
  m.def(
      "kv_block_tables(Tensor lengths, Tensor new_tokens, Tensor(a!) block_tables, Tensor free_blocks, Tensor free_start, int block_size, int num_tokens, Tensor(b!)? status=None) -> (Tensor, Tensor, Tensor, Tensor, Tensor)");
  m.def(
      "kv_cache_append(Tensor key, Tensor value, Tensor(a!) key_cache, Tensor(b!) value_cache, Tensor slots, Tensor(c!)? status=None, int row_bits=8) -> ()");
  m.def(
      "paged_attention(Tensor query, Tensor key_cache, Tensor value_cache, Tensor block_tables, Tensor lengths, float? scale=None, int window=0, float softcap=0.0, int row_bits=8) -> (Tensor, Tensor)");
  m.def(
      "penalize_logits(Tensor logits, Tensor? tokens=None, Tensor? offsets=None, Tensor? prompt_lengths=None, Tensor? repetition=None, Tensor? frequency=None, Tensor? presence=None, Tensor? bias_ids=None, Tensor? bias_values=None, Tensor? bias_offsets=None, Tensor? mask=None) -> Tensor");
  m.def(
      "penalize_logits.out(Tensor logits, Tensor? tokens=None, Tensor? offsets=None, Tensor? prompt_lengths=None, Tensor? repetition=None, Tensor? frequency=None, Tensor? presence=None, Tensor? bias_ids=None, Tensor? bias_values=None, Tensor? bias_offsets=None, Tensor? mask=None, *, Tensor(a!) out) -> Tensor(a!)");
}

TORCH_LIBRARY_IMPL(fbgemm_amd, CUDA, m) {
  m.impl("kv_block_tables", TORCH_FN(kv_block_tables));
  m.impl("kv_cache_append", TORCH_FN(kv_cache_append));
  m.impl("paged_attention", TORCH_FN(paged_attention));
  m.impl("penalize_logits", TORCH_FN(penalize_logits_new));
  m.impl("penalize_logits.out", TORCH_FN(penalize_logits_out));
}
TORCH_LIBRARY_IMPL(fbgemm_amd, Meta, m) {
  m.impl("kv_block_tables", TORCH_FN(kv_block_tables_meta));
  m.impl("kv_cache_append", TORCH_FN(kv_cache_append_meta));
  m.impl("paged_attention", TORCH_FN(paged_attention_meta));
  m.impl("penalize_logits", TORCH_FN(penalize_logits_new_meta));
  m.impl("penalize_logits.out", TORCH_FN(penalize_logits_out_meta));
}
