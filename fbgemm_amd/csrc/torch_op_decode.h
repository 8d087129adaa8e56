// What the torch operators of a decoding step have in common: checks of their tensors, the cache as the C ABI takes it.
#pragma once
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/library.h>

#include <optional>

#include "../../include/fbgemm_amd.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

[[maybe_unused]] void* current_stream(const Tensor& t) { return (void*)c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

#define CHECK_CALL(call)                                              \
  do {                                                                \
    const int rc_ = (int)(call);                                      \
    TORCH_CHECK(rc_ == 0, "fbgemm_amd: ", fbgemm_amd_last_error());   \
  } while (0)

[[maybe_unused]] void on_device(const Tensor& t, const Tensor& like, const char* name) {
  TORCH_CHECK(t.device() == like.device(), "fbgemm_amd: ", name, " must be on ", like.device(), ", got ", t.device());
}
[[maybe_unused]] int32_t index_bits(const Tensor& t, const char* name) {
  TORCH_CHECK(t.scalar_type() == at::kInt || t.scalar_type() == at::kLong, "fbgemm_amd: ", name, " must be int32 or int64");
  return t.scalar_type() == at::kLong ? 64 : 32;
}
[[maybe_unused]] void list_of(const Tensor& t, int64_t numel, const Tensor& like, at::ScalarType type, const char* name) {
  on_device(t, like, name);
  TORCH_CHECK(t.scalar_type() == type, "fbgemm_amd: ", name, " must be ", type, ", got ", t.scalar_type());
  TORCH_CHECK(t.dim() == 1 && t.size(0) == numel, "fbgemm_amd: ", name, " must hold ", numel, " entries, got ", t.sizes());
  TORCH_CHECK(t.is_contiguous(), "fbgemm_amd: ", name, " must be contiguous");
}
[[maybe_unused]] int32_t float_type(at::ScalarType t, const char* name) {
  TORCH_CHECK(t == at::kFloat || t == at::kHalf || t == at::kBFloat16, "fbgemm_amd: ", name, " must be float32, float16 or bfloat16, got ", t);
  return t == at::kFloat ? FBGEMM_AMD_FP32 : t == at::kHalf ? FBGEMM_AMD_FP16 : FBGEMM_AMD_BF16;
}
// a dimension of one entry (or none) has no stride worth looking at
[[maybe_unused]] int64_t stride_of(const Tensor& t, int64_t d) { return t.size(d) > 1 ? t.stride(d) : 0; }
[[maybe_unused]] void rows_dense(const Tensor& t, const char* name) {
  TORCH_CHECK(t.numel() == 0 || t.size(-1) <= 1 || t.stride(-1) == 1, "fbgemm_amd: the elements of a row of ", name, " must be next to each other");
}
[[maybe_unused]] void* status_pointer(const OptTensor& status, const Tensor& like) {
  if (!status.has_value()) return nullptr;
  on_device(*status, like, "status");
  TORCH_CHECK(status->is_contiguous() && status->nbytes() >= FBGEMM_AMD_STATUS_BYTES, "fbgemm_amd: status must be a block of ", FBGEMM_AMD_STATUS_BYTES, " bytes");
  return status->data_ptr();
}
[[maybe_unused]] void* pointer(const OptTensor& t) { return t.has_value() ? t->data_ptr() : nullptr; }

[[maybe_unused]] fbgemm_amd_paged_cache cache_of(const Tensor& key_cache, const Tensor& value_cache, int64_t dim, int64_t row_bits) {
  TORCH_CHECK(key_cache.dim() == 4 && value_cache.dim() == 4, "fbgemm_amd: a cache is [blocks, heads, block_size, row], got ", key_cache.sizes(),
              " and ", value_cache.sizes());
  TORCH_CHECK(key_cache.sizes() == value_cache.sizes() && key_cache.scalar_type() == value_cache.scalar_type(),
              "fbgemm_amd: keys and values must have caches of the same shape and type");
  on_device(value_cache, key_cache, "value_cache");
  rows_dense(key_cache, "key_cache");
  rows_dense(value_cache, "value_cache");
  const bool codes = key_cache.scalar_type() == at::kByte;
  TORCH_CHECK(row_bits == 8 || row_bits == 4, "fbgemm_amd: row_bits must be 8 or 4, got ", row_bits);
  TORCH_CHECK(codes || row_bits == 8, "fbgemm_amd: 4-bit rows are in a uint8 cache, got ", key_cache.scalar_type());
  TORCH_CHECK(row_bits == 8 || dim % 2 == 0, "fbgemm_amd: 4-bit rows hold an even number of elements, got ", dim);
  const int64_t held = row_bits == 8 ? dim + 4 : dim / 2 + 4;
  TORCH_CHECK(codes ? key_cache.size(3) >= held : key_cache.size(3) == dim, "fbgemm_amd: rows of ", key_cache.size(3),
              " do not hold ", dim, " elements", codes ? " and a scale and bias" : "");
  TORCH_CHECK(key_cache.size(1) <= 0x7fffffff && key_cache.size(2) <= 0x7fffffff && dim <= 0x7fffffff, "fbgemm_amd: cache too large");
  fbgemm_amd_paged_cache c;
  c.row_ty = codes ? (row_bits == 8 ? FBGEMM_AMD_INT8 : FBGEMM_AMD_CACHE_INT4) : float_type(key_cache.scalar_type(), "a cache that is not uint8");
  c.blocks = key_cache.size(0);
  c.heads = (int32_t)key_cache.size(1);
  c.block_size = (int32_t)key_cache.size(2);
  c.dim = (int32_t)dim;
  for (int k = 0; k < 3; ++k) {
    c.key_strides[k] = stride_of(key_cache, k);
    c.value_strides[k] = stride_of(value_cache, k);
  }
  return c;
}

} // namespace
