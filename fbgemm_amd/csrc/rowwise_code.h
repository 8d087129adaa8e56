// The arithmetic of the row-wise quantized formats that their producers share: the
// quantizers (quantize_kernels.hip) and the cache rows of a decoding step (kv_append.hip).
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

namespace fbgemm_amd {

__device__ __forceinline__ float q_bits_to_float(uint32_t u) { return __builtin_bit_cast(float, u); }
__device__ __forceinline__ uint32_t q_float_to_bits(float f) { return __builtin_bit_cast(uint32_t, f); }
__device__ __forceinline__ float half_bits_to_float(uint16_t h) { return (float)__builtin_bit_cast(_Float16, h); }
__device__ __forceinline__ uint16_t float_to_half_bits(float f) { return __builtin_bit_cast(uint16_t, (_Float16)f); } // RNE
__device__ __forceinline__ uint16_t float_to_bf16_bits(float f) { return (uint16_t)((q_float_to_bits(f) + 0x8000u) >> 16); }

// What a row's extremes become: the stored scale and bias (bit patterns), what elements are
// subtracted and multiplied by, and the bytes of the stored pair.
struct RowCode {
  uint32_t sb0, sb1;
  float minimum, inverse_scale;
  int sb_bytes;
};
template <int BITS>
__device__ __forceinline__ RowCode row_code(float minimum, float maximum, int sb_float, int layout) {
  constexpr int maxq = (1 << BITS) - 1;
  RowCode c;
  if (sb_float) {
    // QuantUtils.cc:704-715
    const float range = maximum - minimum;
    c.sb0 = q_float_to_bits(range / 255.0f);
    c.sb1 = q_float_to_bits(minimum);
    c.inverse_scale = 255.0f / (range + 1e-8f);
  } else {
    // QuantUtils.cc:573-596
    const uint16_t min16 = float_to_half_bits(minimum);
    minimum = half_bits_to_float(min16);
    const float range = maximum - minimum;
    float scale = range == 0.0f ? 1.0f : range / (float)maxq;
    scale = half_bits_to_float(float_to_half_bits(scale));
    if (scale == 0.0f) scale = 1.0f;
    c.inverse_scale = 1.0f / scale;
    if (__builtin_isinf(c.inverse_scale)) {
      scale = 1.0f;
      c.inverse_scale = 1.0f;
    }
    c.sb0 = float_to_half_bits(scale);
    c.sb1 = min16;
  }
  c.minimum = minimum;
  c.sb_bytes = sb_float ? 8 : 4;
  // TBE rows carry an fp16 pair in front whatever the source format stored
  // (fbgemm_gpu/fbgemm_gpu/tbe/utils/quantize.py:47-70)
  if (layout == 1 && sb_float) {
    c.sb0 = float_to_half_bits(q_bits_to_float(c.sb0));
    c.sb1 = float_to_half_bits(q_bits_to_float(c.sb1));
    c.sb_bytes = 4;
  }
  return c;
}

} // namespace fbgemm_amd
