// Logits in pieces of 16 bytes, for the kernels that read rows of them (penalize_logits.hip, sample_tokens.hip).
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

#include "lookup_common.h"

namespace fbgemm_amd {

// N logits of 16 bytes, wherever a row begins
template <int TY>
struct Piece {
  static constexpr int N = TY == ST_FP32 ? 4 : 8;
  static constexpr int BYTES = TY == ST_FP32 ? 4 : 2;
  typedef __attribute__((ext_vector_type(4))) uint32_t raw_t;
  typedef raw_t __attribute__((aligned(4))) on4_t;
  typedef raw_t __attribute__((aligned(2))) on2_t;
  raw_t raw;
  __device__ __forceinline__ void load(const char* p) {
    if constexpr (BYTES == 4) raw = *reinterpret_cast<const on4_t*>(p);
    else raw = *reinterpret_cast<const on2_t*>(p);
  }
  __device__ __forceinline__ void store(char* p) const {
    if constexpr (BYTES == 4) *reinterpret_cast<on4_t*>(p) = raw;
    else *reinterpret_cast<on2_t*>(p) = raw;
  }
  // the first n
  __device__ __forceinline__ void load_some(const char* p, int n) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (TY == ST_FP32) {
        raw[i] = i < n ? reinterpret_cast<const uint32_t*>(p)[i] : 0;
      } else {
        const uint32_t lo = 2 * i < n ? reinterpret_cast<const uint16_t*>(p)[2 * i] : 0, hi = 2 * i + 1 < n ? reinterpret_cast<const uint16_t*>(p)[2 * i + 1] : 0;
        raw[i] = lo | (hi << 16);
      }
    }
  }
  __device__ __forceinline__ void store_some(char* p, int n) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (TY == ST_FP32) {
        if (i < n) reinterpret_cast<uint32_t*>(p)[i] = raw[i];
      } else {
        if (2 * i < n) reinterpret_cast<uint16_t*>(p)[2 * i] = (uint16_t)raw[i];
        if (2 * i + 1 < n) reinterpret_cast<uint16_t*>(p)[2 * i + 1] = (uint16_t)(raw[i] >> 16);
      }
    }
  }
  __device__ __forceinline__ float get(int i) const {
    if constexpr (TY == ST_FP32) return __builtin_bit_cast(float, (uint32_t)raw[i]);
    const uint16_t h = (uint16_t)(raw[i / 2] >> (i % 2 * 16));
    if constexpr (TY == ST_FP16) return (float)__builtin_bit_cast(_Float16, h);
    else return __builtin_bit_cast(float, (uint32_t)h << 16);
  }
  __device__ __forceinline__ void set(int i, float x) {
    if constexpr (TY == ST_FP32) {
      raw[i] = __builtin_bit_cast(uint32_t, x);
    } else {
      uint32_t h;
      if constexpr (TY == ST_FP16) h = __builtin_bit_cast(uint16_t, (_Float16)x);
      else h = __builtin_bit_cast(uint16_t, (__bf16)x);
      raw[i / 2] = (raw[i / 2] & (i % 2 ? 0xffffu : 0xffff0000u)) | (h << (i % 2 * 16));
    }
  }
};

} // namespace fbgemm_amd
