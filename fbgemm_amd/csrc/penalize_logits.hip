// A step's logits, made ready to sample from: penalties for the tokens that a row has seen, biases
// and a grammar's mask.
//
//   x = seen ? (x > 0 ? x / repetition : x * repetition) : x     seen: among the row's tokens
//   x = x - frequency * count;  x = x - presence * (count > 0)   count: times among those behind its prompt
//   x = x + bias                                                 of several for one token the last one
//   x = -inf                                                     where the mask's bit is 0
//
// in fp32, in this order, rounded once to the logits' type. Bound by memory: logits are read once
// and written once. A workgroup takes a chunk of a row's vocabulary and keeps the chunk's counts in
// LDS (a row's list of tokens is read by each of its workgroups, out of L2), so that nothing of
// the vocabulary's size is ever kept in memory and one launch does it all. Counts are integers and
// a bias is chosen by its place in the list: the order in which LDS is updated changes nothing.
#include "decode.h"

namespace fbgemm_amd {

namespace {

constexpr int THREADS = 256;
constexpr int CHUNK = 8192;
constexpr uint32_t SEEN = 0x80000000u;

template <int TY>
__device__ __forceinline__ float to_float(const void* p, int64_t i) {
  if constexpr (TY == ST_FP32) return reinterpret_cast<const float*>(p)[i];
  else if constexpr (TY == ST_FP16) return (float)reinterpret_cast<const _Float16*>(p)[i];
  else return __builtin_bit_cast(float, (uint32_t)reinterpret_cast<const uint16_t*>(p)[i] << 16);
}
template <int TY>
__device__ __forceinline__ void from_float(void* p, int64_t i, float x) {
  if constexpr (TY == ST_FP32) reinterpret_cast<float*>(p)[i] = x;
  else if constexpr (TY == ST_FP16) reinterpret_cast<_Float16*>(p)[i] = (_Float16)x;
  else reinterpret_cast<__bf16*>(p)[i] = (__bf16)x;
}

// a list's range in [0, numel]
template <typename index_t>
__device__ __forceinline__ void range_of(const void* offsets, int64_t row, int64_t numel, int64_t& begin, int64_t& end) {
  const index_t* o = reinterpret_cast<const index_t*>(offsets);
  begin = (int64_t)o[row];
  end = (int64_t)o[row + 1];
  begin = begin < 0 ? 0 : begin;
  end = end > numel ? numel : end;
}

template <int TY, typename index_t>
__global__ __launch_bounds__(THREADS) void penalize_logits_kernel(const LogitsArgs a) {
  __shared__ uint32_t s_count[CHUNK];
  __shared__ uint32_t s_bias[CHUNK];
  const uint32_t chunks = (uint32_t)((a.vocab + CHUNK - 1) / CHUNK);
  const int64_t row = blockIdx.x / chunks, v0 = (int64_t)(blockIdx.x % chunks) * CHUNK;
  const int width = (int)(a.vocab - v0 < CHUNK ? a.vocab - v0 : CHUNK);
  for (int i = threadIdx.x; i < CHUNK; i += THREADS) {
    s_count[i] = 0;
    s_bias[i] = 0;
  }
  __syncthreads();
  if (a.tokens) {
    int64_t begin, end;
    range_of<index_t>(a.offsets, row, a.tokens_numel, begin, end);
    const int64_t prompt = a.prompt_lengths ? (int64_t)reinterpret_cast<const index_t*>(a.prompt_lengths)[row] : 0;
    for (int64_t i = begin + threadIdx.x; i < end; i += THREADS) {
      const int64_t v = (int64_t)reinterpret_cast<const index_t*>(a.tokens)[i] - v0;
      if (v < 0 || v >= width) continue;
      if (i - begin < prompt) atomicOr(&s_count[v], SEEN);
      else atomicAdd(&s_count[v], 1u);
    }
  }
  int64_t bias0 = 0;
  if (a.bias_ids) {
    int64_t end;
    range_of<index_t>(a.bias_offsets, row, a.bias_numel, bias0, end);
    for (int64_t i = bias0 + threadIdx.x; i < end; i += THREADS) {
      const int64_t v = (int64_t)reinterpret_cast<const index_t*>(a.bias_ids)[i] - v0;
      if (v >= 0 && v < width) atomicMax(&s_bias[v], (uint32_t)(i - bias0) + 1);
    }
  }
  __syncthreads();
  const float repetition = a.repetition ? a.repetition[row] : 1.0f;
  const float frequency = a.frequency ? a.frequency[row] : 0.0f;
  const float presence = a.presence ? a.presence[row] : 0.0f;
  for (int i = threadIdx.x; i < width; i += THREADS) {
    float x = to_float<TY>(a.logits, row * a.logits_stride + v0 + i);
    const uint32_t c = s_count[i];
    if (c) {
      x = x > 0.0f ? x / repetition : x * repetition;
      const uint32_t n = c & ~SEEN;
      if (n) {
        x = x - frequency * (float)n;
        x = x - presence;
      }
    }
    const uint32_t b = s_bias[i];
    if (b) x = x + a.bias_values[bias0 + b - 1];
    if (a.mask && !((a.mask[row * a.mask_stride + ((v0 + i) >> 5)] >> ((v0 + i) & 31)) & 1)) x = -__builtin_inff();
    from_float<TY>(a.out, row * a.out_stride + v0 + i, x);
  }
}

template <int TY>
hipError_t launch(const LogitsArgs& a, bool idx64, hipStream_t stream) {
  const int64_t grid64 = (a.vocab + CHUNK - 1) / CHUNK * a.rows;
  if (grid64 > 0x7fffffff) return hipErrorInvalidValue;
  const unsigned grid = (unsigned)grid64;
  if (idx64) penalize_logits_kernel<TY, int64_t><<<grid, THREADS, 0, stream>>>(a);
  else penalize_logits_kernel<TY, int32_t><<<grid, THREADS, 0, stream>>>(a);
  return hipGetLastError();
}

} // namespace

hipError_t launch_penalize_logits(const LogitsArgs& a, int32_t ty, bool idx64, hipStream_t stream) {
  if (ty == ST_FP32) return launch<ST_FP32>(a, idx64, stream);
  if (ty == ST_FP16) return launch<ST_FP16>(a, idx64, stream);
  return launch<ST_BF16>(a, idx64, stream);
}

} // namespace fbgemm_amd
