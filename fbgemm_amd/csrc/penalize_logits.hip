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
// LDS, so that nothing of the vocabulary's size is ever kept in memory and one launch does it all.
// A row's list of tokens is read by each of its workgroups, out of L2, a batch of eight a thread at
// a time: what counts is how many loads wait for each other, not the instructions. The logits are on
// their way meanwhile and stay in registers. Counts are integers and a bias is chosen by its place in
// the list: the order in which LDS is updated changes nothing.
//
// 256 rows of 131 071 bf16 logits: 28 us with nothing to do (4.8 TB/s), 35 with lists of 0 .. 4 096
// tokens, 48 with biases and a mask too, by then memory and some 25 us of vector instructions one behind the other. Tried: copying all under
// the mask first and writing the named ones again (99), counts and biases in one word (49), a list of
// the named ones made from what the counts' atomics return (58).
#include <type_traits>

#include "decode.h"

namespace fbgemm_amd {

namespace {

constexpr uint32_t SEEN = 0x80000000u;

// PIECE logits of 16 bytes, wherever a row begins
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

// a list's range in [0, numel]
template <typename index_t>
__device__ __forceinline__ void range_of(const void* offsets, int64_t row, int64_t numel, int64_t& begin, int64_t& end) {
  const index_t* o = reinterpret_cast<const index_t*>(offsets);
  begin = (int64_t)o[row];
  end = (int64_t)o[row + 1];
  begin = begin < 0 ? 0 : begin;
  end = end > numel ? numel : end;
}

// f(value, place in the list) for the list's entries, eight a thread in flight
template <typename index_t, int THREADS, typename F>
__device__ __forceinline__ void each_entry(const void* list, int64_t begin, int64_t end, F&& f) {
  constexpr int AT_ONCE = 8;
  const index_t* p = reinterpret_cast<const index_t*>(list) + begin;
  const int64_t n = end - begin;
  for (int64_t i0 = threadIdx.x; i0 < n; i0 += AT_ONCE * THREADS) {
    index_t v[AT_ONCE];
#pragma unroll
    for (int k = 0; k < AT_ONCE; ++k) {
      const int64_t i = i0 + k * THREADS;
      v[k] = p[i < n ? i : n - 1];
    }
#pragma unroll
    for (int k = 0; k < AT_ONCE; ++k)
      if (i0 + k * THREADS < n) f((int64_t)v[k], i0 + k * THREADS);
  }
}

// THREADS threads, PIECES pieces each. The entries of a piece's logits in LDS are its thread's alone, but for the lists' updates.
template <int TY, typename index_t, int THREADS, int PIECES>
__global__ __launch_bounds__(THREADS) void penalize_logits_kernel(const LogitsArgs a) {
  using P = Piece<TY>;
  constexpr int N = P::N, CHUNK = THREADS * PIECES * N;
  typedef __attribute__((ext_vector_type(4))) uint32_t four;
  __shared__ __attribute__((aligned(16))) uint32_t s_count[CHUNK];
  const uint32_t chunks = (uint32_t)((a.vocab + CHUNK - 1) / CHUNK);
  const int64_t row = blockIdx.x / chunks, v0 = (int64_t)(blockIdx.x % chunks) * CHUNK;
  const int width = (int)(a.vocab - v0 < CHUNK ? a.vocab - v0 : CHUNK);
  const char* in = reinterpret_cast<const char*>(a.logits) + (row * a.logits_stride + v0) * P::BYTES;
  char* out = reinterpret_cast<char*>(a.out) + (row * a.out_stride + v0) * P::BYTES;
  // all that waits for nothing: the lists' ranges, the logits, the mask's words
  int64_t begin = 0, end = 0, prompt = 0, bias0 = 0, bias1 = 0;
  if (a.tokens) range_of<index_t>(a.offsets, row, a.tokens_numel, begin, end);
  if (a.tokens && a.prompt_lengths) prompt = (int64_t)reinterpret_cast<const index_t*>(a.prompt_lengths)[row];
  if (a.bias_ids) range_of<index_t>(a.bias_offsets, row, a.bias_numel, bias0, bias1);
  const float repetition = a.repetition ? a.repetition[row] : 1.0f;
  const float frequency = a.frequency ? a.frequency[row] : 0.0f;
  const float presence = a.presence ? a.presence[row] : 0.0f;
  P x[PIECES];
  uint32_t bits[PIECES];
  const auto at = [&](int k) { return (k * THREADS + (int)threadIdx.x) * N; };
#pragma unroll
  for (int k = 0; k < PIECES; ++k) {
    if (at(k) + N <= width) x[k].load(in + (int64_t)at(k) * P::BYTES);
    else if (at(k) < width) x[k].load_some(in + (int64_t)at(k) * P::BYTES, width - at(k));
    const int64_t v = v0 + at(k); // a multiple of N: its bits are in one word
    bits[k] = a.mask && at(k) < width ? a.mask[row * a.mask_stride + (v >> 5)] >> (v & 31) : 0xffffffffu;
  }
#pragma unroll
  for (int k = 0; k < PIECES; ++k)
#pragma unroll
    for (int i = 0; i < N; i += 4) *reinterpret_cast<four*>(&s_count[at(k) + i]) = four{0, 0, 0, 0};
  __syncthreads();
  if (end > begin) {
    each_entry<index_t, THREADS>(a.tokens, begin, end, [&](int64_t v, int64_t i) {
      v -= v0;
      if (v < 0 || v >= width) return;
      if (i < prompt) atomicOr(&s_count[v], SEEN);
      else atomicAdd(&s_count[v], 1u);
    });
    __syncthreads();
  }
  // what happens to a logit: the rounding to its type waits for the end, so 16-bit rows with biases are kept as fp32
  const auto penalized = [&](float y, uint32_t c) {
    if (c) {
      y = y > 0.0f ? y / repetition : y * repetition;
      const uint32_t n = c & ~SEEN;
      if (n) {
        y = y - frequency * (float)n;
        y = y - presence;
      }
    }
    return y;
  };
  const auto finish = [&](int k, const float (&y)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) x[k].set(i, (bits[k] >> i) & 1 ? y[i] : -__builtin_inff());
    if (at(k) + N <= width) x[k].store(out + (int64_t)at(k) * P::BYTES);
    else if (at(k) < width) x[k].store_some(out + (int64_t)at(k) * P::BYTES, width - at(k));
  };
  const auto counts = [&](int k, uint32_t (&c)[N]) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const four w = *reinterpret_cast<const four*>(&s_count[at(k) + i]);
      c[i] = w[0], c[i + 1] = w[1], c[i + 2] = w[2], c[i + 3] = w[3];
    }
  };
  if (bias1 <= bias0) { // the same for the workgroup
#pragma unroll
    for (int k = 0; k < PIECES; ++k) {
      uint32_t c[N];
      float y[N];
      counts(k, c);
#pragma unroll
      for (int i = 0; i < N; ++i) y[i] = penalized(x[k].get(i), c[i]);
      finish(k, y);
    }
    return;
  }
  // biases: the same array holds the last entry of the list for a token, behind the counts, which its thread has read by then
  float y[PIECES][N];
#pragma unroll
  for (int k = 0; k < PIECES; ++k) {
    uint32_t c[N];
    counts(k, c);
#pragma unroll
    for (int i = 0; i < N; ++i) y[k][i] = penalized(x[k].get(i), c[i]);
#pragma unroll
    for (int i = 0; i < N; i += 4) *reinterpret_cast<four*>(&s_count[at(k) + i]) = four{0, 0, 0, 0};
  }
  __syncthreads();
  each_entry<index_t, THREADS>(a.bias_ids, bias0, bias1, [&](int64_t v, int64_t i) {
    v -= v0;
    if (v >= 0 && v < width) atomicMax(&s_count[v], (uint32_t)i + 1);
  });
  __syncthreads();
#pragma unroll
  for (int k = 0; k < PIECES; ++k) {
    uint32_t c[N];
    counts(k, c);
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (c[i]) y[k][i] = y[k][i] + a.bias_values[bias0 + c[i] - 1];
    finish(k, y[k]);
  }
}

// the same from a later row on
LogitsArgs rows_from(LogitsArgs a, int64_t row, int64_t element_bytes, int64_t index_bytes) {
  const auto later = [&](auto*& p, int64_t bytes) {
    if (p) p = reinterpret_cast<std::remove_reference_t<decltype(p)>>(reinterpret_cast<uintptr_t>(p) + row * bytes);
  };
  later(a.logits, a.logits_stride * element_bytes);
  later(a.out, a.out_stride * element_bytes);
  later(a.offsets, index_bytes);
  later(a.prompt_lengths, index_bytes);
  later(a.bias_offsets, index_bytes);
  later(a.repetition, sizeof(float));
  later(a.frequency, sizeof(float));
  later(a.presence, sizeof(float));
  later(a.mask, a.mask_stride * (int64_t)sizeof(uint32_t));
  a.rows -= row;
  return a;
}

template <int TY, int THREADS, int PIECES>
hipError_t launch_shape(const LogitsArgs& all, bool idx64, hipStream_t stream) {
  constexpr int64_t CHUNK = THREADS * PIECES * Piece<TY>::N;
  const int64_t chunks = (all.vocab + CHUNK - 1) / CHUNK;
  const int64_t most = 0xffffffffll / THREADS / chunks; // rows of a launch: fewer than 2^32 threads
  for (int64_t row = 0; row < all.rows; row += most) {
    const LogitsArgs a = rows_from(all, row, Piece<TY>::BYTES, idx64 ? 8 : 4);
    const unsigned grid = (unsigned)(chunks * (a.rows < most ? a.rows : most));
    if (idx64) penalize_logits_kernel<TY, int64_t, THREADS, PIECES><<<grid, THREADS, 0, stream>>>(a);
    else penalize_logits_kernel<TY, int32_t, THREADS, PIECES><<<grid, THREADS, 0, stream>>>(a);
    if (hipError_t e = hipGetLastError()) return e;
  }
  return hipSuccess;
}
template <int TY>
hipError_t launch(const LogitsArgs& a, bool idx64, hipStream_t stream) {
  // Every chunk's workgroup reads the row's whole list: long lists ask for larger chunks, others for more workgroups side by side.
  // 256 rows of 131 071 bf16 logits: lists of 0 .. 4 096 tokens 48.7 us (512 x 32: 57.3), of 0 .. 60 000 tokens 149 us (107)
  if (a.tokens_numel / a.rows > 8192) return launch_shape<TY, 512, 32 / Piece<TY>::N>(a, idx64, stream);
  return launch_shape<TY, 256, 16 / Piece<TY>::N>(a, idx64, stream);
}

} // namespace

hipError_t launch_penalize_logits(const LogitsArgs& a, int32_t ty, bool idx64, hipStream_t stream) {
  if (ty == ST_FP32) return launch<ST_FP32>(a, idx64, stream);
  if (ty == ST_FP16) return launch<ST_FP16>(a, idx64, stream);
  return launch<ST_BF16>(a, idx64, stream);
}

} // namespace fbgemm_amd
