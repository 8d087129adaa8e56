// Rows of requests' tokens out of their pages into dense arrays: with the last request r whose
// offsets[r] <= i, token i is at position p = starts[r] + i - offsets[r] of r, and
//
//   out[i][head] = cache[table[r][p / S]][head][p % S]
//
// as it is, or as the values that 8-bit and 4-bit rows stand for: scale * code + bias in fp32 (the product of an
// fp16 number and a code is exact), rounded once. A token without a page is zeros.
//
// Bound by memory: every row is read once and written once. A workgroup has a run of tokens, whose
// rows' places it finds first, one a thread, by bisection over the offsets; then a thread takes a piece of a row of both keys
// and values at a time.
#include <type_traits>

#include "decode.h"
#include "rowwise_code.h"

namespace fbgemm_amd {

namespace {

constexpr int THREADS = 256;
typedef __attribute__((ext_vector_type(4))) uint32_t piece16;
typedef __attribute__((ext_vector_type(2))) uint32_t piece8;

// A token's rows, without the head: bytes from the caches' beginnings; block < 0: none
struct Rows {
  int32_t block, in_block;
};
template <typename index_t>
__device__ __forceinline__ Rows rows_of(const ReadArgs& a, int64_t token) {
  const index_t* offsets = reinterpret_cast<const index_t*>(a.offsets);
  Rows r{-1, 0};
  if (a.requests == 0 || token >= (int64_t)offsets[a.requests]) return r; // behind the last one: of no request, and nobody's fault
  int lo = 0, hi = a.requests; // the last request that begins at or before the token is in [lo, hi)
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if ((int64_t)offsets[mid] <= token) lo = mid;
    else hi = mid;
  }
  const int64_t in_request = token - (int64_t)offsets[lo];
  const int64_t start = a.starts ? (int64_t)reinterpret_cast<const index_t*>(a.starts)[lo] : 0;
  const int64_t room = a.table_width * a.block.d; // below 2^31, as the number of tokens
  // (sums of 64-bit numbers far from 32-bit ones are no positions)
  if (in_request >= 0 && start > -(1ll << 32) && start < room && start + in_request >= 0 && start + in_request < room) {
    const uint32_t position = (uint32_t)(start + in_request), column = divide(position, a.block);
    const int32_t block = a.tables[lo * a.table_stride + column];
    if (block >= 0 && block < a.blocks) r = Rows{block, (int32_t)(position - column * a.block.d)};
  }
  if (r.block < 0 && a.status) status_index(a.status, token);
  return r;
}

// f(k, piece of a row, where the row begins in cache k or null, where it goes) for a workgroup's pieces
template <int RUN_TOKENS, typename F>
__device__ __forceinline__ void each_piece(const ReadArgs& a, int64_t out_row_bytes, F&& f) {
  __shared__ Rows s_rows[RUN_TOKENS];
  for (int64_t first = (int64_t)blockIdx.x * RUN_TOKENS; first < a.tokens; first += (int64_t)gridDim.x * RUN_TOKENS) {
    const int tokens = (int)(a.tokens - first < RUN_TOKENS ? a.tokens - first : RUN_TOKENS);
    __syncthreads(); // the last run's places have been read
    if ((int)threadIdx.x < tokens) s_rows[threadIdx.x] = a.idx64 ? rows_of<int64_t>(a, first + threadIdx.x) : rows_of<int32_t>(a, first + threadIdx.x);
    __syncthreads();
    const uint32_t items = (uint32_t)tokens * a.per_token.d;
    for (uint32_t i = threadIdx.x; i < items; i += THREADS) {
      const uint32_t token = divide(i, a.per_token), in_token = i - token * a.per_token.d;
      const uint32_t head = divide(in_token, a.per_row), piece = in_token - head * a.per_row.d;
      const Rows r = s_rows[token];
      const int64_t out = ((first + token) * a.heads + head) * out_row_bytes;
      f(r.block >= 0, piece, [&](int k) { return a.cache[k].base + r.block * a.cache[k].block_stride + head * a.cache[k].head_stride + r.in_block * a.cache[k].slot_stride; },
        [&](int k) { return a.out[k] + out; });
    }
  }
}

template <typename piece_t, int RUN_TOKENS>
__global__ __launch_bounds__(THREADS) void kv_read_kernel(const ReadArgs a) {
  each_piece<RUN_TOKENS>(a, (int64_t)a.per_row.d * sizeof(piece_t), [&](bool held, uint32_t piece, auto&& from, auto&& to) {
    piece_t v[2] = {};
    if (held) {
#pragma unroll
      for (int k = 0; k < 2; ++k) v[k] = *reinterpret_cast<const piece_t*>(from(k) + (int64_t)piece * sizeof(piece_t));
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) *reinterpret_cast<piece_t*>(to(k) + (int64_t)piece * sizeof(piece_t)) = v[k];
  });
}

// What a code stands for, in fp32 (said to the compiler, which would else round some of those that become fp16 only once)
__device__ __forceinline__ float value_of(uint32_t code, uint32_t pair) {
  float x = __builtin_fmaf(half_bits_to_float((uint16_t)pair), (float)code, half_bits_to_float((uint16_t)(pair >> 16)));
  asm("" : "+v"(x));
  return x;
}
// values as the output's elements
template <int TY>
__device__ __forceinline__ void put(char* p, float x) {
  if constexpr (TY == ST_FP32) *reinterpret_cast<float*>(p) = x;
  else if constexpr (TY == ST_BF16) *reinterpret_cast<__bf16*>(p) = (__bf16)x;
  else *reinterpret_cast<_Float16*>(p) = (_Float16)x;
}
template <int TY>
__device__ __forceinline__ void put_run(char* p, const float (&x)[READ_RUN]) {
  if constexpr (TY == ST_FP32) {
    typedef __attribute__((ext_vector_type(4))) float four;
    reinterpret_cast<four*>(p)[0] = four{x[0], x[1], x[2], x[3]};
    reinterpret_cast<four*>(p)[1] = four{x[4], x[5], x[6], x[7]};
  } else if constexpr (TY == ST_BF16) {
    typedef __attribute__((ext_vector_type(8))) __bf16 eight;
    *reinterpret_cast<eight*>(p) = eight{(__bf16)x[0], (__bf16)x[1], (__bf16)x[2], (__bf16)x[3], (__bf16)x[4], (__bf16)x[5], (__bf16)x[6], (__bf16)x[7]};
  } else {
    typedef __attribute__((ext_vector_type(8))) _Float16 eight;
    *reinterpret_cast<eight*>(p) =
        eight{(_Float16)x[0], (_Float16)x[1], (_Float16)x[2], (_Float16)x[3], (_Float16)x[4], (_Float16)x[5], (_Float16)x[6], (_Float16)x[7]};
  }
}

// BITS: 8 or 4. WHOLE: rows are whole runs of 8, else an element at a time.
template <int BITS, int TY, bool WHOLE, int RUN_TOKENS>
__global__ __launch_bounds__(THREADS) void kv_read_coded_kernel(const ReadArgs a) {
  constexpr int BYTES = TY == ST_FP32 ? 4 : 2;
  each_piece<RUN_TOKENS>(a, (int64_t)a.dim * BYTES, [&](bool held, uint32_t piece, auto&& from, auto&& to) {
    uint32_t pair[2] = {0, 0}; // scale and bias of 0 where there is no row
    if constexpr (WHOLE) {
      typedef piece8 __attribute__((aligned(4))) on4_t;
      piece8 codes[2] = {};
      if (held) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const char* row = from(k);
          pair[k] = *reinterpret_cast<const uint32_t*>(row);
          if constexpr (BITS == 8) codes[k] = *reinterpret_cast<const on4_t*>(row + 4 + (int64_t)piece * 8);
          else codes[k][0] = *reinterpret_cast<const uint32_t*>(row + 4 + (int64_t)piece * 4);
        }
      }
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        float x[READ_RUN];
#pragma unroll
        for (int e = 0; e < READ_RUN; ++e) {
          const uint32_t code = BITS == 8 ? (codes[k][e / 4] >> (8 * (e % 4))) & 255u : (codes[k][0] >> (4 * e)) & 15u;
          x[e] = value_of(code, pair[k]);
        }
        put_run<TY>(to(k) + (int64_t)piece * READ_RUN * BYTES, x);
      }
    } else {
      uint32_t codes[2] = {};
      if (held) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const char* row = from(k);
          pair[k] = *reinterpret_cast<const uint32_t*>(row);
          const uint32_t byte = reinterpret_cast<const uint8_t*>(row)[4 + (BITS == 8 ? piece : piece / 2)];
          codes[k] = BITS == 8 ? byte : (byte >> (4 * (piece % 2))) & 15u;
        }
      }
#pragma unroll
      for (int k = 0; k < 2; ++k)
        put<TY>(to(k) + (int64_t)piece * BYTES, value_of(codes[k], pair[k]));
    }
  });
}

unsigned grid_for(int64_t tokens, int run) {
  const int64_t runs = (tokens + run - 1) / run;
  return (unsigned)(runs < (1 << 20) ? runs : 1 << 20);
}
// Tokens of a workgroup: enough that a thread has a few pieces, where there are tokens for all of the device
template <typename F>
void by_tokens(const ReadArgs& a, F&& f) {
  if (a.tokens >= 16384 && a.per_token.d <= 1024) f(std::integral_constant<int, 16>());
  else if (a.tokens >= 2048 && a.per_token.d <= 1024) f(std::integral_constant<int, 4>());
  else f(std::integral_constant<int, 1>());
}

template <int BITS, int TY>
void launch_coded(const ReadArgs& a, bool whole, hipStream_t stream) {
  by_tokens(a, [&](auto run) {
    constexpr int RUN = decltype(run)::value;
    if (whole) kv_read_coded_kernel<BITS, TY, true, RUN><<<grid_for(a.tokens, RUN), THREADS, 0, stream>>>(a);
    else kv_read_coded_kernel<BITS, TY, false, RUN><<<grid_for(a.tokens, RUN), THREADS, 0, stream>>>(a);
  });
}
template <int BITS>
void launch_bits(const ReadArgs& a, int32_t ty, bool whole, hipStream_t stream) {
  if (ty == ST_FP32) launch_coded<BITS, ST_FP32>(a, whole, stream);
  else if (ty == ST_FP16) launch_coded<BITS, ST_FP16>(a, whole, stream);
  else launch_coded<BITS, ST_BF16>(a, whole, stream);
}

} // namespace

hipError_t launch_kv_read(const ReadArgs& a, int piece_bytes, hipStream_t stream) {
  by_tokens(a, [&](auto run) {
    constexpr int RUN = decltype(run)::value;
    const unsigned grid = grid_for(a.tokens, RUN);
    switch (piece_bytes) {
      case 16: kv_read_kernel<piece16, RUN><<<grid, THREADS, 0, stream>>>(a); break;
      case 8: kv_read_kernel<piece8, RUN><<<grid, THREADS, 0, stream>>>(a); break;
      case 4: kv_read_kernel<uint32_t, RUN><<<grid, THREADS, 0, stream>>>(a); break;
      default: kv_read_kernel<uint16_t, RUN><<<grid, THREADS, 0, stream>>>(a); break;
    }
  });
  return hipGetLastError();
}

hipError_t launch_kv_read_coded(const ReadArgs& a, int bits, int32_t output_ty, bool whole, hipStream_t stream) {
  if (bits == 8) launch_bits<8>(a, output_ty, whole, stream);
  else launch_bits<4>(a, output_ty, whole, stream);
  return hipGetLastError();
}

} // namespace fbgemm_amd
