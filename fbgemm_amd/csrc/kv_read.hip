// Rows of requests' tokens out of their pages into dense arrays: with the last request r whose
// offsets[r] <= i, token i is at position p = starts[r] + i - offsets[r] of r, and
//
//   out[i][head] = cache[table[r][p / S]][head][p % S]
//
// as it is, or as the values that 8-bit and 4-bit rows stand for: scale * code + bias in fp32 (the product of an
// fp16 number and a code is exact), rounded once. A token without a page is zeros.
//
// Bound by memory: every row is read once and written once. A workgroup has a run of tokens, whose rows' places it finds first, one a
// thread, by bisection over the offsets; then a thread has a piece of a token's rows, of keys and of values, and goes from token to
// token, four of them at a time.
#include <type_traits>

#include "decode.h"
#include "rowwise_code.h"

namespace fbgemm_amd {

namespace {

constexpr int THREADS = 256;
typedef __attribute__((ext_vector_type(4))) uint32_t piece16;
typedef __attribute__((ext_vector_type(2))) uint32_t piece8;

// Where a token's rows begin in the caches, without the head; null: it has none
struct Rows {
  const char* at[2];
};
template <typename index_t>
__device__ __forceinline__ Rows rows_of(const ReadArgs& a, int64_t token) {
  const index_t* offsets = reinterpret_cast<const index_t*>(a.offsets);
  Rows r{{nullptr, nullptr}};
  if (a.requests == 0 || token >= (int64_t)offsets[a.requests]) return r; // behind the last one: of no request, and nobody's fault
  int lo = 0, hi = a.requests; // the last request that begins at or before the token is in [lo, hi)
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if ((int64_t)offsets[mid] <= token) lo = mid;
    else hi = mid;
  }
  const int64_t in_request = (int64_t)((uint64_t)token - (uint64_t)(int64_t)offsets[lo]); // (offsets may be anything; beyond 2^63 it is below 0)
  const int64_t start = a.starts ? (int64_t)reinterpret_cast<const index_t*>(a.starts)[lo] : 0;
  const int64_t room = a.table_width * a.block.d; // below 2^31, as the number of tokens
  // 0 <= start + in_request < room, by differences of numbers that are small: the sum itself could be beyond 2^63, and mean anything to the compiler
  if (in_request >= 0 && start > -(1ll << 32) && start < room && in_request >= -start && in_request < room - start) {
    const uint32_t position = (uint32_t)(start + in_request), column = divide(position, a.block);
    const int32_t block = a.tables[lo * a.table_stride + column];
    if (block >= 0 && block < a.blocks) {
      const int64_t in_block = position - column * a.block.d;
#pragma unroll
      for (int k = 0; k < 2; ++k) r.at[k] = a.cache[k].base + block * a.cache[k].block_stride + in_block * a.cache[k].slot_stride;
    }
  }
  if (!r.at[0] && a.status) status_index(a.status, token);
  return r;
}

// For a workgroup's tokens and a thread's pieces: load(where the row begins, piece), then store(where the row goes, piece, what was loaded,
// or nothing: T{}), AT_ONCE tokens' loads on their way
constexpr int AT_ONCE = 4;
template <int RUN_TOKENS, typename T, typename L, typename S>
__device__ __forceinline__ void each_piece(const ReadArgs& a, int64_t out_row_bytes, L&& load, S&& store) {
  __shared__ Rows s_rows[RUN_TOKENS];
  const uint32_t side = a.per_token.d < THREADS ? THREADS / a.per_token.d : 1; // tokens side by side
  for (int64_t first = (int64_t)blockIdx.x * RUN_TOKENS; first < a.tokens; first += (int64_t)gridDim.x * RUN_TOKENS) {
    const uint32_t tokens = (uint32_t)(a.tokens - first < RUN_TOKENS ? a.tokens - first : RUN_TOKENS);
    __syncthreads(); // the last run's places have been read
    if (threadIdx.x < tokens) s_rows[threadIdx.x] = a.idx64 ? rows_of<int64_t>(a, first + threadIdx.x) : rows_of<int32_t>(a, first + threadIdx.x);
    __syncthreads();
    const uint32_t lead = side > 1 ? divide(threadIdx.x, a.per_token) : 0;
    if (lead >= side) continue;
    for (uint32_t in_token = threadIdx.x - lead * a.per_token.d; in_token < a.per_token.d; in_token += THREADS) {
      const uint32_t head = divide(in_token, a.per_row), piece = in_token - head * a.per_row.d;
      int64_t from[2], to = (first * a.heads + head) * out_row_bytes;
#pragma unroll
      for (int k = 0; k < 2; ++k) from[k] = head * a.cache[k].head_stride;
      for (uint32_t t0 = lead; t0 < tokens; t0 += AT_ONCE * side) {
        T v[AT_ONCE][2];
        const char* at[AT_ONCE][2];
        bool all = true;
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
          const Rows r = s_rows[t0 + i * side < tokens ? t0 + i * side : t0];
          all = all && r.at[0];
#pragma unroll
          for (int k = 0; k < 2; ++k) at[i][k] = r.at[k] ? r.at[k] + from[k] : nullptr;
        }
        if (__builtin_amdgcn_ballot_w64(!all) == 0) { // no branches between the loads: where two ways met they would be waited for
#pragma unroll
          for (int i = 0; i < AT_ONCE; ++i)
#pragma unroll
            for (int k = 0; k < 2; ++k) v[i][k] = load(at[i][k], piece);
        } else {
#pragma unroll
          for (int i = 0; i < AT_ONCE; ++i)
#pragma unroll
            for (int k = 0; k < 2; ++k) v[i][k] = at[i][k] ? load(at[i][k], piece) : T{};
        }
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i)
          if (t0 + i * side < tokens) {
#pragma unroll
            for (int k = 0; k < 2; ++k) store(a.out[k] + to + (int64_t)(t0 + i * side) * a.heads * out_row_bytes, piece, v[i][k]);
          }
      }
    }
  }
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
// Results beyond what the caches hold are marked as not read again soon (STREAMED): 65 552 tokens of 8 heads of 128 out of 4-bit rows, 268 MB of
// bf16, 76 -> 54 us; smaller ones stay where attention over them finds them.
template <bool STREAMED, typename T>
__device__ __forceinline__ void store_to(char* p, T v) {
  if (STREAMED) __builtin_nontemporal_store(v, reinterpret_cast<T*>(p));
  else *reinterpret_cast<T*>(p) = v;
}
template <int TY, bool STREAMED>
__device__ __forceinline__ void put_run(char* p, const float (&x)[READ_RUN]) {
  if constexpr (TY == ST_FP32) {
    typedef __attribute__((ext_vector_type(4))) float four;
    store_to<STREAMED>(p, four{x[0], x[1], x[2], x[3]});
    store_to<STREAMED>(p + 16, four{x[4], x[5], x[6], x[7]});
  } else if constexpr (TY == ST_BF16) {
    typedef __attribute__((ext_vector_type(8))) __bf16 eight;
    store_to<STREAMED>(p, eight{(__bf16)x[0], (__bf16)x[1], (__bf16)x[2], (__bf16)x[3], (__bf16)x[4], (__bf16)x[5], (__bf16)x[6], (__bf16)x[7]});
  } else {
    typedef __attribute__((ext_vector_type(8))) _Float16 eight;
    store_to<STREAMED>(p, eight{(_Float16)x[0], (_Float16)x[1], (_Float16)x[2], (_Float16)x[3], (_Float16)x[4], (_Float16)x[5], (_Float16)x[6], (_Float16)x[7]});
  }
}

// a piece of a row of codes: its row's scale and bias (0 where there is no row), the codes
struct Codes {
  uint32_t pair, code[2];
};

// BITS: 8 or 4. WHOLE: rows are whole runs of 8, else an element at a time.
template <int BITS, int TY, bool WHOLE, int RUN_TOKENS, bool STREAMED>
__global__ __launch_bounds__(THREADS) void kv_read_coded_kernel(const ReadArgs a) {
  constexpr int BYTES = TY == ST_FP32 ? 4 : 2;
  each_piece<RUN_TOKENS, Codes>(
      a, (int64_t)a.dim * BYTES,
      [](const char* row, uint32_t piece) {
        Codes v{0, {0, 0}};
        v.pair = *reinterpret_cast<const uint32_t*>(row);
        if constexpr (!WHOLE) {
          const uint32_t byte = reinterpret_cast<const uint8_t*>(row)[4 + (BITS == 8 ? piece : piece / 2)];
          v.code[0] = BITS == 8 ? byte : (byte >> (4 * (piece % 2))) & 15u;
        } else if constexpr (BITS == 8) {
          typedef piece8 __attribute__((aligned(4))) on4_t;
          const piece8 w = *reinterpret_cast<const on4_t*>(row + 4 + (int64_t)piece * 8);
          v.code[0] = w[0], v.code[1] = w[1];
        } else {
          v.code[0] = *reinterpret_cast<const uint32_t*>(row + 4 + (int64_t)piece * 4);
        }
        return v;
      },
      [](char* row, uint32_t piece, const Codes& v) {
        if constexpr (WHOLE) {
          float x[READ_RUN];
#pragma unroll
          for (int e = 0; e < READ_RUN; ++e) x[e] = value_of(BITS == 8 ? (v.code[e / 4] >> (8 * (e % 4))) & 255u : (v.code[0] >> (4 * e)) & 15u, v.pair);
          put_run<TY, STREAMED>(row + (int64_t)piece * READ_RUN * BYTES, x);
        } else {
          put<TY>(row + (int64_t)piece * BYTES, value_of(v.code[0], v.pair));
        }
      });
}

template <typename piece_t, int RUN_TOKENS, bool STREAMED>
__global__ __launch_bounds__(THREADS) void kv_read_kernel(const ReadArgs a) {
  each_piece<RUN_TOKENS, piece_t>(
      a, (int64_t)a.per_row.d * sizeof(piece_t),
      [](const char* row, uint32_t piece) { return *reinterpret_cast<const piece_t*>(row + (int64_t)piece * sizeof(piece_t)); },
      [](char* row, uint32_t piece, piece_t v) { store_to<STREAMED>(row + (int64_t)piece * sizeof(piece_t), v); });
}

unsigned grid_for(int64_t tokens, int run) {
  const int64_t runs = (tokens + run - 1) / run;
  return (unsigned)(runs < (1 << 20) ? runs : 1 << 20);
}
// f(tokens of a workgroup, whether results are beyond the caches): enough tokens that a thread has a few, where there are some for all of the device.
// us with 1, 4 and 16 of them, of the same caches again and again, 4-bit rows of 8 heads of 128 to bf16, then 16-bit rows of 2 heads of 64:
//    1 024     3.6  3.7  4.7     3.0  2.9  3.1
//    2 048     5.2  4.4  5.2     4.0  3.1  3.1
//    8 192    13.5  9.4  8.7     8.7  4.7  3.9
// With 4 and 16, of other caches in every call, the result of all but the last past the caches from 65 536 on:
//              4 bits, 8 x 128   8 bits, 8 x 128   16 bits, 8 x 128   16 bits, 2 x 64
//    8 192          12.4  11.5        14.2  12.5         14.5  15.7        7.3   7.4
//   65 536          64.8  68.4        81.1  78.2         97.7 104.3       28.5  18.0
// One rule for them all: what 16 lose with long rows, 4 would lose several times over with short ones.
template <typename F>
void by_tokens(const ReadArgs& a, int64_t row_bytes, F&& f) {
  if (2 * a.tokens * a.heads * row_bytes >= (128 << 20)) f(std::integral_constant<int, 16>(), std::true_type());
  else if (a.tokens >= 8192) f(std::integral_constant<int, 16>(), std::false_type());
  else if (a.tokens >= 2048) f(std::integral_constant<int, 4>(), std::false_type());
  else f(std::integral_constant<int, 1>(), std::false_type());
}

template <int BITS, int TY>
void launch_coded(const ReadArgs& a, bool whole, hipStream_t stream) {
  by_tokens(a, (int64_t)a.dim * (TY == ST_FP32 ? 4 : 2), [&](auto run, auto streamed) {
    constexpr int RUN = decltype(run)::value;
    constexpr bool STREAMED = decltype(streamed)::value;
    if (whole) kv_read_coded_kernel<BITS, TY, true, RUN, STREAMED><<<grid_for(a.tokens, RUN), THREADS, 0, stream>>>(a);
    else kv_read_coded_kernel<BITS, TY, false, RUN, false><<<grid_for(a.tokens, RUN), THREADS, 0, stream>>>(a);
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
  by_tokens(a, (int64_t)a.per_row.d * piece_bytes, [&](auto run, auto streamed) {
    constexpr int RUN = decltype(run)::value;
    constexpr bool STREAMED = decltype(streamed)::value;
    const unsigned grid = grid_for(a.tokens, RUN);
    switch (piece_bytes) {
      case 16: kv_read_kernel<piece16, RUN, STREAMED><<<grid, THREADS, 0, stream>>>(a); break;
      case 8: kv_read_kernel<piece8, RUN, false><<<grid, THREADS, 0, stream>>>(a); break;
      case 4: kv_read_kernel<uint32_t, RUN, false><<<grid, THREADS, 0, stream>>>(a); break;
      default: kv_read_kernel<uint16_t, RUN, false><<<grid, THREADS, 0, stream>>>(a); break;
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
