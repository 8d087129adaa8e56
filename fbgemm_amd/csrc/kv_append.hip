// New key and value rows into their slots of a paged cache: cache[slot / S][head][slot % S] = row,
// as they are, or as the framework's 8-bit or 4-bit rows (fp16 scale and bias in front, then the codes).
//
// Bound by memory: every byte is read once and written once (8-bit rows: half of it written, 4-bit rows: a quarter). A
// thread takes a piece of 16 bytes (less where strides or addresses ask for it) of one row of both
// keys and values, so that two loads are in flight and the slot is looked up once for the two.
#include "decode.h"
#include "rowwise_code.h"

namespace fbgemm_amd {

namespace {

constexpr int THREADS = 256;
typedef __attribute__((ext_vector_type(4))) uint32_t piece16;
typedef __attribute__((ext_vector_type(2))) uint32_t piece8;

// Where a slot's rows begin, without the head; -1: the token has none
struct Place {
  int64_t block, in_block;
};
__device__ __forceinline__ bool place_of(const AppendArgs& a, int64_t token, bool report, Place& p) {
  const int64_t slot = a.slots[token];
  if (slot < 0 || slot >= a.total_slots) {
    if (report && slot != -1 && a.status) status_index(a.status, token); // -1: a token of no request
    return false;
  }
  if (a.total_slots <= 0x7fffffff) { // the same for every thread
    p.block = divide((uint32_t)slot, a.block);
    p.in_block = (uint32_t)slot - (uint32_t)p.block * a.block.d;
  } else {
    p.block = slot / a.block.d;
    p.in_block = slot - p.block * a.block.d;
  }
  return true;
}

template <typename piece_t>
__global__ __launch_bounds__(THREADS) void kv_append_kernel(const AppendArgs a) {
  const uint32_t pieces = a.per_row.d * (uint32_t)a.heads; // of a token
  const int64_t n = a.tokens * pieces;
  for (int64_t i = (int64_t)blockIdx.x * THREADS + threadIdx.x; i < n; i += (int64_t)gridDim.x * THREADS) {
    const int64_t token = n <= 0xffffffffll ? (uint32_t)i / pieces : i / pieces;
    const uint32_t in_token = (uint32_t)(i - token * pieces);
    const uint32_t head = divide(in_token, a.per_row), piece = in_token - head * a.per_row.d;
    Place p;
    if (!place_of(a, token, in_token == 0, p)) continue;
    piece_t v[2];
#pragma unroll
    for (int k = 0; k < 2; ++k)
      v[k] = *reinterpret_cast<const piece_t*>(a.in[k] + token * a.token_stride[k] + head * a.head_stride[k] + (int64_t)piece * sizeof(piece_t));
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const CacheRows& c = a.cache[k];
      *reinterpret_cast<piece_t*>(c.base + p.block * c.block_stride + head * c.head_stride + p.in_block * c.slot_stride +
                                  (int64_t)piece * sizeof(piece_t)) = v[k];
    }
  }
}

// Element types of the input: one element, and eight in 16-byte pieces
struct F32 {
  static constexpr int BYTES = 4, PIECES = 2;
  static __device__ __forceinline__ float at(const char* p) { return *reinterpret_cast<const float*>(p); }
  static __device__ __forceinline__ float get(const piece16 (&v)[2], int e) { return q_bits_to_float(v[e / 4][e % 4]); }
};
struct F16 {
  static constexpr int BYTES = 2, PIECES = 1;
  static __device__ __forceinline__ float at(const char* p) { return half_bits_to_float(*reinterpret_cast<const uint16_t*>(p)); }
  static __device__ __forceinline__ float get(const piece16 (&v)[1], int e) { return half_bits_to_float((uint16_t)(v[0][e / 2] >> (e % 2 * 16))); }
};
struct B16 {
  static constexpr int BYTES = 2, PIECES = 1;
  static __device__ __forceinline__ float at(const char* p) { return q_bits_to_float((uint32_t)*reinterpret_cast<const uint16_t*>(p) << 16); }
  static __device__ __forceinline__ float get(const piece16 (&v)[1], int e) { return q_bits_to_float(e % 2 ? v[0][e / 2] & 0xffff0000u : v[0][e / 2] << 16); }
};

constexpr int RUN = 8; // elements of a lane at a time

// The format holds fp16 numbers: elements beyond fp16's largest count as that, NaN as zero
__device__ __forceinline__ float held(float x) { return x != x ? 0.0f : __builtin_amdgcn_fmed3f(x, -65504.0f, 65504.0f); }
// puts an element's byte into place `at` of a word; the conversion stops at 0 and 255
__device__ __forceinline__ uint32_t put_byte(float x, const RowCode& code, uint32_t at, uint32_t word) {
  return __builtin_amdgcn_cvt_pk_u8_f32(__builtin_rintf((x - code.minimum) * code.inverse_scale), at, word);
}
// an element's 4 bits
__device__ __forceinline__ uint32_t code4(float x, const RowCode& code) {
  return (uint32_t)__builtin_amdgcn_fmed3f(__builtin_rintf((x - code.minimum) * code.inverse_scale), 0.0f, 15.0f);
}
template <int CTRL>
__device__ __forceinline__ float other(float x) { // of the lane that a row's permutation puts here
  const int v = __builtin_bit_cast(int, x);
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(v, v, CTRL, 0xf, 0xf, true));
}
// the smallest and largest of a group's lanes, in all of them
__device__ __forceinline__ void extremes_of_group(float& lo, float& hi, int lanes) {
  const auto with = [&](float l, float h) {
    lo = __builtin_fminf(lo, l);
    hi = __builtin_fmaxf(hi, h);
  };
  if (lanes > 1) with(other<0xb1>(lo), other<0xb1>(hi));   // quad_perm 1, 0, 3, 2
  if (lanes > 2) with(other<0x4e>(lo), other<0x4e>(hi));   // quad_perm 2, 3, 0, 1
  if (lanes > 4) with(other<0x141>(lo), other<0x141>(hi)); // row_half_mirror: the other four of eight
  if (lanes > 8) with(other<0x140>(lo), other<0x140>(hi)); // row_mirror: the other eight of sixteen
  for (int m = 16; m < lanes; m <<= 1) with(__shfl_xor(lo, m, 64), __shfl_xor(hi, m, 64));
}

// One row per group of `lanes` lanes (a power of two): rows of any length and alignment, read twice.
template <int BITS, typename T>
__global__ __launch_bounds__(THREADS) void kv_append_coded_kernel(const AppendArgs a, const int lanes) {
  const int sub = threadIdx.x & (lanes - 1);
  const int64_t rows = a.tokens * a.heads;
  const int64_t groups = (int64_t)gridDim.x * (THREADS / lanes);
  for (int64_t row = (int64_t)blockIdx.x * (THREADS / lanes) + threadIdx.x / lanes; row < rows; row += groups) {
    const int64_t token = rows <= 0xffffffffll ? (uint32_t)row / (uint32_t)a.heads : row / a.heads;
    const int64_t head = row - token * a.heads;
    Place p;
    if (!place_of(a, token, head == 0 && sub == 0, p)) continue; // the whole group
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const char* in = a.in[k] + token * a.token_stride[k] + head * a.head_stride[k];
      const CacheRows& c = a.cache[k];
      char* out = c.base + p.block * c.block_stride + head * c.head_stride + p.in_block * c.slot_stride;
      float lo = __builtin_inff(), hi = -__builtin_inff();
      for (int j = sub; j < a.dim; j += lanes) {
        const float x = held(T::at(in + (int64_t)j * T::BYTES));
        lo = __builtin_fminf(lo, x);
        hi = __builtin_fmaxf(hi, x);
      }
      extremes_of_group(lo, hi, lanes);
      const RowCode code = row_code<BITS>(lo, hi, 0, 1);
      if (sub == 0) *reinterpret_cast<uint32_t*>(out) = (code.sb0 & 0xffffu) | (code.sb1 << 16);
      const auto at = [&](int j) { return held(T::at(in + (int64_t)j * T::BYTES)); };
      if constexpr (BITS == 8) {
        for (int j = sub; j < a.dim; j += lanes) out[4 + j] = (char)put_byte(at(j), code, 0, 0);
      } else { // an even number of elements
        for (int j = sub; 2 * j < a.dim; j += lanes) out[4 + j] = (char)(code4(at(2 * j), code) | (code4(at(2 * j + 1), code) << 4));
      }
    }
  }
}

// The common form: rows of whole runs of 8, at most 64 of them, on 16-byte boundaries. The key's and the value's row are
// loaded together and stay in registers between the search for their extremes and the rounding, lane by lane.
// 8 191 tokens x 5 heads x 128 bf16 (32 MB read and written, 6 us at a copy's rate) take 31.5 us by the kernel above and 12.1
// here (13.1 with bytes put together by shifts and extremes exchanged through LDS, 13.3 with two pairs in flight a group). That is 8-bit rows.
template <int BITS, typename T>
__global__ __launch_bounds__(THREADS) void kv_append_coded_runs_kernel(const AppendArgs a, const int lanes) {
  typedef piece8 __attribute__((aligned(4))) on4_t; // a row begins on 4 bytes
  const int sub = threadIdx.x & (lanes - 1);
  const bool mine = sub * RUN < a.dim;
  const int64_t rows = a.tokens * a.heads;
  const int64_t groups = (int64_t)gridDim.x * (THREADS / lanes);
  for (int64_t row = (int64_t)blockIdx.x * (THREADS / lanes) + threadIdx.x / lanes; row < rows; row += groups) {
    const int64_t token = rows <= 0xffffffffll ? (uint32_t)row / (uint32_t)a.heads : row / a.heads;
    const int64_t head = row - token * a.heads;
    piece16 v[2][T::PIECES] = {};
    if (mine) {
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int i = 0; i < T::PIECES; ++i)
          v[k][i] = *reinterpret_cast<const piece16*>(a.in[k] + token * a.token_stride[k] + head * a.head_stride[k] + sub * RUN * T::BYTES + 16 * i);
    }
    Place p;
    if (!place_of(a, token, head == 0 && sub == 0, p)) continue; // the whole group
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      float x[RUN], lo = __builtin_inff(), hi = -__builtin_inff();
#pragma unroll
      for (int e = 0; e < RUN; ++e) {
        x[e] = held(T::get(v[k], e));
        lo = mine ? __builtin_fminf(lo, x[e]) : lo;
        hi = mine ? __builtin_fmaxf(hi, x[e]) : hi;
      }
      extremes_of_group(lo, hi, lanes);
      const RowCode code = row_code<BITS>(lo, hi, 0, 1);
      const CacheRows& c = a.cache[k];
      char* out = c.base + p.block * c.block_stride + head * c.head_stride + p.in_block * c.slot_stride;
      if (sub == 0) *reinterpret_cast<uint32_t*>(out) = (code.sb0 & 0xffffu) | (code.sb1 << 16);
      if constexpr (BITS == 8) {
        piece8 q = {0, 0};
#pragma unroll
        for (int e = 0; e < RUN; ++e) q[e / 4] = put_byte(x[e], code, e % 4, q[e / 4]);
        if (mine) *reinterpret_cast<on4_t*>(out + 4 + sub * RUN) = q;
      } else {
        uint32_t q = 0;
#pragma unroll
        for (int e = 0; e < RUN; ++e) q |= code4(x[e], code) << (4 * e);
        if (mine) *reinterpret_cast<uint32_t*>(out + 4 + sub * RUN / 2) = q;
      }
    }
  }
}

template <int BITS>
void launch_coded(const AppendArgs& a, int32_t input_ty, int lanes, int grid, bool runs, hipStream_t stream) {
  const auto launch = [&](auto type) {
    using T = decltype(type);
    if (runs) kv_append_coded_runs_kernel<BITS, T><<<grid, THREADS, 0, stream>>>(a, lanes);
    else kv_append_coded_kernel<BITS, T><<<grid, THREADS, 0, stream>>>(a, lanes);
  };
  if (input_ty == ST_FP32) launch(F32());
  else if (input_ty == ST_FP16) launch(F16());
  else launch(B16());
}

int grid_for(int64_t items, int per_block) {
  const int64_t want = (items + per_block - 1) / per_block;
  return (int)(want > 8192 ? 8192 : want);
}

} // namespace

hipError_t launch_kv_append(const AppendArgs& a, int piece_bytes, hipStream_t stream) {
  const int grid = grid_for(a.tokens * a.heads * a.per_row.d, THREADS);
  switch (piece_bytes) {
    case 16: kv_append_kernel<piece16><<<grid, THREADS, 0, stream>>>(a); break;
    case 8: kv_append_kernel<piece8><<<grid, THREADS, 0, stream>>>(a); break;
    case 4: kv_append_kernel<uint32_t><<<grid, THREADS, 0, stream>>>(a); break;
    default: kv_append_kernel<uint16_t><<<grid, THREADS, 0, stream>>>(a); break;
  }
  return hipGetLastError();
}

hipError_t launch_kv_append_coded(const AppendArgs& a, int bits, int32_t input_ty, bool aligned16, hipStream_t stream) {
  int lanes = 1;
  while (lanes < 64 && lanes * RUN < a.dim) lanes <<= 1;
  const int grid = grid_for(a.tokens * a.heads, THREADS / lanes);
  const bool runs = aligned16 && a.dim % RUN == 0 && a.dim <= 64 * RUN;
  if (bits == 8) launch_coded<8>(a, input_ty, lanes, grid, runs, stream);
  else launch_coded<4>(a, input_ty, lanes, grid, runs, stream);
  return hipGetLastError();
}

} // namespace fbgemm_amd
