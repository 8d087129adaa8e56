// Rotary positions: a head's first 2 * pairs elements as pairs (a, b), elements (p, p + pairs) or
// neighbours (2 p, 2 p + 1), turned by the angle  position * frequency_p:
//
//   a' = m (a cos - b sin),  b' = m (b cos + a sin)
//
// and the rest of the head as it is. In fp32, rounded once.
//
// Angles are taken in fp64, as quarters of a turn: what is left of a far position's angle behind its whole
// quarters is off by three roundings of 2^-53 of the angle (2 / pi, its product with the frequency, that with the position), less than
// 2^-51; in fp32 it would be 2^-24 of it (262 143 radians: 0.02). Sine and
// cosine of the rest, at most pi/4, are their series.
//
// Bound by memory: every element is read once and written once. 16 384 tokens of 40 heads of 128, bf16: 54.5 us, 6.2 TB/s; 64 of them:
// 2.9 us. A workgroup has a token: it makes its sines once, in LDS, and turns all heads of queries and keys by them, 16 bytes (two of them,
// where a pair's elements are apart) a thread at a time. (Four tokens a workgroup take 8 to 10 % longer.) Pairs that do not fill 16 bytes go
// element by element: those tokens with heads of 96, 24 of it turned, 156 us, 1.6 TB/s.
#include "decode.h"

namespace fbgemm_amd {

namespace {

constexpr int THREADS = 256;
// Bytes of the results from which on they are marked as not read again soon. us without the mark and with it, on other tensors in every call, and
// on the same ones, which the last cache may hold (heads of 128 in bf16, the first row heads of 80 in fp32):
//    31 MB   16.1  17.3   12.3  16.9
//    61 MB   23.4  22.9   19.8  21.9
//    84 MB   29.2  29.4   26.1  28.5
//   123 MB   39.4  41.2   37.4  40.2
//   168 MB   61.8  55.1   60.8  54.2
//   336 MB  120.2 106.3  119.6 105.6
// Between the border and some 130 MB the mark costs a little and leaves the cache to others.
constexpr int64_t STREAM_FROM = 64 << 20;
typedef __attribute__((ext_vector_type(4))) uint32_t piece16;

struct Turn {
  float cosine, sine;
};
// of position * frequency
__device__ __forceinline__ Turn turn_of(double position, double frequency, float magnitude, float sine_magnitude) {
  const double quarters = position * (frequency * 0.63661977236758134308); // 2 / pi
  const double whole = __builtin_rint(quarters);
  const int quadrant = (int)(int64_t)(whole - 4.0 * __builtin_floor(whole * 0.25));
  const float x = (float)(quarters - whole) * 1.5707963267948966f, z = x * x;
  // to z^4 and z^5: the next terms are below 2^-29 at pi/4
  float s = 1.0f / 362880.0f, c = -1.0f / 3628800.0f;
  s = __builtin_fmaf(s, z, -1.0f / 5040.0f);
  s = __builtin_fmaf(s, z, 1.0f / 120.0f);
  s = __builtin_fmaf(s, z, -1.0f / 6.0f);
  s = __builtin_fmaf(s * z, x, x);
  c = __builtin_fmaf(c, z, 1.0f / 40320.0f);
  c = __builtin_fmaf(c, z, -1.0f / 720.0f);
  c = __builtin_fmaf(c, z, 1.0f / 24.0f);
  c = __builtin_fmaf(c, z, -0.5f);
  c = __builtin_fmaf(c, z, 1.0f);
  const float sine = quadrant & 1 ? c : s, cosine = quadrant & 1 ? s : c;
  return Turn{(quadrant == 1 || quadrant == 2 ? -cosine : cosine) * magnitude, (quadrant & 2 ? -sine : sine) * sine_magnitude};
}

// the sines of a token
__device__ __forceinline__ void make_turns(const RotateArgs& a, int64_t token, Turn* turns) {
  const int64_t position = a.idx64 ? reinterpret_cast<const int64_t*>(a.positions)[token] : reinterpret_cast<const int32_t*>(a.positions)[token];
  for (int i = threadIdx.x; i < a.pairs; i += THREADS) turns[i] = turn_of((double)position, a.frequencies[i], a.magnitude, a.sine);
  __syncthreads();
}

// Elements of 16 bytes as fp32, and back
template <int TY>
struct Chunk {
  static constexpr int N = TY == ST_FP32 ? 4 : 8;
  static constexpr int BYTES = 16 / N;
  static __device__ __forceinline__ float get(const piece16& w, int e) {
    if constexpr (TY == ST_FP32) return __builtin_bit_cast(float, (uint32_t)w[e]);
    else if constexpr (TY == ST_BF16) return __builtin_bit_cast(float, e % 2 ? w[e / 2] & 0xffff0000u : w[e / 2] << 16);
    else return (float)__builtin_bit_cast(_Float16, (uint16_t)(w[e / 2] >> (e % 2 * 16)));
  }
  // elements e and e + 1
  static __device__ __forceinline__ void put(piece16& w, int e, float x, float y) {
    if constexpr (TY == ST_FP32) {
      w[e] = __builtin_bit_cast(uint32_t, x);
      w[e + 1] = __builtin_bit_cast(uint32_t, y);
    } else if constexpr (TY == ST_BF16) {
      typedef __attribute__((ext_vector_type(2))) __bf16 pair_t;
      const pair_t v = {(__bf16)x, (__bf16)y};
      w[e / 2] = __builtin_bit_cast(uint32_t, v);
    } else {
      typedef __attribute__((ext_vector_type(2))) _Float16 pair_t;
      const pair_t v = {(_Float16)x, (_Float16)y};
      w[e / 2] = __builtin_bit_cast(uint32_t, v);
    }
  }
  static __device__ __forceinline__ float at(const char* p) {
    if constexpr (TY == ST_FP32) return *reinterpret_cast<const float*>(p);
    else if constexpr (TY == ST_BF16) return __builtin_bit_cast(float, (uint32_t)*reinterpret_cast<const uint16_t*>(p) << 16);
    else return (float)*reinterpret_cast<const _Float16*>(p);
  }
  static __device__ __forceinline__ void set(char* p, float x) {
    if constexpr (TY == ST_FP32) *reinterpret_cast<float*>(p) = x;
    else if constexpr (TY == ST_BF16) *reinterpret_cast<__bf16*>(p) = (__bf16)x;
    else *reinterpret_cast<_Float16*>(p) = (_Float16)x;
  }
};
// (fp32 numbers, said to the compiler: it would else round some, not all, products of fp16 numbers to fp16 at once, and
// results would go by how rows are aligned)
__device__ __forceinline__ float rounded(float x) {
  asm("" : "+v"(x));
  return x;
}
__device__ __forceinline__ float first_of(float a, float b, Turn t) { return rounded(__builtin_fmaf(a, t.cosine, -(b * t.sine))); }
__device__ __forceinline__ float second_of(float a, float b, Turn t) { return rounded(__builtin_fmaf(b, t.cosine, a * t.sine)); }

// where a unit's head is, and its number in it
struct Place {
  const char* in;
  char* out;
  int unit;
  bool same; // out is in
};
__device__ __forceinline__ Place place_of(const RotateArgs& a, int64_t token, uint32_t item) {
  Place p;
  int head = (int)divide(item, a.units);
  p.unit = (int)(item - head * a.units.d);
  const int k = head >= a.heads[0];
  if (k) head -= a.heads[0];
  p.in = a.in[k] + token * a.in_token[k] + head * a.in_head[k];
  p.out = a.out[k] + token * a.out_token[k] + head * a.out_head[k];
  p.same = p.in == p.out;
  return p;
}

// What is far beyond the caches is read and written past them (STREAMED)
template <bool STREAMED>
__device__ __forceinline__ piece16 load_piece(const char* p) {
  return STREAMED ? __builtin_nontemporal_load(reinterpret_cast<const piece16*>(p)) : *reinterpret_cast<const piece16*>(p);
}
template <bool STREAMED>
__device__ __forceinline__ void store_piece(char* p, piece16 v) {
  if (STREAMED) __builtin_nontemporal_store(v, reinterpret_cast<piece16*>(p));
  else *reinterpret_cast<piece16*>(p) = v;
}
// Rows of whole 16-byte pieces on 16-byte boundaries, and pairs that fill whole pieces
template <int TY, bool INTERLEAVED, bool STREAMED>
__device__ __forceinline__ void turn_piece(const RotateArgs& a, const Place& p, const Turn* turns) {
  using C = Chunk<TY>;
  constexpr int N = C::N;
  const int turning = INTERLEAVED ? 2 * a.pairs / N : a.pairs / N; // units; the others are pieces of the rest, behind all pairs
  if (p.unit >= turning) {
    if (p.same) return;
    const int at = 2 * a.pairs * C::BYTES + (p.unit - turning) * 16;
    store_piece<STREAMED>(p.out + at, load_piece<STREAMED>(p.in + at));
  } else if constexpr (INTERLEAVED) {
    const Turn* turn = turns + p.unit * (N / 2);
    piece16 w = load_piece<STREAMED>(p.in + p.unit * 16);
#pragma unroll
    for (int e = 0; e < N; e += 2) {
      const float x = C::get(w, e), y = C::get(w, e + 1);
      C::put(w, e, first_of(x, y, turn[e / 2]), second_of(x, y, turn[e / 2]));
    }
    store_piece<STREAMED>(p.out + p.unit * 16, w);
  } else {
    const Turn* turn = turns + p.unit * N;
    const int other = a.pairs * C::BYTES;
    piece16 v = load_piece<STREAMED>(p.in + p.unit * 16), w = load_piece<STREAMED>(p.in + p.unit * 16 + other);
#pragma unroll
    for (int e = 0; e < N; e += 2) {
      const float x0 = C::get(v, e), x1 = C::get(v, e + 1), y0 = C::get(w, e), y1 = C::get(w, e + 1);
      C::put(v, e, first_of(x0, y0, turn[e]), first_of(x1, y1, turn[e + 1]));
      C::put(w, e, second_of(x0, y0, turn[e]), second_of(x1, y1, turn[e + 1]));
    }
    store_piece<STREAMED>(p.out + p.unit * 16, v);
    store_piece<STREAMED>(p.out + p.unit * 16 + other, w);
  }
}

// Any others: a pair, or an element of the rest
template <int TY>
__device__ __forceinline__ void turn_element(const RotateArgs& a, const Place& p, const Turn* turns) {
  using C = Chunk<TY>;
  if (p.unit < a.pairs) {
    const int e = (a.interleaved ? 2 * p.unit : p.unit) * C::BYTES, f = e + (a.interleaved ? 1 : a.pairs) * C::BYTES;
    const float x = C::at(p.in + e), y = C::at(p.in + f);
    const Turn turn = turns[p.unit];
    C::set(p.out + e, first_of(x, y, turn));
    C::set(p.out + f, second_of(x, y, turn));
  } else if (!p.same) {
    const int e = (p.unit + a.pairs) * C::BYTES; // behind the pairs' second elements
    if constexpr (TY == ST_FP32) *reinterpret_cast<uint32_t*>(p.out + e) = *reinterpret_cast<const uint32_t*>(p.in + e);
    else *reinterpret_cast<uint16_t*>(p.out + e) = *reinterpret_cast<const uint16_t*>(p.in + e);
  }
}

enum { ELEMENTS, HALVES, NEIGHBOURS };
template <int TY, int FORM, bool STREAMED>
__global__ __launch_bounds__(THREADS) void rotate_positions_kernel(const RotateArgs a) {
  extern __shared__ Turn s_turns[];
  const uint32_t items = (uint32_t)(a.heads[0] + a.heads[1]) * a.units.d;
  for (int64_t token = blockIdx.x; token < a.tokens; token += gridDim.x) {
    __syncthreads(); // the last token's turns have been read
    make_turns(a, token, s_turns);
    for (uint32_t i = threadIdx.x; i < items; i += THREADS) {
      const Place p = place_of(a, token, i);
      if constexpr (FORM == ELEMENTS) turn_element<TY>(a, p, s_turns);
      else turn_piece<TY, FORM == NEIGHBOURS, STREAMED>(a, p, s_turns);
    }
  }
}

template <int TY>
void launch(RotateArgs a, bool aligned16, hipStream_t stream) {
  constexpr int N = Chunk<TY>::N;
  // queries and keys share a piece's place in a head
  const bool pieces = aligned16 && a.dim % N == 0 && (a.interleaved ? 2 * a.pairs : a.pairs) % N == 0;
  const int rest = a.dim - 2 * a.pairs;
  const int units = pieces ? (a.interleaved ? 2 * a.pairs / N : a.pairs / N) + rest / N : a.pairs + rest;
  const int heads = a.heads[0] + a.heads[1];
  a.units = make_divisor((uint32_t)units);
  const unsigned grid = (unsigned)(a.tokens < (1 << 22) ? a.tokens : 1 << 22);
  const size_t lds = (size_t)a.pairs * sizeof(Turn);
  const bool streamed = a.tokens * heads * a.dim * Chunk<TY>::BYTES >= STREAM_FROM;
  const auto kernel = !pieces ? rotate_positions_kernel<TY, ELEMENTS, false>
      : a.interleaved ? (streamed ? rotate_positions_kernel<TY, NEIGHBOURS, true> : rotate_positions_kernel<TY, NEIGHBOURS, false>)
                      : (streamed ? rotate_positions_kernel<TY, HALVES, true> : rotate_positions_kernel<TY, HALVES, false>);
  kernel<<<grid, THREADS, lds, stream>>>(a);
}

} // namespace

hipError_t launch_rotate_positions(const RotateArgs& a, int32_t ty, bool aligned16, hipStream_t stream) {
  if (ty == ST_FP32) launch<ST_FP32>(a, aligned16, stream);
  else if (ty == ST_FP16) launch<ST_FP16>(a, aligned16, stream);
  else launch<ST_BF16>(a, aligned16, stream);
  return hipGetLastError();
}

} // namespace fbgemm_amd
