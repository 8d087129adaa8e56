// Attention of one new token per request over a paged key-value cache, on the matrix cores.
//
//   s_t = scale * q . k_t  (or cap * tanh(scale / cap * q . k_t)),  lo <= t < len
//   out = sum_t exp(s_t - m) v_t / sum_t exp(s_t - m),  lse = m + log(sum_t exp(s_t - m)),  m = max_t s_t
//
// in one pass over the tokens with the running m and sum, all in fp32 (exp as exp2 of s * log2 e).
//
// Bound by memory: every row of the cache is read once for up to 16 queries that share its head (more
// read it once per 16). 256 requests of 16 to 8 192 tokens, 64 queries on 8 heads of 128, bf16: 677 us,
// 6.37 TB/s; 64 requests of 1 to 4 096, 32 queries on 8: 92 us, 5.87 TB/s; one of 262 143 in 8-bit rows:
// 103 us, 5.4 TB/s; one of 500: 10.3 us, launches and a chain of dependent steps. That the rows need no staging in LDS, no transposition through it and no exchange between lanes
// is what the operand layouts of the 16x16x32 products give, written here as l = 16 g + n:
//   keys     A = K [token n][8 of dim], B = Q^T [8 of dim][query n]: C holds tokens 4g .. 4g+3 of query n
//   values   A = V^T [a column][8 tokens], B = P^T [8 tokens][query n]: a product sums over tokens in any
//            order that A and B share, so lane group g's 8 tokens are the 4g .. 4g+3 of two 16-token
//            tiles: just the weights that C left in its registers. A lane loads its 8 tokens' rows at
//            columns 8n .. 8n+7 in whole 16-byte pieces (a group covers a row), and product i takes
//            column 8n + i: two bytes of each of 8 registers, put side by side by v_perm_b32.
// The result holds query n and columns 8 (4g + r) + i: rescaling by a query's factor needs no
// exchange, and 8 consecutive columns go out as one piece.
//
// Weights are cut to 16 bits for the products, as two numbers (the rounded weight and what the rounding
// left): 16 bits of them count for bf16 and 22 for fp16, whose weights are 2^14 times larger so that
// those 2^-28 of the largest are still normal numbers. The second product costs matrix time of
// which there is plenty (24 products, 384 cycles, for the 16 KB of 32 tokens x 128 columns).
//
// 8-bit rows (fp16 scale a_t and bias b_t in front): s_t = a_t (q . k8_t) + b_t sum(q); values by c8 = v8 - 128 and
// b'_t = b_t + 128 a_t: weights p_t a_t for c8, p_t b'_t beside them. -128 .. 255 are exact in bf16 and fp16. Rows lie
// about zero, so b' is small and both sums are of the result's size. By v8 and b both are some 128 steps of a row's scale
// and cancel, with what the cut of the weights and the sums' roundings made of them: columns of zeros came out as 2^-18 of
// the scale, not as zeros. Flipping the bytes' top bits costs 0.7 to 2 % (262 143 tokens 101.5 -> 102.2 us). A score's
// rounding is 2^-24 of that anyway; keys are centred where it is free (fp16).
//
// Work: steps of 128 tokens of a (request, key head, 16 queries), 32 for each of a worker's (workgroup's) four waves, numbered in
// that order. Each of W workers takes a W-th of them in a row, whatever requests they are of, so that all end together
// however long the requests are; a pair of request and head weighs one more than its steps, or a worker that meets
// many short ones would be late. The waves' sums of a pair are joined in LDS. A pair that a worker has whole it writes
// out; of one that it shares with its neighbours (its first and its last, at most) it leaves the sums, which a second
// launch adds up in the workers' order: results depend on no order of theirs. (Joining them in the first launch, by the last worker
// to arrive, takes fences that write back and empty whole caches, each die having its own: with those 64 requests of 1 to
// 4 096 tokens took 367 us where two launches took 109 at the time.)
#pragma once
#include <type_traits>

#include "decode.h"

namespace fbgemm_amd {

constexpr int ATT_WAVES = 4;
constexpr int ATT_TILE = 32; // tokens of a wave's step
constexpr int ATT_STEP = ATT_WAVES * ATT_TILE; // of all waves'
static_assert(ATT_STEP == ATTENTION_STEP, "");
constexpr float ATT_LOG2E = 1.4426950408889634f;

#if defined(__HIPCC__)
namespace attention {

typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(2))) _Float16 f16x2;

__device__ __forceinline__ f32x4 product_bf16(uint4 a, uint4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 product_f16(uint4 a, uint4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
template <bool BF16>
__device__ __forceinline__ f32x4 product(uint4 a, uint4 b, f32x4 c) {
  return BF16 ? product_bf16(a, b, c) : product_f16(a, b, c);
}

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) { // to nearest even
  typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
  const bf16x2 v = {(__bf16)a, (__bf16)b};
  return __builtin_bit_cast(uint32_t, v);
}
__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
  const f16x2 v = {(_Float16)a, (_Float16)b};
  return __builtin_bit_cast(uint32_t, v);
}
template <bool BF16>
__device__ __forceinline__ uint32_t pack16(float a, float b) {
  return BF16 ? pack_bf16(a, b) : pack_f16(a, b);
}
template <bool BF16>
__device__ __forceinline__ float unpack16(uint32_t v, int half) {
  if (BF16) return __builtin_bit_cast(float, half ? v & 0xffff0000u : v << 16);
  return (float)__builtin_bit_cast(f16x2, v)[half];
}
// 8 weights as two operands: rounded, and what the rounding left
template <bool BF16>
__device__ __forceinline__ void split(const float (&p)[8], uint4& hi, uint4& lo) {
  uint32_t h[4], l[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    h[i] = pack16<BF16>(p[2 * i], p[2 * i + 1]);
    l[i] = pack16<BF16>(p[2 * i] - unpack16<BF16>(h[i], 0), p[2 * i + 1] - unpack16<BF16>(h[i], 1));
  }
  hi = make_uint4(h[0], h[1], h[2], h[3]);
  lo = make_uint4(l[0], l[1], l[2], l[3]);
}

// Bytes with their top bits flipped are byte - 128 in two's complement. Four at a time, and the compiler is kept from doing it
// byte by byte: then each is one conversion of a signed byte in place, as for plain bytes (else there is a third instruction for each).
__device__ __forceinline__ uint32_t centre(uint32_t bytes) {
  bytes ^= 0x80808080u;
  asm("" : "+v"(bytes));
  return bytes;
}
__device__ __forceinline__ float centred(uint32_t flipped, int i) { return (float)(int8_t)(flipped >> (8 * i)); }

// 8 bytes -> 8 numbers of 16 bits, exactly: byte - 128 for fp16, which a constant gives, the byte for bf16
template <bool BF16>
__device__ __forceinline__ uint4 widen(uint32_t a, uint32_t b) {
  uint32_t r[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t w = i < 2 ? a : b;
    const int s = (i & 1) * 16;
    if (BF16) {
      const float x = (float)((w >> s) & 0xffu), y = (float)((w >> (s + 8)) & 0xffu);
      r[i] = __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, y), __builtin_bit_cast(uint32_t, x), 0x07060302u);
    } else { // 1024 + byte is the byte under fp16's exponent 0x64
      const uint32_t v = __builtin_amdgcn_perm(0x64646464u, w, i & 1 ? 0x04030402u : 0x04010400u);
      const f16x2 off = {(_Float16)1152.0f, (_Float16)1152.0f};
      r[i] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, v) - off);
    }
  }
  return make_uint4(r[0], r[1], r[2], r[3]);
}

__device__ __forceinline__ float half_at(uint32_t pair, int i) { return (float)__builtin_bit_cast(f16x2, pair)[i]; }
// what byte 128 of a row stands for, by its scale and bias
__device__ __forceinline__ float middle(uint32_t pair) { return __builtin_fmaf(128.0f, half_at(pair, 0), half_at(pair, 1)); }
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
// tanh(x) / x = 1 - x^2/3 + 2 x^4/15 - ..., for |x| < TANH_SMALL to 2^-24 (the next term: 0.0036 x^12)
constexpr float TANH_SMALL = 0.35f;
__device__ __forceinline__ float tanh_ratio(float x) {
  const float z = x * x;
  float p = -1382.0f / 155925.0f;
  p = __builtin_fmaf(p, z, 62.0f / 2835.0f);
  p = __builtin_fmaf(p, z, -17.0f / 315.0f);
  p = __builtin_fmaf(p, z, 2.0f / 15.0f);
  p = __builtin_fmaf(p, z, -1.0f / 3.0f);
  return __builtin_fmaf(p, z, 1.0f);
}
// (1 - t) / (1 + t), t = exp(-2 |x|): off by some 2^-23 of 1, so for others than small x
__device__ __forceinline__ float tanh_fast(float x) {
  const float t = exp2_fast(-2.0f * ATT_LOG2E * __builtin_fabsf(x));
  return __builtin_copysignf((1.0f - t) * __builtin_amdgcn_rcpf(1.0f + t), x);
}

// Tables and lengths are written by nobody while a kernel runs: where an address is the same for the
// wave, the scalar unit reads them, apart from the rows' loads and what waits for these.
template <typename T>
using constant = const __attribute__((address_space(4))) T*;
template <typename T>
__device__ __forceinline__ constant<T> as_constant(const void* p) {
  return (constant<T>)reinterpret_cast<uintptr_t>(p);
}

// A tile's rows as a buffer: its address sits in scalar registers, a lane adds 32 bits, a row the scalar offset. Every
// load is inside the tile by the lanes' own offsets; the size is there to be none, for a tile that is not there: its
// loads touch no memory.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_at(const char* p, bool any) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(p), 0, any ? 0x7fffffff : 0, 0x00027000);
}
// Rows of 16-bit numbers are read once, in whole lines, and marked so (non-temporal): 256 requests of 16 to 8 192 tokens,
// 64 queries on 8 heads of 128, 738 -> 677 us. A line of 8-bit rows takes several loads, which then miss it (262 143 tokens
// 110 -> 171 us), and the halves of a line that a key of 64 numbers is loaded in do, a little.
constexpr int READ_ONCE = 2;
template <int AUX, int N>
__device__ __forceinline__ void fetch(uint32_t (&to)[N], __amdgpu_buffer_rsrc_t rows, uint32_t lane, uint32_t row, uint32_t piece) {
  if constexpr (N == 4) {
    const auto w = __builtin_amdgcn_raw_buffer_load_b128(rows, lane + piece, row, AUX);
    to[0] = w[0], to[1] = w[1], to[2] = w[2], to[3] = w[3];
  } else if constexpr (N == 2) {
    const auto w = __builtin_amdgcn_raw_buffer_load_b64(rows, lane + piece, row, AUX);
    to[0] = w[0], to[1] = w[1];
  } else {
    to[0] = __builtin_amdgcn_raw_buffer_load_b32(rows, lane + piece, row, AUX);
  }
}

// the largest over the four lanes n, 16 + n, 32 + n, 48 + n
__device__ __forceinline__ float group_max(float x) {
  const auto a = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x), false, false);
  x = __builtin_fmaxf(__builtin_bit_cast(float, (uint32_t)a[0]), __builtin_bit_cast(float, (uint32_t)a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x), false, false);
  return __builtin_fmaxf(__builtin_bit_cast(float, (uint32_t)b[0]), __builtin_bit_cast(float, (uint32_t)b[1]));
}

// A request's tokens that count, lo <= t < end, in `steps` from `base` on
struct Span {
  int32_t base, lo, end, steps;
};
__device__ __forceinline__ Span span_of(const AttentionArgs& a, int32_t request) {
  int64_t len = a.idx64 ? as_constant<int64_t>(a.lengths)[request] : (int64_t)as_constant<int32_t>(a.lengths)[request];
  len = len < 0 ? 0 : len > a.max_tokens ? a.max_tokens : len;
  Span s;
  s.end = (int32_t)len;
  s.lo = a.window > 0 && len > a.window ? (int32_t)(len - a.window) : 0;
  s.base = s.lo & ~15;
  const int32_t n = (s.end - s.base + ATT_STEP - 1) / ATT_STEP;
  s.steps = n > 0 ? n : 1; // an empty one is somebody's too: its result is zeros
  return s;
}

// U units over W workers: the first U % W have one more
struct Shares {
  uint32_t each, more;
  __device__ __forceinline__ Shares(uint32_t units, uint32_t workers) : each(units / workers), more(units - each * workers) {}
  __device__ __forceinline__ uint32_t begin(uint32_t worker) const { return worker * each + (worker < more ? worker : more); }
  __device__ __forceinline__ uint32_t worker_of(uint32_t unit) const {
    const uint32_t longer = more * (each + 1);
    return unit < longer ? unit / (each + 1) : more + (unit - longer) / each;
  }
};

__device__ __forceinline__ uint32_t inclusive_sum(uint32_t v, int lane) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t o = __shfl_up(v, d, 64);
    v += lane >= d ? o : 0;
  }
  return v;
}

// ROWS8: rows of the 8-bit format. DP: columns the code is laid out for; FULL: dim is DP, else less: lanes that would have the
// columns behind read the row's first ones in their place, which meet zeros in the queries or make outputs that nobody wants.
// PAGE16: pages are whole 16-token tiles, whose addresses are then the same for the wave. PACKED (FULL 8-bit rows, PAGE16): the
// rows of a page's tokens follow each other without gaps. 16 of them are then read as one run of bytes, every line by one
// load and marked as read once, and go through LDS, where a lane finds its pieces: 262 143 tokens 103 us, 118 with a gap
// of 4 bytes behind each row (two tiles ahead instead of one: 2 % more); 256 requests of 16 to 8 192 tokens, 64 queries on 8 heads of 128, 400 us, 459 with gaps.
template <bool BF16, bool ROWS8, int DP, bool FULL, bool PAGE16, bool PACKED>
struct Attention {
  static constexpr int KP = DP / 32;                   // products of a key tile
  static constexpr int HALVES = DP > 128 ? 2 : 1;      // pieces of a value row that a lane holds
  static constexpr int VC = DP / 16 / HALVES;          // columns of a piece: 8, or 4 of DP = 64
  static constexpr int EL = ROWS8 ? 1 : 2;             // bytes of an element
  static constexpr int HEAD = ROWS8 ? 4 : 0;           // of a row, in front of its elements
  static constexpr bool PBF16 = ROWS8 ? true : BF16;   // type of the weights: scales go into them, so 8-bit rows take bf16's range
  static constexpr float SHIFT = PBF16 ? 0.0f : 14.0f; // weights are 2^SHIFT times larger
  static constexpr int VREGS = ROWS8 ? (VC + 3) / 4 : VC / 2; // registers of a value piece
  static constexpr int KREGS = ROWS8 ? 2 : 4;          // registers of a key piece
  static constexpr int DEPTH = 1;                      // tiles loaded ahead
  static constexpr int KEY_AUX = ROWS8 || DP == 64 ? 0 : READ_ONCE, VALUE_AUX = ROWS8 ? 0 : READ_ONCE;

  static constexpr int RUN = 16 * (DP * EL + HEAD);    // PACKED: bytes of 16 rows
  static constexpr int RUN_LOADS = RUN / 1024;         // a wave's loads of one, but for its last 64 bytes
  static_assert(!PACKED || RUN == RUN_LOADS * 1024 + 64, "16 rows of 64, 128 or 256 bytes and a header each");
  static constexpr int STAGE = PACKED ? 4 * RUN : 16;  // bytes of LDS a wave stages a tile in: keys' two runs, values' two

  // a lane's part of 32 tokens
  struct Rows {
    uint32_t k[2][KP][KREGS];
    uint32_t v[HALVES][8][VREGS];
    uint32_t k_pair[ROWS8 ? 8 : 1], v_pair[ROWS8 ? 8 : 1];
  };
  // the same as bytes in a row: keys' runs, values' runs, and the last 64 bytes of the four in lanes 0 .. 15
  struct Runs {
    uint32_t piece[4][RUN_LOADS > 0 ? RUN_LOADS : 1][4], last[4];
  };
  // what a wave has loaded of 32 tokens
  struct Tile : std::conditional_t<PACKED, Runs, Rows> {
    uint32_t seen; // bit j: this lane's token j counts
    bool partial;  // some token of the tile does not (the same for the wave)
  };
  // where its pages are: PAGE16 of the two 16-token halves, else of token `lane & 31`
  struct Pages {
    int block[2];
  };

  const AttentionArgs& a;
  const int lane, n, g;
  uint32_t key_lane, value_lane; // bytes from a row's beginning to the lane's first piece
  uint32_t key_rows, value_rows; // PAGE16: from a tile's, of rows n and 4 g
  const char *key_base, *value_base;
  const int32_t* table;
  Span span;
  int first_column, last_column; // of the tokens that count
  char* stage;                   // PACKED: this wave's STAGE bytes

  __device__ __forceinline__ Attention(const AttentionArgs& args, int lane_, char* stage_)
      : a(args), lane(lane_), n(lane_ & 15), g(lane_ >> 4), stage(stage_) {
    key_lane = HEAD + 8 * g * EL;
    value_lane = HEAD + (FULL || n * VC < a.dim ? n * VC * EL : 0);
    key_rows = n * (uint32_t)a.key.slot_stride + key_lane;
    value_rows = 4 * g * (uint32_t)a.value.slot_stride + value_lane;
  }

  // bytes from the lane's first piece to the next ones
  __device__ __forceinline__ uint32_t key_piece(int i) const { return FULL || 32 * i + 8 * g < a.dim ? 32 * i * EL : 0u - 8 * g * EL; }
  __device__ __forceinline__ uint32_t value_piece(int h) const { return FULL || h == 0 || 128 * h + n * VC < a.dim ? 128 * h * EL : 0u; }

  __device__ __forceinline__ int token_of(int j) const { return (j >> 2) * 16 + 4 * g + (j & 3); } // of this lane's values and scores, in the tile

  __device__ __forceinline__ Pages pages(int t0) const {
    Pages p;
    if (PAGE16) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int column = (int)divide((uint32_t)(t0 + 16 * h), a.block);
        p.block[h] = as_constant<int32_t>(table)[column < last_column ? column : last_column]; // a half behind the end reads rows of the last page
      }
    } else {
      const int column = (int)divide((uint32_t)(t0 + (lane & 31)), a.block); // of a token that counts, or the nearest one that does
      p.block[0] = table[column < first_column ? first_column : column > last_column ? last_column : column];
      p.block[1] = 0;
    }
    return p;
  }

  // `any`: false: PAGE16 loads nothing, else the tile as well (it is there)
  __device__ __forceinline__ void load(Tile& tile, int t0, const Pages& pages, bool any) const {
    typedef __attribute__((ext_vector_type(KREGS))) uint32_t key_t;
    typedef __attribute__((ext_vector_type(VREGS))) uint32_t value_t;
    typedef key_t __attribute__((aligned(ROWS8 ? 4 : 16))) stored_key; // 8-bit rows begin on 4 bytes
    typedef value_t __attribute__((aligned(ROWS8 ? 4 : 2 * VC))) stored_value;
    tile.partial = t0 < span.lo || t0 + ATT_TILE > span.end;
    tile.seen = 0xff;
    [[maybe_unused]] const auto key = [&](auto& tile, int h, int i, const char* p) {
      const auto* at = reinterpret_cast<const stored_key*>(p);
      const key_t w = KEY_AUX ? __builtin_nontemporal_load(at) : *at;
#pragma unroll
      for (int r = 0; r < KREGS; ++r) tile.k[h][i][r] = w[r];
    };
    [[maybe_unused]] const auto value = [&](auto& tile, int h, int j, const char* p) {
      const auto* at = reinterpret_cast<const stored_value*>(p);
      const value_t w = VALUE_AUX ? __builtin_nontemporal_load(at) : *at;
#pragma unroll
      for (int r = 0; r < VREGS; ++r) tile.v[h][j][r] = w[r];
    };
    if constexpr (PACKED) {
      const char* run[4];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int t = t0 + 16 * h;
        const int in_block = t - (int)divide((uint32_t)t, a.block) * a.block_size;
        int block = pages.block[h];
        if ((uint32_t)block >= (uint32_t)a.blocks) {
          block = 0;
          tile.partial = true;
          tile.seen &= h ? 0x0f : 0xf0;
        }
        run[h] = key_base + (block * a.key.block_stride + in_block * a.key.slot_stride);
        run[2 + h] = value_base + (block * a.value.block_stride + in_block * a.value.slot_stride);
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const auto bytes = rows_at(run[r], any);
#pragma unroll
        for (int i = 0; i < RUN_LOADS; ++i) fetch<READ_ONCE>(tile.piece[r][i], bytes, lane * 16, 0, 1024 * i);
      }
      const int r = n >> 2;
      const char* end = (r & 2 ? (r & 1 ? run[3] : run[2]) : (r & 1 ? run[1] : run[0])) + RUN_LOADS * 1024 + (n & 3) * 16;
      typedef __attribute__((ext_vector_type(4))) uint32_t piece_t;
      typedef piece_t __attribute__((aligned(4))) stored_piece;
      const piece_t w = *reinterpret_cast<const stored_piece*>(end);
#pragma unroll
      for (int i = 0; i < 4; ++i) tile.last[i] = w[i];
    } else if constexpr (PAGE16) {
      // addresses are the page's, the same for the wave, and 32 bits that do not change from tile to tile
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int t = t0 + 16 * h;
        const int in_block = t - (int)divide((uint32_t)t, a.block) * a.block_size;
        int block = pages.block[h];
        if ((uint32_t)block >= (uint32_t)a.blocks) {
          block = 0;
          tile.partial = true;
          tile.seen &= h ? 0x0f : 0xf0;
        }
        const auto kb = rows_at(key_base + (block * a.key.block_stride + in_block * a.key.slot_stride), any);
        const auto vb = rows_at(value_base + (block * a.value.block_stride + in_block * a.value.slot_stride), any);
        const uint32_t ks = (uint32_t)a.key.slot_stride, vs = (uint32_t)a.value.slot_stride;
#pragma unroll
        for (int i = 0; i < KP; ++i) fetch<KEY_AUX>(tile.k[h][i], kb, key_rows + (FULL ? 0 : key_piece(i)), 0, FULL ? 32 * i * EL : 0);
        if (ROWS8) {
#pragma unroll
          for (int j = 0; j < 4; ++j) tile.k_pair[4 * h + j] = __builtin_amdgcn_raw_buffer_load_b32(kb, 4 * g * ks, j * ks, 0);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
#pragma unroll
          for (int c = 0; c < HALVES; ++c) fetch<VALUE_AUX>(tile.v[c][4 * h + j], vb, value_rows + (FULL ? 0 : value_piece(c)), j * vs, FULL ? 128 * c * EL : 0);
          if (ROWS8) tile.v_pair[4 * h + j] = __builtin_amdgcn_raw_buffer_load_b32(vb, 4 * g * vs, j * vs, 0);
        }
      }
    } else {
      // lane i finds where the row of token i is, and lanes fetch it from there
      const int t = t0 + (lane & 31);
      const int in_block = t - (int)divide((uint32_t)t, a.block) * a.block_size;
      int block = pages.block[0];
      const bool bad = (uint32_t)block >= (uint32_t)a.blocks;
      if (bad) block = 0;
      const uint32_t bads = (uint32_t)__builtin_amdgcn_ballot_w64(bad);
      if (bads) tile.partial = true;
      const uint64_t kt = (uint64_t)(key_base + (block * a.key.block_stride + in_block * a.key.slot_stride));
      const uint64_t vt = (uint64_t)(value_base + (block * a.value.block_stride + in_block * a.value.slot_stride));
      const auto row = [&](uint64_t v, int src) {
        return reinterpret_cast<const char*>((uint64_t)__shfl((uint32_t)v, src, 64) | ((uint64_t)__shfl((uint32_t)(v >> 32), src, 64) << 32));
      };
      // lanes 16 h + n of either half of the wave have the rows of tokens 16 h + n
      const auto low = __builtin_amdgcn_permlane16_swap((uint32_t)kt, (uint32_t)kt, false, false);
      const auto high = __builtin_amdgcn_permlane16_swap((uint32_t)(kt >> 32), (uint32_t)(kt >> 32), false, false);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const char* p = reinterpret_cast<const char*>((uint64_t)low[h] | ((uint64_t)high[h] << 32)) + key_lane;
#pragma unroll
        for (int i = 0; i < KP; ++i) key(tile, h, i, p + (int32_t)key_piece(i));
      }
      const bool fours = a.block_size % 4 == 0; // four tokens in a row share a page: the first one's row is enough
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const char *kr = nullptr, *vr;
        if (fours) {
          if (ROWS8) kr = row(kt, token_of(j & 4)) + (j & 3) * a.key.slot_stride;
          vr = row(vt, token_of(j & 4)) + (j & 3) * a.value.slot_stride;
        } else {
          if (ROWS8) kr = row(kt, token_of(j));
          vr = row(vt, token_of(j));
        }
        if ((bads >> token_of(j)) & 1) tile.seen &= ~(1u << j);
#pragma unroll
        for (int c = 0; c < HALVES; ++c) value(tile, c, j, vr + value_lane + value_piece(c));
        if (ROWS8) {
          tile.k_pair[j] = *reinterpret_cast<const uint32_t*>(kr);
          tile.v_pair[j] = *reinterpret_cast<const uint32_t*>(vr);
        }
      }
    }
    if (tile.partial) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int t = t0 + token_of(j);
        if (t < span.lo || t >= span.end) tile.seen &= ~(1u << j);
      }
    }
  }

  // the running sums of 16 queries: query n is this lane's
  uint4 q[KP];
  float q_sum;
  f32x4 acc[HALVES][VC];
  float m, l, bias;

  __device__ __forceinline__ void begin(int32_t request, int head, int q0, int rows) {
    q_sum = 0.0f;
#pragma unroll
    for (int c = 0; c < KP; ++c) {
      q[c] = make_uint4(0, 0, 0, 0);
      const int d = 32 * c + 8 * g;
      if (n < rows && d < a.dim)
        q[c] = *reinterpret_cast<const uint4*>(a.query + request * a.query_request_stride + (int64_t)(head * a.group + q0 + n) * a.query_head_stride + d * 2);
      if (ROWS8) {
        const uint32_t w[4] = {q[c].x, q[c].y, q[c].z, q[c].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) q_sum += unpack16<BF16>(w[i], 0) + unpack16<BF16>(w[i], 1);
      }
    }
    if (ROWS8) {
      q_sum += __shfl_xor(q_sum, 16, 64);
      q_sum += __shfl_xor(q_sum, 32, 64);
    }
#pragma unroll
    for (int h = 0; h < HALVES; ++h)
#pragma unroll
      for (int i = 0; i < VC; ++i) acc[h][i] = f32x4{0, 0, 0, 0};
    m = -__builtin_inff();
    l = bias = 0.0f;
  }

  // PACKED: a lane's part of the runs, through LDS, where no other wave looks. Lanes read what others wrote: that the wave's
  // writes and reads keep their order is said to the compiler, for which the addresses of one lane have nothing to do with each other
  static __device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  }
  __device__ __forceinline__ void unpack(const Tile& loaded, Rows& rows) const {
    typedef __attribute__((ext_vector_type(4))) uint32_t piece_t;
    if constexpr (PACKED) {
      wave_sync(); // the last tile's reads, these writes
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int i = 0; i < RUN_LOADS; ++i) {
          const auto& w = loaded.piece[r][i];
          *reinterpret_cast<piece_t*>(stage + r * RUN + 1024 * i + lane * 16) = piece_t{w[0], w[1], w[2], w[3]};
        }
      if (lane < 16)
        *reinterpret_cast<piece_t*>(stage + (n >> 2) * RUN + RUN_LOADS * 1024 + (n & 3) * 16) = piece_t{loaded.last[0], loaded.last[1], loaded.last[2], loaded.last[3]};
      wave_sync();
      constexpr int ROW = DP * EL + HEAD;
      const char *keys = stage, *values = stage + 2 * RUN;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < KP; ++i)
#pragma unroll
          for (int r = 0; r < KREGS; ++r) rows.k[h][i][r] = *reinterpret_cast<const uint32_t*>(keys + (16 * h + n) * ROW + HEAD + 32 * i + 8 * g + 4 * r);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        rows.k_pair[j] = *reinterpret_cast<const uint32_t*>(keys + token_of(j) * ROW);
        rows.v_pair[j] = *reinterpret_cast<const uint32_t*>(values + token_of(j) * ROW);
#pragma unroll
        for (int h = 0; h < HALVES; ++h)
#pragma unroll
          for (int r = 0; r < VREGS; ++r) rows.v[h][j][r] = *reinterpret_cast<const uint32_t*>(values + token_of(j) * ROW + HEAD + 128 * h + n * VC + 4 * r);
      }
    }
  }

  __device__ __forceinline__ void add(Tile& loaded) {
    if constexpr (PACKED) {
      Rows rows;
      unpack(loaded, rows);
      add_rows(rows, loaded.partial, loaded.seen);
    } else {
      add_rows(loaded, loaded.partial, loaded.seen);
    }
  }

  __device__ __forceinline__ void add_rows(Rows& tile, bool partial, uint32_t seen) {
    // ---- scores ----
    float s[8];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      f32x4 r = {0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < KP; ++i) {
        const auto& k = tile.k[h][i];
        if constexpr (ROWS8) r = product<BF16>(widen<BF16>(k[0], k[1]), q[i], r);
        else r = product<BF16>(make_uint4(k[0], k[1], k[2], k[3]), q[i], r);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float y = r[j];
        if (ROWS8) y = __builtin_fmaf(half_at(tile.k_pair[4 * h + j], 0), y, (BF16 ? half_at(tile.k_pair[4 * h + j], 1) : middle(tile.k_pair[4 * h + j])) * q_sum);
        s[4 * h + j] = y * a.scale;
      }
    }
    // cap tanh(s / cap): small scores as s times tanh(x) / x, off by some 2^-22 of themselves, not of the cap, which may be
    // any number. (131 requests of 12 heads, cap 30: 69.2 -> 70.2 us. With the two forms in branches of their own registers spill.)
    if (a.softcap > 0.0f) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float x = s[j] * a.cap_inverse;
        s[j] = __builtin_fabsf(x) < TANH_SMALL ? s[j] * tanh_ratio(x) : a.softcap * tanh_fast(x);
      }
    }
    if (partial) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t keep = (uint32_t)((int32_t)(seen << (31 - j)) >> 31); // all bits or none
        s[j] = keep ? s[j] : -__builtin_inff();
        // what a row without a token holds may be anything: its weight of 0 would not hide it
        if (ROWS8) {
          tile.v_pair[j] &= keep;
        } else {
#pragma unroll
          for (int h = 0; h < HALVES; ++h)
#pragma unroll
            for (int r = 0; r < VREGS; ++r) tile.v[h][j][r] &= keep;
        }
      }
    }
    // ---- running maximum and sum ----
    float most = s[0];
#pragma unroll
    for (int j = 1; j < 8; ++j) most = __builtin_fmaxf(most, s[j]);
    most = group_max(most);
    if (__builtin_amdgcn_ballot_w64(most > m)) {
      const float now = __builtin_fmaxf(m, most);
      const float f = m == now ? 1.0f : exp2_fast(m - now); // m = -inf: 0
      m = now;
      l *= f;
      bias *= f;
#pragma unroll
      for (int h = 0; h < HALVES; ++h)
#pragma unroll
        for (int i = 0; i < VC; ++i) acc[h][i] *= f;
    }
    const float ref = m == -__builtin_inff() ? 0.0f : m - SHIFT; // nothing seen yet: all weights 0
    float p[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      p[j] = exp2_fast(s[j] - ref);
      l += p[j];
    }
    if (ROWS8) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        bias = __builtin_fmaf(p[j], middle(tile.v_pair[j]), bias);
        p[j] *= half_at(tile.v_pair[j], 0);
      }
    }
    uint4 hi, lo;
    split<PBF16>(p, hi, lo);
    // ---- values ----
    if constexpr (ROWS8) {
#pragma unroll
      for (int h = 0; h < HALVES; ++h)
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
          for (int r = 0; r < VREGS; ++r) tile.v[h][j][r] = centre(tile.v[h][j][r]);
    }
#pragma unroll
    for (int h = 0; h < HALVES; ++h)
#pragma unroll
      for (int i = 0; i < VC; ++i) {
        uint32_t t[4]; // column i of tokens 2 j, 2 j + 1
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if constexpr (ROWS8) {
            const float y0 = centred(tile.v[h][2 * j][i / 4], i % 4), y1 = centred(tile.v[h][2 * j + 1][i / 4], i % 4);
            t[j] = __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, y1), __builtin_bit_cast(uint32_t, y0), 0x07060302u);
          } else {
            t[j] = __builtin_amdgcn_perm(tile.v[h][2 * j + 1][i / 2], tile.v[h][2 * j][i / 2], i & 1 ? 0x07060302u : 0x05040100u);
          }
        }
        const uint4 col = make_uint4(t[0], t[1], t[2], t[3]);
        acc[h][i] = product<PBF16>(col, hi, acc[h][i]);
        acc[h][i] = product<PBF16>(col, lo, acc[h][i]);
      }
  }

  // Tiles first, first + STEP, ... up to last. The rows of the DEPTH next ones are on their way while one is added, and the pages of
  // the one behind these are being looked up. There is no branch around the loads: behind the last tile they load nothing
  // (PAGE16) or that tile again, out of the caches. Where two ways met the compiler would wait for the rows of all
  // tiles, and the loads ahead would be none
  int first, last;
  __device__ __forceinline__ void run() {
    if (first > last) return;
    Tile ring[DEPTH + 1];
    const auto clamped = [&](int t) { return t < last ? t : last; };
    Pages p = pages(first);
#pragma unroll
    for (int k = 0; k < DEPTH; ++k) {
      const Pages after = pages(clamped(first + (k + 1) * ATT_STEP));
      load(ring[k], clamped(first + k * ATT_STEP), p, first + k * ATT_STEP <= last);
      p = after;
    }
    for (int t = first;;) {
#pragma unroll
      for (int k = 0; k <= DEPTH; ++k) {
        const int ahead = t + DEPTH * ATT_STEP;
        const Pages after = pages(clamped(ahead + ATT_STEP)); // in front of the rows' loads: waiting for it is not waiting for them
        load(ring[(k + DEPTH) % (DEPTH + 1)], clamped(ahead), p, ahead <= last);
        p = after;
        add(ring[k]);
        t += ATT_STEP;
        if (t > last) return;
      }
    }
  }
};

// Four columns of a row of sums, as they come
struct Sums {
  float m, l;
  f32x4 y;
  __device__ __forceinline__ void add(float om, float ol, f32x4 oy) {
    const float now = __builtin_fmaxf(m, om);
    const float f = m == -__builtin_inff() ? 0.0f : exp2_fast(m - now), of = om == -__builtin_inff() ? 0.0f : exp2_fast(om - now);
    m = now;
    l = l * f + ol * of;
    y = y * f + oy * of;
  }
};

template <bool BF16>
__device__ __forceinline__ void write_out(const AttentionArgs& a, int64_t at, int d, const Sums& s, float shift) {
  const float f = s.l == 0.0f ? 0.0f : 1.0f / s.l; // nothing seen
  uint32_t* o = reinterpret_cast<uint32_t*>(a.out + (at * a.dim + d) * 2);
  o[0] = pack16<BF16>(s.y[0] * f, s.y[1] * f);
  o[1] = pack16<BF16>(s.y[2] * f, s.y[3] * f);
  if (d == 0) a.lse[at] = s.l == 0.0f ? -__builtin_inff() : (s.m - shift + __builtin_amdgcn_logf(s.l)) * (1.0f / ATT_LOG2E);
}

template <bool BF16, bool ROWS8, int DP, bool FULL, bool PAGE16, bool PACKED>
__global__ __launch_bounds__(64 * ATT_WAVES, attention_residents(DP)) void paged_attention_kernel(const AttentionArgs a) {
  using A = Attention<BF16, ROWS8, DP, FULL, PAGE16, PACKED>;
  constexpr int THREADS = 64 * ATT_WAVES;
  __shared__ __attribute__((aligned(16))) float s_acc[ATT_WAVES][ATTENTION_ROWS][DP + 4];
  __shared__ float s_ml[ATT_WAVES][ATTENTION_ROWS][2];
  __shared__ __attribute__((aligned(16))) char s_stage[ATT_WAVES][A::STAGE];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t worker = blockIdx.x;

  // ---- the worker's units: of a pair one for itself, then its steps (every wave finds them by itself: lengths come out of L2) ----
  const uint32_t sets = (uint32_t)(a.kv_heads * a.q_tiles);
  const auto units_of = [&](int32_t b) { return b < a.requests ? (uint32_t)span_of(a, b).steps + 1 : 0u; };
  const uint32_t sum_first = inclusive_sum(units_of(lane), lane); // of the first 64 requests: often all there are
  uint32_t total = 0;
  for (int32_t b = 64 + lane; b < a.requests; b += 64) total += units_of(b);
  total = __builtin_amdgcn_readlane(sum_first, 63) + (a.requests > 64 ? __builtin_amdgcn_readlane(inclusive_sum(total, lane), 63) : 0u);
  const uint32_t U = total * sets;
  const uint32_t W = U < (uint32_t)a.workers ? U : (uint32_t)a.workers; // each has a unit at least
  if (tid == 0) a.joins[worker] = make_int4(-1, 0, 0, 0);
  if (worker >= W) return;
  const Shares shares(U, W);
  uint32_t unit = shares.begin(worker);
  const uint32_t unit_end = shares.begin(worker + 1);
  // the request that holds the first one: the first whose inclusive sum is above unit / sets
  int32_t request = 0;
  uint32_t before = 0; // units (without sets) of the requests before it
  const uint32_t want = unit / sets;
  for (uint32_t sum = sum_first;; sum = inclusive_sum(units_of(request + lane), lane)) {
    const uint64_t above = __builtin_amdgcn_ballot_w64(before + sum > want);
    if (above) {
      const int i = __builtin_ctzll(above);
      if (i > 0) before += __builtin_amdgcn_readlane(sum, i - 1);
      request += i;
      break;
    }
    before += __builtin_amdgcn_readlane(sum, 63);
    request += 64;
  }

  // ---- segment after segment: steps c0 .. c1 - 1 of one pair (request, key head with its tile of queries) ----
  struct Segment {
    int64_t row; // of the output: its first query
    uint32_t c0, c1, steps, first; // first: the unit of the pair's first step
    int rows;
  };
  A x(a, lane, s_stage[wave]);
  const auto set_up = [&]() {
    Segment s;
    x.span = span_of(a, request);
    const uint32_t units = (uint32_t)x.span.steps + 1, in_request = unit - before * sets;
    const uint32_t set = in_request / units, u0 = in_request - set * units;
    const uint32_t u1 = unit_end - unit < units - u0 ? u0 + (unit_end - unit) : units;
    s.steps = (uint32_t)x.span.steps;
    s.c0 = u0 > 0 ? u0 - 1 : 0;
    s.c1 = u1 - 1; // none, where the pair's own unit is all that is left for this worker
    s.first = unit - u0 + 1;
    const int head = (int)(set / (uint32_t)a.q_tiles), q0 = ((int)set - head * a.q_tiles) * ATTENTION_ROWS;
    s.rows = a.group - q0 < ATTENTION_ROWS ? a.group - q0 : ATTENTION_ROWS;
    s.row = request * (int64_t)(a.kv_heads * a.group) + head * a.group + q0;
    x.key_base = a.key.base + head * a.key.head_stride;
    x.value_base = a.value.base + head * a.value.head_stride;
    x.table = a.tables + request * a.table_stride;
    x.first_column = (int)divide((uint32_t)x.span.lo, a.block);
    x.last_column = x.span.end > 0 ? (int)divide((uint32_t)(x.span.end - 1), a.block) : 0;
    // this wave's tiles: one of each step, as long as there are tokens
    x.first = x.span.base + (int)s.c0 * ATT_STEP + wave * ATT_TILE;
    x.last = x.first + (int)(s.c1 - s.c0 - 1) * ATT_STEP;
    if (x.last >= x.span.end) x.last -= ATT_STEP;
    x.begin(request, head, q0, s.rows);
    unit += u1 - u0;
    if (u1 == units && set == sets - 1) {
      before += units;
      ++request;
    }
    return s;
  };
  while (unit < unit_end) {
    const Segment s = set_up();
    if (s.c1 == s.c0) return;
    x.run();
    // ---- the four waves' sums, joined ----
    const int n = x.n, g = x.g;
    x.l += __shfl_xor(x.l, 16, 64);
    x.l += __shfl_xor(x.l, 32, 64);
    if (ROWS8) {
      x.bias += __shfl_xor(x.bias, 16, 64);
      x.bias += __shfl_xor(x.bias, 32, 64);
    }
    if (g == 0) {
      s_ml[wave][n][0] = x.m;
      s_ml[wave][n][1] = x.l;
    }
#pragma unroll
    for (int h = 0; h < A::HALVES; ++h)
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int i = 0; i < A::VC; ++i) s_acc[wave][n][h * 128 + (4 * g + r) * A::VC + i] = x.acc[h][i][r] + x.bias;
    const bool whole = s.c0 == 0 && s.c1 == s.steps;
    __syncthreads();
    const auto each_four = [&](auto&& f) { // f(query, first of four columns)
      for (int i = tid; i < s.rows * (DP / 4); i += THREADS) {
        const int row = i / (DP / 4), d = 4 * (i - row * (DP / 4));
        if (FULL || d < a.dim) f(row, d);
      }
    };
    each_four([&](int row, int d) {
      Sums sum{-__builtin_inff(), 0.0f, {0, 0, 0, 0}};
#pragma unroll
      for (int w = 0; w < ATT_WAVES; ++w) sum.add(s_ml[w][row][0], s_ml[w][row][1], *reinterpret_cast<const f32x4*>(&s_acc[w][row][d]));
      if (whole) {
        write_out<BF16>(a, s.row + row, d, sum, A::SHIFT);
      } else { // a worker's two places: the second for a pair that begins with it
        const int64_t at = ((int64_t)worker * 2 + (s.c0 == 0 ? 1 : 0)) * ATTENTION_ROWS + row;
        *reinterpret_cast<f32x4*>(&a.partial[at * a.dim + d]) = sum.y;
        if (d == 0) {
          a.partial_ml[at * 2] = sum.m;
          a.partial_ml[at * 2 + 1] = sum.l;
        }
      }
    });
    if (!whole && s.c0 == 0 && tid == 0) a.joins[worker] = make_int4((int)shares.worker_of(s.first + s.steps - 1), s.rows, (int)s.row, (int)(s.row >> 32));
    __syncthreads();
  }
}

// Where a pair begins with a worker and goes on with others, their sums are added up. A workgroup has 256 / DP of its
// rows: a thread four columns of one and every fourth worker, sixteen of them at a time where there are many: rounds of
// loads are what it takes, not bytes (64 workers a pair, 8 rows of 128: 11.2 us in rounds of eight).
template <bool BF16, int DP>
__global__ __launch_bounds__(256) void paged_attention_join_kernel(const AttentionArgs a, const int groups, const float shift) {
  constexpr int COLUMNS = DP / 4, ROWS = 64 / COLUMNS, SLICES = 4;
  __shared__ Sums s_sums[SLICES][64];
  const int worker = blockIdx.x / groups, group = blockIdx.x - worker * groups;
  const int4 join = a.joins[worker];
  const int place = threadIdx.x & 63, slice = threadIdx.x >> 6;
  const int row = group * ROWS + place / COLUMNS, d = 4 * (place % COLUMNS);
  if (join.x < 0 || group * ROWS >= join.y) return; // the whole workgroup
  const bool mine = row < join.y && d < a.dim;
  const int parts = join.x - worker + 1;
  Sums sum{-__builtin_inff(), 0.0f, {0, 0, 0, 0}};
  const auto add_all = [&](auto at_once) {
    constexpr int AT_ONCE = decltype(at_once)::value;
    for (int k0 = slice; k0 < parts; k0 += SLICES * AT_ONCE) {
      float m[AT_ONCE], l[AT_ONCE];
      f32x4 y[AT_ONCE];
#pragma unroll
      for (int i = 0; i < AT_ONCE; ++i) {
        const int k = k0 + SLICES * i < parts ? k0 + SLICES * i : k0;
        const int64_t at = ((int64_t)(worker + k) * 2 + (k == 0 ? 1 : 0)) * ATTENTION_ROWS + row;
        m[i] = a.partial_ml[at * 2];
        l[i] = a.partial_ml[at * 2 + 1];
        y[i] = *reinterpret_cast<const f32x4*>(&a.partial[at * a.dim + d]);
      }
#pragma unroll
      for (int i = 0; i < AT_ONCE; ++i)
        if (k0 + SLICES * i < parts) sum.add(m[i], l[i], y[i]);
    }
  };
  if (mine) {
    if (parts <= 2 * SLICES) add_all(std::integral_constant<int, 2>());
    else add_all(std::integral_constant<int, 16>());
  }
  s_sums[slice][place] = sum;
  __syncthreads();
  if (slice || !mine) return;
#pragma unroll
  for (int i = 1; i < SLICES; ++i) sum.add(s_sums[i][place].m, s_sums[i][place].l, s_sums[i][place].y);
  const int64_t first = (int64_t)(uint32_t)join.z | ((int64_t)join.w << 32);
  write_out<BF16>(a, first + row, d, sum, shift);
}

template <bool BF16, bool ROWS8, int DP, bool FULL>
void launch_kernel(const AttentionArgs& a, hipStream_t stream) {
  const dim3 grid(a.workers), block(64 * ATT_WAVES);
  if (a.block_size % 16) {
    paged_attention_kernel<BF16, ROWS8, DP, FULL, false, false><<<grid, block, 0, stream>>>(a);
    return;
  }
  if constexpr (ROWS8 && FULL) {
    if (a.key.slot_stride == DP + 4 && a.value.slot_stride == DP + 4) {
      paged_attention_kernel<BF16, ROWS8, DP, FULL, true, true><<<grid, block, 0, stream>>>(a);
      return;
    }
  }
  paged_attention_kernel<BF16, ROWS8, DP, FULL, true, false><<<grid, block, 0, stream>>>(a);
}

template <bool BF16, bool ROWS8, int DP>
hipError_t launch_dp(const AttentionArgs& a, hipStream_t stream) {
  if (a.dim == DP) launch_kernel<BF16, ROWS8, DP, true>(a, stream);
  else launch_kernel<BF16, ROWS8, DP, false>(a, stream);
  if (hipError_t e = hipGetLastError()) return e;
  if (a.max_tokens <= ATT_STEP - 15) return hipSuccess; // a pair is one step: nobody shares it
  const int rows = a.group < ATTENTION_ROWS ? a.group : ATTENTION_ROWS, groups = (rows + 256 / DP - 1) / (256 / DP);
  paged_attention_join_kernel<BF16, DP><<<a.workers * groups, 256, 0, stream>>>(a, groups, ROWS8 || BF16 ? 0.0f : 14.0f);
  return hipGetLastError();
}

template <bool BF16, bool ROWS8>
hipError_t launch_any(const AttentionArgs& a, hipStream_t stream) {
  if (a.dim <= 64) return launch_dp<BF16, ROWS8, 64>(a, stream);
  if (a.dim <= 128) return launch_dp<BF16, ROWS8, 128>(a, stream);
  return launch_dp<BF16, ROWS8, 256>(a, stream);
}

} // namespace attention
#endif

} // namespace fbgemm_amd
