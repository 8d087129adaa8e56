// Attention of one new token per request over a paged key-value cache, on the matrix cores.
//
//   s_t = scale * q . k_t  (or cap * tanh(scale / cap * q . k_t)),  lo <= t < len
//   out = sum_t exp(s_t - m) v_t / sum_t exp(s_t - m),  lse = m + log(sum_t exp(s_t - m)),  m = max_t s_t
//
// in one pass over the tokens with the running m and sum, all in fp32 (exp as exp2 of s * log2 e).
//
// Bound by memory: every row of the cache is read once for all the queries that share its head.
// That the rows need no staging in LDS, no transposition through it and no exchange between lanes
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
// 8-bit rows (fp16 scale a_t and bias b_t in front): s_t = a_t (q . k8_t) + b_t sum(q), and weights
// p_t a_t for the bytes, p_t b_t for the bias: 0 .. 255 are exact in bf16 and fp16.
//
// Work: units of CHUNK tokens of a (request, key head, 16 queries), numbered in that order; worker w
// of W (at most U) takes units w U / W .. (w + 1) U / W - 1, whatever requests they are of, so that all workers
// end together however long the requests are. A worker's four waves take 32 tokens each in turn and
// are joined in LDS; what a worker has whole it writes out, of what it shares with its neighbours (its
// first and its last pair) it leaves the sums, which a second launch joins in order.
#pragma once
#include "decode.h"

namespace fbgemm_amd {

constexpr int ATT_WAVES = 4;
constexpr int ATT_TILE = 32; // tokens of a wave's step
constexpr int ATT_CHUNK = ATT_WAVES * ATT_TILE;
static_assert(ATT_CHUNK == ATTENTION_CHUNK, "");
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

// 8 bytes -> 8 numbers of 16 bits, exactly
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
      const f16x2 off = {(_Float16)1024.0f, (_Float16)1024.0f};
      r[i] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, v) - off);
    }
  }
  return make_uint4(r[0], r[1], r[2], r[3]);
}

__device__ __forceinline__ float half_at(uint32_t pair, int i) { return (float)__builtin_bit_cast(f16x2, pair)[i]; }
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// n tokens of a request from `lo` on, in units of CHUNK from `base` on
struct Span {
  int32_t base, lo, end, units;
};
__device__ __forceinline__ Span span_of(const AttentionArgs& a, int64_t request) {
  int64_t len = a.idx64 ? reinterpret_cast<const int64_t*>(a.lengths)[request] : (int64_t) reinterpret_cast<const int32_t*>(a.lengths)[request];
  len = len < 0 ? 0 : len > a.max_tokens ? a.max_tokens : len;
  Span s;
  s.end = (int32_t)len;
  s.lo = a.window > 0 && len > a.window ? (int32_t)(len - a.window) : 0;
  s.base = s.lo & ~15;
  const int32_t n = (s.end - s.base + ATT_CHUNK - 1) / ATT_CHUNK;
  s.units = n > 0 ? n : 1; // an empty one is somebody's too: its result is zeros
  return s;
}

__device__ __forceinline__ int64_t wave_sum(int64_t v) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t lo = __shfl_xor((uint32_t)v, d, 64), hi = __shfl_xor((uint32_t)((uint64_t)v >> 32), d, 64);
    v += (int64_t)(((uint64_t)hi << 32) | lo);
  }
  return v;
}

// ROWS8: rows of the 8-bit format. DP: columns the code is laid out for (dim <= DP). PAGE16: pages are
// whole 16-token tiles, whose addresses are then the same for the wave.
template <bool BF16, bool ROWS8, int DP, bool PAGE16>
__global__ __launch_bounds__(64 * ATT_WAVES, DP > 128 ? 1 : 2) void paged_attention_kernel(const AttentionArgs a) {
  constexpr int KP = DP / 32;                   // products of a key tile
  constexpr int VP = DP / 16;                   // columns of a lane in the value products
  constexpr int HALVES = VP > 8 ? 2 : 1;        // pieces of at most 8 columns
  constexpr int VC = VP / HALVES;               // columns of a piece: 8, or 4 of DP = 64
  constexpr int EL = ROWS8 ? 1 : 2;             // bytes of an element
  constexpr int HEAD = ROWS8 ? 4 : 0;           // of a row, in front of its elements
  constexpr bool PBF16 = ROWS8 ? true : BF16;   // type of the weights: scales go into them, so 8-bit rows take bf16's range
  constexpr float SHIFT = PBF16 ? 0.0f : 14.0f; // weights are 2^SHIFT times larger
  constexpr int VREGS = ROWS8 ? (VC + 3) / 4 : VC / 2; // registers of a piece
  __shared__ float s_acc[ATT_WAVES][ATTENTION_ROWS][DP + 4];
  __shared__ float s_ml[ATT_WAVES][ATTENTION_ROWS][2];
  __shared__ int64_t s_scan[64 * ATT_WAVES];
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int worker = blockIdx.x;

  // ---- the worker's units ----
  const int64_t sets = (int64_t)a.kv_heads * a.q_tiles;
  int64_t total = 0;
  for (int64_t b = tid; b < a.requests; b += 64 * ATT_WAVES) total += span_of(a, b).units;
  total = wave_sum(total);
  if (lane == 0) s_scan[wave] = total;
  __syncthreads();
  total = 0;
#pragma unroll
  for (int w = 0; w < ATT_WAVES; ++w) total += s_scan[w];
  __syncthreads();
  const int64_t U = total * sets;
  const int64_t W = U < a.workers ? U : a.workers; // each has a unit at least
  if (tid == 0) a.joins[worker] = make_int4(-1, 0, 0, 0);
  if (worker >= W) return;
  int64_t unit = (int64_t)worker * U / W;
  const int64_t unit_end = (int64_t)(worker + 1) * U / W;
  // the request that holds the first one: the last whose sum of units before it is not above unit / sets
  int64_t request = 0, before = 0; // units (without sets) of the requests before it
  for (int64_t b0 = 0;; b0 += 64 * ATT_WAVES) {
    const int64_t b = b0 + tid;
    int64_t sum = b < a.requests ? span_of(a, b).units : 0;
    s_scan[tid] = sum;
    __syncthreads();
    for (int d = 1; d < 64 * ATT_WAVES; d <<= 1) {
      const int64_t other = tid >= d ? s_scan[tid - d] : 0;
      __syncthreads();
      sum += other;
      s_scan[tid] = sum;
      __syncthreads();
    }
    const int64_t want = unit / sets - before;
    if (want < s_scan[64 * ATT_WAVES - 1]) {
      int lo = 0, hi = 64 * ATT_WAVES - 1; // the first whose inclusive sum is above
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (s_scan[mid] > want) hi = mid;
        else lo = mid + 1;
      }
      request = b0 + lo;
      before += lo ? s_scan[lo - 1] : 0;
      break;
    }
    before += s_scan[64 * ATT_WAVES - 1];
    __syncthreads();
  }
  request = __builtin_amdgcn_readfirstlane((int)request);

  // ---- segment after segment: units of one (request, key head, tile of queries) ----
  while (unit < unit_end) {
    const Span span = span_of(a, request);
    const int64_t in_request = unit - before * sets;
    const int set = (int)(in_request / span.units);
    const int c0 = (int)(in_request - (int64_t)set * span.units);
    const int64_t left = unit_end - unit;
    const int c1 = left < span.units - c0 ? c0 + (int)left : span.units;
    const int head = set / a.q_tiles, q0 = (set - head * a.q_tiles) * ATTENTION_ROWS;
    const int rows = a.group - q0 < ATTENTION_ROWS ? a.group - q0 : ATTENTION_ROWS;

    // queries: lane (n, g) holds columns 32 c + 8 g .. + 7 of query n
    uint4 q[KP];
    float q_sum = 0.0f;
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
    f32x4 acc[HALVES][VC];
#pragma unroll
    for (int h = 0; h < HALVES; ++h)
#pragma unroll
      for (int i = 0; i < VC; ++i) acc[h][i] = f32x4{0, 0, 0, 0};
    float m = -__builtin_inff(), l = 0.0f, bias = 0.0f;

    const char* key_base = a.key.base + head * a.key.head_stride;
    const char* value_base = a.value.base + head * a.value.head_stride;
    const int32_t* table = a.tables + request * a.table_stride;
    const int last_column = span.end > 0 ? (int)divide((uint32_t)(span.end - 1), a.block) : 0;

    for (int c = c0; c < c1; ++c) {
      const int t0 = span.base + c * ATT_CHUNK + wave * ATT_TILE;
      if (t0 >= span.end) continue;
      bool partial = t0 < span.lo || t0 + ATT_TILE > span.end;
      // ---- addresses: of keys, tokens n and 16 + n; of values, tokens 4g .. 4g+3 and 16+4g .. ----
      const char *kp[2], *vp[8];
      uint32_t seen = 0xff; // of this lane's 8 tokens
      if (PAGE16) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int t = t0 + 16 * h;
          int column = (int)divide((uint32_t)t, a.block);
          const int in_block = t - column * a.block_size;
          column = column < last_column ? column : last_column; // a tile behind the end reads rows of the last page
          int block = table[column];
          if ((uint32_t)block >= (uint32_t)a.blocks) {
            block = 0;
            partial = true;
            seen &= h ? 0x0f : 0xf0;
          }
          const char* kt = key_base + block * a.key.block_stride + in_block * a.key.slot_stride;
          const char* vt = value_base + block * a.value.block_stride + in_block * a.value.slot_stride;
          kp[h] = kt + n * a.key.slot_stride;
#pragma unroll
          for (int j = 0; j < 4; ++j) vp[4 * h + j] = vt + (4 * g + j) * a.value.slot_stride;
        }
      } else {
        // lane i (and i + 32) finds token i's page
        int t = t0 + (lane & 31);
        t = t < span.lo ? span.lo : t >= span.end ? span.end - 1 : t;
        const int column = (int)divide((uint32_t)t, a.block);
        const int in_block = t - column * a.block_size;
        int block = table[column];
        const bool bad = (uint32_t)block >= (uint32_t)a.blocks;
        if (bad) block = 0;
        const uint32_t bads = (uint32_t)__builtin_amdgcn_ballot_w64(bad);
        if (bads) partial = true;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int src = 16 * h + n;
          kp[h] = key_base + (int64_t)__shfl(block, src, 64) * a.key.block_stride + (int64_t)__shfl(in_block, src, 64) * a.key.slot_stride;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int sv = 16 * h + 4 * g + j;
            vp[4 * h + j] = value_base + (int64_t)__shfl(block, sv, 64) * a.value.block_stride + (int64_t)__shfl(in_block, sv, 64) * a.value.slot_stride;
            if ((bads >> sv) & 1) seen &= ~(1u << (4 * h + j));
          }
        }
      }
      if (partial) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int t = t0 + (j >> 2) * 16 + 4 * g + (j & 3);
          if (t < span.lo || t >= span.end) seen &= ~(1u << j);
        }
      }
      // ---- loads ----
      uint4 k[2][KP];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < KP; ++i) {
          const int d = 32 * i + 8 * g;
          k[h][i] = make_uint4(0, 0, 0, 0);
          if (d < a.dim) {
            if (ROWS8) {
              const uint32_t* p = reinterpret_cast<const uint32_t*>(kp[h] + HEAD + d);
              k[h][i] = make_uint4(p[0], p[1], 0, 0);
            } else {
              k[h][i] = *reinterpret_cast<const uint4*>(kp[h] + d * 2);
            }
          }
        }
      uint32_t v[HALVES][8][VREGS];
#pragma unroll
      for (int h = 0; h < HALVES; ++h)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int d = h * 128 + n * VC;
#pragma unroll
          for (int r = 0; r < VREGS; ++r) v[h][j][r] = 0;
          if (d < a.dim) {
            typedef __attribute__((ext_vector_type(VREGS))) uint32_t piece_t;
            typedef piece_t __attribute__((aligned(4))) loose_t; // 8-bit rows begin on 4 bytes
            const piece_t w = ROWS8 ? *reinterpret_cast<const loose_t*>(vp[j] + HEAD + d * EL) : *reinterpret_cast<const piece_t*>(vp[j] + d * EL);
#pragma unroll
            for (int r = 0; r < VREGS; ++r) v[h][j][r] = w[r];
          }
        }
      uint32_t k_pair[8], v_pair[8];
      if (ROWS8) {
        const char* kt[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (PAGE16) kt[h] = kp[h] + (4 * g - n) * a.key.slot_stride;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (PAGE16) {
              k_pair[4 * h + j] = *reinterpret_cast<const uint32_t*>(kt[h] + j * a.key.slot_stride);
            } else { // lane 4g + j holds the row of token 4g + j
              const uint64_t at = reinterpret_cast<uint64_t>(kp[h]);
              const uint32_t lo = __shfl((uint32_t)at, 4 * g + j, 64), hi = __shfl((uint32_t)(at >> 32), 4 * g + j, 64);
              k_pair[4 * h + j] = *reinterpret_cast<const uint32_t*>(((uint64_t)hi << 32) | lo);
            }
            v_pair[4 * h + j] = *reinterpret_cast<const uint32_t*>(vp[4 * h + j]);
          }
        }
      }
      // ---- scores ----
      float s[8];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        f32x4 r = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < KP; ++i) r = product<BF16>(ROWS8 ? widen<BF16>(k[h][i].x, k[h][i].y) : k[h][i], q[i], r);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float x = r[j];
          if (ROWS8) x = __builtin_fmaf(half_at(k_pair[4 * h + j], 0), x, half_at(k_pair[4 * h + j], 1) * q_sum);
          x *= a.scale;
          if (a.softcap > 0.0f) x = a.softcap * ATT_LOG2E * tanhf(x);
          s[4 * h + j] = x;
        }
      }
      if (partial) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (!((seen >> j) & 1)) {
            s[j] = -__builtin_inff();
            if (!ROWS8) { // what a row without a token holds may be anything: its weight of 0 would not hide it
#pragma unroll
              for (int h = 0; h < HALVES; ++h)
#pragma unroll
                for (int r = 0; r < VREGS; ++r) v[h][j][r] = 0;
            }
          }
        }
      }
      // ---- running maximum and sum ----
      float most = s[0];
#pragma unroll
      for (int j = 1; j < 8; ++j) most = __builtin_fmaxf(most, s[j]);
      most = __builtin_fmaxf(most, __shfl_xor(most, 16, 64));
      most = __builtin_fmaxf(most, __shfl_xor(most, 32, 64));
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
          const bool live = !partial || ((seen >> j) & 1);
          bias += live ? p[j] * half_at(v_pair[j], 1) : 0.0f;
          p[j] = live ? p[j] * half_at(v_pair[j], 0) : 0.0f;
        }
      }
      uint4 hi, lo;
      split<PBF16>(p, hi, lo);
      // ---- values ----
#pragma unroll
      for (int h = 0; h < HALVES; ++h)
#pragma unroll
        for (int i = 0; i < VC; ++i) {
          uint32_t t[4]; // column i of tokens 2 j, 2 j + 1
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (ROWS8) {
              const float x = (float)((v[h][2 * j][i / 4] >> (i % 4 * 8)) & 0xffu), y = (float)((v[h][2 * j + 1][i / 4] >> (i % 4 * 8)) & 0xffu);
              t[j] = __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, y), __builtin_bit_cast(uint32_t, x), 0x07060302u);
            } else {
              t[j] = __builtin_amdgcn_perm(v[h][2 * j + 1][i / 2], v[h][2 * j][i / 2], i & 1 ? 0x07060302u : 0x05040100u);
            }
          }
          const uint4 col = make_uint4(t[0], t[1], t[2], t[3]);
          acc[h][i] = product<PBF16>(col, hi, acc[h][i]);
          acc[h][i] = product<PBF16>(col, lo, acc[h][i]);
        }
    }

    // ---- the four waves' sums, joined ----
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    if (ROWS8) {
      bias += __shfl_xor(bias, 16, 64);
      bias += __shfl_xor(bias, 32, 64);
    }
    if (g == 0) {
      s_ml[wave][n][0] = m;
      s_ml[wave][n][1] = l;
    }
#pragma unroll
    for (int h = 0; h < HALVES; ++h)
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int i = 0; i < VC; ++i) s_acc[wave][n][h * 128 + (4 * g + r) * VC + i] = acc[h][i][r] + bias;
    __syncthreads();
    const bool whole = c0 == 0 && c1 == span.units;
    const int slot = c0 == 0 ? 1 : 0;
    for (int i = tid; i < rows * DP; i += 64 * ATT_WAVES) {
      const int row = i / DP, d = i - row * DP;
      float M = s_ml[0][row][0];
#pragma unroll
      for (int w = 1; w < ATT_WAVES; ++w) M = __builtin_fmaxf(M, s_ml[w][row][0]);
      float L = 0.0f, x = 0.0f;
#pragma unroll
      for (int w = 0; w < ATT_WAVES; ++w) {
        const float mw = s_ml[w][row][0];
        const float f = mw == -__builtin_inff() ? 0.0f : exp2_fast(mw - M);
        L += f * s_ml[w][row][1];
        x += f * s_acc[w][row][d];
      }
      if (d >= a.dim) continue;
      const int64_t at = request * (int64_t)(a.kv_heads * a.group) + head * a.group + q0 + row;
      if (whole) {
        const float y = L == 0.0f ? 0.0f : x / L;
        char* o = a.out + (at * a.dim + d) * 2;
        *reinterpret_cast<uint16_t*>(o) = (uint16_t)pack16<BF16>(y, y);
        if (d == 0) a.lse[at] = L == 0.0f ? -__builtin_inff() : (M - SHIFT + __builtin_amdgcn_logf(L)) * (1.0f / ATT_LOG2E);
      } else {
        const int64_t part = ((int64_t)worker * 2 + slot) * ATTENTION_ROWS + row;
        a.partial[part * a.dim + d] = x;
        if (d == 0) {
          a.partial_ml[part * 2] = M;
          a.partial_ml[part * 2 + 1] = L;
        }
      }
    }
    if (c0 == 0 && c1 < span.units && tid == 0) {
      // the pair goes on with the next workers; its last unit's is the last worker whose first unit is not behind it
      const int64_t last = unit + span.units - 1;
      a.joins[worker] = make_int4((int)request, set, (int)(((last + 1) * W + U - 1) / U - 1), 0);
    }
    __syncthreads();
    unit += c1 - c0;
    if (c1 == span.units && set == (int)sets - 1) {
      before += span.units;
      ++request;
    }
  }
}

// One workgroup per (worker, query): where a pair of requests and heads begins with this worker and goes on
// with others, its sums are added up in the workers' order.
template <bool BF16>
__global__ __launch_bounds__(256) void paged_attention_join_kernel(const AttentionArgs a, const int rows_max, const float shift) {
  __shared__ float s_acc[4][256];
  __shared__ float s_l[4];
  const int worker = blockIdx.x / rows_max, row = blockIdx.x - worker * rows_max;
  const int4 join = a.joins[worker];
  if (join.x < 0) return;
  const int head = join.y / a.q_tiles, q0 = (join.y - head * a.q_tiles) * ATTENTION_ROWS;
  if (q0 + row >= a.group) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int parts = join.z - worker + 1; // this worker's second place, the others' first
  const auto place = [&](int i) { return ((int64_t)(worker + i) * 2 + (i == 0 ? 1 : 0)) * ATTENTION_ROWS + row; };
  float M = -__builtin_inff();
  for (int i = lane; i < parts; i += 64) M = __builtin_fmaxf(M, a.partial_ml[place(i) * 2]);
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) M = __builtin_fmaxf(M, __shfl_xor(M, d, 64));
  float x[4] = {0, 0, 0, 0}, L = 0.0f;
  for (int i = wave; i < parts; i += 4) {
    const int64_t at = place(i);
    const float mw = a.partial_ml[at * 2];
    const float f = mw == -__builtin_inff() ? 0.0f : exp2_fast(mw - M);
    L += f * a.partial_ml[at * 2 + 1];
#pragma unroll
    for (int c = 0; c < 4; ++c)
      if (lane + 64 * c < a.dim) x[c] += f * a.partial[at * a.dim + lane + 64 * c];
  }
#pragma unroll
  for (int c = 0; c < 4; ++c) s_acc[wave][lane + 64 * c] = x[c];
  if (lane == 0) s_l[wave] = L;
  __syncthreads();
  const int d = threadIdx.x;
  if (d >= a.dim) return;
  L = s_l[0] + s_l[1] + s_l[2] + s_l[3];
  const float y = s_acc[0][d] + s_acc[1][d] + s_acc[2][d] + s_acc[3][d];
  const int64_t at = (int64_t)join.x * (a.kv_heads * a.group) + head * a.group + q0 + row;
  const float r = L == 0.0f ? 0.0f : y / L;
  *reinterpret_cast<uint16_t*>(a.out + (at * a.dim + d) * 2) = (uint16_t)pack16<BF16>(r, r);
  if (d == 0) a.lse[at] = L == 0.0f ? -__builtin_inff() : (M - shift + __builtin_amdgcn_logf(L)) * (1.0f / ATT_LOG2E);
}

template <bool BF16, bool ROWS8, int DP>
hipError_t launch_dp(const AttentionArgs& a, hipStream_t stream) {
  if (a.block_size % 16 == 0) paged_attention_kernel<BF16, ROWS8, DP, true><<<a.workers, 64 * ATT_WAVES, 0, stream>>>(a);
  else paged_attention_kernel<BF16, ROWS8, DP, false><<<a.workers, 64 * ATT_WAVES, 0, stream>>>(a);
  if (hipError_t e = hipGetLastError()) return e;
  if (a.max_tokens <= ATT_CHUNK - 15) return hipSuccess; // every request is one unit
  const int rows = a.group < ATTENTION_ROWS ? a.group : ATTENTION_ROWS;
  paged_attention_join_kernel<BF16><<<a.workers * rows, 256, 0, stream>>>(a, rows, ROWS8 || BF16 ? 0.0f : 14.0f);
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
