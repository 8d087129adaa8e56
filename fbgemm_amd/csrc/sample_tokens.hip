// A token of every row of logits, by a given random number u in [0, 1).
//
// Tokens are put in order: larger logits first, equal ones by their number. With w = exp((x - max) / temperature)
// the ones that may be drawn are a first part of that order:
//
//   top-k    the first k
//   top-p    of those, as few as have a sum of w of at least p times the sum of all of those (one at least)
//   min-p    of those, the ones with w >= min_p
//
// and the token is the first one, by number now, where the running sum of w over what is left is above u times
// its whole. Its probability is w over that whole.
//
// A large vocabulary has a border of two tokens within 1e-6 of almost every u, so sums in fp32 would often draw a
// neighbour. w is a whole number here, 2^fraction times larger and rounded (fraction: 45 bits for
// 131 071 tokens): sums of whole numbers are the same in any order, so lanes, waves and LDS atomics add them as they come,
// and a running sum is off by no more than the w's own roundings, 2^-46 of the largest each (2^-29 if all of them went one way; u has 24 bits).
// exp is made in fp64 (2^-48).
//
// A workgroup has a row. It reads it once to keep the largest logit of every few pieces of 16 bytes, in LDS. Few of these groups
// hold a token that can matter: with top-k those whose largest is above the k-th largest of the groups' largest, without those with a
// weight that is not 0, or enough for min-p. Where a list in LDS takes the tokens of those groups, everything else is done there:
// up to SMALL of them are ranked against each other, more are counted into bins (below). Else (top-p of a flat row) the whole
// row is weighed once, a wave a run of its tokens, into bins of logits of its own, which say the bin where top-p's sum is reached
// and the run where the draw falls; only that bin's tokens and that run are looked at again.
//
// Bound by memory only where rows have little to do: 256 rows of 131 071 logits in bf16 (67 MB, 13 us at a copy's rate), us a call:
// the largest logit 23, the 50 largest 31, 200 and top-p 0.9 of those 36, min-p 0.05 28. A row with all its tokens weighs each of them,
// some 20 fp64 operations: 60, and with top-p 0.9 of a flat row, an LDS atomic for each beside that, and two more looks at parts of
// it: 89. Then it is the compute unit's issue and LDS that bound it. One row: 10.5 to 70 us, a chain of dependent steps.
//
// Finding where a count or a sum is reached, going down from the largest, by bins: of keys (fp32 bits in ascending order), then of
// the keys of the bin that has it, until they are one; then the last token of that key that is within.
#include <type_traits>

#include "decode.h"
#include "logits_piece.h"

namespace fbgemm_amd {

namespace {

typedef uint64_t u64;
constexpr float FLT_BIG = 3.4028234663852886e38f;
constexpr int BINS = 2048;

// fp32 numbers as keys in ascending order. NaN and -inf are no tokens: key 0; +inf counts as the largest finite number.
__device__ __forceinline__ uint32_t key_of(float x) {
  if (!(x > -__builtin_inff())) return 0;
  x = __builtin_fminf(x, FLT_BIG) + 0.0f; // -0 becomes 0
  const uint32_t b = __builtin_bit_cast(uint32_t, x);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float logit_of(uint32_t key) { return __builtin_bit_cast(float, key & 0x80000000u ? key ^ 0x80000000u : ~key); }

// 2^(i / 32)
constexpr int STEPS = 32;
__device__ const double ROOTS[STEPS] = {
    1.0, 1.0218971486541166, 1.0442737824274138, 1.0671404006768237,
    1.0905077326652577, 1.1143867425958924, 1.1387886347566916, 1.1637248587775775,
    1.189207115002721, 1.215247359980469, 1.241857812073484, 1.2690509571917332,
    1.2968395546510096, 1.3252366431597413, 1.3542555469368927, 1.383909881963832,
    1.4142135623730951, 1.4451808069770467, 1.4768261459394993, 1.5091644275934228,
    1.5422108254079407, 1.5759808451078865, 1.6104903319492543, 1.645755478153965,
    1.681792830507429, 1.718619298122478, 1.7562521603732995, 1.7947090750031072,
    1.8340080864093424, 1.8741676341103, 1.9152065613971474, 1.9571441241754002,
};

// exp((x - most) / temperature) in units of 2^-fraction
struct Weights {
  double most, per_logit; // per_logit: log2(e) / temperature
  int fraction;
  const double* roots;    // ROOTS, in LDS: 32 entries lie in different banks
  // x: not +inf; of NaN and -inf: 0
  __device__ __forceinline__ u64 operator()(float x) const {
    // (no branches: weights next to each other are made together)
    const double t = fmax(((double)x - most) * per_logit, -(double)(fraction + 2));
    // a sum with 1.5 * 2^47 is rounded to 32nds, and holds their number in its low bits
    constexpr double ROUND = 211106232532992.0;
    const double steps = t + ROUND, f = t - (steps - ROUND);
    const int n = (int)(uint32_t)__builtin_bit_cast(u64, steps);
    // 2^f, |f| <= 1/64, by its series: the next term is below 2^-48
    double p = 0.0013333558146428443;
    p = __builtin_fma(p, f, 0.009618129107628477);
    p = __builtin_fma(p, f, 0.0555041086648215799);
    p = __builtin_fma(p, f, 0.2402265069591007123);
    p = __builtin_fma(p, f, 0.6931471805599453094);
    const double root = roots[n & (STEPS - 1)];
    p = __builtin_fma(p * f, root, root);
    // times 2^(whole steps + fraction), in the exponent's bits (0.9 < p < 2.1, and the exponent stays that of a normal number)
    u64 bits = __builtin_bit_cast(u64, p);
    bits += (u64)(uint32_t)(((n >> 5) + fraction) << 20) << 32;
    // a double of 2^52 and more holds whole numbers: adding that rounds, and leaves the number in the low bits
    return __builtin_bit_cast(u64, __builtin_bit_cast(double, bits) + 4503599627370496.0) & 0xfffffffffffffull;
  }
};

// Running sums and maxima over a wave by its rows' permutations, which take an instruction each, not a way through LDS: over rows of 16,
// then a row's last lane into the next row, then the first half's into the second
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t moved(uint32_t v) { // 0 where nothing comes
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false);
}
template <typename T, typename F>
__device__ __forceinline__ T wave_running(T v, F&& with) {
  v = with(v, std::integral_constant<int, 0x111>(), std::integral_constant<int, 0xf>()); // row_shr 1, 2, 4, 8
  v = with(v, std::integral_constant<int, 0x112>(), std::integral_constant<int, 0xf>());
  v = with(v, std::integral_constant<int, 0x114>(), std::integral_constant<int, 0xf>());
  v = with(v, std::integral_constant<int, 0x118>(), std::integral_constant<int, 0xf>());
  v = with(v, std::integral_constant<int, 0x142>(), std::integral_constant<int, 0xa>()); // row_bcast 15 into rows 1 and 3
  return with(v, std::integral_constant<int, 0x143>(), std::integral_constant<int, 0xc>()); // row_bcast 31 into rows 2 and 3
}
__device__ __forceinline__ u64 wave_inclusive(u64 v) {
  return wave_running(v, [](u64 x, auto ctrl, auto rows) {
    return x + ((u64)moved<decltype(ctrl)::value, decltype(rows)::value>((uint32_t)x) | ((u64)moved<decltype(ctrl)::value, decltype(rows)::value>((uint32_t)(x >> 32)) << 32));
  });
}
__device__ __forceinline__ uint32_t wave_inclusive32(uint32_t v) {
  return wave_running(v, [](uint32_t x, auto ctrl, auto rows) { return x + moved<decltype(ctrl)::value, decltype(rows)::value>(x); });
}
// (readlane gives an int)
__device__ __forceinline__ uint32_t last_lane32(uint32_t v) { return (uint32_t)__builtin_amdgcn_readlane((int)v, 63); }
__device__ __forceinline__ u64 last_lane(u64 v) { return (u64)last_lane32((uint32_t)v) | ((u64)last_lane32((uint32_t)(v >> 32)) << 32); }
__device__ __forceinline__ u64 wave_sum(u64 v) { return last_lane(wave_inclusive(v)); }
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
  return last_lane32(wave_running(v, [](uint32_t x, auto ctrl, auto rows) {
    const uint32_t o = moved<decltype(ctrl)::value, decltype(rows)::value>(x);
    return x > o ? x : o;
  }));
}

// Orders of numbers of a type: keys of different ones are more than 2^GRAIN apart
template <int TY>
constexpr int GRAIN = TY == ST_FP32 ? 0 : TY == ST_BF16 ? 15 : 12;

// What may be drawn: keys above `hi`, and of those in [lo, hi], which are one, the tokens up to `last`
struct Part {
  uint32_t lo, hi;
  int32_t last;
  __device__ __forceinline__ bool has(uint32_t k, int32_t token) const { return k > hi || (k >= lo && token <= last); }
};

constexpr int GROUPS = 8192; // at most
constexpr int RUN_BINS = 512;
constexpr int FIRST_AHEAD = 8; // pieces that a thread loads together, where they come from memory

template <int THREADS>
struct alignas(16) Shared {
  static constexpr int WAVES = THREADS / 64;
  static constexpr int LIST = THREADS == 1024 ? 320 : 512; // entries of a wave's part of the list
  static constexpr int MOST_GROUPS = THREADS == 1024 ? GROUPS : 1024;
  static constexpr int SMALL = 512; // entries that are ranked
  union {
    struct {
      u64 weight[BINS];
      uint32_t count[BINS];
    };
    u64 run[WAVES][RUN_BINS]; // a run's weights, by bins of logits
    struct {
      u64 ranked[SMALL], amount[SMALL];
      uint32_t small_key[SMALL];
      int32_t small_token[SMALL], rank[SMALL];
    };
  };
  uint32_t group[MOST_GROUPS]; // the largest key of each
  uint16_t chosen[MOST_GROUPS];
  double roots[STEPS];
  u64 sums[WAVES], wave[WAVES];
  uint32_t wave32[WAVES], low32[WAVES];
  u64 found;    // an amount
  uint32_t bin; // a place
  uint32_t found_key;
  int32_t listed[WAVES];
  uint32_t key[WAVES * LIST];
  int32_t token[WAVES * LIST];
};

__device__ __forceinline__ uint32_t group_lanes_max(uint32_t v, int lanes) { // over 1, 2, 4, 8, 16 or 32 lanes
  const auto with = [&](uint32_t o) { v = v > o ? v : o; };
  if (lanes > 1) with(__builtin_amdgcn_update_dpp(0, v, 0xb1, 0xf, 0xf, true));
  if (lanes > 2) with(__builtin_amdgcn_update_dpp(0, v, 0x4e, 0xf, 0xf, true));
  if (lanes > 4) with(__builtin_amdgcn_update_dpp(0, v, 0x141, 0xf, 0xf, true));
  if (lanes > 8) with(__builtin_amdgcn_update_dpp(0, v, 0x140, 0xf, 0xf, true));
  if (lanes > 16) with(__shfl_xor(v, 16, 64));
  return v;
}

// The largest key of a piece. 16-bit numbers as whole numbers of the same order, two at a time; the order puts NaN behind infinity
// (or below its negative): a piece with one such is looked at number by number.
template <int TY>
__device__ __forceinline__ uint32_t largest_of(const Piece<TY>& p) {
  using P = Piece<TY>;
  bool nan;
  float x;
  if constexpr (TY == ST_FP32) {
    int32_t m = INT32_MIN;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int32_t b = (int32_t)p.raw[i], o = b ^ ((b >> 31) & 0x7fffffff);
      m = m > o ? m : o;
    }
    nan = m > 0x7f800000;
    x = __builtin_bit_cast(float, m ^ ((m >> 31) & 0x7fffffff));
  } else {
    typedef __attribute__((ext_vector_type(2))) int16_t pair_t;
    pair_t m = {INT16_MIN, INT16_MIN};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const pair_t b = __builtin_bit_cast(pair_t, (uint32_t)p.raw[i]);
      const uint32_t flip = __builtin_bit_cast(uint32_t, (pair_t)(b >> 15)) & 0x7fff7fffu;
      m = __builtin_elementwise_max(m, __builtin_bit_cast(pair_t, (uint32_t)p.raw[i] ^ flip));
    }
    const int16_t o = m[0] > m[1] ? m[0] : m[1];
    nan = o > (TY == ST_BF16 ? 0x7f80 : 0x7c00);
    const uint16_t b = (uint16_t)(o ^ ((o >> 15) & 0x7fff));
    x = TY == ST_BF16 ? __builtin_bit_cast(float, (uint32_t)b << 16) : (float)__builtin_bit_cast(_Float16, b);
  }
  uint32_t k = key_of(x);
  if (nan) {
    k = 0;
#pragma unroll 1
    for (int i = 0; i < P::N; ++i) {
      const uint32_t o = key_of(p.get(i));
      k = k > o ? k : o;
    }
  }
  return k;
}

// Pieces [first, first + pieces) of a row, a wave a run of `steps` times 64 of them
template <int TY, int THREADS>
struct Row {
  using P = Piece<TY>;
  static constexpr int N = P::N, WAVES = THREADS / 64;
  const char* logits;
  int32_t vocab, first, pieces;
  int steps, lane, wave;
  __device__ __forceinline__ Row(const char* row, int32_t vocab_, int32_t first_, int32_t pieces_)
      : logits(row), vocab(vocab_), first(first_), pieces(pieces_), lane(threadIdx.x & 63), wave(__builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) {
    steps = (pieces + THREADS - 1) / THREADS;
  }
  __device__ __forceinline__ Row run(int w) const { // a wave's run, for all waves
    const int32_t at = w * steps * 64, n = pieces - at;
    return Row(logits, vocab, first + at, n < 0 ? 0 : n < steps * 64 ? n : steps * 64);
  }
  // a lane's piece
  __device__ __forceinline__ int32_t piece_at(int step) const { return (wave * steps + step) * 64 + lane; }
  __device__ __forceinline__ int32_t token_at(int step) const { return (first + piece_at(step)) * N; }
  static __device__ __forceinline__ void load(P& p, const char* logits, int32_t v, int32_t vocab) {
    if (v + N <= vocab) {
      p.load(logits + (int64_t)v * P::BYTES);
    } else { // behind the end: NaN, no token
      p.raw[0] = p.raw[1] = p.raw[2] = p.raw[3] = 0xffffffffu;
      if (v < vocab) {
        const P some = [&] {
          P q;
          q.load_some(logits + (int64_t)v * P::BYTES, vocab - v);
          return q;
        }();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if constexpr (TY == ST_FP32) p.raw[i] = i < vocab - v ? some.raw[i] : 0xffffffffu;
          else p.raw[i] = (2 * i < vocab - v ? some.raw[i] & 0xffffu : 0xffffu) | (2 * i + 1 < vocab - v ? some.raw[i] & 0xffff0000u : 0xffff0000u);
        }
      }
    }
  }
  __device__ __forceinline__ void load(P& p, int step) const {
    const int32_t i = piece_at(step);
    load(p, logits, step < steps && i < pieces ? (first + i) * N : vocab, vocab);
  }
  // f(logit, its token) for those of a piece, in their order (two numbers' code: the piece is turned past them)
  template <typename F>
  static __device__ __forceinline__ void each_of(P p, int32_t v, F&& f) {
#pragma unroll 1
    for (int i = 0; i < N; i += 2) {
      f(p.get(0), v + i);
      f(p.get(1), v + i + 1);
      if constexpr (TY == ST_FP32) p.raw[0] = p.raw[2], p.raw[1] = p.raw[3];
      else p.raw[0] = p.raw[1], p.raw[1] = p.raw[2], p.raw[2] = p.raw[3];
    }
  }
  // f(piece, its first token, its number), step by step; several loads on their way, as long as all lanes have whole pieces
  // (a load that goes to a register by one of two ways is waited for where they meet)
  template <int AHEAD = 4, typename F>
  __device__ __forceinline__ void each_piece(F&& f) const {
    int whole = (vocab / N - first < pieces ? vocab / N - first : pieces) / 64 - wave * steps; // steps
    whole = __builtin_amdgcn_readfirstlane(whole < steps ? whole : steps);
    int k = 0;
    for (; k + AHEAD <= whole; k += AHEAD) {
      P x[AHEAD];
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) x[j].load(logits + (int64_t)token_at(k + j) * P::BYTES);
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) f(x[j], token_at(k + j), piece_at(k + j));
    }
    if constexpr (AHEAD > 4) {
      for (; k + 4 <= whole; k += 4) {
        P x[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j].load(logits + (int64_t)token_at(k + j) * P::BYTES);
#pragma unroll
        for (int j = 0; j < 4; ++j) f(x[j], token_at(k + j), piece_at(k + j));
      }
    }
    for (; k < steps; ++k) {
      P x;
      load(x, k);
      f(x, token_at(k), piece_at(k));
    }
  }
  // f(logit, token) for a thread's tokens (and NaN for what is none)
  template <typename F>
  __device__ __forceinline__ void each_logit(F&& f) const {
    each_piece([&](const P& p, int32_t v, int32_t) { each_of(p, v, f); });
  }
  // f(key, token) for a thread's tokens (and key 0 for what is none)
  template <typename F>
  __device__ __forceinline__ void each(F&& f) const {
    each_piece([&](const P& p, int32_t v, int32_t) { each_of(p, v, [&](float x, int32_t token) { f(key_of(x), token); }); });
  }
  template <typename F>
  __device__ __forceinline__ void each_of_step(int step, F&& f) const {
    P p;
    load(p, step);
    each_of(p, token_at(step), [&](float x, int32_t token) { f(key_of(x), token); });
  }
};

// The list: a wave's entries, in their tokens' order
template <int THREADS>
struct List {
  static constexpr int LIST = Shared<THREADS>::LIST;
  const Shared<THREADS>& s;
  int steps, lane, wave, n;
  __device__ __forceinline__ List(const Shared<THREADS>& shared) : s(shared), lane(threadIdx.x & 63), wave(__builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) {
    n = __builtin_amdgcn_readfirstlane(s.listed[wave]);
    steps = (n + 63) / 64;
  }
  template <typename F>
  __device__ __forceinline__ void each(F&& f) const {
    for (int i = lane; i < n; i += 64) f(s.key[wave * LIST + i], s.token[wave * LIST + i]);
  }
  template <typename F>
  __device__ __forceinline__ void each_of_step(int step, F&& f) const {
    const int i = step * 64 + lane;
    if (i < n) f(s.key[wave * LIST + i], s.token[wave * LIST + i]);
  }
};

// A wave puts those of its 64 pieces' tokens with lo <= logit <= hi for which also(logit) into its part of the list, behind the n that are
// there; the new n, or more than there is room for
template <int TY, int THREADS, typename F>
__device__ __forceinline__ int list_pieces(Shared<THREADS>& s, const Piece<TY>& p, int32_t v, int n, float lo, float hi, F&& also) {
  constexpr int LIST = Shared<THREADS>::LIST, N = Piece<TY>::N;
  const int wave = threadIdx.x >> 6;
  uint32_t in = 0; // few are
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const float x = p.get(e);
    in |= x >= lo && x <= hi ? 1u << e : 0u;
  }
  if (__builtin_amdgcn_ballot_w64(in != 0) == 0) return n;
  const auto at = [&](int e) {
    float x = p.get(0);
#pragma unroll
    for (int i = 1; i < N; ++i) x = e == i ? p.get(i) : x;
    return x;
  };
  for (uint32_t left = in; left; left &= left - 1) {
    const int e = __builtin_ctz(left);
    if (!also(at(e))) in &= ~(1u << e);
  }
  const int mine = __builtin_popcount(in), to = (int)wave_inclusive32((uint32_t)mine), all = (int)last_lane32((uint32_t)to);
  if (n + all > LIST) return LIST + 1;
  int place = wave * LIST + n + to - mine;
  for (; in; in &= in - 1) {
    const int e = __builtin_ctz(in);
    s.key[place] = key_of(at(e));
    s.token[place] = v + e;
    ++place;
  }
  return n + all;
}

// The first token, by number, where the running sum of amount(key, token) is above a target, which is asked for by the whole sum;
// where that is the whole or more, the last one that has an amount. One has at least.
struct Found {
  int32_t token;
  uint32_t key;
  u64 amount, whole;
};
// of `from`, by its waves' sums
template <typename Source, int THREADS, typename F>
__device__ __forceinline__ Found locate_by(const Source& from, Shared<THREADS>& s, F&& amount, u64 mine, u64 whole, u64 target) {
  int in = 0;
  u64 before = 0;
  for (; in < THREADS / 64 - 1 && before + s.sums[in] <= target; ++in) before += s.sums[in];
  if (from.wave == in) {
    for (int k = 0; k < from.steps; ++k) {
      u64 of_step = mine; // of a single step they are known
      if (from.steps > 1) {
        of_step = 0;
        from.each_of_step(k, [&](uint32_t key, int32_t v) { of_step += amount(key, v); });
      }
      const u64 to = before + wave_inclusive(of_step);
      const u64 above = __builtin_amdgcn_ballot_w64(target < to);
      if (above) {
        if (from.lane == __builtin_ctzll(above)) {
          u64 sum = to - of_step;
          bool open = true;
          from.each_of_step(k, [&](uint32_t key, int32_t v) {
            const u64 n = amount(key, v);
            sum += n;
            if (open && target < sum) {
              s.bin = (uint32_t)v;
              s.found = n;
              s.found_key = key;
              open = false;
            }
          });
        }
        break;
      }
      before = last_lane(to);
    }
  }
  __syncthreads();
  const Found r{(int32_t)s.bin, s.found_key, s.found, whole};
  __syncthreads();
  return r;
}
// the waves' sums, and their whole
template <int THREADS>
__device__ __forceinline__ u64 sum_up(Shared<THREADS>& s, u64 mine) {
  mine = wave_sum(mine);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s.sums[threadIdx.x >> 6] = mine;
  __syncthreads();
  u64 whole = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) whole += s.sums[w];
  return whole;
}
template <typename Source, int THREADS, typename F, typename T>
__device__ __forceinline__ Found locate(const Source& from, Shared<THREADS>& s, F&& amount, T&& target_of) {
  u64 mine = 0;
  from.each([&](uint32_t k, int32_t v) { mine += amount(k, v); });
  const u64 whole = sum_up(s, mine);
  const u64 target = target_of(whole);
  return locate_by(from, s, amount, mine, whole, target < whole ? target : whole - 1);
}
// of a row, by its waves' sums in s.sums: the wave's run once more, by all waves
template <int TY, int THREADS, typename F>
__device__ __forceinline__ Found locate_in_run(const Row<TY, THREADS>& row, Shared<THREADS>& s, F&& amount, u64 whole, u64 target) {
  int in = 0;
  for (; in < THREADS / 64 - 1 && s.sums[in] <= target; ++in) target -= s.sums[in];
  Found r = locate(row.run(in), s, amount, [&](u64) { return target; });
  r.whole = whole;
  return r;
}

// s.bin: the first bin where the running sum reaches `target` (asked for by the whole; none does: the last one that is not empty); s.found: the sum
// before it. The target.
template <bool WEIGHTS, int THREADS, typename T>
__device__ __forceinline__ u64 find_bin(Shared<THREADS>& s, T&& target_of) {
  constexpr int EACH = BINS / THREADS;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  u64 n[EACH], mine = 0;
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    n[i] = WEIGHTS ? s.weight[threadIdx.x * EACH + i] : (u64)s.count[threadIdx.x * EACH + i];
    mine += n[i];
  }
  const u64 to = wave_inclusive(mine);
  if (lane == 63) s.wave[wave] = to;
  __syncthreads();
  u64 before = to - mine, whole = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) {
    if (w < wave) before += s.wave[w];
    whole += s.wave[w];
  }
  u64 target = target_of(whole);
  target = target < whole ? target : whole;
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    if (before < target && before + n[i] >= target) {
      s.bin = threadIdx.x * EACH + i;
      s.found = before;
    }
    before += n[i];
  }
  __syncthreads();
  return target;
}
template <bool WEIGHTS, int THREADS>
__device__ __forceinline__ void clear_bins(Shared<THREADS>& s) {
  __syncthreads();
  for (int i = threadIdx.x; i < BINS; i += THREADS) {
    if (WEIGHTS) s.weight[i] = 0;
    else s.count[i] = 0;
  }
  __syncthreads();
}
// bins of keys from `hi` down to `lo`
__device__ __forceinline__ int shift_of(uint32_t lo, uint32_t hi) {
  const uint32_t span = hi - lo;
  return span < BINS ? 0 : 32 - __builtin_clz(span) - 11;
}

// Keys from the largest, `hi`, down to `lo`, until the sum of their amounts reaches a target (at least 1), asked for by the whole: the keys [lo,
// hi], which are one, that do it, the sum before them, the target. WEIGHTS: amounts are sums of u64, else 0 or 1.
struct Border {
  uint32_t lo, hi;
  u64 before, target;
};
template <bool WEIGHTS, int TY, typename Source, int THREADS, typename F, typename T>
__device__ __forceinline__ Border border(const Source& from, Shared<THREADS>& s, uint32_t lo, uint32_t hi, F&& amount, T&& target_of) {
  Border b{0, 0, 0, 0};
  for (bool first = true;; first = false) {
    const int shift = shift_of(lo, hi);
    clear_bins<WEIGHTS>(s);
    from.each([&](uint32_t k, int32_t v) {
      if (k < lo || k > hi) return;
      const u64 n = amount(k, v);
      if (n == 0) return;
      const uint32_t bin = (hi - k) >> shift;
      if (WEIGHTS) atomicAdd((unsigned long long*)&s.weight[bin], (unsigned long long)n);
      else atomicAdd(&s.count[bin], 1u);
    });
    __syncthreads();
    const u64 target = find_bin<WEIGHTS>(s, [&](u64 whole) { return first ? target_of(whole) : b.target - b.before; });
    if (first) b.target = target;
    const uint32_t bin = s.bin;
    b.before += s.found;
    hi -= bin << shift;
    const uint32_t width = (1u << shift) - 1;
    lo = hi - lo > width ? hi - width : lo;
    if (shift <= GRAIN<TY>) {
      b.lo = lo;
      b.hi = hi;
      return b;
    }
  }
}

// What temperature and the filters of a row ask for
struct Filters {
  uint32_t most; // the largest key
  int32_t top_k; // 0: none
  float top_p;
  u64 least;     // min-p, as a weight
  float uniform, min_p;
  Weights weight;
  // the key below which weights are less than a power of two
  __device__ __forceinline__ uint32_t key_below(double power) const {
    const double x = weight.most + power / weight.per_logit;
    const uint32_t k = x > -(double)FLT_BIG ? key_of((float)x) : 1;
    return k > 2 ? k - 1 : 1; // (rounded: one further down)
  }
  __device__ __forceinline__ double min_power() const { return log2((double)fminf(min_p, 1.0f)) - 0.001; } // (and the roundings on its way)
  __device__ __forceinline__ u64 share(u64 whole) const { // top-p's
    const u64 target = (u64)__builtin_ceil((double)top_p * (double)whole);
    return target > 1 ? target : 1;
  }
  __device__ __forceinline__ u64 place(u64 whole) const {
    const u64 target = uniform > 0.0f ? (u64)((double)(uniform < 1.0f ? uniform : 1.0f) * (double)whole) : (u64)0;
    return target < whole ? target : whole - 1;
  }
};

// From whatever holds every token of keys >= lo that may be drawn
template <int TY, typename Source, int THREADS>
__device__ __forceinline__ Found draw(const Source& from, Shared<THREADS>& s, const Filters& f, uint32_t lo, Part part) {
  if (f.top_k > 0) {
    const Border b = border<false, TY>(from, s, lo, f.most, [](uint32_t, int32_t) { return (u64)1; }, [&](u64) { return (u64)f.top_k; });
    // of these keys as many as are missing (where there are fewer than k tokens in all, every one)
    part.lo = b.lo;
    part.hi = b.hi;
    part.last = locate(from, s, [&](uint32_t k, int32_t) { return (u64)(k >= b.lo && k <= b.hi); }, [&](u64) { return b.target - b.before - 1; }).token;
  }
  if (f.top_p < 1.0f) {
    const Part within = part;
    const auto weight = [&](uint32_t k, int32_t v) { return within.has(k, v) ? f.weight(logit_of(k)) : (u64)0; };
    const Border b = border<true, TY>(from, s, lo > within.lo ? lo : within.lo, f.most, weight, [&](u64 whole) { return f.share(whole); });
    part.lo = b.lo;
    part.hi = b.hi;
    part.last = locate(from, s, [&](uint32_t k, int32_t v) { return k >= b.lo && k <= b.hi ? weight(k, v) : (u64)0; }, [&](u64) { return b.target - b.before - 1; }).token;
  }
  return locate(
      from, s,
      [&](uint32_t k, int32_t v) {
        if (!part.has(k, v)) return (u64)0;
        const u64 w = f.weight(logit_of(k));
        return w >= f.least ? w : (u64)0;
      },
      [&](u64 whole) { return f.place(whole); });
}

// Up to SMALL entries of the list: ranked against each other, then the first wave alone, E entries a lane
template <int THREADS>
__device__ __forceinline__ Found draw_small(Shared<THREADS>& s, const Filters& f, int n) {
  const List<THREADS> list(s);
  int at = 0;
  for (int w = 0; w < list.wave; ++w) at += s.listed[w];
  for (int i = list.lane; i < list.n; i += 64) {
    s.small_key[at + i] = s.key[list.wave * List<THREADS>::LIST + i];
    s.small_token[at + i] = s.token[list.wave * List<THREADS>::LIST + i];
  }
  constexpr int SMALL = Shared<THREADS>::SMALL, E = SMALL / 64;
  for (int i = threadIdx.x; i < SMALL; i += THREADS) {
    if (i >= n) s.small_key[i] = 0; // behind all others
    s.rank[i] = 0;
  }
  __syncthreads();
  // 64 entries a wave against a part of all
  const int blocks = (n + 63) / 64, parts = blocks < THREADS / 64 ? THREADS / 64 / blocks : 1, part_of = ((n + 3) / 4 + parts - 1) / parts * 4;
  for (int b = list.wave; b < blocks * parts; b += THREADS / 64) {
    const int each = b % blocks * 64 + list.lane, first = b / blocks * part_of, end = first + part_of < n ? first + part_of : n;
    const uint32_t mine = s.small_key[each];
    int rank = 0;
    // entries of the 64 are before or behind one by their places, all others' places are one side's
    typedef __attribute__((ext_vector_type(4))) uint32_t four;
    const auto count = [&](int from, int to, auto&& before) {
      from = from > first ? from : first;
      to = to < end ? to : end;
#pragma unroll 4
      for (int j = from; j < to; j += 4) { // (behind the last entry: keys of 0)
        const four k = *reinterpret_cast<const four*>(&s.small_key[j]);
#pragma unroll
        for (int e = 0; e < 4; ++e) rank += before(k[e], j + e);
      }
    };
    const int own = b % blocks * 64;
    count(0, own, [&](uint32_t k, int) { return k >= mine; });
    count(own, own + 64, [&](uint32_t k, int j) { return k > mine || (k == mine && j < each); });
    count(own + 64, SMALL, [&](uint32_t k, int) { return k > mine; });
    if (rank) atomicAdd(&s.rank[each], rank);
  }
  __syncthreads();
  for (int each = threadIdx.x; each < SMALL; each += THREADS) {
    const int rank = each < n ? s.rank[each] : each; // (none has a key of 0)
    const u64 w = each < n && (f.top_k == 0 || rank < f.top_k) ? f.weight(logit_of(s.small_key[each])) : (u64)0;
    s.rank[each] = rank;
    s.ranked[rank] = w;
    s.amount[each] = w;
  }
  __syncthreads();
  if (threadIdx.x < 64) {
    const int lane = threadIdx.x;
    // a lane's running sums, behind those of the lanes before
    const auto running = [&](const u64 (&w)[E], u64 (&to)[E]) {
      to[0] = w[0];
#pragma unroll
      for (int e = 1; e < E; ++e) to[e] = to[e - 1] + w[e];
      const u64 before = wave_inclusive(to[E - 1]) - to[E - 1];
#pragma unroll
      for (int e = 0; e < E; ++e) to[e] += before;
      return last_lane(to[E - 1]);
    };
    u64 w[E], to[E];
    int kept = SMALL;
    if (f.top_p < 1.0f) {
#pragma unroll
      for (int e = 0; e < E; ++e) w[e] = s.ranked[E * lane + e];
      const u64 whole = running(w, to), target = f.share(whole);
      int mine = 0;
#pragma unroll
      for (int e = 0; e < E; ++e) mine += to[e] - w[e] < target;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) mine += __shfl_xor(mine, d, 64);
      kept = mine;
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const u64 x = s.amount[E * lane + e];
      w[e] = s.rank[E * lane + e] < kept && x >= f.least ? x : 0;
    }
    const u64 whole = running(w, to), target = f.place(whole);
    const u64 above = __builtin_amdgcn_ballot_w64(target < to[E - 1]);
    if (lane == __builtin_ctzll(above)) {
      bool open = true;
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (open && target < to[e]) {
          s.bin = (uint32_t)s.small_token[E * lane + e];
          s.found = w[e];
          open = false;
        }
      s.wave[0] = whole;
    }
  }
  __syncthreads();
  return Found{(int32_t)s.bin, 0, s.found, s.wave[0]};
}

// No top-k, and more tokens than the list takes: the row is weighed by its waves' runs
template <int TY, int THREADS, typename L>
__device__ __forceinline__ Found draw_weighed(const Row<TY, THREADS>& row, Shared<THREADS>& s, const Filters& f, uint32_t lo, L&& make_list) {
  const float most = logit_of(f.most), least = fmaxf(logit_of(lo), -FLT_BIG); // (the lowest keys are no numbers)
  const auto by_weight = [&]() { // of those that min-p leaves
    const auto amount = [&](uint32_t k, int32_t) {
      const u64 w = k ? f.weight(logit_of(k)) : (u64)0;
      return w >= f.least ? w : (u64)0;
    };
    u64 mine = 0;
    row.each_logit([&](float x, int32_t) {
      const u64 w = f.weight(x);
      mine += w >= f.least ? w : 0;
    });
    const u64 whole = sum_up(s, mine);
    return locate_in_run(row, s, amount, whole, f.place(whole));
  };
  if (f.top_p >= 1.0f) return by_weight();
  // bins of logits, evenly from the largest one down to those that weigh nothing
  const float per_logit = (float)RUN_BINS / fminf(fmaxf(most - least, 1e-30f), FLT_BIG);
  const auto bin_of = [&](float x) { return (int)fminf(fmaxf((most - x) * per_logit, 0.0f), (float)(RUN_BINS - 1)); };
  __syncthreads();
  for (int i = threadIdx.x; i < THREADS / 64 * RUN_BINS; i += THREADS) s.run[0][i] = 0;
  __syncthreads();
  row.each_logit([&](float x, int32_t) {
    const u64 w = f.weight(x);
    if (w) atomicAdd((unsigned long long*)&s.run[row.wave][bin_of(x)], (unsigned long long)w);
  });
  __syncthreads();
  // the bin that has top-p's border: a thread per bin
  u64 to = 0;
  constexpr int EACH = RUN_BINS > THREADS ? RUN_BINS / THREADS : 1;
  u64 n[EACH] = {}, mine = 0;
#pragma unroll
  for (int i = 0; i < EACH; ++i)
    if ((int)threadIdx.x * EACH + i < RUN_BINS) {
#pragma unroll 1
      for (int w = 0; w < THREADS / 64; ++w) n[i] += s.run[w][threadIdx.x * EACH + i];
      mine += n[i];
    }
  const u64 whole = sum_up(s, mine);
  const u64 target = f.share(whole);
  to = wave_inclusive(mine) - mine;
  for (int w = 0; w < row.wave; ++w) to += s.sums[w];
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    if (to < target && to + n[i] >= target) {
      s.bin = threadIdx.x * EACH + i;
      s.found = to;
    }
    to += n[i];
  }
  __syncthreads();
  const int border_bin = (int)s.bin;
  const u64 before = s.found;
  // what each run has above that bin
  u64 above = 0;
  for (int i = row.lane; i < border_bin; i += 64) above += s.run[row.wave][i];
  above = wave_sum(above);
  // its tokens, in a list. (A bin's ends are those of its logits but for roundings, of 2^-22 of the largest number there is.)
  const float off = 2.4e-7f * (fabsf(most) + fabsf(least)), from = border_bin == RUN_BINS - 1 ? least : most - (border_bin + 1) / per_logit - off,
              to_most = most - border_bin / per_logit + off;
  int listed = 0;
  row.each_piece([&](const auto& p, int32_t v, int32_t) {
    if (listed <= Shared<THREADS>::LIST) listed = list_pieces<TY>(s, p, v, listed, from, to_most, [&](float x) { return x >= least && bin_of(x) == border_bin; });
  });
  if (row.lane == 0) s.listed[row.wave] = listed;
  const Part all{lo, lo, row.vocab};
  if (__syncthreads_or(listed > Shared<THREADS>::LIST)) return draw<TY>(row, s, f, lo, all);
  const List<THREADS> list(s);
  const auto weight = [&](uint32_t k, int32_t) { return f.weight(logit_of(k)); };
  const Border b = border<true, TY>(list, s, lo, f.most, weight, [&](u64) { return target - before; });
  const auto tie = locate(list, s, [&](uint32_t k, int32_t v) { return k >= b.lo && k <= b.hi ? weight(k, v) : (u64)0; }, [&](u64) { return b.target - b.before - 1; });
  const Part part{b.lo, b.hi, tie.token};
  const auto amount = [&](uint32_t k, int32_t v) {
    if (!part.has(k, v)) return (u64)0;
    const u64 w = f.weight(logit_of(k));
    return w >= f.least ? w : (u64)0;
  };
  if (tie.amount < f.least) { // min-p leaves less than top-p, and equal ones together
    if (!make_list(f.key_below(f.min_power()))) return by_weight();
    return locate(List<THREADS>(s), s, amount, [&](u64 sum) { return f.place(sum); });
  }
  u64 kept = 0;
  list.each([&](uint32_t k, int32_t v) { kept += part.has(k, v) ? weight(k, v) : (u64)0; });
  const u64 left = sum_up(s, row.lane == 0 ? kept + above : kept);
  return locate_in_run(row, s, amount, left, f.place(left));
}

template <int TY, int THREADS>
__global__ __launch_bounds__(THREADS) void sample_tokens_kernel(const SampleArgs a) {
  using R = Row<TY, THREADS>;
  constexpr int N = R::N, LIST = Shared<THREADS>::LIST, WAVES = THREADS / 64;
  __shared__ Shared<THREADS> s;
  const int64_t at = blockIdx.x;
  const int32_t pieces = (a.vocab + N - 1) / N;
  const R row(reinterpret_cast<const char*>(a.logits) + at * a.stride * R::P::BYTES, a.vocab, 0, pieces);
  const float temperature = a.temperature ? a.temperature[at] : 1.0f, min_p = a.min_p ? a.min_p[at] : 0.0f;
  Filters f;
  f.min_p = min_p;
  f.top_k = a.top_k ? a.top_k[at] : 0;
  f.top_p = a.top_p ? a.top_p[at] : 1.0f;
  f.uniform = a.uniform[at];
  // groups of 1, 2, 4 ... 32 pieces: as many as there is room for
  int log2_lanes = 0;
  while (((pieces - 1) >> log2_lanes) >= Shared<THREADS>::MOST_GROUPS) ++log2_lanes;
  const int lanes = 1 << log2_lanes, groups = ((pieces - 1) >> log2_lanes) + 1;
  if (threadIdx.x < STEPS) s.roots[threadIdx.x] = ROOTS[threadIdx.x];
  for (int i = threadIdx.x; i < BINS; i += THREADS) s.count[i] = 0; // for top-k's groups
  uint32_t high = 0, low = 0; // of the groups' largest: low of the least, as a complement
  row.template each_piece<FIRST_AHEAD>([&](const auto& p, int32_t, int32_t i) {
    const uint32_t k = group_lanes_max(largest_of<TY>(p), lanes);
    high = high > k ? high : k;
    if (k) low = low > ~k ? low : ~k;
    if ((row.lane & (lanes - 1)) == 0 && i < pieces) s.group[i >> log2_lanes] = k;
  });
  high = wave_max(high), low = wave_max(low);
  if (row.lane == 0) s.wave32[row.wave] = high, s.low32[row.wave] = low;
  __syncthreads();
  f.most = 0;
  uint32_t least_group = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    f.most = f.most > s.wave32[w] ? f.most : s.wave32[w];
    least_group = least_group > s.low32[w] ? least_group : s.low32[w];
  }
  least_group = ~least_group;
  __syncthreads(); // (the words are used again)
  const int group_steps = (groups + THREADS - 1) / THREADS; // of a wave, 64 groups each
  const auto group_at = [&](int step) { return (row.wave * group_steps + step) * 64 + row.lane; };
  constexpr int GROUP_STEPS = Shared<THREADS>::MOST_GROUPS / THREADS;
  uint32_t group[GROUP_STEPS]; // a thread's
#pragma unroll
  for (int k = 0; k < GROUP_STEPS; ++k) group[k] = k < group_steps && group_at(k) < groups ? s.group[group_at(k)] : 0;
  const bool greedy = !(temperature > 0.0f) || f.top_k == 1 || !(f.top_p > 0.0f);
  if (f.most == 0) { // nothing to draw from
    if (threadIdx.x == 0) {
      a.tokens[at] = -1;
      a.log_probability[at] = -__builtin_inff();
    }
    return;
  }
  const auto write = [&](int32_t token, float log_probability) {
    a.tokens[at] = token;
    a.log_probability[at] = log_probability;
  };
  // the groups with a key of at least `lo`, in their order; how many
  const auto choose = [&](uint32_t lo) {
    u64 in[GROUP_STEPS];
    int mine = 0; // of the wave
#pragma unroll
    for (int k = 0; k < GROUP_STEPS; ++k) {
      in[k] = __builtin_amdgcn_ballot_w64(group[k] >= lo);
      mine += __builtin_popcountll(in[k]);
    }
    if (row.lane == 0) s.wave32[row.wave] = mine;
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      if (w < row.wave) before += s.wave32[w];
      all += s.wave32[w];
    }
#pragma unroll
    for (int k = 0; k < GROUP_STEPS; ++k) {
      if ((in[k] >> row.lane) & 1) s.chosen[before + __builtin_popcountll(in[k] & ((1ull << row.lane) - 1))] = (uint16_t)group_at(k);
      before += __builtin_popcountll(in[k]);
    }
    __syncthreads();
    return all;
  };
  if (greedy) {
    // the most likely one, the first of equal ones
    choose(f.most);
    if (row.wave == 0) {
      const int32_t i = ((int32_t)s.chosen[0] << log2_lanes) + row.lane;
      typename R::P p;
      R::load(p, row.logits, row.lane < lanes && i < pieces ? i * N : a.vocab, a.vocab);
      int32_t token = -1;
      R::each_of(p, i * N, [&](float x, int32_t v) {
        if (token < 0 && key_of(x) == f.most) token = v;
      });
      const u64 has = __builtin_amdgcn_ballot_w64(token >= 0);
      if (row.lane == __builtin_ctzll(has)) write(token, 0.0f);
    }
    return;
  }
  if (f.top_k <= 0 || f.top_k >= a.vocab) f.top_k = 0;
  const int bits = 32 - __builtin_clz(a.vocab);
  f.weight = Weights{(double)logit_of(f.most), 1.4426950408889634074 / (double)temperature, 62 - bits < 50 ? 62 - bits : 50, s.roots};
  f.least = min_p > 0.0f ? (u64)__builtin_ceil(__builtin_ldexp((double)(min_p < 1.0f ? min_p : 1.0f), f.weight.fraction)) : 0;
  // keys below `lo` take no part
  uint32_t lo = 1;
  if (f.top_k > 0) { // k groups' largest are above them
    const uint32_t least = least_group;
    const int shift = shift_of(least, f.most);
#pragma unroll
    for (int k = 0; k < GROUP_STEPS; ++k)
      if (group[k]) atomicAdd(&s.count[(f.most - group[k]) >> shift], 1u);
    __syncthreads();
    bool enough = false;
    find_bin<false>(s, [&](u64 whole) {
      enough = whole >= (u64)f.top_k;
      return (u64)f.top_k;
    });
    const uint32_t down = (s.bin << shift) + ((1u << shift) - 1); // (a bin is within the keys' span and less than its double)
    if (enough) lo = f.most - least > down ? f.most - down : least;
  } else { // they weigh nothing, or too little for min-p
    lo = f.key_below(-(f.weight.fraction + 2)); // 2^-2 of a unit
    if (f.top_p >= 1.0f && f.min_p > 0.0f) lo = max(lo, f.key_below(f.min_power()));
  }
  // the tokens of those groups, in the list, a wave's share of the groups 64 pieces at a time; false: it does not hold them
  const auto make_list = [&](uint32_t from) {
    const int chosen = choose(from), share = ((chosen << log2_lanes) + THREADS - 1) / THREADS;
    const float least = fmaxf(logit_of(from), -FLT_BIG); // (the lowest keys are no numbers)
    int listed = 0;
    for (int k = 0; k < share && listed <= LIST; ++k) {
      const int32_t item = (row.wave * share + k) * 64 + row.lane, g = item >> log2_lanes;
      const int32_t i = g < chosen ? ((int32_t)s.chosen[g] << log2_lanes) + (item & (lanes - 1)) : pieces;
      typename R::P p;
      R::load(p, row.logits, i < pieces ? i * N : a.vocab, a.vocab);
      listed = list_pieces<TY>(s, p, i * N, listed, least, __builtin_inff(), [](float) { return true; });
    }
    if (row.lane == 0) s.listed[row.wave] = listed;
    return !__syncthreads_or(listed > LIST);
  };
  Found drawn;
  if (make_list(lo)) {
    int n = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) n += s.listed[w];
    if (n <= Shared<THREADS>::SMALL) drawn = draw_small(s, f, n);
    else drawn = draw<TY>(List<THREADS>(s), s, f, lo, Part{lo, lo, a.vocab});
  } else if (f.top_k == 0 && f.weight.most < (double)FLT_BIG) { // (no infinities)
    drawn = draw_weighed(row, s, f, lo, make_list);
  } else {
    drawn = draw<TY>(row, s, f, lo, Part{lo, lo, a.vocab});
  }
  if (threadIdx.x == 0) write(drawn.token, (float)log((double)drawn.amount / (double)drawn.whole));
}

template <int TY, int THREADS>
hipError_t launch_shape(SampleArgs a, hipStream_t stream) {
  constexpr int64_t MOST = 0xffffffffll / THREADS; // rows of a launch: fewer than 2^32 threads
  for (int64_t rows = a.rows; rows > 0; rows -= MOST) {
    sample_tokens_kernel<TY, THREADS><<<(unsigned)(rows < MOST ? rows : MOST), THREADS, 0, stream>>>(a);
    if (hipError_t e = hipGetLastError()) return e;
    const auto later = [](auto*& p) {
      if (p) p += MOST;
    };
    a.logits = reinterpret_cast<const char*>(a.logits) + MOST * a.stride * Piece<TY>::BYTES;
    later(a.uniform), later(a.temperature), later(a.top_k), later(a.top_p), later(a.min_p), later(a.tokens), later(a.log_probability);
  }
  return hipSuccess;
}
template <int TY>
hipError_t launch(const SampleArgs& a, hipStream_t stream) {
  // A row of 16 waves has a compute unit to itself, of rows of 4 waves three are there at once. Small rows are no work for 16 waves, and
  // where there are rows to fill the device several times over, more rows at once are better than each of them faster. us with 16 and with 4
  // waves (bf16; the largest logit, the 50 largest, all, top-p 0.9 of them):
  //   1 row of 8 192             4.7 10.6 12.5 23.7    3.9  9.1 11.8 21.4
  //   1 row of 16 384            5.2 11.4 14.8 26.7    4.8  9.2 17.0 30.8
  //   300 rows of 32 000        11.7 25.9 37.1 65.0    8.9 13.9 39.1 60.8
  //   1 024 rows of 32 000      26.8 54.4 77.0 132     19.0 27.9 70.3 112
  //   300 rows of 65 536        14.5 31.8 51.8 88.9   12.4 17.9 67.6 104
  // (The last, with 16: which rows have a filter is known on the device alone, and those without one take longest.)
  if (a.vocab <= 8192 || (a.rows > a.compute_units && a.vocab <= 32768)) return launch_shape<TY, 256>(a, stream);
  return launch_shape<TY, 1024>(a, stream);
}

} // namespace

hipError_t launch_sample_tokens(const SampleArgs& a, int32_t ty, hipStream_t stream) {
  if (ty == ST_FP32) return launch<ST_FP32>(a, stream);
  if (ty == ST_FP16) return launch<ST_FP16>(a, stream);
  return launch<ST_BF16>(a, stream);
}

} // namespace fbgemm_amd
