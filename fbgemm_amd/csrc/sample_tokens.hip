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
// and a running sum is off by no more than the w's own roundings, some 2^-46 of the largest each. exp is made in fp64 (2^-52).
//
// A workgroup has a row, a wave a run of its tokens, in their order. Passes over the row: the largest logit; then the tokens that
// can matter at all (top-k: the k-th largest of the threads' largest logits is a bound that few others pass; else weights that
// are not 0, or min-p) are put in a list in LDS, if it holds them, and what follows are passes over the list, else over
// the row again, out of the caches. Where the order matters (which of equal ones is within top-k, top-p's sum) the first part
// is found by counting: bins of keys (fp32 bits in ascending order), the bin where the count or sum is reached, bins of that
// bin's keys, until a bin is one key; then the last token of that key that is within.
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

// exp((x - most) / temperature) in units of 2^-fraction
struct Weights {
  double most, per_logit; // per_logit: log2(e) / temperature
  int fraction;
  __device__ __forceinline__ u64 operator()(float x) const {
    const double t = ((double)__builtin_fminf(x, FLT_BIG) - most) * per_logit;
    if (!(t > -(double)(fraction + 2))) return 0;
    const double whole = __builtin_rint(t), f = t - whole;
    // 2^f, |f| <= 1/2, by its series: the next term is below 2^-52
    constexpr double C[12] = {0.6931471805599453094,  0.2402265069591007123,  0.05550410866482157995, 0.009618129107628477162, 0.001333355814642844342, 1.540353039338160995e-4,
                              1.525273380405984028e-5, 1.321548679014430949e-6, 1.017808600923969973e-7, 7.054911620801123329e-9, 4.445538271870811498e-10, 2.567843599348820514e-11};
    double p = C[11];
#pragma unroll
    for (int i = 10; i >= 0; --i) p = __builtin_fma(p, f, C[i]);
    p = __builtin_fma(p, f, 1.0);
    // a double of 2^52 and more holds whole numbers: adding that rounds, and leaves the number in the low bits
    const double w = __builtin_ldexp(p, (int)whole + fraction) + 4503599627370496.0;
    return __builtin_bit_cast(u64, w) & 0xfffffffffffffull;
  }
};

__device__ __forceinline__ u64 shfl_up64(u64 v, int d) {
  return (u64)__shfl_up((uint32_t)v, d, 64) | ((u64)__shfl_up((uint32_t)(v >> 32), d, 64) << 32);
}
__device__ __forceinline__ u64 shfl_xor64(u64 v, int d) {
  return (u64)__shfl_xor((uint32_t)v, d, 64) | ((u64)__shfl_xor((uint32_t)(v >> 32), d, 64) << 32);
}
__device__ __forceinline__ u64 wave_sum(u64 v) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) v += shfl_xor64(v, d);
  return v;
}
__device__ __forceinline__ u64 wave_inclusive(u64 v, int lane) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const u64 o = shfl_up64(v, d);
    v += lane >= d ? o : 0;
  }
  return v;
}
__device__ __forceinline__ u64 last_lane(u64 v) { // (readlane gives an int)
  return (u64)(uint32_t)__builtin_amdgcn_readlane((uint32_t)v, 63) | ((u64)(uint32_t)__builtin_amdgcn_readlane((uint32_t)(v >> 32), 63) << 32);
}
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t o = __shfl_xor(v, d, 64);
    v = v > o ? v : o;
  }
  return v;
}

// What may be drawn: keys above `key`, and of that key the tokens up to `last`
struct Part {
  uint32_t key;
  int32_t last;
  __device__ __forceinline__ bool has(uint32_t k, int32_t token) const { return k > key || (k == key && token <= last); }
};

constexpr int THREADS = 1024, WAVES = THREADS / 64;
constexpr int LIST = 448; // entries of a wave's part of the list
struct Shared {
  u64 weight[BINS];
  uint32_t count[BINS];
  u64 sums[WAVES], wave[WAVES];
  uint32_t wave32[WAVES];
  u64 found;    // an amount
  uint32_t bin; // a place
  int32_t listed[WAVES];
  uint32_t key[WAVES * LIST];
  int32_t token[WAVES * LIST];
};

// The row in memory. A wave's tokens follow each other: `steps` times 64 pieces.
template <int TY>
struct Row {
  using P = Piece<TY>;
  static constexpr int N = P::N, AHEAD = 4; // pieces that are loaded together
  const char* logits;
  int32_t vocab;
  int steps, lane, wave;
  __device__ __forceinline__ Row(const SampleArgs& a, int64_t row)
      : logits(reinterpret_cast<const char*>(a.logits) + row * a.stride * P::BYTES), vocab(a.vocab), lane(threadIdx.x & 63),
        wave(__builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) {
    steps = ((vocab + N - 1) / N + THREADS - 1) / THREADS;
  }
  // the first token of a lane's piece
  __device__ __forceinline__ int32_t at(int step) const { return ((wave * steps + step) * 64 + lane) * N; }
  __device__ __forceinline__ void load(P& p, int step) const {
    const int32_t v = at(step);
    if (step < steps && v + N <= vocab) p.load(logits + (int64_t)v * P::BYTES);
    else p.load_some(logits + (int64_t)v * P::BYTES, step < steps && v < vocab ? vocab - v : 0);
  }
  // f(logit, its token) for those of a lane's piece, in their order
  template <typename F>
  __device__ __forceinline__ void each_of(P p, int32_t v, F&& f) const {
#pragma unroll 1
    for (int i = 0; i < N; i += 2) { // (two elements' code: the piece is turned past them)
      if (v + i < vocab) f(p.get(0), v + i);
      if (v + i + 1 < vocab) f(p.get(1), v + i + 1);
      if constexpr (TY == ST_FP32) p.raw[0] = p.raw[2], p.raw[1] = p.raw[3];
      else p.raw[0] = p.raw[1], p.raw[1] = p.raw[2], p.raw[2] = p.raw[3];
    }
  }
  // f(piece, its first token), step by step; f may end it
  template <typename F>
  __device__ __forceinline__ void each_piece(F&& f) const {
    for (int k = 0; k < steps; k += AHEAD) {
      P x[AHEAD];
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) load(x[j], k + j);
#pragma unroll
      for (int j = 0; j < AHEAD; ++j)
        if (k + j < steps && !f(x[j], at(k + j))) return;
    }
  }
  // f(key, token, step) for a thread's tokens
  template <typename F>
  __device__ __forceinline__ void each(F&& f) const {
    each_piece([&](const P& p, int32_t v) {
      each_of(p, v, [&](float x, int32_t token) { f(key_of(x), token); });
      return true;
    });
  }
  template <typename F>
  __device__ __forceinline__ void each_of_step(int step, F&& f) const {
    P p;
    load(p, step);
    each_of(p, at(step), [&](float x, int32_t token) { f(key_of(x), token); });
  }
};

// The list: a wave's entries, in their tokens' order
struct List {
  const Shared& s;
  int steps, lane, wave, n;
  __device__ __forceinline__ List(const Shared& shared)
      : s(shared), lane(threadIdx.x & 63), wave(__builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) {
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

// The tokens of keys >= lo, into the list; false: it does not hold them
template <int TY>
__device__ __forceinline__ bool make_list(const Row<TY>& row, Shared& s, uint32_t lo) {
  int n = 0; // the same for the wave
  row.each_piece([&](const auto& p, int32_t v) {
    int mine = 0;
    row.each_of(p, v, [&](float x, int32_t) { mine += key_of(x) >= lo; });
    if (__builtin_amdgcn_ballot_w64(mine > 0) == 0) return true;
    int to = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int o = __shfl_up(to, d, 64);
      to += row.lane >= d ? o : 0;
    }
    const int all = __builtin_amdgcn_readlane(to, 63);
    if (n + all > LIST) {
      n = LIST + 1;
      return false;
    }
    int at = row.wave * LIST + n + to - mine;
    if (mine > 0)
      row.each_of(p, v, [&](float x, int32_t token) {
        const uint32_t k = key_of(x);
        if (k >= lo) {
          s.key[at] = k;
          s.token[at] = token;
          ++at;
        }
      });
    n += all;
    return true;
  });
  if (row.lane == 0) s.listed[row.wave] = n;
  return !__syncthreads_or(n > LIST);
}

__device__ __forceinline__ uint32_t block_max(Shared& s, uint32_t v) {
  v = wave_max(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s.wave32[threadIdx.x >> 6] = v;
  __syncthreads();
  v = s.wave32[0];
#pragma unroll
  for (int w = 1; w < WAVES; ++w) v = v > s.wave32[w] ? v : s.wave32[w];
  return v;
}

// The first token, by number, where the running sum of amount(key, token) is above a target, which is asked for by the whole sum;
// where that is the whole or more, the last one that has an amount. One has at least.
struct Found {
  int32_t token;
  u64 amount, whole;
};
template <typename Source, typename F, typename T>
__device__ __forceinline__ Found locate(const Source& from, Shared& s, F&& amount, T&& target_of) {
  u64 mine = 0;
  from.each([&](uint32_t k, int32_t v) { mine += amount(k, v); });
  mine = wave_sum(mine);
  __syncthreads();
  if (from.lane == 0) s.sums[from.wave] = mine;
  __syncthreads();
  u64 whole = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) whole += s.sums[w];
  u64 target = target_of(whole);
  target = target < whole ? target : whole - 1;
  int in = 0;
  u64 before = 0;
  for (; in < WAVES - 1 && before + s.sums[in] <= target; ++in) before += s.sums[in];
  if (from.wave == in) {
    for (int k = 0; k < from.steps; ++k) {
      u64 of_step = 0;
      from.each_of_step(k, [&](uint32_t key, int32_t v) { of_step += amount(key, v); });
      const u64 to = before + wave_inclusive(of_step, from.lane);
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
  const Found r{(int32_t)s.bin, s.found, whole};
  __syncthreads();
  return r;
}

// s.bin: the first bin where the running sum reaches `target` (asked for by the whole; none does: the last one that is not empty); s.found: the sum
// before it. The target.
template <bool WEIGHTS, typename T>
__device__ __forceinline__ u64 find_bin(Shared& s, T&& target_of) {
  constexpr int EACH = BINS / THREADS;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  u64 n[EACH], mine = 0;
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    n[i] = WEIGHTS ? s.weight[threadIdx.x * EACH + i] : (u64)s.count[threadIdx.x * EACH + i];
    mine += n[i];
  }
  const u64 to = wave_inclusive(mine, lane);
  if (lane == 63) s.wave[wave] = to;
  __syncthreads();
  u64 before = to - mine, whole = 0;
  for (int w = 0; w < WAVES; ++w) {
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

// Keys from the largest, `hi`, down to `lo`, until the sum of their amounts reaches a target (at least 1), asked for by the whole: the key that
// does it, the sum before it, the target. WEIGHTS: amounts are sums of u64, else 0 or 1.
struct Border {
  uint32_t key;
  u64 before, target;
};
template <bool WEIGHTS, typename Source, typename F, typename T>
__device__ __forceinline__ Border border(const Source& from, Shared& s, uint32_t lo, uint32_t hi, F&& amount, T&& target_of) {
  Border b{0, 0, 0};
  for (bool first = true;; first = false) {
    const uint32_t span = hi - lo;
    const int shift = span < BINS ? 0 : 32 - __builtin_clz(span) - 11;
    __syncthreads();
    for (int i = threadIdx.x; i < BINS; i += THREADS) {
      if (WEIGHTS) s.weight[i] = 0;
      else s.count[i] = 0;
    }
    __syncthreads();
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
    if (shift == 0) {
      b.key = hi;
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
  float uniform;
  Weights weight;
};

template <typename Source>
__device__ __forceinline__ Found draw(const Source& from, Shared& s, const Filters& f, uint32_t lo, Part part) {
  if (f.top_k > 0) {
    const Border b = border<false>(from, s, lo, f.most, [](uint32_t, int32_t) { return (u64)1; }, [&](u64) { return (u64)f.top_k; });
    // of that key as many as are missing (where there are fewer than k tokens in all, every one)
    part.key = b.key;
    part.last = locate(from, s, [&](uint32_t k, int32_t) { return (u64)(k == b.key); }, [&](u64) { return b.target - b.before - 1; }).token;
  }
  if (f.top_p < 1.0f) {
    const Part within = part;
    const Border b = border<true>(
        from, s, lo > within.key ? lo : within.key, f.most, [&](uint32_t k, int32_t v) { return within.has(k, v) ? f.weight(logit_of(k)) : (u64)0; },
        [&](u64 whole) {
          const u64 target = (u64)__builtin_ceil((double)f.top_p * (double)whole);
          return target > 1 ? target : (u64)1;
        });
    const u64 each = f.weight(logit_of(b.key)), missing = (b.target - b.before + each - 1) / each;
    part.key = b.key;
    part.last = locate(from, s, [&](uint32_t k, int32_t v) { return (u64)(k == b.key && within.has(k, v)); }, [&](u64) { return missing - 1; }).token;
  }
  return locate(
      from, s,
      [&](uint32_t k, int32_t v) {
        if (!part.has(k, v)) return (u64)0;
        const u64 w = f.weight(logit_of(k));
        return w >= f.least ? w : (u64)0;
      },
      [&](u64 whole) { return f.uniform > 0.0f ? (u64)((double)(f.uniform < 1.0f ? f.uniform : 1.0f) * (double)whole) : (u64)0; });
}

template <int TY>
__global__ __launch_bounds__(THREADS) void sample_tokens_kernel(const SampleArgs a) {
  __shared__ Shared s;
  const int64_t at = blockIdx.x;
  const Row<TY> row(a, at);
  uint32_t mine = 0; // the thread's largest key
  row.each([&](uint32_t k, int32_t) { mine = mine > k ? mine : k; });
  Filters f;
  f.most = block_max(s, mine);
  if (f.most == 0) { // nothing to draw from
    if (threadIdx.x == 0) {
      a.tokens[at] = -1;
      a.log_probability[at] = -__builtin_inff();
    }
    return;
  }
  const float temperature = a.temperature ? a.temperature[at] : 1.0f, min_p = a.min_p ? a.min_p[at] : 0.0f;
  f.top_k = a.top_k ? a.top_k[at] : 0;
  f.top_p = a.top_p ? a.top_p[at] : 1.0f;
  f.uniform = a.uniform[at];
  if (!(temperature > 0.0f) || f.top_k == 1 || !(f.top_p > 0.0f)) {
    // the most likely one, the first of equal ones
    const Found first = locate(row, s, [&](uint32_t k, int32_t) { return (u64)(k == f.most); }, [](u64) { return (u64)0; });
    if (threadIdx.x == 0) {
      a.tokens[at] = first.token;
      a.log_probability[at] = 0.0f;
    }
    return;
  }
  if (f.top_k <= 0 || f.top_k >= a.vocab) f.top_k = 0;
  const int bits = 32 - __builtin_clz(a.vocab);
  f.weight = Weights{(double)logit_of(f.most), 1.4426950408889634074 / (double)temperature, 62 - bits < 50 ? 62 - bits : 50};
  f.least = min_p > 0.0f ? (u64)__builtin_ceil(__builtin_ldexp((double)(min_p < 1.0f ? min_p : 1.0f), f.weight.fraction)) : 0;
  // keys below `lo` take no part
  uint32_t lo = 1;
  if (f.top_k > 0 && f.top_k <= THREADS) { // they are not among the first k: k threads' largest are above them. By bisection
    uint32_t high = f.most;
    while (lo < high) {
      const uint32_t mid = lo + (high - lo + 1) / 2;
      if (__syncthreads_count(mine >= mid) >= f.top_k) lo = mid;
      else high = mid - 1;
    }
  } else if (f.top_k == 0) { // they weigh nothing, or too little for min-p
    double below = f.weight.fraction + 2;
    if (min_p > 0.0f && f.top_p >= 1.0f) below = fmin(below, 0.001 - log2((double)fminf(min_p, 1.0f)));
    const double least = f.weight.most - below / f.weight.per_logit;
    if (least > -(double)FLT_BIG) lo = key_of((float)least) - 1; // (rounded: one further down)
  }
  const Part all{lo, a.vocab};
  const Found drawn = make_list(row, s, lo) ? draw(List(s), s, f, lo, all) : draw(row, s, f, lo, all);
  if (threadIdx.x == 0) {
    a.tokens[at] = drawn.token;
    a.log_probability[at] = (float)log((double)drawn.amount / (double)drawn.whole);
  }
}

template <int TY>
hipError_t launch(SampleArgs a, hipStream_t stream) {
  constexpr int64_t MOST = 0xffffffffll / THREADS; // rows of a launch: fewer than 2^32 threads
  for (int64_t rows = a.rows; rows > 0; rows -= MOST) {
    sample_tokens_kernel<TY><<<(unsigned)(rows < MOST ? rows : MOST), THREADS, 0, stream>>>(a);
    if (hipError_t e = hipGetLastError()) return e;
    const auto later = [](auto*& p) {
      if (p) p += MOST;
    };
    a.logits = reinterpret_cast<const char*>(a.logits) + MOST * a.stride * Piece<TY>::BYTES;
    later(a.uniform), later(a.temperature), later(a.top_k), later(a.top_p), later(a.min_p), later(a.tokens), later(a.log_probability);
  }
  return hipSuccess;
}
} // namespace

hipError_t launch_sample_tokens(const SampleArgs& a, int32_t ty, hipStream_t stream) {
  if (ty == ST_FP32) return launch<ST_FP32>(a, stream);
  if (ty == ST_FP16) return launch<ST_FP16>(a, stream);
  return launch<ST_BF16>(a, stream);
}

} // namespace fbgemm_amd
