// Pages, slots and positions of a decoding step, from the requests' lengths.
//
// Request r holds len_r tokens in ceil(len_r / S) pages and gets new_r more:
//   need_r = ceil((len_r + new_r) / S) - ceil(len_r / S)  pages, the free list's entries
//            start + sum_{i<r} need_i and on, in order, at the end of its table;
//   token k of its new ones sits at position len_r + k, in slot table[r][(len_r + k) / S] * S + (len_r + k) % S.
// Two running sums over the requests (tokens, pages) are all there is to it; everything behind
// them is parallel in tokens and in pages.
//
// One launch: every workgroup adds up all requests by itself, a tile of them at a time (lengths come
// out of L2: two loads and two barriers), and then writes those tokens and pages of the tile that its
// place in the grid gives it, finding a token's request by bisection over the tile's sums in LDS.
// A scan in a launch of its own would cost a second launch, and the sums a trip through memory. What
// it costs is a chain of dependent steps, not bytes: sums are 32 bits that stop at the largest
// number (beyond every list there is), and few requests take a smaller workgroup: 64 requests with a
// token each 6.8 -> 4.6 us.
#include "decode.h"

namespace fbgemm_amd {

namespace {

constexpr int ITEMS = 4;

struct Sums {
  uint32_t tokens, pages;
  __device__ __forceinline__ void add(uint32_t t, uint32_t p) {
    tokens = __builtin_elementwise_add_sat(tokens, t);
    pages = __builtin_elementwise_add_sat(pages, p);
  }
};

__device__ __forceinline__ int32_t clipped(uint32_t v, int64_t most) { return (int32_t)((int64_t)v < most ? (int64_t)v : most); }

// the last of `n` ascending entries that is <= v (entry 0 is)
__device__ __forceinline__ int last_not_above(const int32_t* sums, int n, int32_t v) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (sums[mid] <= v) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

template <typename index_t, int THREADS>
__global__ __launch_bounds__(THREADS) void kv_block_tables_kernel(const BlockTablesArgs a) {
  constexpr int TILE = THREADS * ITEMS;
  __shared__ int32_t s_tokens[TILE + 1], s_pages[TILE + 1], s_len[TILE];
  __shared__ Sums s_wave[THREADS / 64];
  const index_t* lengths = reinterpret_cast<const index_t*>(a.lengths);
  const index_t* news = reinterpret_cast<const index_t*>(a.new_tokens);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t me = (int64_t)blockIdx.x * THREADS + tid, all = (int64_t)gridDim.x * THREADS;
  const int64_t limit = a.width * a.block.d; // positions a table has room for
  const int64_t start = *a.free_start;
  const auto free_block = [&](int64_t place) -> int32_t { return place >= 0 && place < a.free_numel ? a.free_blocks[place] : -1; };
  const auto blocks_of = [&](int64_t tokens) { return (int64_t)divide((uint32_t)(tokens + a.block.d - 1), a.block); };
  Sums before{0, 0}; // of all tiles so far
  for (int64_t r0 = 0; r0 < a.R; r0 += TILE) {
    // who reports and writes the tile's per-request results
    const bool owner = (r0 / TILE) % gridDim.x == blockIdx.x;
    int32_t len[ITEMS];
    Sums mine[ITEMS], sum{0, 0};
    int32_t bits = 0;
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
      const int64_t r = r0 + (int64_t)tid * ITEMS + k;
      int64_t held = 0, added = 0;
      if (r < a.R) {
        held = (int64_t)lengths[r];
        added = (int64_t)news[r];
        if (held < 0 || added < 0) bits |= ERR_NEGATIVE_LENGTH;
        held = held < 0 ? 0 : held;
        added = added < 0 ? 0 : added;
        if (owner) reinterpret_cast<index_t*>(a.total_lengths)[r] = (index_t)(held + added);
        // a token beyond the table's room has no page; limit < 2^31
        if (held > limit || added > limit - held) bits |= ERR_BAG_OVERRUN;
      }
      len[k] = (int32_t)(held < limit ? held : limit);
      const int64_t end = added < limit - len[k] ? len[k] + added : limit;
      mine[k].tokens = (uint32_t)(added < 0xffffffffll ? added : 0xffffffffll);
      mine[k].pages = (uint32_t)(blocks_of(end) - blocks_of(len[k]));
      sum.add(mine[k].tokens, mine[k].pages);
    }
    Sums incl = sum; // of this thread's and those in front of it in the wave
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const uint32_t t = __shfl_up(incl.tokens, d, 64), p = __shfl_up(incl.pages, d, 64);
      if (lane >= d) incl.add(t, p);
    }
    Sums at{__shfl_up(incl.tokens, 1, 64), __shfl_up(incl.pages, 1, 64)};
    if (lane == 0) at = Sums{0, 0};
    at.add(before.tokens, before.pages);
    __syncthreads(); // the tile before is done with LDS
    if (lane == 63) s_wave[wave] = incl;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) {
      if (w < wave) at.add(s_wave[w].tokens, s_wave[w].pages);
      before.add(s_wave[w].tokens, s_wave[w].pages);
    }
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
      const int64_t r = r0 + (int64_t)tid * ITEMS + k;
      const int32_t t = clipped(at.tokens, a.num_tokens), p = clipped(at.pages, 0x7fffffff);
      s_tokens[tid * ITEMS + k] = t;
      s_pages[tid * ITEMS + k] = p;
      s_len[tid * ITEMS + k] = len[k];
      if (owner && r < a.R) a.offsets[r] = t;
      at.add(mine[k].tokens, mine[k].pages);
    }
    if (tid == THREADS - 1) {
      s_tokens[TILE] = clipped(before.tokens, a.num_tokens);
      s_pages[TILE] = clipped(before.pages, 0x7fffffff);
    }
    __syncthreads();
    const int count = (int)(a.R - r0 < TILE ? a.R - r0 : TILE);
    const int32_t token0 = s_tokens[0], token1 = s_tokens[TILE], page0 = s_pages[0], page1 = s_pages[TILE];
    for (int64_t p = page0 + me; p < page1; p += all) {
      const int i = last_not_above(s_pages, count, (int32_t)p);
      const int64_t column = blocks_of(s_len[i]) + (p - s_pages[i]);
      a.tables[(r0 + i) * a.table_stride + column] = free_block(start + p);
      if (start + p < 0 || start + p >= a.free_numel) bits |= ERR_OUT_OF_BLOCKS;
    }
    for (int64_t t = token0 + me; t < token1; t += all) {
      const int i = last_not_above(s_tokens, count, (int32_t)t);
      const int64_t position = (int64_t)s_len[i] + (t - s_tokens[i]);
      int64_t slot = -1;
      if (position < limit) {
        const uint32_t column = divide((uint32_t)position, a.block);
        const int64_t old = blocks_of(s_len[i]);
        const int32_t block = column < old ? a.tables[(r0 + i) * a.table_stride + column] : free_block(start + s_pages[i] + (column - old));
        if (block >= 0) slot = (int64_t)block * a.block.d + (position - (int64_t)column * a.block.d);
      }
      a.slots[t] = slot;
      a.positions[t] = position;
    }
    if (a.status && bits && (owner || (bits & ERR_OUT_OF_BLOCKS))) status_or(a.status, bits);
  }
  for (int64_t t = clipped(before.tokens, a.num_tokens) + me; t < a.num_tokens; t += all) {
    a.slots[t] = -1;
    a.positions[t] = 0;
  }
  if (me == 0) {
    a.offsets[a.R] = clipped(before.tokens, a.num_tokens);
    const int64_t next = start + (int64_t)before.pages;
    *a.free_next = (int32_t)(next < 0x7fffffff ? next : 0x7fffffff);
    if (a.status && (int64_t)before.tokens != a.num_tokens) status_or(a.status, ERR_LENGTH_MISMATCH);
  }
}

} // namespace

hipError_t launch_kv_block_tables(const BlockTablesArgs& a, bool idx64, hipStream_t stream) {
  // one token per thread, up to the workgroups that the device holds at once
  const bool few = a.R <= 256 && a.num_tokens <= 4096;
  const int threads = few ? 256 : 1024;
  const int64_t want = (a.num_tokens + threads - 1) / threads;
  const int grid = (int)(want < 1 ? 1 : want > 256 ? 256 : want);
  if (few) {
    if (idx64) kv_block_tables_kernel<int64_t, 256><<<grid, 256, 0, stream>>>(a);
    else kv_block_tables_kernel<int32_t, 256><<<grid, 256, 0, stream>>>(a);
  } else {
    if (idx64) kv_block_tables_kernel<int64_t, 1024><<<grid, 1024, 0, stream>>>(a);
    else kv_block_tables_kernel<int32_t, 1024><<<grid, 1024, 0, stream>>>(a);
  }
  return hipGetLastError();
}

} // namespace fbgemm_amd
