// Host side of the decoding-step operators of the C ABI (include/fbgemm_amd.h): argument checks,
// sizes of launches and workspaces. Nothing is allocated, and nothing of a call is kept.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <limits>
#include <numeric>

#include "../../include/fbgemm_amd.h"
#include "../../include/fbgemm_amd_bench.h"
#include "api_error.h"
#include "decode.h"

using namespace fbgemm_amd;

namespace {

constexpr int64_t MOST = 0x7fffffff;

bool divides(int64_t a, std::initializer_list<int64_t> values) {
  for (int64_t v : values)
    if (v % a) return false;
  return true;
}

// bytes of one stored row; 0: a type a cache cannot hold
int32_t cache_row_bytes(const fbgemm_amd_paged_cache& c) {
  switch (c.row_ty) {
    case ST_FP32: return c.dim * 4;
    case ST_FP16: case ST_BF16: return c.dim * 2;
    case ST_INT8: return c.dim + 4;
    case ST_CACHE_INT4: return c.dim / 2 + 4;
    default: return 0;
  }
}
bool coded(int32_t ty) { return ty == ST_INT8 || ty == ST_CACHE_INT4; }
int32_t storage_bytes(int32_t ty) { return ty == ST_FP32 ? 4 : coded(ty) ? 1 : 2; }

int check_cache(const fbgemm_amd_paged_cache* c) {
  if (!c) return fail(FBGEMM_AMD_E_ARG, "cache is null");
  if (c->dim <= 0 || c->dim > (1 << 16)) return fail(FBGEMM_AMD_E_ARG, "dim must be in 1..65536");
  if (!cache_row_bytes(*c)) return fail(FBGEMM_AMD_E_ARG, "a cache holds FP32, FP16, BF16, INT8 or CACHE_INT4 rows");
  if (c->row_ty == ST_CACHE_INT4 && c->dim % 2) return fail(FBGEMM_AMD_E_ARG, "4-bit rows hold an even number of elements: got dim %d", c->dim);
  if (c->heads <= 0 || c->heads > (1 << 16)) return fail(FBGEMM_AMD_E_ARG, "heads must be in 1..65536");
  if ((int64_t)c->heads * c->dim > (1 << 28)) return fail(FBGEMM_AMD_E_ARG, "heads * dim must not exceed 2^28");
  if (c->block_size <= 0 || c->block_size > (1 << 20)) return fail(FBGEMM_AMD_E_ARG, "block_size must be in 1..1048576");
  if (c->blocks < 0 || c->blocks > MOST) return fail(FBGEMM_AMD_E_ARG, "blocks must be in 0..2^31-1");
  for (int k = 0; k < 3; ++k)
    if (c->key_strides[k] < 0 || c->value_strides[k] < 0) return fail(FBGEMM_AMD_E_ARG, "strides must not be negative");
  if (coded(c->row_ty) && !(divides(4, {c->key_strides[0], c->key_strides[1], c->key_strides[2]}) &&
                                divides(4, {c->value_strides[0], c->value_strides[1], c->value_strides[2]})))
    return fail(FBGEMM_AMD_E_ARG, "8-bit and 4-bit rows begin on 4-byte boundaries: strides must be multiples of 4");
  return 0;
}

// rows of a cache that is written: of two, neither reaches into the other
bool rows_apart(const fbgemm_amd_paged_cache& c, const int64_t (&strides)[3]) {
  const int64_t row = coded(c.row_ty) ? cache_row_bytes(c) : c.dim;
  const int64_t size[3] = {c.blocks, c.heads, c.block_size};
  for (int k = 0; k < 3; ++k)
    if (size[k] > 1 && strides[k] < row) return false;
  return true;
}

typedef __int128 wide; // strides are the caller's

// Rows of `row` bytes, `step` apart
struct Line {
  int64_t count, step;
  wide row;
  wide extent() const { return (wide)(count - 1) * step + row; }
  int64_t moves() const { return count > 1 ? step : 0; }
};
// whether rows of `a` and `b`, where every row begins at a multiple of `every` behind the first one of its kind, can share a byte; b's first is d behind a's
bool rows_within(wide a, wide b, wide d, int64_t every) {
  const wide r = (d % every + every) % every; // of b's rows behind a's, whole steps left out
  return r < a || every - r < b;
}
// Two lines, the second d bytes behind the first, that share a byte (or may, where neither step divides the other)
bool lines_meet(const Line& a, const Line& b, wide d) {
  if (d >= a.extent() || -d >= b.extent()) return false;
  const int64_t every = std::gcd(a.moves(), b.moves());
  return every == 0 || rows_within(a.row, b.row, d, every);
}
wide between(const void* a, const void* b) { return (wide)(uintptr_t)b - (wide)(uintptr_t)a; }
bool bytes_meet(const void* a, wide bytes_a, const void* b, wide bytes_b) { return between(a, b) < bytes_a && between(b, a) < bytes_b; }
// from a cache's first row to its last
wide cache_extent(const fbgemm_amd_paged_cache& c, const int64_t (&strides)[3]) {
  if (c.blocks == 0) return 0;
  return ((wide)(c.blocks - 1) * strides[0] + (wide)(c.heads - 1) * strides[1] + (wide)(c.block_size - 1) * strides[2]) * storage_bytes(c.row_ty) + cache_row_bytes(c);
}

// [tokens][heads][dim] as lines of rows: a token's heads, or a head's tokens, whichever are closer together. outer: these lines as solid rows
struct Grid {
  Line outer, inner;
  // no two elements are one
  bool apart() const { return (inner.count <= 1 || inner.step >= inner.row) && (outer.count <= 1 || outer.step >= outer.row); }
};
Grid grid_of(const fbgemm_amd_head_rows& r, const int64_t (&strides)[2], int64_t tokens, int64_t dim, int64_t element) {
  const int64_t size[2] = {tokens, r.heads};
  const int outer = r.heads == 1 || (tokens > 1 && strides[0] >= strides[1]) ? 0 : 1, inner = 1 - outer;
  Grid g;
  g.inner = Line{size[inner], strides[inner] * element, dim * element};
  g.outer = Line{size[outer], strides[outer] * element, g.inner.extent()};
  return g;
}
// Two grids that share a byte (or may, where they are laid out differently). What one has between its rows may be the other's: queries and
// keys of a projection [tokens][heads][3][dim] do not meet.
bool grids_meet(const void* a, const Grid& x, const void* b, const Grid& y) {
  const wide d = between(a, b);
  if (!lines_meet(x.outer, y.outer, d)) return false;
  const int64_t every = std::gcd(std::gcd(x.outer.moves(), x.inner.moves()), std::gcd(y.outer.moves(), y.inner.moves()));
  if (every != 0 && !rows_within(x.inner.row, y.inner.row, d, every)) return false;
  if (x.outer.moves() && y.outer.moves() && x.outer.step != y.outer.step) return true;
  const int64_t step = std::max(x.outer.moves(), y.outer.moves());
  if (step == 0) return lines_meet(x.inner, y.inner, d);
  // line j of y begins d + (j - i) * step behind line i of x: those that are near enough, of lines inside one step no more than two
  wide k = std::max<wide>(-(wide)(x.outer.count - 1), (-y.outer.row - d) / step - 1);
  const wide last = std::min<wide>(y.outer.count - 1, (x.outer.row - d) / step + 1);
  if (last - k > 8) return true;
  for (; k <= last; ++k)
    if (lines_meet(x.inner, y.inner, d + k * step)) return true;
  return false;
}

// a status block holds a 64-bit number that kernels update atomically
int check_status(const void* d_status) {
  return (uintptr_t)d_status % 8 ? fail(FBGEMM_AMD_E_ARG, "a status block begins on an 8-byte boundary") : 0;
}

CacheRows rows_of(void* base, const int64_t (&strides)[3], int32_t ty) {
  const int64_t e = storage_bytes(ty);
  return CacheRows{(char*)base, strides[0] * e, strides[1] * e, strides[2] * e};
}

// The device's compute units; the answer does not change, and a device that cannot be asked is taken for whole
int compute_units() {
  static thread_local int of[64] = {};
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 256;
  if (!of[dev]) {
    int n = 0;
    of[dev] = hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) == hipSuccess && n > 0 ? n : 256;
  }
  return of[dev];
}

// Workgroups of the attention kernel: as many as the device holds at once, but no more than there can be units of work
int attention_workers(const fbgemm_amd_paged_cache& c, int64_t requests, int32_t query_heads, int64_t max_tokens) {
  const int64_t sets = (int64_t)c.heads * ((query_heads / c.heads + ATTENTION_ROWS - 1) / ATTENTION_ROWS);
  const int64_t each = std::max<int64_t>(1, (max_tokens + 15 + ATTENTION_STEP - 1) / ATTENTION_STEP);
  const int64_t most = (int64_t)compute_units() * attention_residents(c.dim, c.row_ty == ST_CACHE_INT4 ? 4 : c.row_ty == ST_INT8 ? 8 : 16, c.block_size % 16 == 0);
  if (requests * sets >= most || each >= most) return (int)most;
  return (int)std::min(most, requests * sets * each);
}

int64_t attention_max_tokens(const fbgemm_amd_paged_cache& c, int64_t table_width) {
  if (c.blocks == 0) return 0;
  return std::min<int64_t>(table_width, (MOST - 4096) / c.block_size) * c.block_size;
}

struct AttentionSpace {
  int64_t partial, ml, joins, total;
};
AttentionSpace attention_space(int workers, int32_t dim) {
  AttentionSpace s;
  s.partial = (int64_t)workers * 2 * ATTENTION_ROWS * dim * (int64_t)sizeof(float);
  s.ml = (int64_t)workers * 2 * ATTENTION_ROWS * 2 * (int64_t)sizeof(float);
  s.joins = (int64_t)workers * (int64_t)sizeof(int4);
  s.total = s.partial + s.ml + s.joins;
  return s;
}

int check_attention(const fbgemm_amd_paged_cache* cache, int64_t requests, int32_t query_heads, int64_t table_width) {
  if (int rc = check_cache(cache)) return rc;
  if (cache->row_ty == ST_FP32) return fail(FBGEMM_AMD_E_UNSUPPORTED, "attention reads FP16, BF16 or INT8 rows, or CACHE_INT4 ones");
  if (cache->dim % 8 || cache->dim > 256) return fail(FBGEMM_AMD_E_UNSUPPORTED, "attention takes a dim that is a multiple of 8, up to 256: got %d", cache->dim);
  if (requests < 0 || requests > (1 << 24)) return fail(FBGEMM_AMD_E_ARG, "requests must be in 0..2^24");
  if (query_heads <= 0 || query_heads > (1 << 20) || query_heads % cache->heads)
    return fail(FBGEMM_AMD_E_ARG, "query heads must be a multiple of the cache's heads");
  if (table_width < 0) return fail(FBGEMM_AMD_E_ARG, "table_width must not be negative");
  const int64_t sets = (int64_t)cache->heads * ((query_heads / cache->heads + ATTENTION_ROWS - 1) / ATTENTION_ROWS);
  const int64_t units = attention_max_tokens(*cache, table_width) / ATTENTION_STEP + 3;
  if (requests > 0 && units > MOST / (requests * sets)) // requests * sets < 2^45
    return fail(FBGEMM_AMD_E_UNSUPPORTED, "tables for fewer than 2^31 times %d tokens, over all requests and heads, are supported", ATTENTION_STEP);
  return 0;
}

} // namespace

extern "C" {

int fbgemm_amd_kv_block_tables(
    const void* d_lengths, const void* d_new_tokens, int32_t index_bits, int64_t requests, int32_t* d_block_tables,
    int64_t table_stride, int64_t table_width, const int32_t* d_free_blocks, int64_t free_numel, const int32_t* d_free_start,
    int32_t block_size, int64_t num_tokens, int64_t* d_slots, int64_t* d_positions, int32_t* d_offsets, void* d_total_lengths,
    int32_t* d_free_next, void* d_status, void* stream) {
  if (index_bits != 32 && index_bits != 64) return fail(FBGEMM_AMD_E_ARG, "index_bits must be 32 or 64");
  if (requests < 0 || requests > MOST) return fail(FBGEMM_AMD_E_ARG, "requests must be in 0..2^31-1");
  if (block_size <= 0 || block_size > (1 << 20)) return fail(FBGEMM_AMD_E_ARG, "block_size must be in 1..1048576");
  if (table_width < 0 || table_width > (MOST - block_size) / block_size) return fail(FBGEMM_AMD_E_ARG, "a table must hold fewer than 2^31 tokens");
  if (requests > 1 && table_stride < table_width) return fail(FBGEMM_AMD_E_ARG, "tables must not overlap");
  if (free_numel < 0 || free_numel > MOST) return fail(FBGEMM_AMD_E_ARG, "the free list must hold fewer than 2^31 blocks");
  if (num_tokens < 0 || num_tokens > MOST) return fail(FBGEMM_AMD_E_ARG, "num_tokens must be in 0..2^31-1");
  if (!d_offsets || !d_free_start || !d_free_next || (requests > 0 && (!d_lengths || !d_new_tokens || !d_total_lengths)) ||
      (requests > 0 && table_width > 0 && !d_block_tables) || (free_numel > 0 && !d_free_blocks) || (num_tokens > 0 && (!d_slots || !d_positions)))
    return fail(FBGEMM_AMD_E_ARG, "null data pointer");
  if (int rc = check_status(d_status)) return rc;
  BlockTablesArgs a;
  a.lengths = d_lengths;
  a.new_tokens = d_new_tokens;
  a.R = requests;
  a.tables = d_block_tables;
  a.table_stride = table_stride;
  a.width = table_width;
  a.free_blocks = d_free_blocks;
  a.free_numel = free_numel;
  a.free_start = d_free_start;
  a.block = make_divisor((uint32_t)block_size);
  a.num_tokens = num_tokens;
  a.slots = d_slots;
  a.positions = d_positions;
  a.offsets = d_offsets;
  a.total_lengths = d_total_lengths;
  a.free_next = d_free_next;
  a.status = (Status*)d_status;
  HIP_TRY(launch_kv_block_tables(a, index_bits == 64, (hipStream_t)stream));
  return 0;
}

int fbgemm_amd_kv_cache_append(
    const fbgemm_amd_paged_cache* cache, const void* d_key, const void* d_value, int32_t input_ty, int64_t tokens,
    const int64_t* key_strides, const int64_t* value_strides, const int64_t* d_slots, void* d_key_cache, void* d_value_cache,
    void* d_status, void* stream) {
  if (int rc = check_cache(cache)) return rc;
  const bool codes = coded(cache->row_ty);
  if (input_ty != ST_FP32 && input_ty != ST_FP16 && input_ty != ST_BF16) return fail(FBGEMM_AMD_E_ARG, "keys and values are FP32, FP16 or BF16");
  if (!codes && input_ty != cache->row_ty) return fail(FBGEMM_AMD_E_ARG, "rows are stored as they come: the cache's type must be the keys'");
  if (tokens < 0 || tokens > MOST) return fail(FBGEMM_AMD_E_ARG, "tokens must be in 0..2^31-1");
  if (tokens == 0) return 0;
  if (!key_strides || !value_strides || !d_key || !d_value || !d_slots) return fail(FBGEMM_AMD_E_ARG, "null data pointer");
  if (cache->blocks > 0 && (!d_key_cache || !d_value_cache)) return fail(FBGEMM_AMD_E_ARG, "null data pointer");
  if (int rc = check_status(d_status)) return rc;
  AppendArgs a;
  const int64_t e = storage_bytes(input_ty);
  a.in[0] = (const char*)d_key;
  a.in[1] = (const char*)d_value;
  for (int k = 0; k < 2; ++k) {
    const int64_t* s = k ? value_strides : key_strides;
    if (s[0] < 0 || s[1] < 0) return fail(FBGEMM_AMD_E_ARG, "strides must not be negative");
    a.token_stride[k] = s[0] * e;
    a.head_stride[k] = s[1] * e;
  }
  a.cache[0] = rows_of(d_key_cache, cache->key_strides, cache->row_ty);
  a.cache[1] = rows_of(d_value_cache, cache->value_strides, cache->row_ty);
  a.slots = d_slots;
  a.tokens = tokens;
  a.total_slots = cache->blocks * cache->block_size;
  a.heads = cache->heads;
  a.dim = cache->dim;
  a.row_bytes = (int32_t)(cache->dim * e);
  a.block = make_divisor((uint32_t)cache->block_size);
  a.per_row = make_divisor(1);
  a.status = (Status*)d_status;
  // one cache for both holds the same rows twice, or which of the two is left to chance
  const auto check_shared = [&]() -> int {
    const bool same = d_key == d_value && key_strides[0] == value_strides[0] && key_strides[1] == value_strides[1];
    return d_key_cache == d_value_cache && cache->blocks > 0 && !same ? fail(FBGEMM_AMD_E_ARG, "keys and values that differ must not overlap in the cache") : 0;
  };
  if (!rows_apart(*cache, cache->key_strides) || !rows_apart(*cache, cache->value_strides)) return fail(FBGEMM_AMD_E_ARG, "rows of a cache must not overlap");
  if (codes) {
    if ((uintptr_t)d_key_cache % 4 || (uintptr_t)d_value_cache % 4) return fail(FBGEMM_AMD_E_ARG, "8-bit and 4-bit rows begin on 4-byte boundaries");
    if (int rc = check_shared()) return rc;
    const bool aligned16 = (uintptr_t)d_key % 16 == 0 && (uintptr_t)d_value % 16 == 0 &&
        divides(16, {a.token_stride[0], a.head_stride[0], a.token_stride[1], a.head_stride[1]});
    HIP_TRY(launch_kv_append_coded(a, cache->row_ty == ST_INT8 ? 8 : 4, input_ty, aligned16, (hipStream_t)stream));
    return 0;
  }
  // the largest piece that every row is made of and begins at
  int piece = 16;
  const auto fits = [&](int p) {
    bool ok = a.row_bytes % p == 0;
    for (int k = 0; k < 2; ++k)
      ok = ok && divides(p, {a.token_stride[k], a.head_stride[k], a.cache[k].block_stride, a.cache[k].head_stride, a.cache[k].slot_stride}) &&
          (uintptr_t)a.in[k] % p == 0 && (uintptr_t)a.cache[k].base % p == 0;
    return ok;
  };
  while (piece > 2 && !fits(piece)) piece >>= 1;
  if (!fits(piece)) return fail(FBGEMM_AMD_E_ARG, "rows are not aligned to their elements");
  if (int rc = check_shared()) return rc;
  a.per_row = make_divisor((uint32_t)(a.row_bytes / piece));
  HIP_TRY(launch_kv_append(a, piece, (hipStream_t)stream));
  return 0;
}

int fbgemm_amd_kv_cache_read(
    const fbgemm_amd_paged_cache* cache, const void* d_key_cache, const void* d_value_cache, const int32_t* d_block_tables,
    int64_t table_stride, int64_t table_width, const void* d_offsets, const void* d_starts, int32_t index_bits, int64_t requests,
    int64_t tokens, int32_t output_ty, void* d_key, void* d_value, void* d_status, void* stream) {
  if (int rc = check_cache(cache)) return rc;
  const bool codes = coded(cache->row_ty);
  if (output_ty != ST_FP32 && output_ty != ST_FP16 && output_ty != ST_BF16) return fail(FBGEMM_AMD_E_ARG, "keys and values are FP32, FP16 or BF16");
  if (!codes && output_ty != cache->row_ty) return fail(FBGEMM_AMD_E_ARG, "rows come as they are stored: the keys' type must be the cache's");
  if (index_bits != 32 && index_bits != 64) return fail(FBGEMM_AMD_E_ARG, "index_bits must be 32 or 64");
  if (requests < 0 || requests > MOST - 1) return fail(FBGEMM_AMD_E_ARG, "requests must be in 0..2^31-2");
  if (tokens < 0 || tokens > MOST) return fail(FBGEMM_AMD_E_ARG, "tokens must be in 0..2^31-1");
  if (table_width < 0 || table_width > (MOST - cache->block_size) / cache->block_size) return fail(FBGEMM_AMD_E_ARG, "a table must hold fewer than 2^31 tokens");
  if (tokens == 0) return 0;
  if (!d_key || !d_value || !d_offsets || (requests > 0 && table_width > 0 && !d_block_tables) || (cache->blocks > 0 && (!d_key_cache || !d_value_cache)))
    return fail(FBGEMM_AMD_E_ARG, "null data pointer");
  if ((uintptr_t)d_key % 16 || (uintptr_t)d_value % 16) return fail(FBGEMM_AMD_E_ARG, "keys and values must begin on 16-byte boundaries");
  if (int rc = check_status(d_status)) return rc;
  ReadArgs a;
  a.cache[0] = rows_of(const_cast<void*>(d_key_cache), cache->key_strides, cache->row_ty);
  a.cache[1] = rows_of(const_cast<void*>(d_value_cache), cache->value_strides, cache->row_ty);
  a.out[0] = (char*)d_key;
  a.out[1] = (char*)d_value;
  a.tables = d_block_tables;
  a.table_stride = table_stride;
  a.table_width = table_width;
  a.offsets = d_offsets;
  a.starts = d_starts;
  a.idx64 = index_bits == 64;
  a.requests = (int32_t)requests;
  a.heads = cache->heads;
  a.dim = cache->dim;
  a.blocks = (int32_t)cache->blocks;
  a.tokens = tokens;
  a.block = make_divisor((uint32_t)cache->block_size);
  a.status = (Status*)d_status;
  const auto pieces = [&](int32_t of_row) {
    a.per_row = make_divisor((uint32_t)of_row);
    a.per_token = make_divisor((uint32_t)(of_row * cache->heads)); // heads * dim is at most 2^28
  };
  const auto on = [&](int64_t p) {
    bool ok = true;
    for (const CacheRows& c : a.cache) ok = ok && divides(p, {c.block_stride, c.head_stride, c.slot_stride}) && (uintptr_t)c.base % p == 0;
    return ok;
  };
  const auto check_apart = [&]() { // a row may be read after another one's thread has written
    const wide bytes = (wide)tokens * cache->heads * cache->dim * storage_bytes(output_ty);
    if (bytes_meet(d_key, bytes, d_value, bytes)) return fail(FBGEMM_AMD_E_ARG, "keys and values must not overlap");
    for (const char* out : a.out)
      if (bytes_meet(out, bytes, d_key_cache, cache_extent(*cache, cache->key_strides)) || bytes_meet(out, bytes, d_value_cache, cache_extent(*cache, cache->value_strides)))
        return fail(FBGEMM_AMD_E_ARG, "keys and values must not overlap the cache");
    return 0;
  };
  if (codes) {
    if (!on(4)) return fail(FBGEMM_AMD_E_ARG, "8-bit and 4-bit rows begin on 4-byte boundaries");
    if (int rc = check_apart()) return rc;
    const bool whole = cache->dim % READ_RUN == 0;
    pieces(whole ? cache->dim / READ_RUN : cache->dim);
    HIP_TRY(launch_kv_read_coded(a, cache->row_ty == ST_INT8 ? 8 : 4, output_ty, whole, (hipStream_t)stream));
    return 0;
  }
  const int32_t row_bytes = cache_row_bytes(*cache);
  int piece = 16;
  const auto fits = [&](int p) { return row_bytes % p == 0 && on(p); };
  while (piece > 2 && !fits(piece)) piece >>= 1;
  if (!fits(piece)) return fail(FBGEMM_AMD_E_ARG, "rows are not aligned to their elements");
  if (int rc = check_apart()) return rc;
  pieces(row_bytes / piece);
  HIP_TRY(launch_kv_read(a, piece, (hipStream_t)stream));
  return 0;
}

int fbgemm_amd_rotate_positions(
    const fbgemm_amd_head_rows* query, const fbgemm_amd_head_rows* key, int32_t ty, int64_t tokens, int32_t dim,
    const void* d_positions, int32_t index_bits, const double* d_frequencies, int32_t pairs, int32_t interleaved,
    float magnitude, int32_t inverse, void* stream) {
  if (!query) return fail(FBGEMM_AMD_E_ARG, "query is null");
  if (ty != ST_FP32 && ty != ST_FP16 && ty != ST_BF16) return fail(FBGEMM_AMD_E_ARG, "queries and keys are FP32, FP16 or BF16");
  if (index_bits != 32 && index_bits != 64) return fail(FBGEMM_AMD_E_ARG, "index_bits must be 32 or 64");
  if (tokens < 0 || tokens > MOST) return fail(FBGEMM_AMD_E_ARG, "tokens must be in 0..2^31-1");
  if (dim <= 0 || dim > (1 << 16)) return fail(FBGEMM_AMD_E_ARG, "dim must be in 1..65536");
  if (pairs < 0 || 2 * (int64_t)pairs > dim || pairs > ROTATE_MOST_PAIRS) return fail(FBGEMM_AMD_E_ARG, "a head of %d has at most %d pairs, and no more than %d are turned", dim, dim / 2, ROTATE_MOST_PAIRS);
  if (!std::isfinite(magnitude)) return fail(FBGEMM_AMD_E_ARG, "magnitude must be finite");
  const fbgemm_amd_head_rows* of[2] = {query, key};
  int64_t heads = 0;
  for (const auto* r : of) {
    if (!r) continue;
    if (r->heads < 0 || r->heads > (1 << 16)) return fail(FBGEMM_AMD_E_ARG, "heads must be in 0..65536");
    for (int k = 0; k < 2; ++k)
      if (r->in_strides[k] < 0 || r->out_strides[k] < 0) return fail(FBGEMM_AMD_E_ARG, "strides must not be negative");
    heads += r->heads;
  }
  if (heads * dim > (1 << 28)) return fail(FBGEMM_AMD_E_ARG, "heads * dim must not exceed 2^28");
  if (tokens == 0 || heads == 0) return 0;
  if (!d_positions || (pairs > 0 && !d_frequencies)) return fail(FBGEMM_AMD_E_ARG, "null data pointer");
  RotateArgs a = {};
  const int64_t e = storage_bytes(ty);
  bool aligned16 = true;
  for (int k = 0; k < 2; ++k) {
    const auto* r = of[k];
    if (!r || r->heads == 0) continue;
    if (!r->in || !r->out) return fail(FBGEMM_AMD_E_ARG, "null data pointer");
    if ((uintptr_t)r->in % e || (uintptr_t)r->out % e) return fail(FBGEMM_AMD_E_ARG, "rows are not aligned to their elements");
    if (!grid_of(*r, r->out_strides, tokens, dim, e).apart()) return fail(FBGEMM_AMD_E_ARG, "rows of a result must not overlap");
    a.in[k] = (const char*)r->in;
    a.out[k] = (char*)r->out;
    a.in_token[k] = r->in_strides[0] * e;
    a.in_head[k] = r->in_strides[1] * e;
    a.out_token[k] = r->out_strides[0] * e;
    a.out_head[k] = r->out_strides[1] * e;
    a.heads[k] = r->heads;
    aligned16 = aligned16 && divides(16, {a.in_token[k], a.in_head[k], a.out_token[k], a.out_head[k]}) && (uintptr_t)r->in % 16 == 0 && (uintptr_t)r->out % 16 == 0;
  }
  for (int k = 0; k < 2; ++k)
    for (int i = 0; i < 2; ++i) {
      if (!a.heads[k] || !a.heads[i]) continue;
      const bool in_place = i == k && a.in[k] == a.out[k] && (tokens == 1 || a.in_token[k] == a.out_token[k]) && (a.heads[k] == 1 || a.in_head[k] == a.out_head[k]);
      const Grid out = grid_of(*of[k], of[k]->out_strides, tokens, dim, e);
      if (!in_place && grids_meet(a.in[i], grid_of(*of[i], of[i]->in_strides, tokens, dim, e), a.out[k], out))
        return fail(FBGEMM_AMD_E_ARG, "a result may be its own input, but must not overlap inputs otherwise");
      if (i < k && grids_meet(a.out[i], grid_of(*of[i], of[i]->out_strides, tokens, dim, e), a.out[k], out))
        return fail(FBGEMM_AMD_E_ARG, "the results must not overlap each other");
    }
  a.dim = dim;
  a.pairs = pairs;
  a.tokens = tokens;
  a.positions = d_positions;
  a.idx64 = index_bits == 64;
  a.interleaved = interleaved != 0;
  a.frequencies = d_frequencies;
  a.magnitude = magnitude;
  a.sine = inverse ? -magnitude : magnitude;
  HIP_TRY(launch_rotate_positions(a, ty, aligned16, (hipStream_t)stream));
  return 0;
}

int64_t fbgemm_amd_paged_attention_workspace(const fbgemm_amd_paged_cache* cache, int64_t requests, int32_t query_heads, int64_t table_width) {
  if (int rc = check_attention(cache, requests, query_heads, table_width)) return rc;
  if (requests == 0) return 0;
  return attention_space(attention_workers(*cache, requests, query_heads, attention_max_tokens(*cache, table_width)), cache->dim).total;
}

int fbgemm_amd_paged_attention_form(const fbgemm_amd_paged_cache* cache) {
  if (int rc = check_attention(cache, 1, cache ? cache->heads : 1, 1)) return rc;
  const int64_t e = storage_bytes(cache->row_ty);
  return attention_form(cache->dim, cache->row_ty == ST_CACHE_INT4 ? 4 : cache->row_ty == ST_INT8 ? 8 : 16, cache->block_size, cache->key_strides[2] * e, cache->value_strides[2] * e);
}

int fbgemm_amd_paged_attention(
    const fbgemm_amd_paged_cache* cache, const void* d_query, int32_t query_ty, int64_t requests, int32_t query_heads,
    int64_t query_request_stride, int64_t query_head_stride, const void* d_key_cache, const void* d_value_cache,
    const int32_t* d_block_tables, int64_t table_stride, int64_t table_width, const void* d_lengths, int32_t index_bits,
    float scale, int64_t window, float softcap, void* d_output, float* d_lse, void* d_workspace, int64_t workspace_bytes, void* stream) {
  if (int rc = check_attention(cache, requests, query_heads, table_width)) return rc;
  const bool codes = coded(cache->row_ty);
  if (query_ty != ST_FP16 && query_ty != ST_BF16) return fail(FBGEMM_AMD_E_UNSUPPORTED, "queries are FP16 or BF16");
  if (!codes && query_ty != cache->row_ty) return fail(FBGEMM_AMD_E_ARG, "16-bit rows must have the queries' type");
  if (index_bits != 32 && index_bits != 64) return fail(FBGEMM_AMD_E_ARG, "index_bits must be 32 or 64");
  if (window < 0) return fail(FBGEMM_AMD_E_ARG, "window must not be negative");
  if (!std::isfinite(scale)) return fail(FBGEMM_AMD_E_ARG, "scale must be finite");
  if (!(softcap >= 0.0f) || !std::isfinite(softcap)) return fail(FBGEMM_AMD_E_ARG, "softcap must be finite and not negative");
  if (requests == 0) return 0;
  const int64_t max_tokens = attention_max_tokens(*cache, table_width);
  if (!d_query || !d_lengths || !d_output || !d_lse || !d_workspace || (max_tokens > 0 && (!d_block_tables || !d_key_cache || !d_value_cache)))
    return fail(FBGEMM_AMD_E_ARG, "null data pointer");
  AttentionArgs a;
  a.query = (const char*)d_query;
  a.query_request_stride = query_request_stride * 2;
  a.query_head_stride = query_head_stride * 2;
  a.key = rows_of(const_cast<void*>(d_key_cache), cache->key_strides, cache->row_ty);
  a.value = rows_of(const_cast<void*>(d_value_cache), cache->value_strides, cache->row_ty);
  const int64_t row_align = codes ? 4 : 16;
  bool aligned = divides(16, {a.query_request_stride, a.query_head_stride}) && (uintptr_t)d_query % 16 == 0;
  if (a.key.slot_stride >= (1 << 26) || a.value.slot_stride >= (1 << 26)) return fail(FBGEMM_AMD_E_UNSUPPORTED, "tokens of a block must be less than 64 MiB apart");
  for (const CacheRows* r : {&a.key, &a.value})
    aligned = aligned && divides(row_align, {r->block_stride, r->head_stride, r->slot_stride}) && (uintptr_t)r->base % row_align == 0;
  if (!aligned) return fail(FBGEMM_AMD_E_ARG, "queries and 16-bit rows must begin on 16-byte boundaries, 8-bit and 4-bit rows on 4-byte ones");
  if ((uintptr_t)d_output % 16 || (uintptr_t)d_workspace % 16) return fail(FBGEMM_AMD_E_ARG, "output and workspace must begin on 16-byte boundaries");
  a.tables = d_block_tables;
  a.table_stride = table_stride;
  a.lengths = d_lengths;
  a.idx64 = index_bits == 64;
  a.requests = (int32_t)requests;
  a.kv_heads = cache->heads;
  a.group = query_heads / cache->heads;
  a.q_tiles = (a.group + ATTENTION_ROWS - 1) / ATTENTION_ROWS;
  a.dim = cache->dim;
  a.blocks = (int32_t)cache->blocks;
  a.block_size = cache->block_size;
  a.max_tokens = max_tokens;
  a.block = make_divisor((uint32_t)cache->block_size);
  constexpr double LOG2E = 1.4426950408889634;
  a.scale = (float)(scale * LOG2E);
  int up = 0;
  a.scale_part = (float)std::frexp(std::max(std::fabs(scale * LOG2E), (double)std::numeric_limits<float>::min()), &up);
  a.scale_up = up;
  // normal and of a finite inverse for the smallest cap too: a score of zero times infinity would be none
  const double cap = softcap > 0.0f ? std::max(softcap * LOG2E, (double)std::numeric_limits<float>::min()) : 0.0;
  a.softcap = (float)cap;
  a.cap_inverse = softcap > 0.0f ? (float)(1.0 / cap) : 0.0f;
  a.window = window;
  a.out = (char*)d_output;
  a.lse = d_lse;
  a.workers = attention_workers(*cache, requests, query_heads, max_tokens);
  const AttentionSpace space = attention_space(a.workers, cache->dim);
  if (workspace_bytes < space.total) return fail(FBGEMM_AMD_E_ARG, "workspace of %lld bytes: %lld are needed", (long long)workspace_bytes, (long long)space.total);
  a.partial = (float*)d_workspace;
  a.partial_ml = (float*)((char*)d_workspace + space.partial);
  a.joins = (int4*)((char*)d_workspace + space.partial + space.ml);
  const bool bf16 = query_ty == ST_BF16;
  hipError_t (*const launch)(const AttentionArgs&, hipStream_t) =
      cache->row_ty == ST_INT8 ? (bf16 ? launch_paged_attention_bf16_rows8 : launch_paged_attention_fp16_rows8)
      : cache->row_ty == ST_CACHE_INT4 ? (bf16 ? launch_paged_attention_bf16_rows4 : launch_paged_attention_fp16_rows4)
                                       : (bf16 ? launch_paged_attention_bf16 : launch_paged_attention_fp16);
  HIP_TRY(launch(a, (hipStream_t)stream));
  return 0;
}

int fbgemm_amd_penalize_logits(
    const void* d_logits, int32_t logits_ty, int64_t rows, int64_t vocab, int64_t logits_stride, const void* d_tokens,
    int64_t tokens_numel, const void* d_offsets, const void* d_prompt_lengths, int32_t index_bits, const float* d_repetition,
    const float* d_frequency, const float* d_presence, const void* d_bias_ids, const float* d_bias_values, int64_t bias_numel,
    const void* d_bias_offsets, const int32_t* d_mask, int64_t mask_stride, void* d_output, int64_t output_stride, void* stream) {
  if (logits_ty != ST_FP32 && logits_ty != ST_FP16 && logits_ty != ST_BF16) return fail(FBGEMM_AMD_E_ARG, "logits are FP32, FP16 or BF16");
  if (index_bits != 32 && index_bits != 64) return fail(FBGEMM_AMD_E_ARG, "index_bits must be 32 or 64");
  if (rows < 0 || rows > (1 << 24) || vocab < 0 || vocab > MOST) return fail(FBGEMM_AMD_E_ARG, "rows must be in 0..2^24, vocab in 0..2^31-1");
  if (tokens_numel < 0 || tokens_numel > MOST || bias_numel < 0 || bias_numel > MOST) return fail(FBGEMM_AMD_E_ARG, "lists must hold fewer than 2^31 entries");
  if (rows == 0 || vocab == 0) return 0;
  if (!d_logits || !d_output) return fail(FBGEMM_AMD_E_ARG, "null data pointer");
  if (rows > 1 && ((logits_stride != 0 && logits_stride < vocab) || output_stride < vocab)) return fail(FBGEMM_AMD_E_ARG, "rows must not overlap");
  if (tokens_numel > 0 && (!d_tokens || !d_offsets)) return fail(FBGEMM_AMD_E_ARG, "tokens need their offsets");
  if (bias_numel > 0 && (!d_bias_ids || !d_bias_values || !d_bias_offsets)) return fail(FBGEMM_AMD_E_ARG, "biases need ids, values and offsets");
  if (d_mask && rows > 1 && mask_stride != 0 && mask_stride < (vocab + 31) / 32) return fail(FBGEMM_AMD_E_ARG, "a row of the mask has one bit per token of the vocabulary");
  const int64_t e = storage_bytes(logits_ty);
  const bool in_place = d_output == d_logits && (rows == 1 || output_stride == logits_stride);
  if (!in_place && lines_meet(Line{rows, logits_stride * e, vocab * e}, Line{rows, output_stride * e, vocab * e}, between(d_logits, d_output)))
    return fail(FBGEMM_AMD_E_ARG, "the result may be the logits themselves, but must not overlap them otherwise");
  LogitsArgs a;
  a.logits = d_logits;
  a.out = d_output;
  a.rows = rows;
  a.vocab = vocab;
  a.logits_stride = logits_stride;
  a.out_stride = output_stride;
  a.tokens = tokens_numel > 0 ? d_tokens : nullptr;
  a.offsets = d_offsets;
  a.prompt_lengths = d_prompt_lengths;
  a.tokens_numel = tokens_numel;
  a.repetition = d_repetition;
  a.frequency = d_frequency;
  a.presence = d_presence;
  a.bias_ids = bias_numel > 0 ? d_bias_ids : nullptr;
  a.bias_values = d_bias_values;
  a.bias_offsets = d_bias_offsets;
  a.bias_numel = bias_numel;
  a.mask = (const uint32_t*)d_mask;
  a.mask_stride = mask_stride;
  HIP_TRY(launch_penalize_logits(a, logits_ty, index_bits == 64, (hipStream_t)stream));
  return 0;
}

int fbgemm_amd_sample_tokens(
    const void* d_logits, int32_t logits_ty, int64_t rows, int64_t vocab, int64_t logits_stride, const float* d_uniform,
    const float* d_temperature, const int32_t* d_top_k, const float* d_top_p, const float* d_min_p, int64_t* d_tokens,
    float* d_log_probability, void* stream) {
  if (logits_ty != ST_FP32 && logits_ty != ST_FP16 && logits_ty != ST_BF16) return fail(FBGEMM_AMD_E_ARG, "logits are FP32, FP16 or BF16");
  if (rows < 0 || rows > (1 << 24)) return fail(FBGEMM_AMD_E_ARG, "rows must be in 0..2^24");
  if (vocab < 1 || vocab > SAMPLE_MOST_VOCAB) return fail(FBGEMM_AMD_E_ARG, "vocab must be in 1..2^20");
  if (rows == 0) return 0;
  if (!d_logits || !d_uniform || !d_tokens || !d_log_probability) return fail(FBGEMM_AMD_E_ARG, "null data pointer");
  if (logits_stride < 0) return fail(FBGEMM_AMD_E_ARG, "strides must not be negative");
  if ((uintptr_t)d_logits % storage_bytes(logits_ty)) return fail(FBGEMM_AMD_E_ARG, "rows are not aligned to their elements");
  SampleArgs a;
  a.logits = d_logits;
  a.rows = rows;
  a.stride = rows > 1 ? logits_stride : 0;
  a.vocab = (int32_t)vocab;
  a.compute_units = compute_units();
  a.uniform = d_uniform;
  a.temperature = d_temperature;
  a.top_k = d_top_k;
  a.top_p = d_top_p;
  a.min_p = d_min_p;
  a.tokens = d_tokens;
  a.log_probability = d_log_probability;
  HIP_TRY(launch_sample_tokens(a, logits_ty, (hipStream_t)stream));
  return 0;
}

} // extern "C"
