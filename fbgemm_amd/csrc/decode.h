// Arguments and launchers of the operators of a decoding step over a paged key-value cache
// (host side: decode_api.cpp).
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

#include "lookup_common.h"

namespace fbgemm_amd {

// n / d for 0 <= n < 2^31 as (n * magic) >> shift
struct Divisor {
  uint32_t d, magic, shift;
};
inline Divisor make_divisor(uint32_t d) {
  uint32_t s = 0;
  while ((1ull << s) < d) ++s;
  // ceil(2^(31 + s) / d) <= 2^32 - 1 for d >= 2; one has to be its own case
  return d == 1 ? Divisor{1, 1, 0} : Divisor{d, (uint32_t)(((1ull << (31 + s)) + d - 1) / d), 31 + s};
}
#if defined(__HIPCC__)
__device__ __forceinline__ uint32_t divide(uint32_t n, const Divisor& v) { return (uint32_t)(((uint64_t)n * v.magic) >> v.shift); }
#endif

struct BlockTablesArgs {
  const void* lengths;    // [R]
  const void* new_tokens; // [R]
  int64_t R;
  int32_t* tables; // [R][table_stride], width entries each
  int64_t table_stride, width;
  const int32_t* free_blocks;
  int64_t free_numel;
  const int32_t* free_start;
  Divisor block;
  int64_t num_tokens;
  int64_t* slots;
  int64_t* positions;
  int32_t* offsets;    // [R + 1]
  void* total_lengths; // [R]
  int32_t* free_next;
  Status* status;
};
hipError_t launch_kv_block_tables(const BlockTablesArgs& a, bool idx64, hipStream_t stream);

// A cache is [blocks][heads][block_size][row]; strides (in bytes) of the first three, rows without gaps.
struct CacheRows {
  char* base;
  int64_t block_stride, head_stride, slot_stride;
};
struct AppendArgs {
  const char* in[2]; // key, value: [tokens][heads][dim]
  int64_t token_stride[2], head_stride[2]; // bytes
  CacheRows cache[2];
  const int64_t* slots;
  int64_t tokens, total_slots;
  int32_t heads, dim, row_bytes; // of one input row
  Divisor block, per_row;        // per_row: pieces of a row
  Status* status;
};
hipError_t launch_kv_append(const AppendArgs& a, int piece_bytes, hipStream_t stream);
// rows of `bits` (8 or 4); aligned16: input rows are
hipError_t launch_kv_append_coded(const AppendArgs& a, int bits, int32_t input_ty, bool aligned16, hipStream_t stream);

// Rows of requests' tokens, out of their pages into dense arrays
struct ReadArgs {
  CacheRows cache[2]; // key, value
  char* out[2];       // [tokens][heads][dim], dense
  const int32_t* tables;
  int64_t table_stride, table_width;
  const void* offsets; // [requests + 1]
  const void* starts;  // [requests] or null: zeros
  int32_t idx64;
  int32_t requests, heads, dim, blocks;
  int64_t tokens;
  Divisor block, per_row, per_token; // per_row, per_token: pieces of a row, and of a token's rows
  Status* status;
};
constexpr int READ_RUN = 8; // codes of a piece
hipError_t launch_kv_read(const ReadArgs& a, int piece_bytes, hipStream_t stream);                          // rows as they are
hipError_t launch_kv_read_coded(const ReadArgs& a, int bits, int32_t output_ty, bool whole, hipStream_t stream); // whole: rows are whole pieces

// Queries and keys turned by their positions
struct RotateArgs {
  const char* in[2]; // queries, keys: [tokens][heads][dim]
  char* out[2];
  int64_t in_token[2], in_head[2], out_token[2], out_head[2]; // bytes
  int32_t heads[2], dim, pairs;                                // heads[1] may be 0
  int64_t tokens;
  const void* positions;
  int32_t idx64, interleaved;
  const double* frequencies; // [pairs], radians a position
  float magnitude, sine;     // of cosines and sines: sine is -magnitude where turning back
  Divisor units;             // pieces of work of a head
};
constexpr int ROTATE_MOST_PAIRS = 1024; // their sines are in LDS
hipError_t launch_rotate_positions(const RotateArgs& a, int32_t ty, bool aligned16, hipStream_t stream);

struct AttentionArgs {
  const char* query; // [requests][heads][dim], 16 bits
  int64_t query_request_stride, query_head_stride; // bytes
  CacheRows key, value;
  const int32_t* tables;
  int64_t table_stride;
  const void* lengths;
  int32_t idx64;
  int32_t requests, kv_heads, group, q_tiles, dim;
  int32_t blocks, block_size;
  int64_t max_tokens; // table width * block size
  Divisor block;
  float scale;       // of the scores, times log2(e)
  float scale_part;  // |scale| (but at least the smallest normal number) is scale_part * 2^scale_up, scale_part in [1/2, 1]
  int32_t scale_up;
  float softcap;     // times log2(e); 0: none
  float cap_inverse; // 1 / softcap
  int64_t window; // 0: none
  char* out; // [requests][heads][dim], dense
  float* lse; // [requests][heads]
  // workspace
  int32_t workers;
  float* partial;     // [workers][2][rows][dim]
  float* partial_ml;  // [workers][2][rows][2]
  int4* joins;        // [workers]: the last worker of the pair that begins with this one (-1: none goes on), its rows, the first of them
};
constexpr int ATTENTION_STEP = 128; // tokens of a unit of work
// Workgroups of the attention kernel that a compute unit holds at once: what its registers leave room for. bits: of an element of the
// rows; pages: whole tiles of 16 tokens. 4-bit rows in such pages, 256 requests of 16 to 8 192 tokens, times three with one tile on its way: two
// with two tiles 1.06, with three 1.11; three with two tiles do not fit the registers, 1.40.
constexpr int attention_residents(int dim, int bits, bool pages) {
  if (dim > 128) return 1;
  if (bits == 4) return pages ? 3 : 2;
  return dim > 64 ? 2 : 3;
}
// How the attention kernel finds rows of `bits` bits: lane by lane; in pages of whole tiles of 16 tokens, whose addresses are the wave's; or there as
// runs of bytes, where a page's rows follow each other without gaps and 16 of them are what its loads are laid out for (however far apart
// pages are, of keys or of values).
enum AttentionForm : int { ATTENTION_LANES, ATTENTION_PAGES, ATTENTION_RUNS };
constexpr bool attention_has_runs(int dim, int bits) { return bits == 8 ? dim == 64 || dim == 128 || dim == 256 : bits == 4 && (dim == 128 || dim == 256); }
inline AttentionForm attention_form(int dim, int bits, int block_size, int64_t key_slot_stride, int64_t value_slot_stride) {
  if (block_size % 16) return ATTENTION_LANES;
  const int64_t row = dim * bits / 8 + 4;
  return attention_has_runs(dim, bits) && key_slot_stride == row && value_slot_stride == row ? ATTENTION_RUNS : ATTENTION_PAGES;
}
constexpr int ATTENTION_ROWS = 16; // queries of a key head that one tile of the matrix cores takes
hipError_t launch_paged_attention_bf16(const AttentionArgs& a, hipStream_t stream);
hipError_t launch_paged_attention_fp16(const AttentionArgs& a, hipStream_t stream);
hipError_t launch_paged_attention_bf16_rows8(const AttentionArgs& a, hipStream_t stream);
hipError_t launch_paged_attention_fp16_rows8(const AttentionArgs& a, hipStream_t stream);
hipError_t launch_paged_attention_bf16_rows4(const AttentionArgs& a, hipStream_t stream);
hipError_t launch_paged_attention_fp16_rows4(const AttentionArgs& a, hipStream_t stream);

struct LogitsArgs {
  const void* logits;
  void* out;
  int64_t rows, vocab, logits_stride, out_stride; // elements
  const void* tokens;
  const void* offsets;        // [rows + 1]
  const void* prompt_lengths; // [rows] or null
  int64_t tokens_numel;
  const float* repetition;
  const float* frequency;
  const float* presence;
  const void* bias_ids;
  const float* bias_values;
  const void* bias_offsets;
  int64_t bias_numel;
  const uint32_t* mask;
  int64_t mask_stride; // words
};
hipError_t launch_penalize_logits(const LogitsArgs& a, int32_t ty, bool idx64, hipStream_t stream);

struct SampleArgs {
  const void* logits;
  int64_t rows, stride; // stride: elements
  int32_t vocab, compute_units; // the device's
  const float* uniform;
  const float* temperature; // [rows] or null, as the next ones
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  int64_t* tokens;
  float* log_probability;
};
constexpr int SAMPLE_MOST_VOCAB = 1 << 20;
hipError_t launch_sample_tokens(const SampleArgs& a, int32_t ty, hipStream_t stream);

} // namespace fbgemm_amd
