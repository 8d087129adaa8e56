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
hipError_t launch_kv_append_rows8(const AppendArgs& a, int32_t input_ty, bool aligned16, hipStream_t stream); // aligned16: input rows are

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
// workgroups of the attention kernel that a compute unit holds at once: what its registers leave room for
constexpr int attention_residents(int dim) { return dim > 128 ? 1 : dim > 64 ? 2 : 3; }
constexpr int ATTENTION_ROWS = 16; // queries of a key head that one tile of the matrix cores takes
hipError_t launch_paged_attention_bf16(const AttentionArgs& a, hipStream_t stream);
hipError_t launch_paged_attention_fp16(const AttentionArgs& a, hipStream_t stream);
hipError_t launch_paged_attention_bf16_rows8(const AttentionArgs& a, hipStream_t stream);
hipError_t launch_paged_attention_fp16_rows8(const AttentionArgs& a, hipStream_t stream);

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

} // namespace fbgemm_amd
