/*
 * fbgemm_amd -- C ABI of the MI355X (gfx950) quantized embedding-bag library.
 *
 * Every data pointer named d_* is a DEVICE pointer (HBM). `stream` is a
 * hipStream_t passed as void* (NULL = the default stream). Launch calls are
 * asynchronous: they enqueue on `stream` and return. Nothing is allocated per
 * call except where a function says so.
 *
 * Return values: 0 = enqueued / done, < 0 = FBGEMM_AMD_E_* (bad argument or a
 * HIP error). Input errors that the reference reports by returning false
 * (index out of range, bag overrun, length mismatch) are detected ON THE
 * DEVICE and recorded in a 16-byte status block the caller owns; read it back
 * with fbgemm_amd_status_read (this is the only call that synchronizes).
 */
#ifndef FBGEMM_AMD_H_
#define FBGEMM_AMD_H_

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Element types; values follow the reference's SparseType
 * (fbgemm_gpu/include/fbgemm_gpu/embedding_common.h:20-32). */
enum {
  FBGEMM_AMD_FP32 = 0,
  FBGEMM_AMD_FP16 = 1,
  FBGEMM_AMD_INT8 = 2,
  FBGEMM_AMD_INT4 = 3,
  FBGEMM_AMD_INT2 = 4,
  FBGEMM_AMD_BF16 = 5,
  FBGEMM_AMD_FP8 = 6
};

/* Pooling modes (embedding_common.h:34). NONE (one output row per index) has its own entry point,
 * fbgemm_amd_tbe_forward_nobag. */
enum { FBGEMM_AMD_POOL_SUM = 0, FBGEMM_AMD_POOL_MEAN = 1, FBGEMM_AMD_POOL_NONE = 2 };

/* Error codes returned by the entry points. */
enum {
  FBGEMM_AMD_OK = 0,
  FBGEMM_AMD_E_ARG = -1,      /* invalid argument combination */
  FBGEMM_AMD_E_HIP = -2,      /* a HIP runtime call failed; see fbgemm_amd_last_error */
  FBGEMM_AMD_E_UNSUPPORTED = -3
};

/* Bits of the device status word (what made the reference return false). */
enum {
  FBGEMM_AMD_ERR_INDEX_OUT_OF_RANGE = 1,
  FBGEMM_AMD_ERR_BAG_OVERRUN = 2,
  FBGEMM_AMD_ERR_LENGTH_MISMATCH = 4,
  FBGEMM_AMD_ERR_NEGATIVE_LENGTH = 8,
  FBGEMM_AMD_ERR_OUT_OF_BLOCKS = 16 /* fbgemm_amd_kv_block_tables only */
};

#define FBGEMM_AMD_STATUS_BYTES 16

/* Human-readable text of the last FBGEMM_AMD_E_* on this thread. */
const char* fbgemm_amd_last_error(void);

/* Library version, "major.minor". */
const char* fbgemm_amd_version(void);

/* ---- status block ------------------------------------------------------- */

/* Reset a status block (launches a one-thread fill kernel; capture-safe). */
int fbgemm_amd_status_clear(void* d_status, void* stream);

/* Synchronize `stream`, copy the block back. *bits = OR of FBGEMM_AMD_ERR_*;
 * *first_bad_pos = smallest position in the index array holding an
 * out-of-range index, or -1. Either out pointer may be NULL. */
int fbgemm_amd_status_read(const void* d_status, void* stream, int32_t* bits, int64_t* first_bad_pos);

/* The calling thread's own block, for calls that wait for their result: begin hands
 * out the block (cleared), the launches of this thread that follow take it as their
 * d_status, end waits for `stream` and returns what they recorded (bits, and the
 * first offending position or -1). One pair at a time per thread, on one device.
 * Costs a one-thread kernel on the stream, and more only if something was recorded. A begin whose
 * launches were all refused needs no end; one whose launches were enqueued and
 * that is not ended makes the thread's next begin wait for the device. The block
 * is the library's: beside the launches, status_clear and status_read may be
 * called on it, and nothing else may write it. */
int fbgemm_amd_status_begin(void** d_status);
int fbgemm_amd_status_end(void* stream, int32_t* bits, int64_t* first_bad_pos);

/* ---- single-table pooled lookup ----------------------------------------- *
 *
 * Replaces the kernels returned by fbgemm::GenerateEmbeddingSpMDMWithStrides,
 * GenerateEmbeddingSpMDMNBitWithStrides, GenerateEmbeddingSpMDMFP8WithStrides,
 * GenerateEmbeddingSpMDMRowWiseSparse and GenerateEmbeddingSpMDMNBitRowWiseSparse
 * (include/fbgemm/FbgemmEmbedding.h:94-117,151-174,185-203,229-262): the config holds
 * what those factories fix at generation time, the launch takes what
 * EmbeddingSpMDMKernelSignature::Type takes (FbgemmEmbedding.h:41-49,211-221).
 */
typedef struct fbgemm_amd_spmdm_config {
  int32_t weight_ty;            /* FBGEMM_AMD_INT8/INT4/INT2/FP16/BF16/FP32/FP8 */
  int32_t output_ty;            /* FBGEMM_AMD_FP32/FP16/BF16 (no_bag: also INT8/INT4) */
  int32_t index_bits;           /* 32 or 64 */
  int32_t offset_bits;          /* 32 or 64 */
  int64_t block_size;           /* elements per row (D) */
  int64_t output_stride;        /* elements between output rows; -1 = block_size */
  int64_t input_stride;         /* storage elements between table rows (bytes for the
                                   integer formats, halfs for fp16/bf16, floats for
                                   fp32); -1 = densely packed rows */
  int32_t normalize_by_lengths; /* mean pooling */
  int32_t is_weight_positional; /* weights[i] belongs to entry i of every bag */
  int32_t use_offsets;          /* 1: offsets[output_size+1]; 0: lengths[output_size] */
  int32_t scale_bias_last;      /* 1: scale/bias after the row data (fp32 pair for
                                   INT8, fp16 pair for INT4/INT2); 0: fp16 pair in
                                   front of the data, and index -1 is skipped */
  int32_t no_bag;               /* 1: no pooling, one output row per index (the
                                   factories' no_bag flag, FbgemmEmbedding.h:113,170;
                                   src/RefImplementations.cc:1235-1288,1352-1376,
                                   1466-1484): output_size indices, offsets unused,
                                   d_weights[m] scales row m, -1 is out of range.
                                   output_ty INT8 (8-bit rows) copies the first
                                   min(output_stride, input_stride) bytes of each row
                                   to rows output_stride bytes apart; output_ty INT4
                                   (4-bit rows, the only output they have) copies
                                   input_stride bytes to rows input_stride apart */
  int32_t fp8_exponent_bits;    /* weight_ty FP8 (GenerateEmbeddingSpMDMFP8WithStrides, */
  int32_t fp8_exponent_bias;    /* FbgemmEmbedding.h:185-203): the format of the rows */
  int32_t accumulate;           /* FBGEMM_AMD_ACC_EXACT (0, the default) or
                                   FBGEMM_AMD_ACC_FAST, see below */
} fbgemm_amd_spmdm_config;

/* How 4- and 8-bit rows are accumulated. No counterpart in the reference.
 * EXACT: the reference's own sequence of fp32 roundings, acc = fma(scale, q,
 *   acc + bias) per element in index order (src/RefImplementations.cc:1326-1333,
 *   1519-1527): results are bit-identical to the CPU path.
 * FAST: the biases of a bag are summed apart, acc = fma(scale, q, acc) per
 *   element, out = acc + sum of the biases: a third fewer vector instructions
 *   per 4-bit element. Same index order, one lane per output column, so results
 *   are deterministic and differ from the reference's by a few fp32 roundings of
 *   the partial sums (tests hold every element that is not a cancellation to
 *   1e-5 relative for fp32 output and to one unit in the last place of fp16 /
 *   bf16 output). A call of few, long bags (fewer than 256 waves, 32 rows per
 *   bag and more) over such rows is cut into segments whose fp32 partial sums
 *   are added in order afterwards: still deterministic, another association of
 *   the same sum.
 * Only 4- and 8-bit rows of the regular shapes (whole 16-byte chunks, 32
 * columns per lane) have the FAST arithmetic; 4- and 8-bit rows of other widths
 * are summed the EXACT way inside a segment but may still be cut into segments.
 * 2-bit, fp16 / bf16 / fp32 / fp8 rows are computed the EXACT way in either
 * mode and never in segments: a table-batched plan cuts bags only when every
 * one of its tables has 4- or 8-bit rows. */
enum { FBGEMM_AMD_ACC_EXACT = 0, FBGEMM_AMD_ACC_FAST = 1 };

/* Enqueue one pooled lookup. d_weights may be NULL (unweighted).
 * d_compressed_indices_table, when non-NULL, selects the row-wise-sparse
 * variant: data_size then bounds the LOGICAL ids and the table maps them to
 * physical rows (-1 = pruned). d_status must be a cleared status block.
 * With use_offsets == 0 the call makes a prefix sum of the lengths into a
 * library-owned scratch buffer first (grown with hipMalloc when too small).
 * The library keeps one set of scratch buffers (and one status block for
 * fbgemm_amd_spmdm_run) per host thread and device: host threads may call
 * concurrently, each on its own stream; the calls of one thread that use
 * scratch must be ordered on one stream. */
int fbgemm_amd_spmdm_launch(
    const fbgemm_amd_spmdm_config* cfg, int64_t output_size, int64_t index_size,
    int64_t data_size, const void* d_input, const void* d_indices,
    const void* d_offsets_or_lengths, const float* d_weights, void* d_out,
    const int32_t* d_compressed_indices_table, void* d_status, void* stream);

/* fbgemm_amd_spmdm_launch for callers that cannot allocate device memory (code
 * under HIP graph capture, tight serving loops, harnesses that forbid
 * hipMalloc). It has no counterpart in the reference. Same arguments, same
 * kernels; the same results bit for bit with FBGEMM_AMD_ACC_EXACT, and with
 * FBGEMM_AMD_ACC_FAST whenever the call above does not cut the bags into
 * segments (this entry point never does: the segments' partial sums need
 * scratch of a size it has no place for). The two pieces of scratch the call above
 * takes from hipMalloc'ed buffers (the prefix sum of the lengths when
 * use_offsets == 0, and the bag order of the scheduler for calls of 2^21
 * lookups and more) live in a static device array of the library instead
 * (about 1.5 MiB, held by every GPU the library runs on until the process
 * ends). Limit: output_size <= FBGEMM_AMD_NOALLOC_MAX_BAGS, larger calls are
 * rejected with FBGEMM_AMD_E_ARG. It calls no hipMalloc / hipFree and no
 * allocating library routine; its first call on a device asks the runtime for
 * the array's device address (no allocation, but make that call outside a
 * graph capture). All calls on one GPU share the array: two of them that
 * overlap in time (different streams, or host threads without ordering) race;
 * order them on one stream. Nothing in the array has to start at zero (every
 * call writes what it reads). */
#define FBGEMM_AMD_NOALLOC_MAX_BAGS 65536
int fbgemm_amd_spmdm_launch_noalloc(
    const fbgemm_amd_spmdm_config* cfg, int64_t output_size, int64_t index_size,
    int64_t data_size, const void* d_input, const void* d_indices,
    const void* d_offsets_or_lengths, const float* d_weights, void* d_out,
    const int32_t* d_compressed_indices_table, void* d_status, void* stream);
/* The limit above, for callers that bind the library without its header. */
int64_t fbgemm_amd_noalloc_max_bags(void);

/* Same, synchronous, with the reference's return convention: 1 = true,
 * 0 = false (the inputs were rejected; output unspecified), < 0 = API error.
 * Uses a library-owned status block. */
int fbgemm_amd_spmdm_run(
    const fbgemm_amd_spmdm_config* cfg, int64_t output_size, int64_t index_size,
    int64_t data_size, const void* d_input, const void* d_indices,
    const void* d_offsets_or_lengths, const float* d_weights, void* d_out,
    const int32_t* d_compressed_indices_table, void* stream);

/* ---- table-batched forward ----------------------------------------------- *
 *
 * Replaces int_nbit_split_embedding_codegen_lookup_function
 * (fbgemm_gpu/codegen/inference/embedding_forward_quantized_host_cpu.cpp:84-227,
 * embedding_forward_quantized_cpu_template.cpp:208-520; GPU dispatcher
 * embedding_forward_quantized_host.cpp:259-370). A plan is made once from the
 * operator's metadata tensors (HOST copies), then reused for every forward.
 */
typedef struct fbgemm_amd_tbe_plan fbgemm_amd_tbe_plan;

/* weights_offsets[T] (bytes), weights_tys[T] (element types), D_offsets[T+1],
 * weights_placements[T] (0 = dev_weights, anything else = uvm_weights) are the
 * operator's tensors of the same names, on the host. *_weights_bytes are the
 * sizes of the two weights buffers (they bound the last table's row count, as
 * embedding_forward_quantized_cpu_template.cpp:372-380 does). row_alignment
 * is the operator's argument (16 on GPU builds of the reference). */
int fbgemm_amd_tbe_plan_create(
    fbgemm_amd_tbe_plan** plan, int32_t T, const int64_t* weights_offsets,
    const uint8_t* weights_tys, const int32_t* D_offsets,
    const int32_t* weights_placements, int64_t dev_weights_bytes,
    int64_t uvm_weights_bytes, int64_t row_alignment);

void fbgemm_amd_tbe_plan_destroy(fbgemm_amd_tbe_plan* plan);

/* Enqueue the forward of all T tables in ONE kernel launch.
 * d_offsets holds T*B+1 entries in (table, bag) order with the width of the
 * indices (index_bits). d_indice_weights NULL = unweighted. d_output is
 * [B, total_D] of output_ty, row-major; columns of table t start at
 * D_offsets[t]. The first forward with a new B uploads a per-wave work list
 * (allocates); later ones reuse it.
 * output_ty FBGEMM_AMD_INT8 is the reference GPU operator's quantized pooled
 * output (embedding_forward_quantized_split_nbit_kernel_template.cu:535-566;
 * shape: fbgemm_gpu/fbgemm_gpu/sparse_ops.py:571-577): d_output is uint8
 * [B, total_D + 8 T]; per bag and table, the pooled fp32 vector quantized
 * row-wise to 8 bits as FloatToFused8BitRowwiseQuantized does (D_t bytes, fp32
 * scale, fp32 bias), table t starting at byte D_offsets[t] + 8 t. Tables of
 * the regular shapes are quantized in the lookup kernel's own output stage, as
 * in the reference; tables of other shapes (and forwards that cut their bags
 * into segments) go as floats through a plan-owned fp32 [B, total_D] scratch
 * and one more launch. */
int fbgemm_amd_tbe_forward(
    fbgemm_amd_tbe_plan* plan, const void* d_dev_weights, const void* d_uvm_weights,
    const void* d_indices, const void* d_offsets, int32_t index_bits,
    int64_t indices_numel, int64_t offsets_numel, int32_t pooling_mode,
    const float* d_indice_weights, int32_t output_ty, void* d_output,
    void* d_status, void* stream);

/* The same forward with the pruned-row remap fused in: d_indices hold LOGICAL
 * ids; for a table with a mapping (index_remappings_offsets[t+1] >
 * index_remappings_offsets[t], both as in pruned_array_lookup) the physical
 * row is index_remappings[offsets[t] + id], -1 = pruned = skipped; tables
 * without a mapping take their ids as they are. Equal, bit for bit, to
 * fbgemm_amd_pruned_array_lookup followed by fbgemm_amd_tbe_forward (the order
 * of split_table_batched_embeddings_ops_inference.py:1067-1152) without the
 * round trip of the dense indices through HBM. A logical id outside its
 * mapping is reported as out of range. index_remappings_offsets_numel must be
 * T + 1 with T the plan's tables (the operator's features). No counterpart as
 * one call in the reference. */
int fbgemm_amd_tbe_forward_pruned(
    fbgemm_amd_tbe_plan* plan, const void* d_dev_weights, const void* d_uvm_weights,
    const void* d_indices, const void* d_offsets, int32_t index_bits,
    int64_t indices_numel, int64_t offsets_numel, int32_t pooling_mode,
    const float* d_indice_weights, int32_t output_ty, void* d_output,
    const void* d_index_remappings, int32_t remap_bits,
    const int64_t* d_index_remappings_offsets, int64_t index_remappings_offsets_numel,
    void* d_status, void* stream);

/* The forward above with the checks of fbgemm_amd_check_remap_indices in it, on inputs as the caller
 * has them: the lookup kernels judge every index as they read it (rows_per_table; with a mapping the rows
 * before pruning first), take row 0 for one outside its table and, in mode 1 (WARNING), leave the number of
 * those in *d_warning. Waits for the result: returns 0 when the output is what the check and the forward one
 * after the other make. Otherwise the caller makes the two calls: 1, and nothing was done, for the 8-bit output, a
 * plan in the tolerance-grade mode, a mapping over tables of other widths than the kernels' regular ones (unless
 * the forward is small), a table without rows, a stream that is being captured; 2, with an output and a *d_warning that mean nothing, for
 * offsets that are not in order from at least 0 to indices_numel, which the check repairs, and row counts below 1. */
int fbgemm_amd_tbe_forward_checked(
    fbgemm_amd_tbe_plan* plan, const void* d_dev_weights, const void* d_uvm_weights,
    const void* d_indices, const void* d_offsets, int32_t index_bits,
    int64_t indices_numel, int64_t offsets_numel, int32_t pooling_mode,
    const float* d_indice_weights, int32_t output_ty, void* d_output,
    const int64_t* d_rows_per_table, int32_t bounds_check_mode, int64_t* d_warning,
    const int64_t* d_logical_rows_per_table, const void* d_index_remappings, int32_t remap_bits,
    const int64_t* d_index_remappings_offsets, int64_t index_remappings_offsets_numel, void* stream);

/* A compact form of the mappings for the forward before it. No counterpart in the
 * reference. For every table whose mapping is order-preserving (its kept rows
 * are numbered 0, 1, 2, ... in logical order: what embedding_bag_rowwise_prune
 * and the inference converter produce) the plan builds, on the device, 2 bits per
 * logical row (a kept-row bitmap with a running count per 32 rows) and the
 * forwards compute the physical row from that instead of fetching a 4- or 8-byte
 * entry of a table-sized array: the same integers, from a structure that fits
 * the caches. Tables whose mapping is anything else keep reading the array.
 * d_index_remappings / remap_bits as in the forward; index_remappings_offsets is
 * the HOST copy of the T+1 offsets. The forwards use the records whenever they
 * are passed the same d_index_remappings pointer, and then bound and slice the
 * mappings with the offsets given HERE (the plan keeps a device copy), whatever
 * offsets the forward is handed; call this again after the array's contents or
 * its offsets change (NULL array = drop the records). Allocates; synchronizes
 * `stream`. fbgemm_amd_tbe_plan_rank_tables returns how many tables use records. */
int fbgemm_amd_tbe_plan_set_index_remappings(
    fbgemm_amd_tbe_plan* plan, const void* d_index_remappings, int32_t remap_bits,
    const int64_t* index_remappings_offsets, int64_t index_remappings_offsets_numel, void* stream);
int32_t fbgemm_amd_tbe_plan_rank_tables(const fbgemm_amd_tbe_plan* plan);

/* Select FBGEMM_AMD_ACC_EXACT (the default of a new plan) or FBGEMM_AMD_ACC_FAST
 * for the forwards of a plan. No counterpart in the reference. */
int fbgemm_amd_tbe_plan_set_accumulate(fbgemm_amd_tbe_plan* plan, int32_t mode);

/* A plan caches, per (batch size, stream), the work lists of its forwards and the
 * scratch of the bag scheduler; past 16 entries the least recently used one that
 * no forward under stream capture has touched is dropped. This call drops ALL of
 * them (after a device synchronize), including those a captured graph may hold:
 * graphs that contain forwards of this plan must be captured again afterwards.
 * fbgemm_amd_tbe_plan_cached_work returns the number of cached entries. No
 * counterpart in the reference. */
int fbgemm_amd_tbe_plan_trim(fbgemm_amd_tbe_plan* plan);
int64_t fbgemm_amd_tbe_plan_cached_work(const fbgemm_amd_tbe_plan* plan);
/* How many of the cached entries a forward under stream capture has touched (a
 * graph may hold their addresses): a cache of plans must not destroy a plan
 * while this is not 0 unless its owner knows the graphs are gone. */
int64_t fbgemm_amd_tbe_plan_pinned_work(fbgemm_amd_tbe_plan* plan);

/* Tables of FBGEMM_AMD_FP8 rows (D bytes per row, no scale/bias) are decoded
 * with the operator's fp8_exponent_bits / fp8_exponent_bias
 * (Float8ToFloat_ref, src/RefImplementations.cc:184-214; the pooled arithmetic
 * is EmbeddingSpMDMFP8_ref's, :1544-1616: acc = fma(w, value, acc)). Set them
 * before the first forward of a plan that holds such tables; an index of -1 is
 * skipped as for every other row type. */
int fbgemm_amd_tbe_plan_set_fp8(fbgemm_amd_tbe_plan* plan, int32_t exponent_bits, int32_t exponent_bias);

/* The forward without pooling (PoolingMode.NONE, "sequence" output;
 * embedding_forward_quantized_host_cpu.cpp:113-139 and
 * embedding_forward_quantized_cpu_template.cpp:283-296,390-420): d_output is
 * [indices_numel, D] of output_ty, row i the row d_indices[i] of the table
 * whose slice of d_offsets holds position i, converted like a bag of one
 * (unweighted); an index of -1 gives a row of zeros. All tables share D (the
 * operator passes the largest of its max_*_D). output_ty FBGEMM_AMD_INT8 /
 * FBGEMM_AMD_INT4 copies the stored row (fp16 scale, fp16 bias, elements:
 * D + 4 bytes, resp. (D + 8) / 2 bytes per output row) and needs every table
 * to be of that type (src/RefImplementations.cc:1235-1253,1466-1484). */
int fbgemm_amd_tbe_forward_nobag(
    fbgemm_amd_tbe_plan* plan, const void* d_dev_weights, const void* d_uvm_weights,
    const void* d_indices, const void* d_offsets, int32_t index_bits,
    int64_t indices_numel, int64_t offsets_numel, int32_t D, int32_t output_ty,
    void* d_output, void* d_status, void* stream);

/* Rows the plan inferred for table t (what an index is checked against). */
int64_t fbgemm_amd_tbe_plan_num_rows(const fbgemm_amd_tbe_plan* plan, int32_t t);
/* Padded row bytes of table t. */
int64_t fbgemm_amd_tbe_plan_row_bytes(const fbgemm_amd_tbe_plan* plan, int32_t t);

/* ---- pruned-row remap ------------------------------------------------------ *
 * Replaces pruned_array_lookup
 * (embedding_forward_quantized_cpu_template.cpp:605-659,
 * embedding_forward_quantized_split_lookup.cu:120-168): position-preserving,
 * d_dense[i] = remap[remap_offsets[t] + indices[i]] for tables that own a
 * mapping (remap_offsets[t+1] > remap_offsets[t]), a copy otherwise. An id
 * outside its table's mapping yields -1 (the reference reads out of bounds). */
int fbgemm_amd_pruned_array_lookup(
    const void* d_indices, const void* d_offsets, int32_t index_bits,
    int64_t offsets_numel, const void* d_index_remappings, int32_t remap_bits,
    const int64_t* d_index_remappings_offsets, int32_t T, void* d_dense,
    void* stream);

/* ---- in-place row update of a table-batched weights buffer ----------------- *
 * Replaces emb_inplace_update
 * (fbgemm_gpu/src/embedding_inplace_ops/embedding_inplace_update.cu:28-101,207-282,
 * CPU form embedding_inplace_update_cpu.cpp:25-70; schema :257-258; caller
 * embedding_inplace_update_internal,
 * fbgemm_gpu/fbgemm_gpu/split_table_batched_embeddings_ops_inference.py:2057-2144):
 * for update i the padded row d_update_row_idx[i] of table d_update_table_idx[i]
 * (fbgemm_amd_tbe_plan_row_bytes bytes) is overwritten with the bytes at
 * d_update_weights + d_update_offsets[i]. Tables, row sizes, placements and row
 * counts come from the plan. Beyond the reference, which checks nothing: a row id
 * of -1 (a pruned row, see below) is skipped; a table outside [0, T), another row
 * outside its table, or an update that would read past update_weights_bytes is
 * skipped and recorded in d_status (out-of-range / overrun bits; may be NULL:
 * then it is only skipped). Two updates of one row in a call race, as in the
 * reference's kernel. Asynchronous; forwards that should see the rows must be
 * ordered after it on `stream`. */
int fbgemm_amd_tbe_inplace_update(
    fbgemm_amd_tbe_plan* plan, void* d_dev_weights, void* d_uvm_weights,
    const void* d_update_weights, int64_t update_weights_bytes,
    const int32_t* d_update_table_idx, const void* d_update_row_idx, int32_t row_index_bits,
    const int64_t* d_update_offsets, int64_t n, void* d_status, void* stream);

/* Replaces pruned_array_lookup_from_row_idx (embedding_inplace_update.cu:359-465,
 * embedding_inplace_update_cpu.cpp:199-251): the logical rows of an update become
 * physical rows, d_dense[i] = index_remappings[offsets[t_i] + row_i] where table
 * t_i owns a mapping and row_i otherwise. A row outside its mapping or a table
 * outside [0, T) yields -1 (the reference reads out of bounds). */
int fbgemm_amd_pruned_array_lookup_from_row_idx(
    const void* d_update_row_idx, int32_t index_bits, const int32_t* d_update_table_idx, int64_t n,
    const void* d_index_remappings, int32_t remap_bits, const int64_t* d_index_remappings_offsets,
    int32_t T, void* d_dense, void* stream);

/* ---- index operators that run before the lookup ---------------------------- *
 *
 * bounds_check_indices (fbgemm_gpu/codegen/utils/embedding_bounds_check_host_cpu.cpp:76-219,
 * schema :240-256; the step before the lookup in
 * split_table_batched_embeddings_ops_inference.py:1067-1124). In place on
 * d_indices / d_offsets (same width). bounds_check_mode: 0 FATAL, 1 WARNING,
 * 2 IGNORE (embedding_common.h:44-48).
 *   WARNING / IGNORE: offsets[last] becomes indices_numel; every offset is
 *     clamped to [0, indices_numel] and raised to the largest offset before it
 *     (what the reference's sequential loop leaves); an index other than -1
 *     outside [0, rows_per_table[t]) becomes 0. WARNING zeroes d_warning[0]
 *     first and counts one per repaired last offset, per bad bag and per bad
 *     index, like the reference's counter.
 *   FATAL: nothing is modified; the conditions the reference raises on are
 *     ORed into d_status (FBGEMM_AMD_ERR_LENGTH_MISMATCH: last offset !=
 *     indices_numel; FBGEMM_AMD_ERR_BAG_OVERRUN: offsets negative, decreasing
 *     or beyond indices_numel; FBGEMM_AMD_ERR_INDEX_OUT_OF_RANGE, with the
 *     first offending position). The reference's GPU kernel asserts on the
 *     device instead, which takes the process down.
 * d_B_offsets: NULL, or int32[T+1] first bag of every table (variable batch
 * sizes). Uses library-owned scratch: calls must be ordered on one stream. */
int fbgemm_amd_bounds_check_indices(
    const int64_t* d_rows_per_table, int32_t T, void* d_indices, void* d_offsets, int32_t index_bits,
    int64_t indices_numel, int64_t offsets_numel, int32_t bounds_check_mode, int64_t* d_warning,
    const int32_t* d_B_offsets, void* d_status, void* stream);

/* bounds_check_indices in WARNING or IGNORE mode on copies of the inputs, with the
 * array-based pruned-row mapping in the same pass when there is one: the check
 * against d_logical_rows_per_table, pruned_array_lookup, and the check against
 * d_rows_per_table, each index read and written once. d_index_remappings_offsets
 * (T + 1 entries) may be NULL: then only the check. d_out_indices and d_out_offsets
 * have the inputs' sizes and must not overlap them; d_warning ends as the last check
 * of the separate calls would leave it. B must not be zero. Calls on several streams
 * may overlap, and captured calls be replayed beside them, as long as their outputs
 * and warning counters are their own. */
int fbgemm_amd_check_remap_indices(
    const int64_t* d_rows_per_table, int32_t T, const void* d_indices, const void* d_offsets, int32_t index_bits,
    int64_t indices_numel, int64_t offsets_numel, int32_t bounds_check_mode, int64_t* d_warning,
    const int64_t* d_logical_rows_per_table, const void* d_index_remappings, int32_t remap_bits,
    const int64_t* d_index_remappings_offsets, void* d_out_indices, void* d_out_offsets, void* stream);

/* The compact form of pruned-row mappings that keep the rows' order, 2 bits per logical
 * row, for the check above: made once from d_index_remappings (T + 1 offsets on the
 * host; waits for `stream`) and made anew by the caller whenever its contents change.
 * Returns for how many tables there is one; *out is NULL where there is none. destroy
 * waits for the device. The ranked check is the check above and, where `ranks`
 * (NULL: none) was made from the very array it is handed, asks it instead of the
 * array, whose random 4-byte reads cost a line each: the same results. A call under
 * stream capture reads the array. */
typedef struct fbgemm_amd_rank_records fbgemm_amd_rank_records;
int fbgemm_amd_rank_records_create(
    fbgemm_amd_rank_records** out, const void* d_index_remappings, int32_t remap_bits,
    const int64_t* index_remappings_offsets, int64_t index_remappings_offsets_numel, void* stream);
void fbgemm_amd_rank_records_destroy(fbgemm_amd_rank_records* ranks);
int fbgemm_amd_check_remap_indices_ranked(
    const fbgemm_amd_rank_records* ranks,
    const int64_t* d_rows_per_table, int32_t T, const void* d_indices, const void* d_offsets, int32_t index_bits,
    int64_t indices_numel, int64_t offsets_numel, int32_t bounds_check_mode, int64_t* d_warning,
    const int64_t* d_logical_rows_per_table, const void* d_index_remappings, int32_t remap_bits,
    const int64_t* d_index_remappings_offsets, void* d_out_indices, void* d_out_offsets, void* stream);

/* pruned_hashmap_lookup (embedding_forward_quantized_cpu_template.cpp:524-603; GPU
 * embedding_forward_quantized_split_lookup.cu:19-118): d_hash_table holds
 * [slots][2] (sparse id, dense id) pairs of hash_bits each, -1 = empty, built by
 * the reference's pruned_hashmap_insert (linear probing from MurmurHash3's
 * finalizer of the id, 32- or 64-bit after the index width, modulo the table's
 * capacity). d_dense[i] = the dense id of d_indices[i], -1 when absent, a copy
 * for tables with an empty slot range. */
int fbgemm_amd_pruned_hashmap_lookup(
    const void* d_indices, const void* d_offsets, int32_t index_bits, int64_t offsets_numel,
    const void* d_hash_table, int32_t hash_bits, const int64_t* d_hash_table_offsets, int32_t T,
    void* d_dense, void* stream);

/* pruned_hashmap_insert (embedding_forward_quantized_cpu_template.cpp:124-201;
 * the reference has this operator on the CPU only and its GPU module calls
 * it there, split_table_batched_embeddings_ops_inference.py:2001-2010): HOST
 * pointers, runs on the calling thread. Inserts (indices[i], dense_indices[i])
 * of every table's slice into that table's slots of h_hash_table ([slots][2],
 * -1 = empty), skipping pairs whose dense id is -1, by linear probing from the
 * same hash as the lookup. Returns FBGEMM_AMD_E_ARG when a table has no empty
 * slot left (the reference would not return). */
int fbgemm_amd_pruned_hashmap_insert_host(
    const void* h_indices, const void* h_dense_indices, const void* h_offsets, int32_t index_bits,
    int64_t offsets_numel, void* h_hash_table, int32_t hash_bits, const int64_t* h_hash_table_offsets, int32_t T);

/* ---- row-wise quantizers: producers and readers of the row formats ---------- *
 *
 * fp32 / fp16 rows [rows][cols] -> fused quantized rows, bit for bit what the
 * reference's CPU routines write:
 *   bit_rate 2 / 4 / 8, sb_float 0: FloatOrHalfToFusedNBitRowwiseQuantizedSBHalf
 *     (src/QuantUtils.cc:534-611): packed elements, then fp16 scale, fp16 bias;
 *   bit_rate 8, sb_float 1: FloatOrHalfToFused8BitRowwiseQuantizedSBFloat
 *     (src/QuantUtils.cc:677-718): bytes, then fp32 scale, fp32 bias.
 * layout FBGEMM_AMD_QLAYOUT_TRAILER keeps that order; FBGEMM_AMD_QLAYOUT_TBE
 * writes the table-batched operator's rows, fp16 scale and bias FIRST, then
 * the elements, as quantize_embs rearranges them
 * (fbgemm_gpu/fbgemm_gpu/tbe/utils/quantize.py:47-70; with sb_float 1 the fp32
 * pair is rounded to fp16, as there). out_row_stride is in bytes (>= the row's
 * size: padding bytes are left alone). */
enum { FBGEMM_AMD_QLAYOUT_TRAILER = 0, FBGEMM_AMD_QLAYOUT_TBE = 1 };
int fbgemm_amd_quantize_rowwise(
    const void* d_input, int32_t input_ty, int64_t rows, int32_t cols, int32_t bit_rate, int32_t sb_float,
    int32_t layout, int64_t out_row_stride, void* d_output, void* stream);

/* The same with extremes the caller brings: the `rowwise_min_max` argument of
 * FloatOrHalfToFusedNBitRowwiseQuantizedSBHalf / FloatOrHalfToFused8BitRowwiseQuantizedSBFloat
 * (include/fbgemm/QuantUtils.h:277-283, :311-317; src/QuantUtilsAvx2.cc:1605-1628, :1831-1853).
 * d_rowwise_min_max holds [rows][2] values of the input's type, minimum then
 * maximum, which take the place of the row's own extremes; null means "find
 * them", as the call above. Elements outside the extremes given: the 2 / 4 / 8
 * bit fp16-pair formats saturate to 0 .. 2^bit_rate - 1; the 8-bit fp32-pair
 * format does what the reference's vector code does, saturate in the leading
 * whole groups of 32 columns and keep the low byte of the rounded integer in
 * the columns behind them. */
int fbgemm_amd_quantize_rowwise_min_max(
    const void* d_input, int32_t input_ty, int64_t rows, int32_t cols, int32_t bit_rate, int32_t sb_float,
    int32_t layout, int64_t out_row_stride, void* d_output, const void* d_rowwise_min_max, void* stream);

/* The inverses (src/QuantUtils.cc:743-789 FusedNBitRowwiseQuantizedSBHalfToFloatOrHalf,
 * :847-892 Fused8BitRowwiseQuantizedSBFloatToFloatOrHalf): element =
 * float(double(scale) * q + double(bias)), written as fp32, fp16 (round to
 * nearest even) or bf16 ((bits + 0x8000) >> 16); output [rows][cols], dense. */
int fbgemm_amd_dequantize_rowwise(
    const void* d_input, int64_t rows, int64_t in_row_stride, int32_t cols, int32_t bit_rate, int32_t sb_float,
    int32_t layout, int32_t output_ty, void* d_output, void* stream);

/* fp32 <-> 8-bit float (hfp8) element-wise, `n` elements: the operators
 * FloatToHFP8Quantized / HFP8QuantizedToFloat
 * (fbgemm_gpu/src/quantize_ops/quantize_ops_cpu.cpp:531-620,
 * fbgemm_gpu/include/fbgemm_gpu/quantize_ops_utils.h:29-110; the same arithmetic as
 * FloatToFloat8_ref / Float8ToFloat_ref, src/RefImplementations.cc:126-214), which
 * produce and read back the rows of FP8 tables (quantize_embs,
 * fbgemm_gpu/fbgemm_gpu/tbe/utils/quantize.py:36-45). |x| is clamped to max_pos,
 * rounding is to nearest even, values below the smallest normal keep gradual
 * underflow. */
int fbgemm_amd_float_to_hfp8(const float* d_input, int64_t n, int32_t ebits, int32_t exponent_bias, float max_pos,
                             uint8_t* d_output, void* stream);
int fbgemm_amd_hfp8_to_float(const uint8_t* d_input, int64_t n, int32_t ebits, int32_t exponent_bias, float* d_output,
                             void* stream);

/* fbgemm::compressed_indices_remap (include/fbgemm/FbgemmEmbedding.h:392-401,
 * src/RefImplementations.cc:2308-2333): the core library's pruned-row remap, which
 * compacts. Entries whose row is pruned (d_mapping[index] == -1) are dropped, the
 * others become their physical row and move up, per-sample weights (optional) move
 * with them; d_out_offsets[i] = entries that stay before bag i, d_out_offsets[0] =
 * offsets[0]. Indices and offsets share index_bits; offsets must not decrease (the
 * reference then walks positions offsets[0] .. offsets[last]-1 in order). Beyond the
 * reference: mapping_numel bounds the indices (an index outside the mapping is dropped
 * and recorded in d_status instead of being read; d_status may be NULL: then it is
 * only dropped). Outputs must not alias inputs.
 * Reads offsets[0] and offsets[last] back first (synchronizes `stream`), then runs
 * asynchronously; uses library-owned scratch (calls must be ordered on one stream). */
int fbgemm_amd_compressed_indices_remap(
    int32_t offsets_numel, const void* d_indices, int32_t index_bits, const int32_t* d_mapping, int64_t mapping_numel,
    const void* d_offsets, const float* d_weights, void* d_out_indices, void* d_out_offsets, float* d_out_weights,
    void* d_status, void* stream);

/* embedding_bag_rowwise_prune (fbgemm_gpu/src/sparse_ops/sparse_ops_cpu.cpp:2836-2893,
 * which ends in at::native::_rowwise_prune; the converter's pruning step,
 * fbgemm_gpu/fbgemm_gpu/split_embedding_inference_converter.py:75-93), in two calls
 * because the size of the result depends on the data.
 * _map: row i stays when indicator[i] (|indicator[i]| with use_abs) > threshold, or
 * when the rows kept so far plus all rows still to come do not exceed
 * min_non_pruned_rows; d_remap[rows] (int32 or int64) receives the new row id or -1,
 * *num_kept (host) the number of rows that stay. Synchronizes `stream`.
 * _gather: d_output[remap[i]] = d_weights[i] for the rows that stay; rows of
 * row_bytes bytes, output_rows = the num_kept the map gave. */
int fbgemm_amd_rowwise_prune_map(const float* d_indicator, int64_t rows, double threshold, int32_t use_abs,
                                 int64_t min_non_pruned_rows, int32_t index_bits, void* d_remap, int64_t* num_kept,
                                 void* stream);
int fbgemm_amd_rowwise_prune_gather(const void* d_weights, int64_t rows, int64_t row_bytes, const void* d_remap,
                                    int32_t index_bits, void* d_output, int64_t output_rows, void* stream);

/* ---- a decoding step over a paged key-value cache ---------------------------- *
 *
 * Operators of language-model serving that have no counterpart in the reference's
 * quantized-embedding path. A cache is an array of blocks (pages) of block_size
 * tokens; a request's tokens are those of the blocks its table lists, in order.
 * Asynchronous, capture-safe; nothing is allocated and nothing waits. Lengths and
 * lists live on the device, so a step needs no copy to the host.
 *
 * fbgemm_amd_kv_block_tables: pages, slots and positions for the tokens a step adds.
 * Request r holds d_lengths[r] tokens and gets d_new_tokens[r] (both int32 or int64).
 * Its table (table_width entries, table_stride apart; those of the tokens it holds
 * are read, the entries behind them written) gets the next blocks of d_free_blocks,
 * requests in order, from *d_free_start on; *d_free_next is the place behind the last
 * block taken (beyond free_numel: that many are missing). New token k of request r is
 * number d_offsets[r] + k of the step, its position is d_lengths[r] + k, its slot
 * table[position / block_size] * block_size + position % block_size, or -1 where
 * there is no block for it (table too narrow, free list exhausted, a negative entry).
 * Positions count from the table's room where a request holds more than that: from
 * table_width * block_size on they are no tokens' places, and their slots are -1.
 * d_slots and d_positions hold num_tokens entries: those behind the last token are -1
 * and 0; tokens beyond num_tokens get none. d_total_lengths = lengths + new tokens.
 * Called again with the same inputs it writes the same. d_status (may be NULL: then
 * the entries say it all): NEGATIVE_LENGTH (counted as 0), BAG_OVERRUN (a table too
 * narrow), OUT_OF_BLOCKS, LENGTH_MISMATCH (the new tokens' sum is not num_tokens: set
 * by a step that is padded on purpose too, whose d_offsets[requests] is below
 * num_tokens; of a list that is cut it is num_tokens).
 * d_free_next must not be d_free_start, nor d_total_lengths d_lengths. */
int fbgemm_amd_kv_block_tables(
    const void* d_lengths, const void* d_new_tokens, int32_t index_bits, int64_t requests, int32_t* d_block_tables,
    int64_t table_stride, int64_t table_width, const int32_t* d_free_blocks, int64_t free_numel, const int32_t* d_free_start,
    int32_t block_size, int64_t num_tokens, int64_t* d_slots, int64_t* d_positions, int32_t* d_offsets, void* d_total_lengths,
    int32_t* d_free_next, void* d_status, void* stream);

/* Keys and values are two arrays [blocks][heads][block_size][row]; strides (blocks,
 * heads, slots) in elements of storage (INT8: bytes), a row's elements next to each
 * other. INT8 rows are the table-batched operator's: fp16 scale, fp16 bias, dim bytes
 * (dim + 4 bytes, on 4-byte boundaries). CACHE_INT4 rows are its 4-bit ones: scale and
 * bias, then two elements a byte, the first in the low bits (dim / 2 + 4 bytes, strides
 * in bytes, on 4-byte boundaries too; dim is even). */
enum { FBGEMM_AMD_CACHE_INT4 = 16 }; /* a cache's row_ty alone: a table's type is no cache's */
typedef struct fbgemm_amd_paged_cache {
  int32_t row_ty;     /* FBGEMM_AMD_FP32/FP16/BF16/INT8, FBGEMM_AMD_CACHE_INT4 */
  int32_t block_size; /* tokens of a block */
  int32_t heads, dim; /* of keys and values */
  int64_t blocks;
  int64_t key_strides[3], value_strides[3];
} fbgemm_amd_paged_cache;

/* New rows into their slots: cache[slot / block_size][head][slot % block_size] = row.
 * d_key and d_value are [tokens][heads][dim] with the strides (tokens, heads) given in
 * elements. A cache of FP32 / FP16 / BF16 rows takes rows of its own type as they are;
 * an INT8 or CACHE_INT4 cache takes any of the three and stores what fbgemm_amd_quantize_rowwise
 * (bit_rate 8 or 4, sb_float 0, FBGEMM_AMD_QLAYOUT_TBE) makes of them, with elements beyond
 * fp16's range at its end and NaN as 0 (a zero bias may have either sign). Slot -1 is
 * skipped; another slot outside the cache too, and is recorded in d_status (may be
 * NULL) as INDEX_OUT_OF_RANGE with the token's number. Slots differ from each other
 * (but for -1): a slot that several tokens have ends as a mixture of their rows, which
 * are written by many threads in no order; no other slot is touched. Rows of the cache
 * must not overlap. */
int fbgemm_amd_kv_cache_append(
    const fbgemm_amd_paged_cache* cache, const void* d_key, const void* d_value, int32_t input_ty, int64_t tokens,
    const int64_t* key_strides, const int64_t* value_strides, const int64_t* d_slots, void* d_key_cache, void* d_value_cache,
    void* d_status, void* stream);

/* Rows of requests' tokens, out of their pages into dense arrays d_key and d_value
 * [tokens][heads][dim] on 16-byte boundaries, which overlap neither each other nor what lies
 * between a cache's first row and its last: what attention of a prompt's later part
 * reads of its earlier one. Token i belongs to the request r with d_offsets[r] <= i <
 * d_offsets[r + 1] (requests + 1 entries, ascending, int32 or int64 by index_bits) and is at position
 * d_starts[r] + i - d_offsets[r] of it (d_starts NULL: 0). Rows come as they are, in the cache's type;
 * INT8 and CACHE_INT4 rows as the values they stand for, scale * code + bias, in
 * FP32, FP16 or BF16. A token whose block the table or the cache does not have is zeros, and is
 * recorded in d_status (may be NULL) as INDEX_OUT_OF_RANGE with its number; tokens
 * from d_offsets[requests] on are zeros. table_width * block_size is below 2^31. */
int fbgemm_amd_kv_cache_read(
    const fbgemm_amd_paged_cache* cache, const void* d_key_cache, const void* d_value_cache, const int32_t* d_block_tables,
    int64_t table_stride, int64_t table_width, const void* d_offsets, const void* d_starts, int32_t index_bits, int64_t requests,
    int64_t tokens, int32_t output_ty, void* d_key, void* d_value, void* d_status, void* stream);

/* Rows [tokens][heads][dim] that go in and come out; strides (tokens, heads) in elements */
typedef struct fbgemm_amd_head_rows {
  const void* in;
  void* out; /* may be in, with the same strides */
  int64_t in_strides[2], out_strides[2];
  int32_t heads;
} fbgemm_amd_head_rows;

/* Queries and keys turned by their positions (rotary positions). Of the first 2 * pairs
 * elements of a head pair p is (p, p + pairs), or with `interleaved` (2 p, 2 p + 1):
 *   (a, b) -> magnitude * (a cos - b sin, b cos + a sin) of position * d_frequencies[p]
 * (radians, fp64); the elements behind them stay as they are. With `inverse` the other
 * way round, with the same magnitude: the way a gradient takes. d_positions [tokens],
 * int32 or int64 by index_bits; FP32, FP16 or BF16 rows, in fp32 and rounded once;
 * angles in fp64. pairs: at most 1024; `key` may be NULL. What is written must not
 * overlap what else is read or written. */
int fbgemm_amd_rotate_positions(
    const fbgemm_amd_head_rows* query, const fbgemm_amd_head_rows* key, int32_t ty, int64_t tokens, int32_t dim,
    const void* d_positions, int32_t index_bits, const double* d_frequencies, int32_t pairs, int32_t interleaved,
    float magnitude, int32_t inverse, void* stream);

/* Attention of one new token per request. d_query [requests][query_heads][dim] (FP16
 * or BF16; strides in elements, rows on 16-byte boundaries), query head h reads key
 * head h / (query_heads / heads). Of request r's d_lengths[r] tokens (the new one
 * among them; more than its table has room for count as that many) all are read, or
 * with window > 0 the last `window`:
 *   s_t = scale * q . k_t, with softcap > 0 softcap * tanh(s_t / softcap),
 *   d_output [requests][query_heads][dim] (the queries' type, dense) = softmax(s) v,
 *   d_lse [requests][query_heads] = log(sum_t exp(s_t)).
 * Tokens of a block outside [0, blocks) are left out; where no token is left the output
 * is 0 and d_lse -inf. What the cache holds where no token is may be anything. A score
 * of NaN, or of +inf without a cap, and a value that is not finite make their queries'
 * outputs not finite; a score of -inf weighs 0. Tokens of a block are less than 64 MiB
 * apart. A
 * cache of FP16 / BF16 rows must have the queries' type and rows on 16-byte boundaries,
 * one of INT8 or CACHE_INT4 rows goes with either. dim: a multiple of 8, at most 256;
 * requests * heads * table_width * block_size below some 2^37. Scores, weights
 * and sums are fp32 (weights go to the matrix cores as two 16-bit numbers); results do
 * not depend on the order in which workgroups run. d_workspace: scratch of
 * fbgemm_amd_paged_attention_workspace bytes that no other call uses at the same time. */
int64_t fbgemm_amd_paged_attention_workspace(const fbgemm_amd_paged_cache* cache, int64_t requests, int32_t query_heads, int64_t table_width);
int fbgemm_amd_paged_attention(
    const fbgemm_amd_paged_cache* cache, const void* d_query, int32_t query_ty, int64_t requests, int32_t query_heads,
    int64_t query_request_stride, int64_t query_head_stride, const void* d_key_cache, const void* d_value_cache,
    const int32_t* d_block_tables, int64_t table_stride, int64_t table_width, const void* d_lengths, int32_t index_bits,
    float scale, int64_t window, float softcap, void* d_output, float* d_lse, void* d_workspace, int64_t workspace_bytes, void* stream);

/* Logits [rows][vocab] (FP32, FP16 or BF16) made ready to sample from. A row's tokens
 * are d_tokens[d_offsets[row] .. d_offsets[row + 1] - 1], the first
 * d_prompt_lengths[row] (NULL: none) of them its prompt; tokens outside the vocabulary
 * are passed over. In fp32, in this order, rounded once at the end:
 *   a token of the list:              x = x > 0 ? x / repetition : x * repetition
 *   n > 0 times behind the prompt:    x = x - frequency * n, then x = x - presence
 *   a bias for it (the last one):     x = x + bias
 *   its bit of the mask is 0:         x = -inf, whatever x was
 * The three penalties are one fp32 number per row (NULL: 1, 0, 0), biases a list of
 * (id, value) per row like the tokens' (all lists have index_bits), the mask one bit
 * per token, bit v % 32 of word v / 32 of a row (mask_stride words apart). With a stride
 * of 0 all rows share the logits, or the mask. d_output may be d_logits (with the same
 * stride, not 0); rows of the two that overlap otherwise are refused. */
int fbgemm_amd_penalize_logits(
    const void* d_logits, int32_t logits_ty, int64_t rows, int64_t vocab, int64_t logits_stride, const void* d_tokens,
    int64_t tokens_numel, const void* d_offsets, const void* d_prompt_lengths, int32_t index_bits, const float* d_repetition,
    const float* d_frequency, const float* d_presence, const void* d_bias_ids, const float* d_bias_values, int64_t bias_numel,
    const void* d_bias_offsets, const int32_t* d_mask, int64_t mask_stride, void* d_output, int64_t output_stride, void* stream);

/* A token of every row of logits [rows][vocab] (FP32, FP16 or BF16), drawn by a number
 * d_uniform[row] in [0, 1). With tokens in order, larger logits first, equal ones by
 * number, and w = exp((x - max) / temperature), those that may be drawn are the first
 * top_k; of these the fewest first ones whose w add up to top_p times the sum of all of
 * these (one at least); of these the ones with w >= min_p. d_tokens[row] is the
 * first of them, by number, where the running sum of w is above uniform times the whole
 * (or the last one), d_log_probability[row] the logarithm of its w over the whole. Of
 * the four lists, one number per row, each may be NULL: temperature 1, top_k and min_p
 * 0, top_p 1. top_k <= 0 or >= vocab, top_p >= 1 and min_p <= 0 leave every token (min_p
 * >= 1: those of the largest logit, and any so near it by the temperature that its w is
 * rounded to the same); with a temperature or top_p that is not above 0 it is the first
 * of the largest ones, of probability 1. NaN and -inf are never drawn,
 * +inf counts as the largest finite fp32 number; a row with nothing else gives -1 and
 * -inf. Sums are of whole numbers, w rounded to units of 2^-f of the largest, f the
 * smaller of 50 and 62 - bits of vocab (45 for 131 071 tokens, 41 for 2^20): the same in
 * any order, and off by little more than half a unit a token. A draw is that of exact
 * sums but within some vocab / 2 units of a border of two tokens (2^-29 of the largest w
 * for 131 071 tokens, 2^-22 for 2^20). vocab: 1..2^20, rows up to 2^24; a row stride of 0 shares the
 * logits. */
int fbgemm_amd_sample_tokens(
    const void* d_logits, int32_t logits_ty, int64_t rows, int64_t vocab, int64_t logits_stride, const float* d_uniform,
    const float* d_temperature, const int32_t* d_top_k, const float* d_top_p, const float* d_min_p, int64_t* d_tokens,
    float* d_log_probability, void* stream);

/* Wait for everything enqueued on `stream` (hipStreamSynchronize), for callers
 * of the asynchronous entry points that hold no HIP headers. */
int fbgemm_amd_stream_synchronize(void* stream);

/* ---- row-size arithmetic (host, no GPU) ------------------------------------ *
 * embedding_common.h:189-225. */
int32_t fbgemm_amd_unpadded_row_size_in_bytes(int32_t dim, int32_t weight_ty, int32_t scale_bias_bytes);
int32_t fbgemm_amd_padded_row_size_in_bytes(int32_t dim, int32_t weight_ty, int32_t row_alignment, int32_t scale_bias_bytes);

#ifdef __cplusplus
}
#endif
#endif /* FBGEMM_AMD_H_ */
