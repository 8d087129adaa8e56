// One instance of the attention kernels (paged_attention.h): fp16 queries, 4-bit rows.
#include "paged_attention.h"

namespace fbgemm_amd {
hipError_t launch_paged_attention_fp16_rows4(const AttentionArgs& a, hipStream_t stream) { return attention::launch_any<false, 4>(a, stream); }
} // namespace fbgemm_amd
