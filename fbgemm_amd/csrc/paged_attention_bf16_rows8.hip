// One instance of the attention kernels (paged_attention.h): bf16 queries, 8-bit rows.
#include "paged_attention.h"

namespace fbgemm_amd {
hipError_t launch_paged_attention_bf16_rows8(const AttentionArgs& a, hipStream_t stream) { return attention::launch_any<true, 8>(a, stream); }
} // namespace fbgemm_amd
