// One instance of the attention kernels (paged_attention.h): fp16 queries, rows of the same type.
#include "paged_attention.h"

namespace fbgemm_amd {
hipError_t launch_paged_attention_fp16(const AttentionArgs& a, hipStream_t stream) { return attention::launch_any<false, 16>(a, stream); }
} // namespace fbgemm_amd
