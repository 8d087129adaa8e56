// How an entry point of the C ABI fails: the code it returns, with the text that
// fbgemm_amd_last_error() hands the calling thread (c_api.cpp keeps it).
#pragma once
#include <hip/hip_runtime.h>

#include "../../include/fbgemm_amd.h"

namespace fbgemm_amd {
int fail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
} // namespace fbgemm_amd

#define HIP_TRY(expr)                                                                   \
  do {                                                                                  \
    hipError_t e_ = (expr);                                                             \
    if (e_ != hipSuccess) return fbgemm_amd::fail(FBGEMM_AMD_E_HIP, "%s: %s", #expr, hipGetErrorString(e_)); \
  } while (0)
