// internal.h -- what the library's translation units share and do not export.
#pragma once
#include <hip/hip_runtime.h>

namespace ggq {

// true for hipSuccess; otherwise stores the text that ggq_last_error() returns on this thread
__attribute__((visibility("hidden"))) bool report_hip(hipError_t e, const char *what);

}  // namespace ggq
