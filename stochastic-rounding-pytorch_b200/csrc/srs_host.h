// Host-side helpers shared by the units that define extern "C" entry points:
// error text, the device check and the SM count (implemented in srs_abi.cu).
#pragma once

#include <cstdint>
#include <cuda_runtime.h>

#include "srs_b200.h"

namespace srs {

// Sets the calling thread's error text and returns `code`.
int fail(int code, const char* fmt, ...);
int cuda_fail(cudaError_t e, const char* what);
void clear_error();

// SRS_OK if the current device runs the kernels (compute capability 10.0).
int check_device();

// Multiprocessors of the current device (after a successful check_device()).
int sm_count();

inline bool valid_format(int f) { return f >= SRS_FMT_F32 && f <= SRS_FMT_E5M2; }
inline bool valid_rule(int r) {
  return r == SRS_RULE_NEAREST || r == SRS_RULE_STOCHASTIC || r == SRS_RULE_TOWARD_ZERO;
}
inline int fmt_bytes(int f) { return f == SRS_FMT_F32 ? 4 : (f <= SRS_FMT_F16 ? 2 : 1); }

}  // namespace srs
