// hprms_host.h - what the translation units of libhprms.so share on the host:
// the calling thread's error text, the launch check, the CU count and the
// bounds of sizes and strides.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "hp_rms_norm_amd.h"

namespace hprms {

// Not exported: the product and the bench library, loaded into one process,
// each keep their own.
#define HPRMS_LOCAL __attribute__((visibility("hidden")))

// A whole MI355X: what the row-count rules were measured on.
constexpr int kRefCUs = 256;

// Sets the calling thread's error text (hprms_last_error) and returns `code`.
HPRMS_LOCAL __attribute__((format(printf, 2, 3))) int fail(int code, const char* fmt, ...);

// HPRMS_OK, or HPRMS_E_LAUNCH with the runtime's message about the last launch.
HPRMS_LOCAL int check_launch(const char* what);

// CUs of the current device; 256 when there is no device to ask (a launch
// would then fail and report why)
HPRMS_LOCAL int current_cus();

// No buffer on any GPU spans more bytes (virtual addresses have at most 57
// bits), and under this bound the kernels' 64-bit row offsets cannot overflow.
constexpr int64_t kMaxExtentBytes = int64_t(1) << 56;

// `rows` rows of `width` elements of `elem` bytes, `stride` elements apart,
// span at most kMaxExtentBytes
inline bool extent_ok(int64_t rows, int64_t stride, int64_t elem, int64_t width) {
  if (rows <= 1) return true;
  if (stride > kMaxExtentBytes / elem) return false;
  return rows - 1 <= (kMaxExtentBytes / elem - width) / stride;
}

}  // namespace hprms
