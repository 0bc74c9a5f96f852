// What the files of the C boundary share: the calling thread's error message and
// the argument checks.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/cpab_hip.h"

namespace cpab {

// Sets the calling thread's message and returns `code`.
int fail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
int check_hip(hipError_t e, const char* what);
// Compute units of the current device.
int compute_units();

}  // namespace cpab

#define CPAB_REQUIRE(ptr) \
  do { if (!(ptr)) return fail(CPAB_ERR_INVALID, "%s must not be NULL", #ptr); } while (0)

// Per-cell tables are read as 8- and 16-byte vectors; every float array must
// be at least float-aligned.
#define CPAB_ALIGNED(ptr, bytes)                                                      \
  do {                                                                                \
    if ((ptr) && (reinterpret_cast<uintptr_t>(ptr) % (bytes)) != 0)                  \
      return fail(CPAB_ERR_INVALID, "%s must be %d-byte aligned", #ptr, (int)(bytes)); \
  } while (0)
