// Host-side helpers of the translation units that implement the C ABI: the message of the last
// error (kept by mccl_kernels.hip) and the checks that entry points share.
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

#include "mccl.h"

// Stores the message that mccl_last_error() returns on this thread and returns `code`.
__attribute__((visibility("hidden"), format(printf, 2, 3))) int mccl_report_error(int code, const char* fmt, ...);

namespace {

inline bool ranges_overlap(const void* a, size_t a_bytes, const void* b, size_t b_bytes) {
  const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
  return a && b && a_bytes && b_bytes && x < y + b_bytes && y < x + a_bytes;
}

inline bool misaligned(const void* p, size_t to) { return (uintptr_t)p % to != 0; }

}  // namespace
