// kb200_internal.h -- host-side helpers shared by the C-ABI entry points.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>
#include <stddef.h>
#include <atomic>
#include "../../include/kb200.h"

namespace kb {
// Records a message for kb200_last_error() and returns `code`.
int set_error(int code, const char* fmt, ...);
inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
inline size_t align_up(size_t x, size_t a = 256) { return (x + a - 1) / a * a; }
// Lets `kernel` use `bytes` of dynamic shared memory on the current device.  `done` is the
// kernel's own mask of the devices where that is set already (setting it twice does no harm).
int allow_smem(const void* kernel, size_t bytes, std::atomic<uint64_t>& done);
// SMs of the current device (148 without one).
int sm_count();
// Checks the result of the launches just issued.
int check_launch(const char* what);
}  // namespace kb
