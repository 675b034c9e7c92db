// Host-side plumbing shared by the C entry points: status codes, the per-thread
// error message, argument checks and the post-launch check.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <cstdarg>

#include "qwen35_hip.h"

namespace qk {

// Records a printf-style message for the calling thread and returns `status`.
int fail(int status, const char* fmt, ...) __attribute__((format(printf, 2, 3)));

// Clears the calling thread's message and returns QWEN_STATUS_OK.
int ok();

// QWEN_STATUS_LAUNCH_FAILED with the runtime's message if the last launch on
// this thread was rejected, else ok().
int check_launch(const char* what);

inline hipStream_t as_stream(void* s) { return reinterpret_cast<hipStream_t>(s); }

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Whether na bytes from a and nb bytes from b have none in common.
inline bool apart(const void* a, size_t na, const void* b, size_t nb) {
    const uintptr_t p = reinterpret_cast<uintptr_t>(a), q = reinterpret_cast<uintptr_t>(b);
    return na == 0 || nb == 0 || p + na <= q || q + nb <= p;
}

// Number of blocks for `items` work items at `per_block` per block.
inline unsigned blocks_for(int64_t items, int64_t per_block) {
    return static_cast<unsigned>((items + per_block - 1) / per_block);
}

// A grid for n workgroups, n below 2^31, of up to 512 threads, along x and, past 2^22 of them, y: one axis of 2^32 threads or more
// runs short without an error. Kernels number their workgroups blockIdx.y * gridDim.x + blockIdx.x and leave from n on.
inline dim3 grid_of(int64_t n) {
    constexpr int64_t kMost = 1 << 22;
    return dim3(static_cast<unsigned>(n < kMost ? n : kMost), blocks_for(n, kMost));
}

}  // namespace qk

#define QK_REQUIRE(cond, ...)                                          \
    do {                                                               \
        if (!(cond)) return ::qk::fail(QWEN_STATUS_INVALID_ARGUMENT, __VA_ARGS__); \
    } while (0)
