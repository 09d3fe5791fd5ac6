// launch_common.hpp -- what the entry points of cache.cpp and decode.cpp do
// alike around a launch (internal to libmanta_rocm.so).
#pragma once

#include <hip/hip_runtime.h>

#include "manta_cache.h"
#include "runtime_internal.hpp"

#define TRY_HIP(call, what)                                                             \
    do {                                                                                \
        hipError_t e_ = (call);                                                         \
        if (e_ != hipSuccess)                                                           \
            return manta_rt::fail(err, MANTA_ROCM_ERROR, "%s: %s (%s)", what, hipGetErrorName(e_), \
                                  hipGetErrorString(e_));                               \
    } while (0)

namespace manta_rt {

// A launch, counted and timed as the runtime's other kernels are.
template <class F>
int launch(MantaRocm* rt, const char* what, char** err, F f) {
    void* ev = launch_begin(rt);
    const hipError_t e = f((hipStream_t)runtime_stream(rt));
    launch_end(rt, what, ev);
    TRY_HIP(e, what);
    return MANTA_ROCM_OK;
}

inline bool aligned16(const void* p, int64_t a, int64_t b, int size) {
    return ((uintptr_t)p % 16) == 0 && (a * size) % 16 == 0 && (b * size) % 16 == 0;
}

inline int element_size(int dtype) { return dtype == MANTA_ROCM_F32 ? 4 : 2; }

}  // namespace manta_rt
