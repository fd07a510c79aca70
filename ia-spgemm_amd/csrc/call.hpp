// call.hpp — what the entry points on a caller's device and stream share (attention.hip,
// rel_bias.hip): the device, refusals, limits of a launch, and the buckets of a distance.
#pragma once

#include "ias.h"
#include "ias_internal.hpp"

#include <hip/hip_runtime.h>

#include <cstdint>

#define HIPC(x)                                                                   \
    do {                                                                          \
        hipError_t _e = (x);                                                      \
        if (_e != hipSuccess) {                                                   \
            ias::set_last_error("%s failed: %s", #x, hipGetErrorString(_e));      \
            return _e == hipErrorOutOfMemory ? IAS_ERROR_OUT_OF_MEMORY : IAS_ERROR_DEVICE; \
        }                                                                         \
    } while (0)

#define REFUSE(status, ...)               \
    do {                                  \
        ias::set_last_error(__VA_ARGS__); \
        return status;                    \
    } while (0)

namespace ias {

// Makes `device` current for the call and puts the caller's back.
struct OnDevice {
    int before = -1;
    hipError_t to(int device) {
        hipError_t e = hipGetDevice(&before);
        if (e == hipSuccess && before != device) e = hipSetDevice(device);
        else if (e == hipSuccess) before = -1;
        return e;
    }
    ~OnDevice() {
        if (before >= 0) (void)hipSetDevice(before);
    }
};

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

inline ias_status launched() {
    HIPC(hipGetLastError());
    return IAS_SUCCESS;
}

// A launch holds fewer than 2^32 threads.
inline ias_status check_grid(int64_t grid, int threads) {
    if (grid > (int64_t)UINT32_MAX / threads) REFUSE(IAS_ERROR_OVERFLOW, "%lld workgroups of %d threads in a launch", (long long)grid, threads);
    return IAS_SUCCESS;
}

namespace dev {

// How many of the ascending edges are <= d.
__device__ inline int bucket_of(int64_t d, const int32_t *edges, int num_buckets) {
    int lo = 0, hi = num_buckets - 1;
    while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (edges[mid] <= d) lo = mid + 1;
        else hi = mid;
    }
    return lo;
}

}  // namespace dev
}  // namespace ias
