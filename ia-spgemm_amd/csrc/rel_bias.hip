// rel_bias.hip — relative position bias by buckets as a dense matrix, and its
// gradient (ias_rel_bias* of include/ias.h).  The reference has no counterpart.
#include "ias.h"
#include "ias_internal.hpp"

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include <algorithm>

namespace ias {
namespace {

#define HIPC(x)                                                                   \
    do {                                                                          \
        hipError_t _e = (x);                                                      \
        if (_e != hipSuccess) {                                                   \
            set_last_error("%s failed: %s", #x, hipGetErrorString(_e));           \
            return _e == hipErrorOutOfMemory ? IAS_ERROR_OUT_OF_MEMORY : IAS_ERROR_DEVICE; \
        }                                                                         \
    } while (0)

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

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

__device__ inline float up(float x) { return x; }
__device__ inline float up(__hip_bfloat16 x) { return __bfloat162float(x); }
__device__ inline float up(__half x) { return __half2float(x); }
__device__ inline void down(float x, float *o) { *o = x; }
__device__ inline void down(float x, __hip_bfloat16 *o) { *o = __float2bfloat16(x); }
__device__ inline void down(float x, __half *o) { *o = __float2half(x); }

__device__ inline int bucket_of(int64_t d, const int32_t *edges, int nb) {
    int lo = 0, hi = nb - 1;
    while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (edges[mid] <= d) lo = mid + 1;
        else hi = mid;
    }
    return lo;
}

template <class T>
__global__ __launch_bounds__(256) void k_rel_bias(int32_t heads, int64_t q_len, int64_t k_len, int32_t nb,
                                                  const T *__restrict__ table, const int32_t *__restrict__ edges,
                                                  T *__restrict__ out) {
    const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (e >= q_len * k_len) return;
    const int64_t i = e / k_len, j = e % k_len;
    const int n = bucket_of(j - i - (k_len - q_len), edges, nb);
    for (int h = 0; h < heads; ++h) out[h * q_len * k_len + e] = table[n * heads + h];
}

// Rows of one head, each lane's sums by bucket in its own column of LDS.
template <class T>
__global__ __launch_bounds__(64) void k_rel_bias_grad(int64_t batch, int32_t heads, int64_t q_len, int64_t k_len,
                                                      int32_t nb, const T *__restrict__ grad, int64_t sb, int64_t sh,
                                                      int64_t sr, const int32_t *__restrict__ edges,
                                                      int32_t per, float *__restrict__ part) {
    extern __shared__ float hist[];   // nb x 64
    __shared__ int32_t es[64];
    const int lane = threadIdx.x, h = blockIdx.x % heads;
    const int64_t chunk = blockIdx.x / heads, rows = batch * q_len;
    if (lane < nb - 1) es[lane] = edges[lane];
    for (int n = 0; n < nb; ++n) hist[n * 64 + lane] = 0.0f;
    __syncthreads();
    for (int64_t r = chunk * per; r < min(rows, (chunk + 1) * per); ++r) {
        const int64_t b = r / q_len, i = r % q_len;
        const T *x = grad + b * sb + h * sh + i * sr;
        for (int64_t j = lane; j < k_len; j += 64) hist[bucket_of(j - i - (k_len - q_len), es, nb) * 64 + lane] += up(x[j]);
    }
    __syncthreads();
    if (lane < nb) {
        float t = 0.0f;
        for (int n = 0; n < 64; ++n) t += hist[lane * 64 + n];
        part[(chunk * heads + h) * nb + lane] = t;
    }
}

template <class T>
__global__ __launch_bounds__(64) void k_rel_bias_sum(int64_t chunks, int32_t heads, int32_t nb,
                                                     const float *__restrict__ part, T *__restrict__ dtable) {
    const int h = blockIdx.x % heads, n = blockIdx.x / heads;
    float t = 0.0f;
    for (int64_t c = threadIdx.x; c < chunks; c += 64) t += part[(c * heads + h) * nb + n];
    for (int d = 32; d; d >>= 1) t += __shfl_xor(t, d);
    if (threadIdx.x == 0) down(t, dtable + (int64_t)n * heads + h);
}

#define REFUSE(status, ...)          \
    do {                             \
        set_last_error(__VA_ARGS__); \
        return status;               \
    } while (0)

ias_status check_bias(int32_t dtype, int64_t batch, int32_t heads, int64_t q_len, int64_t k_len, int32_t nb, int32_t device) {
    if (dtype < IAS_DTYPE_F32 || dtype > IAS_DTYPE_F16) REFUSE(IAS_ERROR_UNSUPPORTED, "dtype %d", dtype);
    if (batch < 0 || heads < 0 || q_len < 0 || k_len < 0 || device < 0)
        REFUSE(IAS_ERROR_INVALID_ARGUMENT, "batch %lld, heads %d, q_len %lld, k_len %lld, device %d", (long long)batch, heads,
               (long long)q_len, (long long)k_len, device);
    if (nb < 1 || nb > 64) REFUSE(IAS_ERROR_UNSUPPORTED, "%d buckets: 1 to 64", nb);
    if (batch > INT32_MAX || q_len > INT32_MAX / 2 || k_len > INT32_MAX / 2 ||
        (q_len > 0 && batch * heads > INT64_MAX / 16 / q_len / std::max<int64_t>(1, k_len)))
        REFUSE(IAS_ERROR_OVERFLOW, "batch x heads x q_len x k_len is too large");
    return IAS_SUCCESS;
}

constexpr int ROWS = 16;   // rows of a workgroup of the gradient
int64_t chunks_of(int64_t batch, int64_t q_len) { return ceil_div(batch * q_len, ROWS); }

ias_status launched() {
    HIPC(hipGetLastError());
    return IAS_SUCCESS;
}

template <class T>
ias_status bias(int32_t heads, int64_t q_len, int64_t k_len, int32_t nb, const void *table, const int32_t *edges,
                void *out, hipStream_t st) {
    const int64_t grid = ceil_div(q_len * k_len, 256);
    k_rel_bias<T><<<dim3((unsigned)grid), 256, 0, st>>>(heads, q_len, k_len, nb, (const T *)table, edges, (T *)out);
    return launched();
}

template <class T>
ias_status bias_grad(int64_t batch, int32_t heads, int64_t q_len, int64_t k_len, int32_t nb, const void *grad,
                     int64_t sb, int64_t sh, int64_t sr, const int32_t *edges, void *dtable, float *part, hipStream_t st) {
    const int64_t chunks = k_len > 0 ? chunks_of(batch, q_len) : 0;
    if (chunks * heads > 0) {
        k_rel_bias_grad<T><<<dim3((unsigned)(chunks * heads)), 64, (size_t)nb * 256, st>>>(batch, heads, q_len, k_len, nb, (const T *)grad,
                                                                                           sb, sh, sr, edges, ROWS, part);
        IAS_TRY(launched());
    }
    k_rel_bias_sum<T><<<dim3((unsigned)(heads * nb)), 64, 0, st>>>(chunks, heads, nb, part, (T *)dtable);
    return launched();
}

}  // namespace
}  // namespace ias

using namespace ias;

extern "C" ias_status ias_rel_bias(int32_t dtype, int32_t heads, int64_t q_len, int64_t k_len, int32_t num_buckets,
                                   const void *table, const int32_t *edges, void *out, int32_t device, void *stream) {
    IAS_TRY(check_bias(dtype, 1, heads, q_len, k_len, num_buckets, device));
    if (heads == 0 || q_len == 0 || k_len == 0) return IAS_SUCCESS;
    if (!table || (num_buckets > 1 && !edges) || !out) REFUSE(IAS_ERROR_INVALID_ARGUMENT, "no table, edges or out");
    OnDevice on;
    HIPC(on.to(device));
    hipStream_t st = (hipStream_t)stream;
    if (dtype == IAS_DTYPE_F32) return bias<float>(heads, q_len, k_len, num_buckets, table, edges, out, st);
    if (dtype == IAS_DTYPE_BF16) return bias<__hip_bfloat16>(heads, q_len, k_len, num_buckets, table, edges, out, st);
    return bias<__half>(heads, q_len, k_len, num_buckets, table, edges, out, st);
}

extern "C" ias_status ias_rel_bias_grad_workspace(int64_t batch, int32_t heads, int64_t q_len, int64_t k_len,
                                                  int32_t num_buckets, int64_t *bytes) {
    IAS_TRY(check_bias(IAS_DTYPE_F32, batch, heads, q_len, k_len, num_buckets, 0));
    if (!bytes) REFUSE(IAS_ERROR_INVALID_ARGUMENT, "no bytes");
    *bytes = chunks_of(batch, q_len) * heads * num_buckets * (int64_t)sizeof(float);
    return IAS_SUCCESS;
}

extern "C" ias_status ias_rel_bias_grad(int32_t dtype, int64_t batch, int32_t heads, int64_t q_len, int64_t k_len,
                                        int32_t num_buckets, const void *grad, int64_t stride_batch, int64_t stride_head,
                                        int64_t stride_row, const int32_t *edges, void *dtable, void *workspace,
                                        int64_t workspace_bytes, int32_t device, void *stream) {
    IAS_TRY(check_bias(dtype, batch, heads, q_len, k_len, num_buckets, device));
    if (heads == 0) return IAS_SUCCESS;
    const bool any = batch > 0 && q_len > 0 && k_len > 0;
    if (!dtable || (any && !grad) || (num_buckets > 1 && !edges)) REFUSE(IAS_ERROR_INVALID_ARGUMENT, "no grad, edges or dtable");
    int64_t need = 0;
    IAS_TRY(ias_rel_bias_grad_workspace(batch, heads, q_len, k_len, num_buckets, &need));
    if (any && (!workspace || workspace_bytes < need))
        REFUSE(IAS_ERROR_INSUFFICIENT_CAPACITY, "workspace of %lld bytes: %lld are needed", (long long)(workspace ? workspace_bytes : 0), (long long)need);
    if ((uintptr_t)workspace & 15) REFUSE(IAS_ERROR_INVALID_ARGUMENT, "the workspace has to be 16-byte aligned");
    OnDevice on;
    HIPC(on.to(device));
    hipStream_t st = (hipStream_t)stream;
    float *part = static_cast<float *>(workspace);
    if (dtype == IAS_DTYPE_F32)
        return bias_grad<float>(batch, heads, q_len, k_len, num_buckets, grad, stride_batch, stride_head, stride_row, edges, dtable, part, st);
    if (dtype == IAS_DTYPE_BF16)
        return bias_grad<__hip_bfloat16>(batch, heads, q_len, k_len, num_buckets, grad, stride_batch, stride_head, stride_row, edges, dtable, part, st);
    return bias_grad<__half>(batch, heads, q_len, k_len, num_buckets, grad, stride_batch, stride_head, stride_row, edges, dtable, part, st);
}
