// rel_bias.hip — relative position bias by buckets as a dense matrix, and its
// gradient (ias_rel_bias* of include/ias.h).  The reference has no counterpart.
#include "ias.h"
#include "ias_internal.hpp"
#include "call.hpp"

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

namespace ias {
namespace {

__device__ inline float up(float x) { return x; }
__device__ inline float up(__hip_bfloat16 x) { return __bfloat162float(x); }
__device__ inline float up(__half x) { return __half2float(x); }
__device__ inline void down(float x, float *o) { *o = x; }
__device__ inline void down(float x, __hip_bfloat16 *o) { *o = __float2bfloat16(x); }
__device__ inline void down(float x, __half *o) { *o = __float2half(x); }

constexpr int V = 8;         // consecutive values of a thread of k_rel_bias
constexpr int HEADS = 16;    // heads of a workgroup
constexpr int E = 2;         // neighbouring diagonals of a thread of k_rel_bias_grad
constexpr int SPAN = 256 * E;

// out[h][i][j] = table[bucket(j - i - shift)][h].  A thread has 8 consecutive values
// of one matrix (counted through its rows) and writes them for 16 heads: their
// buckets are found once, by one search and steps from edge to edge, and a head costs
// 8 reads of the table in LDS and one 16-byte store (32 for f32).  Bound by the
// stores: 2048 x 2048, 16 heads, bf16, 134 MB in 24 us, 5.6 TB/s.
template <class T>
__global__ __launch_bounds__(256) void k_rel_bias(int32_t heads, int64_t q_len, int64_t k_len, int32_t nb,
                                                  const T *__restrict__ table, const int32_t *__restrict__ edges,
                                                  T *__restrict__ out) {
    typedef uint32_t Packed __attribute__((ext_vector_type(sizeof(T) * V / 4), aligned(sizeof(T))));
    __shared__ T ts[64 * HEADS];
    __shared__ int32_t es[64];
    const int h0 = blockIdx.y * HEADS, hn = min(HEADS, heads - h0);
    for (int e = threadIdx.x; e < nb * HEADS; e += 256)
        if (e % HEADS < hn) ts[e] = table[(e / HEADS) * heads + h0 + e % HEADS];
    if ((int)threadIdx.x < nb - 1) es[threadIdx.x] = edges[threadIdx.x];
    __syncthreads();
    const int64_t size = q_len * k_len, e0 = ((int64_t)blockIdx.x * 256 + threadIdx.x) * V;
    if (e0 >= size) return;
    const int64_t i = e0 / k_len;
    int64_t j = e0 - i * k_len, d = j - i - (k_len - q_len);
    int at[V], n = dev::bucket_of(d, es, nb);
#pragma unroll
    for (int v = 0; v < V; ++v) {
        at[v] = n * HEADS;
        if (++j < k_len) {
            ++d;
            while (n < nb - 1 && es[n] <= d) ++n;
        } else {   // on to the next row
            j = 0;
            d -= k_len;
            n = dev::bucket_of(d, es, nb);
        }
    }
    for (int h = 0; h < hn; ++h) {
        alignas(16) T y[V];
#pragma unroll
        for (int v = 0; v < V; ++v) y[v] = ts[at[v] + h];
        T *to = out + (h0 + h) * size + e0;
        if (e0 + V <= size) {
            *reinterpret_cast<Packed *>(to) = *reinterpret_cast<Packed *>(y);   // vector stores, whatever their alignment
        } else {
#pragma unroll
            for (int v = 0; v < V; ++v)
                if (e0 + v < size) to[v] = y[v];
        }
    }
}

// Values of a diagonal are summed by eights, and 2048 or more of them (batch elements of short
// matrices) by themselves: 2^16 added one by one to what has grown to their sum can be off by
// 2^-9 of it.
constexpr int RUN = 2048;

// Sums over diagonals.  A thread has 2 neighbouring diagonals and goes down some rows
// of every batch element, its loads moving one to the right with each row: the sums
// stay in registers, and buckets matter only at the end, where each is one stretch of
// the workgroup's 512 diagonals.  part: [chunk][head][bucket].  Bound by the read of
// the gradient: 2 x 16 x 2048 x 2048, bf16, 268 MB in 49 us (part of it from the cache; 66
// us with k_rel_bias_sum and gradients that are not in it, 4 TB/s).  Four or eight
// diagonals a thread took 81 to 116 us: fewer workgroups, unaligned loads that cross lines.
template <class T>
__global__ __launch_bounds__(256) void k_rel_bias_grad(int64_t batch, int32_t heads, int64_t q_len, int64_t k_len,
                                                       int32_t nb, const T *__restrict__ grad, int64_t sb, int64_t sh,
                                                       int64_t sr, const int32_t *__restrict__ edges, int32_t spans,
                                                       int32_t rows, float *__restrict__ part) {
    __shared__ float sums[SPAN];
    __shared__ int32_t es[64];
    const int tid = threadIdx.x, h = blockIdx.x % heads;
    const int64_t chunk = blockIdx.x / heads;
    const int64_t r0 = chunk / spans * rows, r1 = min(q_len, r0 + rows);
    // column of the thread's first diagonal in row i: c0 + i
    const int64_t first = chunk % spans * SPAN - (q_len - 1), c0 = first + tid * E;
    if (tid < nb - 1) es[tid] = edges[tid];
    float all[E] = {}, acc[E] = {};
    int64_t held = 0;   // values in acc
    // rows where both columns are there, and those beside them where one is
    const int64_t ia = max(r0, -c0), ib = min(r1, k_len - E + 1 - c0);
    for (int64_t b = 0; b < batch; ++b) {
        const T *x = grad + b * sb + h * sh + c0;
        int64_t i = ia;
        auto rows_down = [&](auto some) {   // rows whose loads are in flight together
            constexpr int U = decltype(some)::value;
            for (; i + U <= ib; i += U) {
                T y[U][E];
#pragma unroll
                for (int u = 0; u < U; ++u) __builtin_memcpy(y[u], x + (i + u) * (sr + 1), sizeof y[u]);
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    float z[U];
#pragma unroll
                    for (int u = 0; u < U; ++u) z[u] = up(y[u][e]);
#pragma unroll
                    for (int n = 1; n < U; n *= 2)
#pragma unroll
                        for (int u = 0; u < U; u += 2 * n) z[u] += z[u + n];
                    acc[e] += z[0];
                }
            }
        };
        rows_down(std::integral_constant<int, 8>{});
        rows_down(std::integral_constant<int, 2>{});
        rows_down(std::integral_constant<int, 1>{});
        for (int side = 0; side < 2; ++side) {
            const int64_t from = side ? max(r0, max(ia, ib)) : max(r0, -c0 - (E - 1)), to = side ? min(r1, k_len - c0) : min(min(r1, ia), k_len - c0);
            for (int64_t n = from; n < to; ++n)
#pragma unroll
                for (int e = 0; e < E; ++e)
                    if (c0 + n + e >= 0 && c0 + n + e < k_len) acc[e] += up(x[n * (sr + 1) + e]);
        }
        if ((held += r1 - r0) >= RUN) {
#pragma unroll
            for (int e = 0; e < E; ++e) {
                all[e] += acc[e];
                acc[e] = 0.0f;
            }
            held = 0;
        }
    }
#pragma unroll
    for (int e = 0; e < E; ++e) sums[tid * E + e] = all[e] + acc[e];
    __syncthreads();
    // bucket n is the stretch of diagonals from edge n - 1 to edge n
    const int lane = tid % 64;
    const int64_t d0 = first - (k_len - q_len);   // distance of the first diagonal
    for (int n = tid / 64; n < nb; n += 4) {
        const int64_t lo = n == 0 ? 0 : max((int64_t)0, es[n - 1] - d0), hi = n == nb - 1 ? SPAN : min((int64_t)SPAN, es[n] - d0);
        float t = 0.0f;
        for (int64_t k = lo + lane; k < hi; k += 64) t += sums[k];
        for (int d = 32; d; d >>= 1) t += __shfl_xor(t, d);
        if (lane == 0) part[(chunk * heads + h) * nb + n] = t;
    }
}

// dtable[n][h]: one wave for each, in a fixed order.
template <class T>
__global__ __launch_bounds__(64) void k_rel_bias_sum(int64_t chunks, int32_t heads, int32_t nb,
                                                     const float *__restrict__ part, T *__restrict__ dtable) {
    const int h = blockIdx.x % heads, n = blockIdx.x / heads;
    float t = 0.0f;
    for (int64_t c = threadIdx.x; c < chunks; c += 64) t += part[(c * heads + h) * nb + n];
    for (int d = 32; d; d >>= 1) t += __shfl_xor(t, d);
    if (threadIdx.x == 0) down(t, dtable + (int64_t)n * heads + h);
}

ias_status check_bias(int32_t dtype, int64_t batch, int32_t heads, int64_t q_len, int64_t k_len, int32_t nb, int32_t device) {
    if (dtype < IAS_DTYPE_F32 || dtype > IAS_DTYPE_F16) REFUSE(IAS_ERROR_UNSUPPORTED, "dtype %d", dtype);
    if (batch < 0 || heads < 0 || q_len < 0 || k_len < 0 || device < 0)
        REFUSE(IAS_ERROR_INVALID_ARGUMENT, "batch %lld, heads %d, q_len %lld, k_len %lld, device %d", (long long)batch, heads,
               (long long)q_len, (long long)k_len, device);
    if (nb < 1 || nb > 64) REFUSE(IAS_ERROR_UNSUPPORTED, "%d buckets: 1 to 64", nb);
    if (batch > INT32_MAX || heads > 1 << 16 || q_len > 1 << 24 || k_len > 1 << 24 ||
        (q_len > 0 && k_len > (1ll << 34) / q_len) || (q_len > 0 && batch * heads > INT64_MAX / 16 / q_len / std::max<int64_t>(1, k_len)))
        REFUSE(IAS_ERROR_OVERFLOW, "batch x heads x q_len x k_len is too large");
    return IAS_SUCCESS;
}

// How the gradient is shared out: spans of 512 diagonals, and so many rows that
// about 4096 workgroups are there (half of them hold corners outside the matrix), 16
// at least (each ends in sums of its own) and all that there are at most (2^24: the
// kernel takes 32 bits; a tall matrix of many heads would ask for 2^31 and more).
struct Chunks {
    int64_t spans = 0, rows = 1, all = 0;
    Chunks(int64_t batch, int32_t heads, int64_t q_len, int64_t k_len) {
        if (batch == 0 || heads == 0 || q_len == 0 || k_len == 0) return;
        spans = ceil_div(q_len + k_len - 1, SPAN);
        rows = std::min<int64_t>(q_len, std::max<int64_t>(16, ceil_div(q_len * spans * heads, 4096)));
        all = spans * ceil_div(q_len, rows);
    }
};

template <class T>
ias_status bias(int32_t heads, int64_t q_len, int64_t k_len, int32_t nb, const void *table, const int32_t *edges,
                void *out, hipStream_t st) {
    const dim3 grid((unsigned)ceil_div(q_len * k_len, 256 * V), (unsigned)ceil_div(heads, HEADS));
    k_rel_bias<T><<<grid, 256, 0, st>>>(heads, q_len, k_len, nb, (const T *)table, edges, (T *)out);
    return launched();
}

template <class T>
ias_status bias_grad(int64_t batch, int32_t heads, int64_t q_len, int64_t k_len, int32_t nb, const void *grad,
                     int64_t sb, int64_t sh, int64_t sr, const int32_t *edges, void *dtable, float *part, hipStream_t st) {
    const Chunks c(batch, heads, q_len, k_len);
    if (c.all > 0) {
        k_rel_bias_grad<T><<<dim3((unsigned)(c.all * heads)), 256, 0, st>>>(batch, heads, q_len, k_len, nb, (const T *)grad, sb, sh, sr, edges,
                                                                            (int32_t)c.spans, (int32_t)c.rows, part);
        IAS_TRY(launched());
    }
    k_rel_bias_sum<T><<<dim3((unsigned)(heads * nb)), 64, 0, st>>>(c.all, heads, nb, part, (T *)dtable);
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
    const int64_t parts = Chunks(batch, heads, q_len, k_len).all * heads;
    if (parts >= 1 << 24) REFUSE(IAS_ERROR_OVERFLOW, "%lld workgroups of 256 threads in a launch", (long long)parts);
    *bytes = parts * num_buckets * (int64_t)sizeof(float);
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
