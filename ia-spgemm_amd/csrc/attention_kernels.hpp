// attention_kernels.hpp — device code of the block-sparse attention (attention.hip).
#pragma once

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include <cstdint>

#include "call.hpp"

namespace ias {
namespace dev {

// A call's shapes, strides and pointers, as the kernels take them.
struct Side {
    const uint16_t *p;
    int64_t batch, token, head;
    __device__ const uint16_t *at(int64_t b, int64_t n, int64_t h) const { return p + b * batch + n * token + h * head; }
};
struct SideOut {
    uint16_t *p;
    int64_t batch, token, head;
    __device__ uint16_t *at(int64_t b, int64_t n, int64_t h) const { return p + b * batch + n * token + h * head; }
};
struct AttnShape {
    int64_t q_len, k_len;
    int32_t batch, q_heads, k_heads, group, dim, block, keep, causal, nblocks, num_buckets, clear;
    uint32_t inverse, inverse_keep;   // ceil(2^16 / group), ceil(2^32 / keep) (0 for keep = 1)
    float scale;
    const int32_t *q_lens, *k_lens;
    const uint16_t *table;
    const int32_t *edges;
    const uint8_t *map;       // bucket of each distance, map[d + k_len - 1]
    // r / group for r < 64 (group <= 64: the inverse is off by less than 2^-16)
    __device__ int per_group(int r) const { return (int)((uint32_t)r * inverse >> 16); }
    // e / keep for e < 2^14 (keep <= 256)
    __device__ int per_keep(int e) const { return inverse_keep ? (int)__umulhi((uint32_t)e, inverse_keep) : e; }
    __device__ int32_t ql(int b) const {
        return q_lens ? min(max(q_lens[b], 0), (int32_t)q_len) : (int32_t)q_len;
    }
    __device__ int32_t kl(int b) const {
        return k_lens ? min(max(k_lens[b], 0), (int32_t)k_len) : (int32_t)k_len;
    }
};

struct Bf16 {
    static constexpr bool NARROW = false;   // 8 bits of exponent, as fp32
    static __device__ float up(uint16_t x) { return __uint_as_float((uint32_t)x << 16); }
    static __device__ uint16_t down(float f) {
        __hip_bfloat16 h = __float2bfloat16(f);
        return *reinterpret_cast<uint16_t *>(&h);
    }
};
struct Fp16 {
    static constexpr bool NARROW = true;    // 5 bits of exponent
    static __device__ float up(uint16_t x) { return __half2float(*reinterpret_cast<__half *>(&x)); }
    static __device__ uint16_t down(float f) {
        __half h = __float2half(f);
        return *reinterpret_cast<uint16_t *>(&h);
    }
};

// ------------------------------------------------------------------ summary
// Mean of each block's keys.  256 threads: 16-byte chunks of the head
// dimension across, rows of the block down, one f64 sum each; the rows'
// partial sums meet in LDS.  Sums of 8- or 11-bit significands over one block
// are exact in 53 bits for all but absurdly spread values, so the order does
// not show.  Bound by the one read of K, and below some 10 MB by the launch (4096 keys,
// 8 heads of 128, 8 MB: 4.2 us; all 32768 keys of 16 users' 8 heads are 1 GB, so a step
// of single tokens renews one block each: 4.1 us).
template <class T>
__global__ __launch_bounds__(256) void k_block_summary(AttnShape s, Side k, int64_t fresh, int32_t per,
                                                       uint16_t *__restrict__ out) {
    __shared__ double part[16][128];
    const uint32_t head = blockIdx.x / (uint32_t)per;
    const int c0 = (int)(blockIdx.x - head * per), b = head / (uint32_t)s.k_heads, g = head - b * s.k_heads;
    const int kl = s.kl(b);
    int c = c0;
    if (fresh > 0) {
        c += (int)(max((int64_t)0, (int64_t)kl - fresh) / s.block);
        if ((int64_t)c * s.block >= kl) return;
    }
    const int chunks = s.dim / 8, lane = threadIdx.x % 16, row = threadIdx.x / 16;
    const int64_t j0 = (int64_t)c * s.block;
    const int n = (int)max((int64_t)0, min((int64_t)s.block, kl - j0));
    double sum[8] = {};
    if (lane < chunks)
        for (int r = row; r < n; r += 16) {
            const uint4 x = *reinterpret_cast<const uint4 *>(k.at(b, j0 + r, g) + 8 * lane);
            const uint32_t u[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                sum[2 * e] += (double)T::up((uint16_t)u[e]);
                sum[2 * e + 1] += (double)T::up((uint16_t)(u[e] >> 16));
            }
        }
#pragma unroll
    for (int e = 0; e < 8; ++e) part[row][8 * lane + e] = sum[e];
    __syncthreads();
    if ((int)threadIdx.x < s.dim) {
        double t = 0.0;
        for (int r = 0; r < 16; ++r) t += part[r][threadIdx.x];
        const uint16_t m = T::down((float)(t / (double)max(n, 1)));
        out[(((int64_t)b * s.k_heads + g) * s.nblocks + c) * s.dim + threadIdx.x] = m;
    }
}

// ------------------------------------------------------------------ buckets
// The buckets of d .. d + 3, a byte each.
__device__ inline uint32_t four_buckets(int d, const int32_t *edges, int num_buckets) {
    int n = bucket_of(d, edges, num_buckets);
    uint32_t got = n;
    for (int e = 1; e < 4; ++e) {
        while (n < num_buckets - 1 && edges[n] <= d + e) ++n;
        got |= (uint32_t)n << (8 * e);
    }
    return got;
}

// map[d + k_len - 1] = how many edges are <= d, for every distance of a call; clears
// `count` for a backward pass, which saves it a launch.  4.5 us: the launch.
__global__ __launch_bounds__(256) void k_bucket_map(int64_t k_len, int64_t n, int32_t num_buckets,
                                                    const int32_t *__restrict__ edges, uint8_t *__restrict__ map,
                                                    int32_t *__restrict__ count, int64_t entries) {
    const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
    for (int64_t c = e; c < entries; c += (int64_t)gridDim.x * 256) count[c] = 0;
    if (e >= n) return;
    map[e] = (uint8_t)bucket_of(e - (k_len - 1), edges, num_buckets);
}

}  // namespace dev
}  // namespace ias
