// attention_kernels.hpp — device code of the block-sparse attention (attention.hip).
#pragma once

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include <cstdint>

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
    int32_t batch, q_heads, k_heads, group, dim, block, keep, causal, nblocks, num_buckets;
    float scale;
    const int32_t *q_lens, *k_lens;
    const uint16_t *table;
    const uint8_t *map;       // bucket of each distance, map[d + k_len - 1]
    __device__ int32_t ql(int b) const {
        return q_lens ? min(max(q_lens[b], 0), (int32_t)q_len) : (int32_t)q_len;
    }
    __device__ int32_t kl(int b) const {
        return k_lens ? min(max(k_lens[b], 0), (int32_t)k_len) : (int32_t)k_len;
    }
};

struct Bf16 {
    static __device__ float up(uint16_t x) { return __uint_as_float((uint32_t)x << 16); }
    static __device__ uint16_t down(float f) {
        __hip_bfloat16 h = __float2bfloat16(f);
        return *reinterpret_cast<uint16_t *>(&h);
    }
};
struct Fp16 {
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
// not show.  Bound by the one read of K.
template <class T>
__global__ __launch_bounds__(256) void k_block_summary(AttnShape s, Side k, int64_t fresh, int32_t per,
                                                       uint16_t *__restrict__ out) {
    __shared__ double part[16][128];
    int64_t w = blockIdx.x;
    const int c0 = (int)(w % per);
    w /= per;
    const int g = (int)(w % s.k_heads), b = (int)(w / s.k_heads);
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

// ------------------------------------------------------------------ selection
__device__ inline unsigned long long order_key(double x) {
    x = x + 0.0;   // -0 ranks as +0
    const unsigned long long u = (unsigned long long)__double_as_longlong(x);
    return (u >> 63) ? ~u : u | (1ull << 63);
}

template <class T>
__global__ __launch_bounds__(64) void k_block_select(AttnShape s, Side q, const uint16_t *__restrict__ summary,
                                                     int32_t first, int32_t local, int32_t *__restrict__ blocks) {
    extern __shared__ unsigned long long key[];   // nblocks, then the chosen bits
    uint32_t *chosen = reinterpret_cast<uint32_t *>(key + s.nblocks);
    int64_t w = blockIdx.x;
    const int i = (int)(w % s.q_len);
    w /= s.q_len;
    const int g = (int)(w % s.k_heads), b = (int)(w / s.k_heads), lane = threadIdx.x;
    const int ql = s.ql(b), kl = s.kl(b);
    if (i >= ql) return;
    const int p = i + kl - ql;
    const int seen = s.causal ? (p < 0 ? 0 : p / s.block + 1) : (kl + s.block - 1) / s.block;
    for (int n = lane; n < (s.nblocks + 31) / 32; n += 64) chosen[n] = 0;
    for (int c = lane; c < seen; c += 64) {
        const uint16_t *m = summary + (((int64_t)b * s.k_heads + g) * s.nblocks + c) * s.dim;
        double best = -INFINITY;
        for (int h = 0; h < s.group; ++h) {
            const uint16_t *x = q.at(b, i, g * s.group + h);
            double t = 0.0;
            for (int d = 0; d < s.dim; ++d) t += (double)T::up(x[d]) * (double)T::up(m[d]);
            if (t > best) best = t;
        }
        key[c] = order_key(best);
    }
    __syncthreads();
    int left = min(s.keep, seen);
    auto take = [&](int c) {
        if (lane == 0) {
            chosen[c / 32] |= 1u << (c % 32);
            key[c] = 0;
        }
        --left;
        __syncthreads();
    };
    for (int c = 0; c < min(first, seen); ++c) take(c);
    for (int c = max(min(first, seen), seen - local); c < seen; ++c) take(c);
    while (left > 0) {
        unsigned long long top = 0;
        int at = INT32_MAX;
        for (int c = lane; c < seen; c += 64)
            if (key[c] > top) { top = key[c]; at = c; }
        for (int d = 32; d; d >>= 1) {
            const unsigned long long t = __shfl_xor(top, d);
            const int a = __shfl_xor(at, d);
            if (t > top || (t == top && a < at)) { top = t; at = a; }
        }
        take(at);
    }
    int32_t *row = blocks + ((((int64_t)b * s.k_heads + g) * s.q_len) + i) * s.keep;
    int n = 0;
    for (int c0 = 0; c0 < seen; c0 += 64) {
        const int c = c0 + lane;
        const bool on = c < seen && (chosen[c / 32] >> (c % 32) & 1);
        const unsigned long long m = __ballot(on);
        if (on) row[n + __popcll(m & ((1ull << lane) - 1))] = c;
        n += __popcll(m);
    }
    for (int t = n + lane; t < s.keep; t += 64) row[t] = -1;
}

// ------------------------------------------------------------------ bucket map
// map[d + k_len - 1] = how many edges are <= d, for every distance of a call.
__global__ __launch_bounds__(256) void k_bucket_map(int64_t k_len, int64_t n, int32_t num_buckets,
                                                    const int32_t *__restrict__ edges, uint8_t *__restrict__ map) {
    const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (e >= n) return;
    const int64_t d = e - (k_len - 1);
    int lo = 0, hi = num_buckets - 1;
    while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (edges[mid] <= d) lo = mid + 1;
        else hi = mid;
    }
    map[e] = (uint8_t)lo;
}

// ------------------------------------------------------------------ plain forms
// One wave for each (batch, query, head): 64 keys at a time, a key per lane.
__device__ inline float wave_max(float x) {
    for (int d = 32; d; d >>= 1) x = fmaxf(x, __shfl_xor(x, d));
    return x;
}
__device__ inline float wave_sum(float x) {
    for (int d = 32; d; d >>= 1) x += __shfl_xor(x, d);
    return x;
}

template <class T> __device__ float dot_row(const float *a, const uint16_t *x, int dim) {
    float t = 0.0f;
    for (int d = 0; d < dim; ++d) t += a[d] * T::up(x[d]);
    return t;
}

__device__ inline bool first_entry(const int32_t *row, int t, int nblocks) {
    const int c = row[t];
    if (c < 0 || c >= nblocks) return false;
    for (int u = 0; u < t; ++u)
        if (row[u] == c) return false;
    return true;
}

// dq and the row's sums by bucket (sums: batch x q_len x q_heads x buckets), and delta.
template <class T>
__global__ __launch_bounds__(64) void k_grad_q_plain(AttnShape s, Side dout, Side q, Side k, Side v, Side out,
                                                     const float *__restrict__ lse, const int32_t *__restrict__ blocks,
                                                     SideOut dq, float *__restrict__ delta, float *__restrict__ sums) {
    __shared__ float qs[128], ds[128], ps[64], hist[64];
    int64_t w = blockIdx.x;
    const int h = (int)(w % s.q_heads);
    w /= s.q_heads;
    const int i = (int)(w % s.q_len), b = (int)(w / s.q_len), lane = threadIdx.x, g = h / s.group;
    const int ql = s.ql(b), kl = s.kl(b);
    hist[lane] = 0.0f;
    __syncthreads();
    if (i < ql) {
        const int p = i + kl - ql, end = s.causal ? min(kl, p + 1) : kl;
        float part = 0.0f;
        for (int d = lane; d < s.dim; d += 64) {
            qs[d] = T::up(q.at(b, i, h)[d]);
            ds[d] = T::up(dout.at(b, i, h)[d]);
            part += ds[d] * T::up(out.at(b, i, h)[d]);
        }
        const float dl = wave_sum(part), l = lse[((int64_t)b * s.q_heads + h) * s.q_len + i];
        if (lane == 0) delta[((int64_t)b * s.q_heads + h) * s.q_len + i] = dl;
        __syncthreads();
        const int32_t *row = blocks + ((((int64_t)b * s.k_heads + g) * s.q_len) + i) * s.keep;
        float o[2] = {0.0f, 0.0f};
        for (int t = 0; t < s.keep; ++t) {
            if (!first_entry(row, t, s.nblocks)) continue;
            for (int64_t j0 = (int64_t)row[t] * s.block; j0 < (int64_t)(row[t] + 1) * s.block && j0 < end; j0 += 64) {
                const int64_t j = j0 + lane;
                float e = 0.0f;
                if (j < end && l != -INFINITY) {
                    float x = dot_row<T>(qs, k.at(b, j, g), s.dim) * s.scale;
                    const int bucket = s.table ? s.map[j - p + s.k_len - 1] : 0;
                    if (s.table) x += T::up(s.table[bucket * s.q_heads + h]);
                    e = expf(x - l) * (dot_row<T>(ds, v.at(b, j, g), s.dim) - dl);
                }
                ps[lane] = e;
                __syncthreads();
                for (int u = 0; u < 2; ++u) {
                    const int d = lane + 64 * u;
                    if (d >= s.dim) continue;
                    for (int n = 0; n < 64 && j0 + n < end; ++n) o[u] += ps[n] * T::up(k.at(b, j0 + n, g)[d]);
                }
                if (s.table && lane == 0)
                    for (int n = 0; n < 64 && j0 + n < end; ++n) hist[s.map[j0 + n - p + s.k_len - 1]] += ps[n];
                __syncthreads();
            }
        }
        for (int u = 0; u < 2; ++u)
            if (lane + 64 * u < s.dim) dq.at(b, i, h)[lane + 64 * u] = T::down(o[u] * s.scale);
    }
    if (sums && lane < s.num_buckets)
        sums[(((int64_t)b * s.q_len + i) * s.q_heads + h) * s.num_buckets + lane] = hist[lane];
}

// One wave for each (batch, key head, key): every query that reads its block.
template <class T>
__global__ __launch_bounds__(64) void k_grad_kv_plain(AttnShape s, Side dout, Side q, Side k, Side v,
                                                      const float *__restrict__ lse, const float *__restrict__ delta,
                                                      const int32_t *__restrict__ blocks, SideOut dk, SideOut dv) {
    __shared__ float ks[128], vs[128];
    int64_t w = blockIdx.x;
    const int g = (int)(w % s.k_heads);
    w /= s.k_heads;
    const int j = (int)(w % s.k_len), b = (int)(w / s.k_len), lane = threadIdx.x;
    const int ql = s.ql(b), kl = s.kl(b);
    if (j >= kl) return;
    for (int d = lane; d < s.dim; d += 64) {
        ks[d] = T::up(k.at(b, j, g)[d]);
        vs[d] = T::up(v.at(b, j, g)[d]);
    }
    __syncthreads();
    const int c = j / s.block;
    float ok[2] = {}, ov[2] = {};
    for (int i0 = 0; i0 < ql; i0 += 64) {
        const int i = i0 + lane;
        bool on = false;
        if (i < ql && (!s.causal || j <= i + kl - ql)) {
            const int32_t *row = blocks + ((((int64_t)b * s.k_heads + g) * s.q_len) + i) * s.keep;
            for (int t = 0; t < s.keep; ++t) on = on || row[t] == c;
        }
        for (unsigned long long m = __ballot(on); m; m &= m - 1) {
            const int r = i0 + __ffsll(m) - 1;
            for (int h = g * s.group; h < (g + 1) * s.group; ++h) {
                const int64_t at = ((int64_t)b * s.q_heads + h) * s.q_len + r;
                float a = 0.0f, e = 0.0f, x[2] = {}, y[2] = {};
                for (int u = 0; u < 2; ++u) {
                    const int d = lane + 64 * u;
                    if (d >= s.dim) continue;
                    x[u] = T::up(q.at(b, r, h)[d]);
                    y[u] = T::up(dout.at(b, r, h)[d]);
                    a += x[u] * ks[d];
                    e += y[u] * vs[d];
                }
                a = wave_sum(a) * s.scale;
                e = wave_sum(e);
                if (s.table) a += T::up(s.table[s.map[j - (r + kl - ql) + s.k_len - 1] * s.q_heads + h]);
                if (lse[at] == -INFINITY) continue;
                const float pr = expf(a - lse[at]), dsv = pr * (e - delta[at]);
                for (int u = 0; u < 2; ++u) {
                    ov[u] += pr * y[u];
                    ok[u] += dsv * x[u];
                }
            }
        }
    }
    for (int u = 0; u < 2; ++u)
        if (lane + 64 * u < s.dim) {
            dk.at(b, j, g)[lane + 64 * u] = T::down(ok[u] * s.scale);
            dv.at(b, j, g)[lane + 64 * u] = T::down(ov[u]);
        }
}

// dtable from the rows' sums, in a fixed order.
template <class T>
__global__ __launch_bounds__(256) void k_grad_table(int64_t rows, int32_t heads, int32_t nb,
                                                    const float *__restrict__ sums, uint16_t *__restrict__ dtable) {
    __shared__ float part[256];
    const int h = blockIdx.x % heads, n = blockIdx.x / heads;
    float t = 0.0f;
    for (int64_t r = threadIdx.x; r < rows; r += 256) t += sums[(r * heads + h) * nb + n];
    part[threadIdx.x] = t;
    __syncthreads();
    for (int d = 128; d; d >>= 1) {
        if ((int)threadIdx.x < d) part[threadIdx.x] += part[threadIdx.x + d];
        __syncthreads();
    }
    if (threadIdx.x == 0) dtable[(int64_t)n * heads + h] = T::down(part[0]);
}

}  // namespace dev
}  // namespace ias
