// attention_select.hpp — which blocks each query reads (k_block_select).
//
// The order of the scores q . mean has to be that of 64-bit sums, but only near
// the last place does that matter.  So the scores come from the matrix
// instructions first, in fp32, with a bound of their error, and only candidates
// within twice the bound of the last chosen place are computed again in 64 bits
// (a few queries in a hundred have one, where the scores are spread at all).
//
// A workgroup takes up to 16 * MT rows (row r is query r / group, head r % group)
// against all blocks: each wave has every n-th tile of 16 blocks; the maximum over
// a query's heads is taken in LDS on the scores as ordered integers.  Then each
// wave picks the blocks of one query at a time.
//
// Error of the fp32 score: at most 128 sums, each off by 2^-23 of the sum of
// |q_d m_d| if it truncates, so 2^-16 |q| |m|.  Where the norms' squares are not
// comfortably inside fp32 (infinities, NaN, zeros), every candidate is computed in
// 64 bits.
#pragma once

#include "attention_fwd.hpp"

namespace ias {
namespace dev {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

template <class T> __device__ float square_sum(s16x8 x, float t);
template <> __device__ inline float square_sum<Bf16>(s16x8 x, float t) {
    const bf16x8 y = __builtin_bit_cast(bf16x8, x);
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
        const bf16x2 z = {y[e], y[e + 1]};
        t = __builtin_amdgcn_fdot2_f32_bf16(z, z, t, false);
    }
    return t;
}
template <> __device__ inline float square_sum<Fp16>(s16x8 x, float t) {
    const f16x8 y = __builtin_bit_cast(f16x8, x);
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
        const f16x2 z = {y[e], y[e + 1]};
        t = __builtin_amdgcn_fdot2(z, z, t, false);
    }
    return t;
}

// Ordered integers: a < b as numbers = key(a) < key(b); NaN and -inf lowest, 0 below all.
__device__ inline uint32_t order_key(float x) {
    const uint32_t u = __float_as_uint(x == x ? x + 0.0f : -INFINITY);
    return (u >> 31) ? ~u : u | 0x80000000u;
}
__device__ inline float of_key(uint32_t k) { return __uint_as_float((k >> 31) ? k & 0x7fffffffu : ~k); }
__device__ inline unsigned long long order_key(double x) {
    const unsigned long long u = (unsigned long long)__double_as_longlong(x + 0.0);   // -0 ranks as +0
    return (u >> 63) ? ~u : u | (1ull << 63);
}

struct SelectPlan {
    int32_t nq, tiles, first, local, stride;   // queries of a workgroup, workgroups of a key head, words of a query's keys
};
inline size_t select_lds(int nq, int stride, int waves) { return 4 * ((size_t)nq * stride + nq + 1 + 2 * (size_t)waves * ((stride + 31) / 32)); }

// The largest 64-bit score of the query's heads with block c, for 4 blocks at a
// time: 16 lanes each, 8 channels a lane.  Every lane of a group returns it.
template <class T>
__device__ double exact_score(const AttnShape &s, const Side &q, const uint16_t *__restrict__ mean, int b, int i, int g, int c, int lane) {
    const int d = 8 * (lane & 15);
    const bool on = d < s.dim;
    const s16x8 m = on ? load8(mean + (int64_t)c * s.dim + d) : s16x8{};
    double best = -INFINITY;
    for (int h0 = 0; h0 < s.group; h0 += 4) {
        s16x8 x[4];
#pragma unroll
        for (int n = 0; n < 4; ++n)
            x[n] = on ? load8(q.at(b, i, (int64_t)g * s.group + min(h0 + n, s.group - 1)) + d) : s16x8{};
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            double t = 0.0;
#pragma unroll
            for (int e = 0; e < 8; ++e) t += (double)T::up((uint16_t)x[n][e]) * (double)T::up((uint16_t)m[e]);
            for (int k = 8; k; k >>= 1) t += __shfl_xor(t, k);
            if (t > best) best = t;
        }
    }
    return best;
}

template <class T, int DP, int MT>
__global__ __launch_bounds__(MT == 1 ? 1024 : 256) void k_block_select(AttnShape s, SelectPlan plan, Side q, const uint16_t *__restrict__ summary,
                                                       int32_t *__restrict__ blocks) {
    constexpr int KS = DP / 32;
    extern __shared__ uint32_t keys[];                       // [nq][stride], then the norms, then each wave's bits
    uint32_t *qnorm = keys + plan.nq * plan.stride, *mnorm = qnorm + plan.nq;
    int64_t w = work_of((int64_t)s.batch * s.k_heads * plan.tiles);
    if (w >= (int64_t)s.batch * s.k_heads * plan.tiles) return;
    const int i0 = (int)(w % plan.tiles) * plan.nq;
    w /= plan.tiles;
    const int g = (int)(w % s.k_heads), b = (int)(w / s.k_heads);
    const int ql = s.ql(b), kl = s.kl(b);
    if (i0 >= ql) return;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / 64), waves = blockDim.x / 64;
    const int lane = tid % 64, col = lane & 15, quad = lane >> 4;
    const int nq = min(plan.nq, ql - i0), rows = nq * s.group;
    const int p0 = i0 + kl - ql, pl = p0 + nq - 1;
    auto blocks_seen = [&](int p) { return s.causal ? (p < 0 ? 0 : p / s.block + 1) : (kl + s.block - 1) / s.block; };
    const int all = blocks_seen(pl);
    const uint16_t *mean = summary + ((int64_t)b * s.k_heads + g) * s.nblocks * s.dim;

    if (all > s.keep) {   // else every query reads all that it may
        for (int e = tid; e < plan.nq * plan.stride + plan.nq + 1; e += blockDim.x) keys[e] = 0;
        s16x8 qf[MT][KS];
        int qrow[MT][4];
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            const int r = m * 16 + col;
            const uint16_t *row = q.at(b, i0 + (r < rows ? r / s.group : 0), (int64_t)g * s.group + (r < rows ? r % s.group : 0));
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                const int d = 32 * ks + 8 * quad;
                qf[m][ks] = r < rows && d < s.dim ? load8(row + d) : s16x8{};
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int rr = m * 16 + 4 * quad + e;
                qrow[m][e] = rr < rows ? rr / s.group : -1;
            }
        }
        __syncthreads();
        if (wave == 0) {
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                float t = 0.0f;
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) t = square_sum<T>(qf[m][ks], t);
                t += __shfl_xor(t, 16);
                t += __shfl_xor(t, 32);
                const int r = m * 16 + col;
                if (r < rows && quad == 0) atomicMax(&qnorm[r / s.group], __float_as_uint(t) & 0x7fffffffu);
            }
        }
        uint32_t largest = 0;
        const bool fours = s.group % 4 == 0;
        s16x8 mf[KS];
        auto fetch = [&](int c0) {
            const int c = c0 + col;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                const int d = 32 * ks + 8 * quad;
                mf[ks] = c < all && d < s.dim ? load8(mean + (int64_t)c * s.dim + d) : s16x8{};
            }
        };
        if (wave * 16 < all) fetch(wave * 16);
        for (int c0 = wave * 16; c0 < all; c0 += waves * 16) {
            const int c = c0 + col;
            float t = 0.0f;
            f32x4 x[MT];
#pragma unroll
            for (int m = 0; m < MT; ++m) x[m] = f32x4{};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                t = square_sum<T>(mf[ks], t);
#pragma unroll
                for (int m = 0; m < MT; ++m) x[m] = Mma<T>::run(qf[m][ks], mf[ks], x[m]);
            }
            if (c0 + waves * 16 < all) fetch(c0 + waves * 16);
            t += __shfl_xor(t, 16);
            t += __shfl_xor(t, 32);
            largest = max(largest, __float_as_uint(t) & 0x7fffffffu);
            if (c < all) {
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    uint32_t k[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) k[e] = order_key(x[m][e]);
                    if (fours) {   // four rows of one query
                        if (qrow[m][0] >= 0) atomicMax(&keys[qrow[m][0] * plan.stride + c], max(max(k[0], k[1]), max(k[2], k[3])));
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (qrow[m][e] >= 0) atomicMax(&keys[qrow[m][e] * plan.stride + c], k[e]);
                    }
                }
            }
        }
        for (int n = 32; n; n >>= 1) largest = max(largest, (uint32_t)__shfl_xor((int)largest, n));
        if (lane == 0) atomicMax(mnorm, largest);
        __syncthreads();
    }

    constexpr int HELD = 8;   // 64-block pieces of the keys in registers; more are read from LDS
    const int words = (plan.stride + 31) / 32;
    uint32_t *taken = mnorm + 1 + wave * 2 * words, *open = taken + words;
    for (int qi = wave; qi < nq; qi += waves) {
        const int i = i0 + qi, seen = blocks_seen(p0 + qi);
        int32_t *row = blocks + ((((int64_t)b * s.k_heads + g) * s.q_len) + i) * s.keep;
        if (seen <= s.keep) {
            for (int t = lane; t < s.keep; t += 64) row[t] = t < seen ? t : -1;
            continue;
        }
        uint32_t *key = keys + qi * plan.stride;
        // first + local <= keep < seen: the two do not meet
        const int lo = plan.first, hi = seen - plan.local, pieces = (seen + 63) / 64;
        int left = s.keep - plan.first - plan.local;
        uint32_t held[HELD];
        auto load = [&]() {
#pragma unroll
            for (int n = 0; n < HELD; ++n) {
                const int c = n * 64 + lane;
                held[n] = c >= lo && c < hi ? key[c] : 0;
            }
        };
        auto count = [&](uint32_t least) {   // candidates with a key of at least that (least > 0)
            int t = 0;
#pragma unroll
            for (int n = 0; n < HELD; ++n)
                if (n < pieces) t += __popcll(__ballot(held[n] >= least));
            for (int n = HELD; n < pieces; ++n) {
                const int c = n * 64 + lane;
                t += __popcll(__ballot(c < hi && c >= lo && key[c] >= least));
            }
            return t;
        };
        // the largest key that at least `left` candidates have
        auto place = [&]() {
            uint32_t high = 0, low = 0xffffffffu;
#pragma unroll
            for (int n = 0; n < HELD; ++n) {
                high = max(high, held[n]);
                if (held[n]) low = min(low, held[n]);
            }
            for (int n = HELD; n < pieces; ++n) {
                const int c = n * 64 + lane;
                const uint32_t k = c >= lo && c < hi ? key[c] : 0;
                high = max(high, k);
                if (k) low = min(low, k);
            }
            for (int d = 32; d; d >>= 1) {
                high = max(high, (uint32_t)__shfl_xor((int)high, d));
                low = min(low, (uint32_t)__shfl_xor((int)low, d));
            }
            high = __builtin_amdgcn_readfirstlane(high);
            low = __builtin_amdgcn_readfirstlane(low);
            if (high == low) return high;
            // all keys agree above this bit
            const int top = 31 - __clz(high ^ low);
            uint32_t at = high >> top >> 1 << top << 1;
            for (int bit = top; bit >= 0; --bit) {
                const uint32_t up = at | 1u << bit;
                const int n = count(up);
                if (n >= left) at = up;
                if (n == left) {   // these and no others: their smallest key
                    uint32_t least = 0xffffffffu;
#pragma unroll
                    for (int m = 0; m < HELD; ++m)
                        if (held[m] >= up) least = min(least, held[m]);
                    for (int m = HELD; m < pieces; ++m) {
                        const int c = m * 64 + lane;
                        if (c >= lo && c < hi && key[c] >= up) least = min(least, key[c]);
                    }
                    for (int d = 32; d; d >>= 1) least = min(least, (uint32_t)__shfl_xor((int)least, d));
                    return least;
                }
            }
            return at;
        };
        // marks what is above `over` as taken and what is in [from, over] as open; returns how many are open
        auto split = [&](uint32_t from, uint32_t over, bool start) {
            int opened = 0, sure = 0;
            for (int n = 0; n < pieces; ++n) {
                const int c = n * 64 + lane;
                const uint32_t k = c >= lo && c < hi ? key[c] : 0;
                const unsigned long long up = __ballot(k > over), on = __ballot(k >= from && k <= over && k > 0);
                const unsigned long long forced = __ballot(start && c < seen && (c < lo || c >= hi));
                sure += __popcll(up);
                opened += __popcll(on);
                if (lane < 2) {
                    const uint32_t u = (uint32_t)((up | forced) >> (32 * lane)), o = (uint32_t)(on >> (32 * lane));
                    if (n * 2 + lane < (plan.stride + 31) / 32) {
                        taken[n * 2 + lane] = start ? u : taken[n * 2 + lane] | u;
                        open[n * 2 + lane] = o;
                    }
                }
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            left -= sure;
            return opened;
        };
        int opened;
        if (left > 0) {
            load();
            const float qq = __uint_as_float(qnorm[qi]), mm = __uint_as_float(*mnorm);
            if (qq > 1e-30f && qq < 1e30f && mm > 1e-30f && mm < 1e30f) {
                const float off = 2.0f * 1.6e-5f * sqrtf(qq) * sqrtf(mm), last = of_key(place());
                opened = split(order_key(last - off), order_key(last + off), true);
            } else {
                opened = split(1, 0xffffffffu, true);
            }
        } else {
            opened = split(0xffffffffu, 0xffffffffu, true);
            opened = 0;
        }
        // the open ones by their 64-bit scores.  Up to 64, as nearly always: candidate n's
        // score to lane n, and its place is the number of those before it.
        if (opened > left && left > 0 && opened <= 64) {
            unsigned long long mine = 0;
            int where = 0, n = 0;
            for (int p = 0; p < pieces; ++p) {
                unsigned long long on = (unsigned long long)(2 * p + 1 < words ? open[2 * p + 1] : 0) << 32 | open[2 * p];
                while (on) {
                    int c[4];
                    const int n0 = n;
#pragma unroll
                    for (int d = 0; d < 4; ++d) {
                        c[d] = on ? p * 64 + __ffsll(on) - 1 : -1;
                        n += on != 0;
                        on &= on - 1;
                    }
                    const int group = lane / 16, own = group == 0 ? c[0] : group == 1 ? c[1] : group == 2 ? c[2] : c[3];
                    const unsigned long long k = order_key(exact_score<T>(s, q, mean, b, i, g, max(own, 0), lane));
#pragma unroll
                    for (int d = 0; d < 4; ++d) {
                        const unsigned long long kd = __shfl(k, 16 * d);
                        if (lane == n0 + d && c[d] >= 0) {
                            mine = kd;
                            where = c[d];
                        }
                    }
                }
            }
            int before = 0;
            for (int d = 0; d < opened; ++d) {
                const unsigned long long k = __shfl(mine, d);
                before += k > mine || (k == mine && d < lane);
            }
            if (lane < opened && before < left) atomicOr(&taken[where >> 5], 1u << (where & 31));
            left = 0;
        }
        // more: high half, then the low one's halves
        for (int level = 0; level < 3 && opened > left && left > 0; ++level) {
            for (int n = 0; n < pieces; ++n) {
                const uint32_t low = open[2 * n], high = 2 * n + 1 < (plan.stride + 31) / 32 ? open[2 * n + 1] : 0;
                unsigned long long on = (unsigned long long)high << 32 | low;
                if (n * 64 + lane >= lo && n * 64 + lane < hi && !(on >> lane & 1)) key[n * 64 + lane] = 0;
                while (on) {
                    int mine = -1;
                    for (int d = 0; d < 4 && on; ++d, on &= on - 1)
                        if (lane / 16 == d) mine = __ffsll(on) - 1;
                    const double x = exact_score<T>(s, q, mean, b, i, g, n * 64 + max(mine, 0), lane);
                    const unsigned long long k = order_key(x);
                    const uint32_t part = level == 0 ? (uint32_t)(k >> 32) : level == 1 ? (uint32_t)(k >> 16 & 0xffff) + 1 : (uint32_t)(k & 0xffff) + 1;
                    if (mine >= 0 && col == 0) key[n * 64 + mine] = part;
                }
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            load();
            const uint32_t last = place();
            opened = split(last, last, false);
        }
        // taken, and of the open ones the first
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        int n = 0;
        for (int m = 0; m < pieces; ++m) {
            const int c = m * 64 + lane;
            const bool in = c < seen && (taken[c / 32] >> (c & 31) & 1), may = left > 0 && c < seen && (open[c / 32] >> (c & 31) & 1);
            const unsigned long long maybe = __ballot(may);
            const bool on = in || (may && __popcll(maybe & ((1ull << lane) - 1)) < left);
            left -= min(left, __popcll(maybe));
            const unsigned long long got = __ballot(on);
            if (on) row[n + __popcll(got & ((1ull << lane) - 1))] = c;
            n += __popcll(got);
        }
        for (int t = n + lane; t < s.keep; t += 64) row[t] = -1;
    }
}

}  // namespace dev
}  // namespace ias
