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
//
// Bound by the picking of each query, a wave's chain of some 20 counts by ballots with
// half of the time waiting, not by the scores' products (4096 tokens, 32/8 heads of 128,
// 16 of 64 blocks: 36 us; 16 single tokens, 32 of 512 blocks: 16 us).  Blocks that a
// bisection of keys held in registers decides cost less than sorting or a pass over LDS
// for each bit (72 -> 42 us).
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

// One of 64 lanes' maximum / minimum in all of them.
template <class F> __device__ inline uint32_t wave_reduce(uint32_t x, F f) {
    x = f(x, (uint32_t)__builtin_amdgcn_update_dpp((int)x, (int)x, 0xb1, 0xf, 0xf, false));    // lanes 1 apart
    x = f(x, (uint32_t)__builtin_amdgcn_update_dpp((int)x, (int)x, 0x4e, 0xf, 0xf, false));    // 2
    x = f(x, (uint32_t)__builtin_amdgcn_update_dpp((int)x, (int)x, 0x141, 0xf, 0xf, false));   // mirrored in 8
    x = f(x, (uint32_t)__builtin_amdgcn_update_dpp((int)x, (int)x, 0x140, 0xf, 0xf, false));   // in 16
    const auto a = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    x = f(a[0], a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return __builtin_amdgcn_readfirstlane(f(b[0], b[1]));
}

// What a wave needs to pick one query's blocks.  off: twice the bound of the scores'
// errors, infinite where there is none.  keep < seen here, so the first and the local
// blocks do not meet.
struct Pick {
    const AttnShape &s;
    const SelectPlan &plan;
    const Side &q;
    const uint16_t *mean;
    int b, i, g, seen, lane;
    uint32_t *key;
    float off;
    int32_t *row;
};

// Up to 64 NP blocks: keys in registers, sets of blocks in masks.  False, and nothing
// written, if more than 64 candidates are too close to call (equal blocks, say).
template <class T, int NP> __device__ bool pick_held(const Pick &p) {
    const int lane = p.lane, lo = p.plan.first, hi = p.seen - p.plan.local;
    int left = p.s.keep - p.plan.first - p.plan.local;
    uint32_t held[NP];
    unsigned long long taken[NP], open[NP];
#pragma unroll
    for (int n = 0; n < NP; ++n) {
        const int c = n * 64 + lane;
        const bool free = c >= lo && c < hi;
        held[n] = free ? p.key[c] : 0;
        taken[n] = __ballot(c < p.seen && !free);
        open[n] = 0;
    }
    if (left > 0) {
        auto count = [&](uint32_t least) {
            int t = 0;
#pragma unroll
            for (int n = 0; n < NP; ++n) t += __popcll(__ballot(held[n] >= least));
            return t;
        };
        uint32_t from = 1, over = 0xffffffffu;
        if (p.off < INFINITY) {
            // the key in the last place: bits from the top, below those that all keys share
            uint32_t high = 0, low = 0xffffffffu;
#pragma unroll
            for (int n = 0; n < NP; ++n) {
                high = max(high, held[n]);
                low = min(low, held[n] ? held[n] : 0xffffffffu);
            }
            high = wave_reduce(high, [](uint32_t x, uint32_t y) { return max(x, y); });
            low = wave_reduce(low, [](uint32_t x, uint32_t y) { return min(x, y); });
            uint32_t at = high;
            if (high != low) {
                const int top = 31 - __clz(high ^ low);
                at = high >> top >> 1 << top << 1;
                for (int bit = top; bit >= 0; --bit) {
                    const int n = count(at | 1u << bit);
                    if (n >= left) at |= 1u << bit;
                    if (n == left) {   // these and no others: the smallest of their keys
                        uint32_t least = 0xffffffffu;
#pragma unroll
                        for (int m = 0; m < NP; ++m) least = min(least, held[m] >= at ? held[m] : 0xffffffffu);
                        at = wave_reduce(least, [](uint32_t x, uint32_t y) { return min(x, y); });
                        break;
                    }
                }
            }
            const float last = of_key(at);
            from = order_key(last - p.off);
            over = order_key(last + p.off);
        }
        int opened = 0;
#pragma unroll
        for (int n = 0; n < NP; ++n) {
            const unsigned long long up = __ballot(held[n] > over);
            open[n] = __ballot(held[n] >= from) & ~up;
            taken[n] |= up;
            left -= __popcll(up);
            opened += __popcll(open[n]);
        }
        if (opened > left) {
            if (opened > 64) return false;
            // candidate n's 64-bit score to lane n; its place is the number of those before it
            unsigned long long mine = 0;
            int where = 0, n = 0;
#pragma unroll
            for (int m = 0; m < NP; ++m)
                for (unsigned long long on = open[m]; on;) {
                    int c[4];
                    const int n0 = n;
#pragma unroll
                    for (int d = 0; d < 4; ++d) {
                        c[d] = on ? m * 64 + __ffsll(on) - 1 : -1;
                        n += on != 0;
                        on &= on - 1;
                    }
                    const int group = lane / 16, own = group == 0 ? c[0] : group == 1 ? c[1] : group == 2 ? c[2] : c[3];
                    const unsigned long long k = order_key(exact_score<T>(p.s, p.q, p.mean, p.b, p.i, p.g, max(own, 0), lane));
#pragma unroll
                    for (int d = 0; d < 4; ++d) {
                        const unsigned long long kd = __shfl(k, 16 * d);
                        if (lane == n0 + d && c[d] >= 0) {
                            mine = kd;
                            where = c[d];
                        }
                    }
                }
            int before = 0;
            for (int d = 0; d < opened; ++d) {
                const unsigned long long k = __shfl(mine, d);
                before += k > mine || (k == mine && d < lane);
            }
            for (unsigned long long on = __ballot(lane < opened && before < left); on; on &= on - 1) {
                const int c = __shfl(where, __ffsll(on) - 1);
#pragma unroll
                for (int m = 0; m < NP; ++m)
                    if (c / 64 == m) taken[m] |= 1ull << (c & 63);
            }
        } else {
#pragma unroll
            for (int n = 0; n < NP; ++n) taken[n] |= open[n];
        }
    }
    int n = 0;
#pragma unroll
    for (int m = 0; m < NP; ++m) {
        if (taken[m] >> lane & 1) p.row[n + __popcll(taken[m] & ((1ull << lane) - 1))] = m * 64 + lane;
        n += __popcll(taken[m]);
    }
    for (int t = n + lane; t < p.s.keep; t += 64) p.row[t] = -1;
    return true;
}

// Any number of blocks: keys and sets in LDS (taken, open: a bit for each block).
template <class T> __device__ void pick_any(const Pick &p, uint32_t *taken, uint32_t *open) {
    const AttnShape &s = p.s;
    const SelectPlan &plan = p.plan;
    const Side &q = p.q;
    const uint16_t *mean = p.mean;
    const int b = p.b, i = p.i, g = p.g, seen = p.seen, lane = p.lane, col = lane & 15;
    uint32_t *key = p.key;
    int32_t *row = p.row;
    const float off = p.off;
    const int words = (plan.stride + 31) / 32, pieces = (seen + 63) / 64;
    const int lo = plan.first, hi = seen - plan.local;
    int left = s.keep - plan.first - plan.local;
    auto count = [&](uint32_t least) {   // candidates with a key of at least that (least > 0)
        int t = 0;
        for (int n = 0; n < pieces; ++n) {
            const int c = n * 64 + lane;
            t += __popcll(__ballot(c < hi && c >= lo && key[c] >= least));
        }
        return t;
    };
    // the largest key that at least `left` candidates have
    auto place = [&]() {
        uint32_t at = 0;
        for (int bit = 31; bit >= 0; --bit)
            if (count(at | 1u << bit) >= left) at |= 1u << bit;
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
                if (n * 2 + lane < words) {
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
        if (off < INFINITY) {
            const float last = of_key(place());
            opened = split(order_key(last - off), order_key(last + off), true);
        } else {
            opened = split(1, 0xffffffffu, true);
        }
    } else {
        opened = split(0xffffffffu, 0xffffffffu, true);
        opened = 0;
    }
    // the open ones by their 64-bit scores: high half, then the low one's halves
    for (int level = 0; level < 3 && opened > left && left > 0; ++level) {
        for (int n = 0; n < pieces; ++n) {
            const uint32_t low = open[2 * n], high = 2 * n + 1 < words ? open[2 * n + 1] : 0;
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

template <class T, int DP, int MT>
__global__ __launch_bounds__(MT == 1 ? 1024 : 256) void k_block_select(AttnShape s, SelectPlan plan, Side q, const uint16_t *__restrict__ summary,
                                                       int32_t *__restrict__ blocks) {
    constexpr int KS = DP / 32;
    extern __shared__ uint32_t keys[];                       // [nq][stride], then the norms, then each wave's bits
    uint32_t *qnorm = keys + plan.nq * plan.stride, *mnorm = qnorm + plan.nq;
    const Part part = tile_of(s.batch * s.k_heads, plan.tiles);
    if (part.head < 0) return;
    const int i0 = part.tile * plan.nq, b = (uint32_t)part.head / (uint32_t)s.k_heads, g = part.head - b * s.k_heads;
    const int ql = s.ql(b), kl = s.kl(b);
    if (s.clear && i0 + plan.nq > ql) {   // queries behind the sequence's end
        const int64_t from = max(i0, ql), to = min((int64_t)i0 + plan.nq, s.q_len);
        for (int64_t e = threadIdx.x; e < (to - from) * s.keep; e += blockDim.x)
            blocks[((((int64_t)b * s.k_heads + g) * s.q_len) + from) * s.keep + e] = -1;
    }
    if (i0 >= ql) return;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / 64), waves = blockDim.x / 64;
    const int lane = tid % 64, col = lane & 15, quad = lane >> 4;
    const int nq = min(plan.nq, ql - i0), rows = nq * s.group;
    const int p0 = i0 + kl - ql, pl = p0 + nq - 1;
    auto blocks_seen = [&](int p) { return s.causal ? (p < 0 ? 0 : (int)((uint32_t)p / (uint32_t)s.block) + 1) : (int)((uint32_t)(kl + s.block - 1) / (uint32_t)s.block); };
    const int all = blocks_seen(pl);
    const uint16_t *mean = summary + ((int64_t)b * s.k_heads + g) * s.nblocks * s.dim;

    if (all > s.keep) {   // else every query reads all that it may
        for (int e = tid; e < plan.nq * plan.stride + plan.nq + 1; e += blockDim.x) keys[e] = 0;
        s16x8 qf[MT][KS];
        int qrow[MT][4];
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            const int r = m * 16 + col;
            const uint16_t *row = q.at(b, i0 + (r < rows ? s.per_group(r) : 0), (int64_t)g * s.group + (r < rows ? r - s.per_group(r) * s.group : 0));
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                const int d = 32 * ks + 8 * quad;
                qf[m][ks] = r < rows && d < s.dim ? load8(row + d) : s16x8{};
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int rr = m * 16 + 4 * quad + e;
                qrow[m][e] = rr < rows ? s.per_group(rr) : -1;
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

    const int words = (plan.stride + 31) / 32;
    uint32_t *taken = mnorm + 1 + wave * 2 * words, *open = taken + words;
    for (int qi = wave; qi < nq; qi += waves) {
        const int i = i0 + qi, seen = blocks_seen(p0 + qi);
        int32_t *row = blocks + ((((int64_t)b * s.k_heads + g) * s.q_len) + i) * s.keep;
        if (seen <= s.keep) {
            for (int t = lane; t < s.keep; t += 64) row[t] = t < seen ? t : -1;
            continue;
        }
        const float qq = __uint_as_float(__builtin_amdgcn_readfirstlane(qnorm[qi])), mm = __uint_as_float(__builtin_amdgcn_readfirstlane(*mnorm));
        const bool tame = qq > 1e-30f && qq < 1e30f && mm > 1e-30f && mm < 1e30f;
        const Pick p{s, plan, q, mean, b, i, g, seen, lane, keys + qi * plan.stride, tame ? 2.0f * 1.6e-5f * sqrtf(qq) * sqrtf(mm) : INFINITY, row};
        const bool done = seen <= 64 ? pick_held<T, 1>(p) : seen <= 128 ? pick_held<T, 2>(p) : seen <= 512 ? pick_held<T, 8>(p) : false;
        if (!done) pick_any<T>(p, taken, open);
    }
}

}  // namespace dev
}  // namespace ias
