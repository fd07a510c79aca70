// attention_fwd.hpp — block-sparse attention, forward (k_attend, k_attend_join).
//
// A workgroup takes up to 16 * MT rows of one key head: its query heads for a few
// consecutive queries (row r is query r / span, head r % span), or some of the heads
// of one query where there are more of them than rows.  It walks the union of the blocks that these queries chose, each block once:
// neighbouring queries choose mostly the same blocks, and where they do not the
// walk reads no more than the queries would one by one.  A row that did not
// choose a block masks it.  The four waves share nothing while they walk: wave w
// takes every fourth piece of 32 keys and keeps its own running maximum, sum and
// output (softmax in one pass), and the four meet once at the end.
//
// Per piece: S^T = K Q^T with K straight from memory into the matrix
// instruction's registers (a lane holds 8 consecutive channels of one key) and
// Q^T resident.  In S^T's result a lane holds one row and 2 x 4 keys, which is
// just what the right operand of O^T += V^T P^T asks for, so P never leaves the
// registers; it is rounded to the inputs' type for that product (off by half a
// step relative to each probability, as the values are), everything else is
// fp32.  V^T's fragments need the keys of one channel side by side: V goes
// through a wave's own LDS tile and comes back by transposed reads.  The tile's
// 32-byte columns are permuted by row, so that the 8 rows which half a wave
// reads lie in 8 different groups of banks.
#pragma once

#include "attention_kernels.hpp"

namespace ias {
namespace dev {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

template <class T> struct Mma;
template <> struct Mma<Bf16> {
    static __device__ f32x4 run(s16x8 a, s16x8 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
    static __device__ s16x8 pack(const float *x) {
        bf16x8 y;
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = (__bf16)x[e];
        return __builtin_bit_cast(s16x8, y);
    }
};
template <> struct Mma<Fp16> {
    static __device__ f32x4 run(s16x8 a, s16x8 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
    static __device__ s16x8 pack(const float *x) {
        f16x8 y;
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = (_Float16)x[e];
        return __builtin_bit_cast(s16x8, y);
    }
};

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

__device__ inline s16x8 load8(const uint16_t *p) { return *reinterpret_cast<const s16x8 *>(p); }

// A tile of DP channels (16 bits) by rows in LDS, 32-byte columns permuted by row.
template <int DP> struct Tile {
    static constexpr int ROW = DP * 2;   // bytes
    static __device__ int column(int row, int c) { return DP == 128 ? c ^ (row & 7) : c ^ ((row >> 1) & 3); }
    // 16-byte chunk `c` of a row
    static __device__ char *chunk(char *t, int row, int c) { return t + row * ROW + column(row, c >> 1) * 32 + (c & 1) * 16; }
    // Fragment of the transposed tile: channel 16 * col + (lane & 15), keys
    // row0 + 4 * (lane >> 4) + 0..3 and 16 more.
    static __device__ s16x8 transposed(char *t, int row0, int col, int lane) {
        typedef __attribute__((address_space(3))) s16x4 lds4;
        const int r = row0 + 4 * (lane >> 4) + ((lane & 15) >> 2);
        char *a = t + r * ROW + column(r, col) * 32 + (lane & 3) * 8;
        const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4 *)a);
        const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4 *)(a + 16 * ROW));   // 16 rows on, the same columns
        return __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
    }
};

// Which part of the call a workgroup has.  Consecutive ids go to the 8 dies in
// turn; each die gets a contiguous stretch of the work, so that the tiles of one
// key head, which read the same K and V, meet in one L2.
__device__ inline int64_t work_of(int64_t total) {
    const int64_t per = (total + 7) / 8;
    return (int64_t)(blockIdx.x % 8) * per + blockIdx.x / 8;
}

// The union of the blocks that the queries [i0, i0 + nq) chose and can read:
// ids ascending, for each the queries (bits) that chose it.  All threads call it.
// words: LDS, (nblocks + 31) / 32 bits, then that many counts.
__device__ inline int block_union(const AttnShape &s, const int32_t *__restrict__ blocks, int b, int g, int64_t i0, int nq,
                                  int ql, int kl, uint32_t *words, int32_t *ids, uint32_t *masks, int32_t *total) {
    const int nw = (s.nblocks + 31) / 32, tid = threadIdx.x;
    uint32_t *before = words + nw;
    for (int n = tid; n < nw; n += blockDim.x) words[n] = 0;
    __syncthreads();
    const int64_t row0 = ((int64_t)b * s.k_heads + g) * s.q_len + i0;
    const int n = nq * s.keep;
    for (int e = tid; e < n; e += blockDim.x) {
        const int qi = e / s.keep, c = blocks[row0 * s.keep + e];
        const int end = s.causal ? min(kl, (int)(i0 + qi) + kl - ql + 1) : kl;
        if (c >= 0 && c < s.nblocks && (int64_t)c * s.block < end) atomicOr(&words[c >> 5], 1u << (c & 31));
    }
    __syncthreads();
    if (tid < 64) {
        int at = 0;
        for (int w0 = 0; w0 < nw; w0 += 64) {
            const int mine = w0 + tid < nw ? __popc(words[w0 + tid]) : 0;
            int sum = mine;
            for (int d = 1; d < 64; d <<= 1) {
                const int t = __shfl_up(sum, d);
                if (tid >= d) sum += t;
            }
            if (w0 + tid < nw) before[w0 + tid] = at + sum - mine;
            at += __shfl(sum, 63);
        }
        if (tid == 0) *total = at;
    }
    __syncthreads();
    const int found = *total;
    for (int k = tid; k < found; k += blockDim.x) masks[k] = 0;
    __syncthreads();
    for (int e = tid; e < n; e += blockDim.x) {
        const int qi = e / s.keep, c = blocks[row0 * s.keep + e];
        const int end = s.causal ? min(kl, (int)(i0 + qi) + kl - ql + 1) : kl;
        if (c >= 0 && c < s.nblocks && (int64_t)c * s.block < end) {
            const int k = before[c >> 5] + __popc(words[c >> 5] & ((1u << (c & 31)) - 1));
            ids[k] = c;
            atomicOr(&masks[k], 1u << qi);
        }
    }
    __syncthreads();
    return found;
}

struct RowPlan {
    int32_t nq, span, parts;   // queries and heads of a workgroup, workgroups of one query's heads
    int32_t tiles;     // per batch element and key head
    int32_t splits;    // workgroups that share a tile's walk
    int32_t most;      // bound on the blocks of a union
    float *part;       // splits > 1: [tile][split][16 MT rows][DP] sums
    float *stat;       //             [tile][split][16 MT rows][2] maximum and sum
};

// LDS of k_attend: the end's sums (the waves' V tiles lie in the same place),
// the lists, the rows' figures, the bias table.
template <int DP, int MT> constexpr int attend_out_bytes() { return 4 * 16 * MT * (DP + 4) * 4; }
inline size_t attend_lds(int dp, int mt, int nblocks, int most, int table) {
    const size_t v = 4 * 32 * (size_t)dp * 2, o = 4 * 16 * (size_t)mt * (dp + 4) * 4;
    return (v > o ? v : o) + 8 * (size_t)((nblocks + 31) / 32) + 8 * (size_t)most + 4 * 16 * (size_t)mt * 2 * 4 + 16 + 4 * (size_t)table;
}

template <class T, int DP, int MT, bool BIAS>
__global__ __launch_bounds__(256, 2) void k_attend(AttnShape s, RowPlan plan, Side q, Side k, Side v,
                                                const int32_t *__restrict__ blocks, SideOut out, float *__restrict__ lse) {
    constexpr int R = 16 * MT, KS = DP / 32, DT = DP / 16, VL = 32 * DP * 2 / 1024, CH = DP / 8;
    constexpr int AREA = attend_out_bytes<DP, MT>() > 4 * 32 * DP * 2 ? attend_out_bytes<DP, MT>() : 4 * 32 * DP * 2;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    float *sums = reinterpret_cast<float *>(lds);                       // [4][R][DP + 4]
    float *stat = reinterpret_cast<float *>(lds + AREA);                // [4][R][2]
    int32_t *scratch = reinterpret_cast<int32_t *>(stat + 4 * R * 2);   // total, flag
    int32_t *ids = scratch + 4;
    uint32_t *masks = reinterpret_cast<uint32_t *>(ids + plan.most);
    uint32_t *words = masks + plan.most;
    float *table = reinterpret_cast<float *>(words + 2 * ((s.nblocks + 31) / 32));

    int64_t w = work_of((int64_t)s.batch * s.k_heads * plan.tiles * plan.splits);
    if (w >= (int64_t)s.batch * s.k_heads * plan.tiles * plan.splits) return;
    const int split = (int)(w % plan.splits);
    w /= plan.splits;
    const int64_t tile_id = w;
    const int64_t i0 = (w % plan.tiles) / plan.parts * plan.nq;
    const int h0 = (int)(w % plan.tiles % plan.parts) * plan.span;   // of the key head's query heads
    w /= plan.tiles;
    const int g = (int)(w % s.k_heads), b = (int)(w / s.k_heads);
    const int ql = s.ql(b), kl = s.kl(b);
    if (i0 >= ql) return;
    const int nq = min(plan.nq, ql - (int)i0), rows = (nq - 1) * plan.span + min(plan.span, s.group - h0);
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / 64), lane = tid % 64, col = lane & 15, quad = lane >> 4;
    char *tile = lds + wave * 32 * DP * 2;

    if (BIAS)
        for (int e = tid; e < s.num_buckets * s.group; e += 256)
            table[e] = T::up(s.table[(e / s.group) * s.q_heads + g * s.group + e % s.group]);
    const int found = __builtin_amdgcn_readfirstlane(block_union(s, blocks, b, g, i0, nq, ql, kl, words, ids, masks, scratch));

    // this lane's rows
    s16x8 qf[MT][KS];
    int qi[MT], end[MT], pos[MT], hr[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        const int r = m * 16 + col;
        const bool there = r < rows;
        qi[m] = there ? r / plan.span : 0;
        hr[m] = h0 + (there ? r % plan.span : 0);
        pos[m] = (int)i0 + qi[m] + kl - ql;
        end[m] = !there ? 0 : s.causal ? min(kl, pos[m] + 1) : kl;
        const uint16_t *row = q.at(b, i0 + qi[m], (int64_t)g * s.group + hr[m]);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const int d = 32 * ks + 8 * quad;
            qf[m][ks] = there && d < s.dim ? load8(row + d) : s16x8{};
        }
    }
    const int per_block = s.block / 32;
    const int share = (found + plan.splits - 1) / plan.splits;
    const int u0 = min(found, split * share) * per_block, u1 = min(found, (split + 1) * share) * per_block;
    const float c = BIAS ? s.scale : s.scale * LOG2E;

    // turn 0: all queries together.  Zeros of P times infinities of V make NaN
    // in rows that do not read them: if anything in the result is not finite, each
    // query is done again by itself with the values that it does not read cleared.
    for (int turn = 0; turn <= nq; ++turn) {
        const uint32_t only = turn == 0 ? ~0u : 1u << (turn - 1);
        const int vend = turn == 0 || !s.causal ? kl : min(kl, (int)i0 + turn - 1 + kl - ql + 1);
        f32x4 o[MT][DT];
        float top[MT], sum[MT];
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            top[m] = -INFINITY;
            sum[m] = 0.0f;
#pragma unroll
            for (int t = 0; t < DT; ++t) o[m][t] = f32x4{};
        }
        s16x8 kf[2][KS], vf[VL];
        auto at = [&](int u) { return __builtin_amdgcn_readfirstlane(ids[u / per_block]) * s.block + (u % per_block) * 32; };
        auto chose = [&](int u) { return (uint32_t)__builtin_amdgcn_readfirstlane(masks[u / per_block]) & only; };
        auto next = [&](int u) {   // the next piece of this wave that anyone here reads
            while (u < u1 && !chose(u)) u += 4;
            return u;
        };
        auto fetch_k = [&](int u) {
            const int j0 = at(u);
#pragma unroll
            for (int sub = 0; sub < 2; ++sub) {
                const uint16_t *row = k.at(b, min(j0 + 16 * sub + col, kl - 1), g);
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    const int d = 32 * ks + 8 * quad;
                    kf[sub][ks] = d < s.dim ? load8(row + d) : s16x8{};
                }
            }
        };
        auto fetch_v = [&](int u) {
            const int j0 = at(u);
            const int ch = lane % CH;
#pragma unroll
            for (int n = 0; n < VL; ++n) {
                const int j = j0 + n * (64 / CH) + lane / CH;
                vf[n] = j < vend && ch * 8 < s.dim ? load8(v.at(b, j, g) + ch * 8) : s16x8{};
            }
        };
        int u = next(u0 + wave);
        if (u < u1) {
            fetch_k(u);
            fetch_v(u);
        }
        while (u < u1) {
            const int j0 = at(u);
            const uint32_t mask = chose(u);
#pragma unroll
            for (int n = 0; n < VL; ++n)
                *reinterpret_cast<s16x8 *>(Tile<DP>::chunk(tile, n * (64 / CH) + lane / CH, lane % CH)) = vf[n];
            f32x4 x[MT][2];
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int sub = 0; sub < 2; ++sub) {
                    f32x4 acc{};
#pragma unroll
                    for (int ks = 0; ks < KS; ++ks) acc = Mma<T>::run(kf[sub][ks], qf[m][ks], acc);
                    x[m][sub] = acc;
                }
            const int un = next(u + 4);
            if (un < u1) {
                fetch_k(un);
                fetch_v(un);
            }
            s16x8 pf[MT];
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                const int lim = (mask >> qi[m] & 1u) ? end[m] - j0 - 4 * quad : INT32_MIN;
                float y[8], big = -INFINITY;
#pragma unroll
                for (int sub = 0; sub < 2; ++sub) {
                    uint32_t bucket = 0;
                    if (BIAS) __builtin_memcpy(&bucket, s.map + ((int64_t)j0 + 16 * sub + 4 * quad - pos[m] + s.k_len - 1), 4);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float t = x[m][sub][e] * c;
                        if (BIAS) t += table[(bucket >> (8 * e) & 255) * s.group + hr[m]];
                        t = 16 * sub + e < lim ? t : -INFINITY;
                        y[4 * sub + e] = t;
                        big = fmaxf(big, t);
                    }
                }
                big = fmaxf(big, __shfl_xor(big, 16));
                big = fmaxf(big, __shfl_xor(big, 32));
                const float was = top[m], now = fmaxf(was, big), base = now == -INFINITY ? 0.0f : now;
                if (__any(now > was)) {
                    const float f = BIAS ? __builtin_amdgcn_exp2f((was - base) * LOG2E) : __builtin_amdgcn_exp2f(was - base);
                    sum[m] *= f;
#pragma unroll
                    for (int t = 0; t < DT; ++t) o[m][t] *= f;
                    top[m] = now;
                }
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    y[e] = BIAS ? __builtin_amdgcn_exp2f((y[e] - base) * LOG2E) : __builtin_amdgcn_exp2f(y[e] - base);
                    sum[m] += y[e];
                }
                pf[m] = Mma<T>::pack(y);
            }
#pragma unroll
            for (int t = 0; t < DT; ++t) {
                const s16x8 vt = Tile<DP>::transposed(tile, 0, t, lane);
#pragma unroll
                for (int m = 0; m < MT; ++m) o[m][t] = Mma<T>::run(vt, pf[m], o[m][t]);
            }
            u = un;
        }
        // the waves meet
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            sum[m] += __shfl_xor(sum[m], 16);
            sum[m] += __shfl_xor(sum[m], 32);
            if (quad == 0) {
                stat[(wave * R + m * 16 + col) * 2] = top[m];
                stat[(wave * R + m * 16 + col) * 2 + 1] = sum[m];
            }
        }
        if (tid == 0) scratch[1] = 0;
        __syncthreads();
        const float unit = BIAS ? LOG2E : 1.0f;
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            float all = -INFINITY;
            for (int n = 0; n < 4; ++n) all = fmaxf(all, stat[(n * R + m * 16 + col) * 2]);
            const float f = top[m] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((top[m] - all) * unit);
#pragma unroll
            for (int t = 0; t < DT; ++t) {
                float *to = sums + (wave * R + m * 16 + col) * (DP + 4) + 16 * t + 4 * quad;
                // a wave that read nothing for a row adds nothing
                *reinterpret_cast<f32x4 *>(to) = top[m] == -INFINITY && !(sum[m] != sum[m]) ? f32x4{} : o[m][t] * f;
            }
        }
        __syncthreads();
        bool fine = true;
        for (int e = tid; e < R * CH; e += 256) {
            const int r = e / CH, ch = e % CH;
            if (r >= rows || ch * 8 >= s.dim) continue;
            const int rq = r / plan.span;
            if (!(only >> rq & 1u)) continue;
            float all = -INFINITY, l = 0.0f, y[8] = {};
            for (int n = 0; n < 4; ++n) all = fmaxf(all, stat[(n * R + r) * 2]);
            for (int n = 0; n < 4; ++n) {
                const float m = stat[(n * R + r) * 2], x = stat[(n * R + r) * 2 + 1];
                if (m != -INFINITY || x != x) l += x * __builtin_amdgcn_exp2f((m - all) * unit);
#pragma unroll
                for (int d = 0; d < 8; ++d) y[d] += sums[(n * R + r) * (DP + 4) + ch * 8 + d];
            }
            if (plan.splits > 1) {
                const int64_t at = (tile_id * plan.splits + split) * R + r;
#pragma unroll
                for (int d = 0; d < 8; ++d) plan.part[at * DP + ch * 8 + d] = y[d];
                if (ch == 0) {
                    plan.stat[at * 2] = all;
                    plan.stat[at * 2 + 1] = l;
                }
            } else {
                const float inv = l == 0.0f ? 0.0f : 1.0f / l;
                float z[8];
#pragma unroll
                for (int d = 0; d < 8; ++d) z[d] = y[d] * inv;
                const int64_t h = (int64_t)g * s.group + h0 + r % plan.span;
                *reinterpret_cast<s16x8 *>(out.at(b, i0 + rq, h) + ch * 8) = Mma<T>::pack(z);
                if (lse && ch == 0)
                    lse[((int64_t)b * s.q_heads + h) * s.q_len + i0 + rq] =
                        l == 0.0f ? -INFINITY : (BIAS ? all : all * LN2) + __builtin_amdgcn_logf(l) * LN2;
            }
#pragma unroll
            for (int d = 0; d < 8; ++d) fine = fine && fabsf(y[d]) < INFINITY;
        }
        if (turn == 0) {
            if (!fine) scratch[1] = 1;
            __syncthreads();
            const bool again = scratch[1] != 0;
            if (!again) break;
        }
        __syncthreads();
    }
}

// Joins the splits of a tile: one wave for each row.
template <class T>
__global__ __launch_bounds__(64) void k_attend_join(AttnShape s, RowPlan plan, int32_t dp, int32_t tile_rows, float unit,
                                                    SideOut out, float *__restrict__ lse) {
    int64_t w = blockIdx.x;
    const int r = (int)(w % (plan.nq * plan.span));
    w /= plan.nq * plan.span;
    const int64_t tile_id = w, i = (w % plan.tiles) / plan.parts * plan.nq + r / plan.span;
    const int hh = (int)(w % plan.tiles % plan.parts) * plan.span + r % plan.span;
    w /= plan.tiles;
    const int g = (int)(w % s.k_heads), b = (int)(w / s.k_heads), lane = threadIdx.x;
    if (i >= s.ql(b) || hh >= s.group) return;
    float all = -INFINITY, l = 0.0f, y[2] = {};
    for (int n = 0; n < plan.splits; ++n) all = fmaxf(all, plan.stat[((tile_id * plan.splits + n) * tile_rows + r) * 2]);
    for (int n = 0; n < plan.splits; ++n) {
        const int64_t at = (tile_id * plan.splits + n) * tile_rows + r;
        const float m = plan.stat[at * 2], x = plan.stat[at * 2 + 1];
        if (m == -INFINITY && !(x != x)) continue;
        const float f = __builtin_amdgcn_exp2f((m - all) * unit);
        l += x * f;
        for (int u = 0; u < 2; ++u)
            if (2 * lane + u < s.dim) y[u] += plan.part[at * dp + 2 * lane + u] * f;
    }
    const int64_t h = (int64_t)g * s.group + hh;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    if (2 * lane < s.dim) {
        uint16_t *to = out.at(b, i, h) + 2 * lane;
        *reinterpret_cast<uint32_t *>(to) = (uint32_t)T::down(y[0] * inv) | (uint32_t)T::down(y[1] * inv) << 16;
    }
    if (lse && lane == 0)
        lse[((int64_t)b * s.q_heads + h) * s.q_len + i] = l == 0.0f ? -INFINITY : (all * unit + __builtin_amdgcn_logf(l)) * LN2;
}

}  // namespace dev
}  // namespace ias
