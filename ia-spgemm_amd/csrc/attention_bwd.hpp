// attention_bwd.hpp — block-sparse attention, backward.
//
// dS = P (dP - delta), with P = exp(x - lse) recomputed and delta = dout . out.
// k_grad_q walks as the forward pass does (rows of a few queries, the union of
// their blocks, one piece of 32 keys per wave): dQ^T += K^T dS^T, and the
// bias's gradient by bucket.  k_grad_kv takes a block of keys and the queries that
// chose it, which the pattern's transpose lists: dV += P^T dO, dK += dS^T Q.
// Nothing is added atomically in floating point, every sum has a fixed order.
//
// P and dS are rounded to the inputs' type for the matrix products, off by half a step of
// each, and delta is taken from `out` as it was rounded; all sums are fp32.  Of a bf16
// gradient of the queries that makes an error of 0.0026 to 0.0032 of its largest entry
// (bound: 0.005) where the formula in separate fp32 operators has 0.0017.  dS in two parts brought
// it to 0.0024, since delta's part stays, and cost 8 to 13 % of a training step.
//
// 8192 tokens, 16/2 heads of 128, 16 blocks a query, 0.83 to 0.85 ms with the forward's 228 us:
// k_grad_q 282 us and k_grad_kv 271 us, both bound by latency at two and three waves a SIMD
// as the forward is (together 7 products where the forward makes 2; matrix units busy in 28
// and 19 % of the cycles, LDS in 44 and 28 %), k_grad_kv_join 49 us, bound
// by its read of partial results (64 KB an item); the pattern's transpose 18 us in three
// launches.
#pragma once

#include "attention_fwd.hpp"

namespace ias {
namespace dev {

// ------------------------------------------------------------------ dq
struct GradPlan {
    int32_t nq, span, parts, tiles, most;   // as RowPlan
    uint32_t inverse;
    float *delta;                           // [batch][q_heads][q_len]
    float *sums;                            // [tile][span][num_buckets], null: no dtable
    float *shift, *corr;                    // as delta, with a bias only: P = exp2((x - shift) log2(e) - corr)
    __device__ int per_span(int r) const { return (int)((uint32_t)r * inverse >> 16); }
};

// LDS of k_grad_q: the waves' K and V tiles and the lanes' sums by bucket, over which
// the end's sums are laid; the lists; the bias table.
inline int grad_q_area(int dp, int rows, int waves, int buckets, bool sums) {
    const int v = waves * 2 * 32 * dp * 2 + (sums ? buckets * 64 * waves * 4 : 0), o = walk_area(dp, rows, waves);
    return v > o ? v : o;
}
inline size_t grad_q_lds(int area, int nblocks, int most, int span, int buckets) {
    return area + 8 * (size_t)((nblocks + 31) / 32) + 8 * (size_t)most + 16 + 4 * (size_t)span * buckets;
}

// fp16 holds 65504 at most and 11 bits only down to 2^-14, and dS goes by the size of dout
// and v: 160000 from values and gradients of 200, 2^-24 from a small loss over many keys.
// So before it is rounded a row (a key, in k_grad_kv) multiplies it by a power of two, which
// its sum loses again at the end.  It starts with 2^80 (dS is below 2^40: 128 products of two
// fp16) and is lowered, with what was summed by then, only where a dS would pass 2^15, so
// that the largest comes to [2^11, 2^12): that is the first piece and hardly ever another.  Of
// the largest that the row has met, everything down to 2^-25 keeps its 11 bits.  bf16 has the
// range of fp32 and needs none of this.
constexpr int FACTOR_START = 80;   // exponents of the factors
constexpr float FACTOR_TOP = 0x1p15f;
__device__ inline float times(float x, int exponent) { return __builtin_amdgcn_ldexpf(x, exponent); }
__device__ inline int factor_for(float big) { return 11 + 127 - (int)(__float_as_uint(big) >> 23); }   // infinite: -117
// k_grad_kv's P is at most 1 (up to roundings) and as small as one over the keys: 2^15 times
// it keeps its 11 bits down to 2^-29.  The exponentials' argument takes the 15.
template <class T> constexpr float LIFT = T::NARROW ? 15.0f : 0.0f;
template <class T> __device__ inline float unscaled(float x, int exponent) { return T::NARROW ? times(x, -exponent) : x; }
template <int N> __device__ inline float largest(const float *y) {
    float big = 0.0f;   // NaN is passed over: it stays NaN whatever the factor
#pragma unroll
    for (int e = 0; e < N; ++e) big = fmaxf(big, fabsf(y[e]));
    return big;
}

// The largest score of a row over its part of the union and log2 of the sum of
// exponentials beside it, by one wave.
struct RowSum {
    float top, log;
};
template <class T>
__device__ RowSum row_sums(const AttnShape &s, const uint16_t *__restrict__ q, const Side &k, int b, int g, int end, int pos, int found,
                           const int32_t *ids, const uint32_t *masks, int query, const float *table, int span, int lane) {
    float top = -INFINITY, sum = 0.0f;
    for (int n = 0; n < found; ++n) {
        if (!(masks[n] >> query & 1u)) continue;
        const int j0 = ids[n] * s.block;
        for (int j = j0 + lane; j < min(end, j0 + s.block); j += 64) {
            const uint16_t *row = k.at(b, j, g);
            float x = 0.0f;
            for (int d = 0; d < s.dim; d += 8) {
                const s16x8 u = load8(q + d), v = load8(row + d);
#pragma unroll
                for (int e = 0; e < 8; ++e) x = __builtin_fmaf(T::up((uint16_t)u[e]), T::up((uint16_t)v[e]), x);
            }
            x = __builtin_fmaf(x, s.scale, table[s.map[(int64_t)j - pos + s.k_len - 1] * span]);
            if (!(x > -INFINITY)) continue;
            if (x > top) {
                sum *= __builtin_amdgcn_exp2f((top - x) * LOG2E);
                top = x;
            }
            sum += __builtin_amdgcn_exp2f((x - top) * LOG2E);
        }
    }
    float all = top;
    for (int d = 32; d; d >>= 1) all = fmaxf(all, __shfl_xor(all, d));
    sum = top == -INFINITY ? 0.0f : sum * __builtin_amdgcn_exp2f((top - all) * LOG2E);
    for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
    return {all, __builtin_amdgcn_logf(sum)};
}

template <class T, int DP, int ROWS, int W, bool BIAS>
__global__ __launch_bounds__(64 * W, 2) void k_grad_q(AttnShape s, GradPlan plan, int32_t area, Side dout, Side q, Side k,
                                                      Side v, Side out, const float *__restrict__ lse,
                                                      const int32_t *__restrict__ blocks, SideOut dq) {
    typedef Form<ROWS> F;
    constexpr int THREADS = 64 * W, CH = DP / 8, N = F::N, VL = Tile<DP>::N;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    float *sums = reinterpret_cast<float *>(lds);                           // [W][ROWS][DP + 4], at the end
    float *hist = reinterpret_cast<float *>(lds + W * 2 * Tile<DP>::BYTES);   // [buckets][64 W]
    int32_t *scratch = reinterpret_cast<int32_t *>(lds + area);             // total, flag
    int32_t *ids = scratch + 4;
    uint32_t *masks = reinterpret_cast<uint32_t *>(ids + plan.most);
    uint32_t *words = masks + plan.most;
    float *table = reinterpret_cast<float *>(words + 2 * ((s.nblocks + 31) / 32));

    const Part part = tile_of(s.batch * s.k_heads, plan.tiles);
    if (part.head < 0) return;
    const uint32_t step = (uint32_t)part.tile / (uint32_t)plan.parts;
    const int64_t tile_id = (int64_t)part.head * plan.tiles + part.tile, i0 = (int64_t)step * plan.nq;
    const int h0 = (int)(part.tile - step * plan.parts) * plan.span;
    const int b = (uint32_t)part.head / (uint32_t)s.k_heads, g = part.head - b * s.k_heads;
    const int ql = s.ql(b), kl = s.kl(b);
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / 64), lane = tid % 64;
    if (s.clear && i0 + plan.nq > ql)
        clear_rows(s, b, g, h0, min(plan.span, s.group - h0), max(i0, (int64_t)ql), min(i0 + plan.nq, s.q_len), dq, nullptr);
    if (i0 >= ql) {
        if (BIAS && plan.sums)
            for (int e = tid; e < plan.span * s.num_buckets; e += THREADS) plan.sums[tile_id * plan.span * s.num_buckets + e] = 0.0f;
        return;
    }
    const int nq = min(plan.nq, ql - (int)i0), rows = (nq - 1) * plan.span + min(plan.span, s.group - h0);
    const Tile<DP, ROWS> tile(lds + wave * 2 * Tile<DP>::BYTES, lane);   // K, then V
    constexpr int KT = 0, VT = Tile<DP>::BYTES;

    if (BIAS) {
        for (int e = tid; e < s.num_buckets * plan.span; e += THREADS)
            if (h0 + e % plan.span < s.group) table[e] = T::up(s.table[(e / plan.span) * s.q_heads + g * s.group + h0 + e % plan.span]);
        if (plan.sums)
            for (int e = tid; e < s.num_buckets * THREADS; e += THREADS) hist[e] = 0.0f;
    }
    const int found = __builtin_amdgcn_readfirstlane(block_union(s, blocks, b, g, i0, nq, ql, kl, words, ids, masks, scratch));

    const Row<DP, ROWS> row(lane, rows, plan.per_span(lane % ROWS), h0, plan.span, (int)i0, kl, ql, s.causal);
    float delta = 0.0f, shift, corr = 0.0f;
    // a row that read nothing has lse = -inf: exp(x - inf) = 0
    if (BIAS) {
        const int64_t at = ((int64_t)b * s.q_heads + (int64_t)g * s.group + row.head) * s.q_len + i0 + row.query;
        const float l = row.there ? lse[at] : -INFINITY;
        shift = l == -INFINITY ? INFINITY : l;
        // Beside a bias of the type's lowest value fp32 holds no log of a sum: at 4096 lse is off
        // by up to 2^-13, far beyond it a row of equals would get P = 1 for each.  Such rows (hardly
        // ever any) find their maximum and sum again.
        for (unsigned long long wild = __ballot(lane < ROWS && fabsf(l) >= 4096.0f && fabsf(l) < INFINITY); wild; wild &= wild - 1) {
            const int r = __ffsll(wild) - 1, rq = plan.per_span(r), hr = r - rq * plan.span, pos = (int)i0 + rq + kl - ql;
            const RowSum got = row_sums<T>(s, q.at(b, i0 + rq, (int64_t)g * s.group + h0 + hr), k, b, g, s.causal ? min(kl, pos + 1) : kl, pos,
                                           found, ids, masks, rq, table + hr, plan.span, lane);
            if (lane % ROWS == r && got.top > -INFINITY) {
                shift = got.top;
                corr = got.log;
            }
        }
        if (wave == 0 && row.part == 0 && row.there) {
            plan.shift[at] = shift;
            plan.corr[at] = corr;
        }
    }
    s16x8 qf[DP / F::K], df[DP / F::K];
    {
        const int64_t h = (int64_t)g * s.group + row.head, at = ((int64_t)b * s.q_heads + h) * s.q_len + i0 + row.query;
        row.load(df, dout.at(b, i0 + row.query, h), s.dim);
        row.load(qf, out.at(b, i0 + row.query, h), s.dim);
#pragma unroll
        for (int ks = 0; ks < DP / F::K; ++ks)
#pragma unroll
            for (int e = 0; e < 8; ++e) delta = __builtin_fmaf(T::up((uint16_t)df[ks][e]), T::up((uint16_t)qf[ks][e]), delta);
        delta = row_sum<F::PARTS>(delta);
        row.load(qf, q.at(b, i0 + row.query, h), s.dim);
        if (s.scale < 0.0f)
#pragma unroll
            for (int ks = 0; ks < DP / F::K; ++ks) qf[ks] = negated(qf[ks]);
        if (!BIAS) {
            const float l = row.there ? lse[at] : -INFINITY;
            shift = l == -INFINITY ? INFINITY : l * LOG2E;
        }
        if (wave == 0 && row.part == 0 && row.there) plan.delta[at] = delta;
    }
    const float c = fabsf(BIAS ? s.scale : s.scale * LOG2E);
    const int per_block = s.block / 32;
    const int sure = s.causal ? min(kl, (int)i0 + kl - ql + 1) : kl;
    const Piece<DP> kp(k, b, g, lane, s.dim, kl), vp(v, b, g, lane, s.dim, kl);

    // turn 0 and the rest as in k_attend: here it is zeros of dS times infinities of K
    for (int turn = 0; turn <= nq; ++turn) {
        const uint32_t only = turn == 0 ? ~0u : 1u << (turn - 1);
        const int vend = turn == 0 || !s.causal ? kl : min(kl, (int)i0 + turn - 1 + kl - ql + 1);
        typename F::Acc o[DP / ROWS];
#pragma unroll
        for (int t = 0; t < DP / ROWS; ++t) o[t] = typename F::Acc{};
        int factor = FACTOR_START;   // of the row's dS and o
        s16x8 kr[VL], vr[VL];
        Walk<W> at(wave, per_block);
        auto skip = [&]() {
            while (turn > 0 && at.step < found && !(masks[at.step] & only)) at.on();
        };
        skip();
        int j0 = 0;
        uint32_t mask = 0;
        if (at.step < found) {
            j0 = __builtin_amdgcn_readfirstlane(ids[at.step]) * s.block + at.part * 32;
            mask = __builtin_amdgcn_readfirstlane(masks[at.step]) & only;
            kp.load(kr, j0, vend);
            vp.load(vr, j0, vend);
        }
        while (at.step < found) {
            at.on();
            skip();
            const bool more = at.step < found;
            const int id = more ? ids[at.step] : 0;
            const uint32_t chose = more ? masks[at.step] : 0;
            tile.fill(kr, KT);
            tile.fill(vr, VT);
            float x[N], y[N];
            __builtin_amdgcn_s_setprio(1);
            scores<T, DP, ROWS, false>(tile, KT, qf, x);
            scores<T, DP, ROWS, false>(tile, VT, df, y);
            __builtin_amdgcn_s_setprio(0);
            const int jn = __builtin_amdgcn_readfirstlane(id) * s.block + at.part * 32;
            const uint32_t maskn = __builtin_amdgcn_readfirstlane(chose) & only;
            if (more) {
                kp.load(kr, jn, vend);
                vp.load(vr, jn, vend);
            }
            const bool sel = mask >> row.query & 1u;
            // exp(x - inf) = 0; a row's factor lies in its exponentials
            const float off = !sel ? INFINITY : T::NARROW && !BIAS ? shift - (float)factor : shift;
            const float less = T::NARROW ? corr - (float)factor : corr;
            uint32_t bucket[N / 4];
#pragma unroll
            for (int n = 0; n < N; n += 4) {
                if (BIAS) __builtin_memcpy(&bucket[n / 4], s.map + ((int64_t)j0 + row.key(n) + 4 * row.part - row.pos + s.k_len - 1), 4);
#pragma unroll
                for (int e = n; e < n + 4; ++e) {
                    float p;
                    if (BIAS)
                        p = __builtin_amdgcn_exp2f(__builtin_fmaf(__builtin_fmaf(x[e], c, table[(bucket[n / 4] >> (8 * (e - n)) & 255) * plan.span + row.head - h0]) - off, LOG2E, -less));
                    else
                        p = __builtin_amdgcn_exp2f(__builtin_fmaf(x[e], c, -off));
                    y[e] = p * (y[e] - delta);
                }
            }
            if (j0 + 32 > sure) {
                const int lim = row.end - j0 - 4 * row.part;
#pragma unroll
                for (int e = 0; e < N; ++e) y[e] = row.key(e) < lim ? y[e] : 0.0f;
            }
            if (BIAS && plan.sums && turn == 0) {
                // Each lane has a column of its own, so plain sums do, in the walk's order (an
                // atomic LDS add takes some 200 cycles a wave).  Far keys share a bucket, mostly
                // for a whole wave: then their sum goes in at once.
                float *mine = hist + tid;
                if (!sel)
#pragma unroll
                    for (int e = 0; e < N; ++e) y[e] = 0.0f;
#pragma unroll
                for (int n = 0; n < N; n += 4) {
                    const uint32_t to = bucket[n / 4] & 255;
                    if (__all(bucket[n / 4] == to * 0x01010101u)) {
                        mine[to * THREADS] += unscaled<T>((y[n] + y[n + 1]) + (y[n + 2] + y[n + 3]), factor);
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e) mine[(bucket[n / 4] >> (8 * e) & 255) * THREADS] += unscaled<T>(y[n + e], factor);
                    }
                }
            }
            if (T::NARROW) {
                float big = largest<N>(y);
                if (__builtin_expect(__any(big > FACTOR_TOP) != 0, 0)) {
                    big = row_max<F::PARTS>(big);
                    const int down = big > FACTOR_TOP ? factor_for(big) : 0;
                    const float f = times(1.0f, down);
#pragma unroll
                    for (int t = 0; t < DP / ROWS; ++t) o[t] *= f;
#pragma unroll
                    for (int e = 0; e < N; ++e) y[e] *= f;
                    factor += down;
                    if (more) {   // again, so that their registers are free here (else 24 more are spilled)
                        kp.load(kr, jn, vend);
                        vp.load(vr, jn, vend);
                    }
                }
            }
            __builtin_amdgcn_s_setprio(1);
            products<T, DP, ROWS>(tile, KT, y, o);
            __builtin_amdgcn_s_setprio(0);
            j0 = jn;
            mask = maskn;
        }
        if (tid == 0) scratch[1] = 0;
        __syncthreads();
        if (BIAS && plan.sums && turn == 0) {
            // a row's columns first: ROWS threads take a bucket, starting at different columns so
            // that those of a wave lie in different banks
            constexpr int COLS = THREADS / ROWS;
            for (int n = tid / ROWS; n < s.num_buckets; n += COLS) {
                float t = 0.0f;
                for (int a = 0; a < COLS; ++a) t += hist[n * THREADS + ((a + n) & (COLS - 1)) * ROWS + tid % ROWS];
                hist[n * THREADS + tid % ROWS] = t;   // read by this thread alone (column 0) up to here
            }
            __syncthreads();
            for (int e = tid; e < plan.span * s.num_buckets; e += THREADS) {
                const int h = e / s.num_buckets, n = e % s.num_buckets;
                float t = 0.0f;
                for (int r = h; r < rows; r += plan.span) t += hist[n * THREADS + r];
                plan.sums[tile_id * plan.span * s.num_buckets + e] = t;
            }
            __syncthreads();
        }
        const int r0 = lane % ROWS;
        const float back = T::NARROW ? times(1.0f, -factor) : 1.0f;
#pragma unroll
        for (int t = 0; t < DP / ROWS; ++t)
#pragma unroll
            for (int n = 0; n < (int)(sizeof(typename F::Acc) / 4); n += 4) {
                f32x4 z;
#pragma unroll
                for (int e = 0; e < 4; ++e) z[e] = T::NARROW ? o[t][n + e] * back : o[t][n + e];
                *reinterpret_cast<f32x4 *>(sums + (wave * ROWS + r0) * (DP + 4) + ROWS * t + row.key(n) + 4 * row.part) = z;
            }
        __syncthreads();
        bool fine = true;
        for (int e = tid; e < ROWS * CH; e += THREADS) {
            const int r = e / CH, ch = e % CH;
            if (r >= rows || ch * 8 >= s.dim) continue;
            const int rq = plan.per_span(r);
            if (!(only >> rq & 1u)) continue;
            float y[8] = {};
            for (int n = 0; n < W; ++n)
#pragma unroll
                for (int d = 0; d < 8; ++d) y[d] += sums[(n * ROWS + r) * (DP + 4) + ch * 8 + d];
#pragma unroll
            for (int d = 0; d < 8; ++d) {
                fine = fine && fabsf(y[d]) < INFINITY;
                y[d] *= s.scale;
            }
            *reinterpret_cast<s16x8 *>(dq.at(b, i0 + rq, (int64_t)g * s.group + h0 + r - rq * plan.span) + ch * 8) = Mma<T>::pack(y);
        }
        if (turn == 0) {
            if (!fine) scratch[1] = 1;
            __syncthreads();
            if (scratch[1] == 0) break;
        }
        __syncthreads();
    }
}

// dtable[n][h]: the tiles' sums, one workgroup for each (bucket, head), at the end of
// k_grad_kv_join's where that is launched (2 x 2048 tokens of 16 heads, 32 buckets: a
// launch of its own is 4.6 us).
template <class T> __device__ void sum_table(const AttnShape &s, const GradPlan &plan, uint32_t w, uint16_t *__restrict__ dtable) {
    __shared__ float part[256];
    const int h = w % (uint32_t)s.q_heads, n = w / (uint32_t)s.q_heads, g = h / s.group, hh = h % s.group;
    const int32_t each = plan.tiles / plan.parts;   // tiles with this head, of a batch element and key head
    float t = 0.0f;
    for (int64_t r = threadIdx.x; r < (int64_t)s.batch * each; r += 256) {
        const int64_t tile = (r / each * s.k_heads + g) * plan.tiles + r % each * plan.parts + hh / plan.span;
        t += plan.sums[(tile * plan.span + hh % plan.span) * s.num_buckets + n];
    }
    part[threadIdx.x] = t;
    __syncthreads();
    for (int d = 128; d; d >>= 1) {
        if ((int)threadIdx.x < d) part[threadIdx.x] += part[threadIdx.x + d];
        __syncthreads();
    }
    if (threadIdx.x == 0) dtable[(int64_t)n * s.q_heads + h] = T::down(part[0]);
}
template <class T>
__global__ __launch_bounds__(256) void k_grad_table(AttnShape s, GradPlan plan, uint16_t *__restrict__ dtable) {
    sum_table<T>(s, plan, blockIdx.x, dtable);
}

// ------------------------------------------------------------------ the pattern's transpose
// bits[batch x k_heads][block][q_len / 32]: who chose the block and can read of
// it; count[..][block]: how many.  One workgroup for 32 queries, so that a block's word
// has one writer; integer atomics, whose order does not show.  8192 queries, 2 heads, 128
// blocks: 6.8 us.
__global__ __launch_bounds__(256) void k_invert(AttnShape s, int32_t nw, const int32_t *__restrict__ blocks,
                                                       uint32_t *__restrict__ bits, int32_t *__restrict__ count) {
    extern __shared__ uint32_t word[];   // nblocks
    const uint32_t head = blockIdx.x / (uint32_t)nw;
    const int64_t bh = head;
    const int q32 = (int)(blockIdx.x - head * nw), b = (int)(head / (uint32_t)s.k_heads);
    const int ql = s.ql(b), kl = s.kl(b), i0 = q32 * 32;
    for (int c = threadIdx.x; c < s.nblocks; c += 256) word[c] = 0;
    __syncthreads();
    const int n = max(0, min(32, ql - i0)) * s.keep;
    for (int e = threadIdx.x; e < n; e += 256) {
        const int i = i0 + s.per_keep(e), c = blocks[(bh * s.q_len + i0) * s.keep + e];
        const int end = s.causal ? min(kl, i + kl - ql + 1) : kl;
        if (c >= 0 && c < s.nblocks && (int64_t)c * s.block < end) atomicOr(&word[c], 1u << (i - i0));
    }
    __syncthreads();
    for (int c = threadIdx.x; c < s.nblocks; c += 256) {
        const uint32_t x = word[c];
        bits[(bh * s.nblocks + c) * nw + q32] = x;
        if (x) atomicAdd(&count[bh * s.nblocks + c], __popc(x));
    }
}

// first[e] = items of the blocks before e, an item being up to `per` queries of a block;
// slot[e] = items before e of blocks with more than one, whose results are joined.
// first[n], slot[n] = all.  One workgroup's scan: 5 us up to some thousand blocks.
__global__ __launch_bounds__(1024) void k_items(int64_t n, int32_t per, const int32_t *__restrict__ count, int32_t *__restrict__ first,
                                                       int32_t *__restrict__ slot) {
    __shared__ int32_t part[2][1024];
    const int tid = threadIdx.x;
    const int64_t share = (n + 1023) / 1024, lo = min(n, tid * share), hi = min(n, lo + share);
    int32_t sum = 0, many = 0;
    for (int64_t e = lo; e < hi; ++e) {
        const int32_t items = (count[e] + per - 1) / per;
        sum += items;
        many += items > 1 ? items : 0;
    }
    part[0][tid] = sum;
    part[1][tid] = many;
    __syncthreads();
    for (int d = 1; d < 1024; d <<= 1) {
        const int32_t s = tid >= d ? part[0][tid - d] : 0, m = tid >= d ? part[1][tid - d] : 0;
        __syncthreads();
        part[0][tid] += s;
        part[1][tid] += m;
        __syncthreads();
    }
    int32_t at = part[0][tid] - sum, of = part[1][tid] - many;
    for (int64_t e = lo; e < hi; ++e) {
        const int32_t items = (count[e] + per - 1) / per;
        first[e] = at;
        slot[e] = of;
        at += items;
        of += items > 1 ? items : 0;
    }
    if (tid == 1023) {
        first[n] = part[0][1023];
        slot[n] = part[1][1023];
    }
}

__global__ __launch_bounds__(256) void k_clear(int64_t n, int32_t *__restrict__ p) {
    const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (e < n) p[e] = 0;
}

// ------------------------------------------------------------------ dk, dv
struct KeyPlan {
    int32_t nw, per, subs;      // words of a block's bits, queries of an item, 64-key parts of a block
    int64_t entries;            // batch x k_heads x nblocks
    const uint32_t *bits;
    const int32_t *count, *first, *slot;
    const float *delta, *shift, *corr;
    float *part;                // [slot][sub][dk, dv][64][DP]: items of blocks with more than one
};

constexpr int FIGURES = 6;   // of each row in k_grad_kv's LDS

// One workgroup for an item and 64 of its block's keys; wave w has 16 of them,
// with K and V resident as the right operands of S = Q K^T and dP = dO V^T.
// Their results hold one key and 2 x 4 rows in a lane, as the left operands of
// dV += P^T dO and dK += dS^T Q want them; dO and Q come from LDS both ways.
// P and dS are rounded to the inputs' type for these products (half a step of
// each), sums are fp32.  Three workgroups a CU need at most 168 registers, hence the
// barriers that keep the compiler from reading ahead (with 35 spilled 1.29 ms, with few
// 1.16 ms for 8192 tokens' training step then; 2 are left for bf16 heads of 128, 6 for fp16).
template <class T, int DP, bool BIAS>
__global__ __launch_bounds__(256, BIAS && DP == 128 ? 2 : 3) void k_grad_kv(AttnShape s, KeyPlan plan, Side dout, Side q, Side k, Side v,
                                                    const float *__restrict__ lse, SideOut dk, SideOut dv) {
    constexpr int KS = DP / 32, DT = DP / 16, CH = DP / 8, TILE = 32 * DP * 2, LD = 32 * CH / 256;
    extern __shared__ __attribute__((aligned(16))) char lds[];   // [2][Q, dO] tiles
    float *fig = reinterpret_cast<float *>(lds + 4 * TILE);       // [2][32] of (shift, delta, end, position, head, corr)
    int32_t *list = reinterpret_cast<int32_t *>(fig + 2 * FIGURES * 32);
    int32_t *scratch = list + plan.per;                           // flag, prefix of the list's words
    float *table = reinterpret_cast<float *>(scratch + 8);

    const int32_t w = work_of((uint32_t)plan.first[plan.entries] * plan.subs);
    if (w < 0) return;
    const int32_t item = (uint32_t)w / (uint32_t)plan.subs;
    const int sub = w - item * plan.subs;
    uint32_t lo = 0, hi = (uint32_t)plan.entries;   // the block with first[e] <= item < first[e + 1]
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (plan.first[mid] <= item) lo = mid;
        else hi = mid;
    }
    const uint32_t head = lo / (uint32_t)s.nblocks;
    const int64_t entry = lo;
    const int part = item - plan.first[entry], items = plan.first[entry + 1] - plan.first[entry];
    const int c = (int)(lo - head * s.nblocks), b = head / (uint32_t)s.k_heads, g = head - b * s.k_heads;
    const int ql = s.ql(b), kl = s.kl(b), j0 = c * s.block + sub * 64;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / 64), lane = tid % 64, col = lane & 15, quad = lane >> 4;
    const int nqueries = min(plan.per, plan.count[entry] - part * plan.per);

    if (BIAS)
        for (int e = tid; e < s.num_buckets * s.group; e += 256)
            table[e] = T::up(s.table[(e / s.group) * s.q_heads + g * s.group + e % s.group]);
    // the queries of this item: those whose rank among the block's bits is in [part * per, + per)
    if (wave == 0) {
        int before = 0;
        const uint32_t *bits = plan.bits + entry * plan.nw;
        for (int w0 = 0; w0 < plan.nw && before < part * plan.per + nqueries; w0 += 64) {
            uint32_t x = w0 + lane < plan.nw ? bits[w0 + lane] : 0;
            int sum = __popc(x);
            const int mine = sum;
            for (int d = 1; d < 64; d <<= 1) {
                const int t = __shfl_up(sum, d);
                if (lane >= d) sum += t;
            }
            int rank = before + sum - mine - part * plan.per;
            for (; x; x &= x - 1, ++rank)
                if (rank >= 0 && rank < nqueries) list[rank] = (w0 + lane) * 32 + __ffs(x) - 1;
            before += __shfl(sum, 63);
        }
    }
    const Tile<DP> tile(lds, lane);
    // this wave's keys
    const int key = j0 + 16 * wave + col;
    s16x8 kf[KS], vf[KS];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
        const int d = 32 * ks + 8 * quad;
        const bool on = key < kl && d < s.dim;
        kf[ks] = on ? load8(k.at(b, key, g) + d) : s16x8{};
        vf[ks] = on ? load8(v.at(b, key, g) + d) : s16x8{};
    }
    __syncthreads();
    const int rows = nqueries * s.group;
    const float cs = BIAS ? s.scale : s.scale * LOG2E;

    f32x4 ak[DT], av[DT];
#pragma unroll
    for (int t = 0; t < DT; ++t) ak[t] = av[t] = f32x4{};
    int factor = FACTOR_START - (int)LIFT<T>;   // of this lane's key: its dS and its sum of them
    s16x8 qn[LD], dn[LD];
    float fn[FIGURES];
    auto fetch = [&](int r0) {
#pragma unroll
        for (int n = 0; n < LD; ++n) {
            const int r = r0 + (n * 256 + tid) / CH, ch = tid % CH;
            const bool on = r < rows && ch * 8 < s.dim;
            const int rr = min(r, rows - 1), rq = (uint32_t)rr / (uint32_t)s.group, i = list[rq], d = ch * 8 < s.dim ? ch * 8 : 0;
            const int64_t h = (int64_t)g * s.group + rr - rq * s.group;
            const s16x8 x = load8(q.at(b, i, h) + d), y = load8(dout.at(b, i, h) + d);
            qn[n] = on ? x : s16x8{};
            dn[n] = on ? y : s16x8{};
        }
        if (tid < 32) {
            const int r = r0 + tid;
            const bool on = r < rows;
            const int rr = min(r, rows - 1), rq = (uint32_t)rr / (uint32_t)s.group, i = list[rq], p = i + kl - ql;
            const int64_t at = ((int64_t)b * s.q_heads + (int64_t)g * s.group + rr - rq * s.group) * s.q_len + i;
            if (BIAS) {
                fn[0] = on ? plan.shift[at] : INFINITY;
                fn[5] = plan.corr[at] - LIFT<T>;
            } else {
                const float l = on ? lse[at] : -INFINITY;
                fn[0] = l == -INFINITY ? INFINITY : l * LOG2E - LIFT<T>;
            }
            fn[1] = plan.delta[at];
            fn[2] = __int_as_float(!on ? 0 : s.causal ? min(kl, p + 1) : kl);
            fn[3] = __int_as_float(p);
            fn[4] = __int_as_float(rr - rq * s.group);
        }
    };
    auto put = [&](int buf) {
#pragma unroll
        for (int n = 0; n < LD; ++n) {
            const int e = n * 256 + tid;
            char *to = lds + buf * 2 * TILE + Tile<DP>::chunk(e / CH, e % CH);
            *reinterpret_cast<s16x8 *>(to) = qn[n];
            *reinterpret_cast<s16x8 *>(to + TILE) = dn[n];
        }
        if (tid < 32)
#pragma unroll
            for (int f = 0; f < (BIAS ? 6 : 3); ++f) fig[(buf * FIGURES + f) * 32 + tid] = fn[f];
    };
    fetch(0);
    int buf = 0;
    for (int r0 = 0; r0 < rows; r0 += 32, buf ^= 1) {
        put(buf);
        __syncthreads();
        if (r0 + 32 < rows) fetch(r0 + 32);
        const int qt = buf * 2 * TILE, dt = qt + TILE;
        const float *f = fig + buf * FIGURES * 32;
        float p[8], ds[8];
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            __builtin_amdgcn_sched_barrier(0);
            f32x4 x{}, dp{};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                x = Mma<T>::run(tile.natural(qt, 16 * m, ks), kf[ks], x);
                dp = Mma<T>::run(tile.natural(dt, 16 * m, ks), vf[ks], dp);
            }
            const int at = 16 * m + 4 * quad;
            const f32x4 shift = *reinterpret_cast<const f32x4 *>(f + at), delta = *reinterpret_cast<const f32x4 *>(f + 32 + at);
            const f32x4 end = *reinterpret_cast<const f32x4 *>(f + 64 + at);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float y;
                if (BIAS) {
                    const int pos = __float_as_int(f[96 + at + e]), hr = __float_as_int(f[128 + at + e]);
                    y = __builtin_amdgcn_exp2f(__builtin_fmaf(__builtin_fmaf(x[e], cs, table[s.map[(int64_t)key - pos + s.k_len - 1] * s.group + hr]) - shift[e], LOG2E, -f[160 + at + e]));
                } else {
                    y = __builtin_amdgcn_exp2f(__builtin_fmaf(x[e], cs, -shift[e]));
                }
                const bool on = key < __float_as_int(end[e]);
                p[4 * m + e] = on ? y : 0.0f;
                ds[4 * m + e] = on ? y * (dp[e] - delta[e]) : 0.0f;
            }
        }
        if (T::NARROW) {
#pragma unroll
            for (int e = 0; e < 8; ++e) ds[e] = times(ds[e], factor);
            float big = largest<8>(ds);
            if (__any(big > FACTOR_TOP)) {
                big = row_max<4>(big);
                const int down = big > FACTOR_TOP ? factor_for(big) : 0;
                const float f = times(1.0f, down);
#pragma unroll
                for (int e = 0; e < 8; ++e) ds[e] *= f;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float c = __shfl(f, 4 * quad + e);
#pragma unroll
                    for (int t = 0; t < DT; ++t) ak[t][e] *= c;
                }
                factor += down;
            }
        }
        const s16x8 pf = Mma<T>::pack(p), sf = Mma<T>::pack(ds);
#pragma unroll
        for (int t = 0; t < DT; ++t) {
            if (t % 2 == 0) __builtin_amdgcn_sched_barrier(0);   // else every fragment is read ahead and spilled
            av[t] = Mma<T>::run(pf, tile.transposed(dt, t), av[t]);
            ak[t] = Mma<T>::run(sf, tile.transposed(qt, t), ak[t]);
        }
    }
    if (T::NARROW)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float back = times(1.0f, -__shfl(factor, 4 * quad + e) - (int)LIFT<T>);
#pragma unroll
            for (int t = 0; t < DT; ++t) {
                ak[t][e] *= back;
                av[t][e] = times(av[t][e], -(int)LIFT<T>);
            }
        }
    if (tid == 0) scratch[0] = 0;
    __syncthreads();
    const bool alone = items == 1;
    float *const parts = plan.part + ((int64_t)(plan.slot[entry] + part) * plan.subs + sub) * 2 * 64 * DP;   // not if alone
    bool fine = true;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        __builtin_amdgcn_sched_barrier(0);   // one row's addresses at a time
        const int n = 16 * wave + 4 * quad + e, j = j0 + n;
        uint16_t *tk = dk.at(b, min(j, kl - 1), g) + col, *tv = dv.at(b, min(j, kl - 1), g) + col;
        float *to = parts + n * DP + col;
#pragma unroll
        for (int t = 0; t < DT; ++t) {
            if (16 * t + col >= s.dim) continue;
            fine = fine && fabsf(ak[t][e]) < INFINITY && fabsf(av[t][e]) < INFINITY;
            if (!alone) {
                to[16 * t] = ak[t][e];
                to[64 * DP + 16 * t] = av[t][e];
            } else if (j < kl) {
                tk[16 * t] = T::down(ak[t][e] * s.scale);
                tv[16 * t] = T::down(av[t][e]);
            }
        }
    }
    if (!fine) scratch[0] = 1;
    __syncthreads();
    if (scratch[0] == 0) return;

    // Something is not finite.  Zeros of P and dS times a row's infinities make NaN in keys that
    // the row does not read, so once more without products of what is masked: four threads for a
    // key, a quarter of the channels each, the rows one by one.
    constexpr int C = DP / 4;
    const int n = tid / 4, j = j0 + n, d0 = tid % 4 * C;
    float bk[C], bv[C];
#pragma unroll
    for (int d = 0; d < C; ++d) bk[d] = bv[d] = 0.0f;
    if (j < kl) {
        const uint16_t *kr = k.at(b, j, g), *vr = v.at(b, j, g);
        for (int r = 0; r < rows; ++r) {
            const int i = list[r / s.group], pos = i + kl - ql, hr = r % s.group;
            const int64_t h = (int64_t)g * s.group + hr, at = ((int64_t)b * s.q_heads + h) * s.q_len + i;
            const float l = lse[at], shift = BIAS ? plan.shift[at] : l, corr = BIAS ? plan.corr[at] : 0.0f;
            if ((s.causal && j > pos) || l == -INFINITY) continue;
            const uint16_t *qr = q.at(b, i, h), *dr = dout.at(b, i, h);
            float x = 0.0f, dp = 0.0f;
#pragma unroll
            for (int d = 0; d < C; ++d)
                if (d0 + d < s.dim) {
                    x = __builtin_fmaf(T::up(qr[d0 + d]), T::up(kr[d0 + d]), x);
                    dp = __builtin_fmaf(T::up(dr[d0 + d]), T::up(vr[d0 + d]), dp);
                }
            for (int m = 1; m < 4; m <<= 1) {
                x += __shfl_xor(x, m);
                dp += __shfl_xor(dp, m);
            }
            x *= s.scale;
            if (BIAS) x += table[s.map[(int64_t)j - pos + s.k_len - 1] * s.group + hr];
            const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(x - shift, LOG2E, -corr)), ds = p * (dp - plan.delta[at]);
#pragma unroll
            for (int d = 0; d < C; ++d)
                if (d0 + d < s.dim) {
                    bv[d] = __builtin_fmaf(p, T::up(dr[d0 + d]), bv[d]);
                    bk[d] = __builtin_fmaf(ds, T::up(qr[d0 + d]), bk[d]);
                }
        }
#pragma unroll
        for (int d = 0; d < C; ++d) {
            if (d0 + d >= s.dim) continue;
            if (!alone) {
                parts[n * DP + d0 + d] = bk[d];
                parts[(64 + n) * DP + d0 + d] = bv[d];
            } else {
                dk.at(b, j, g)[d0 + d] = T::down(bk[d] * s.scale);
                dv.at(b, j, g)[d0 + d] = T::down(bv[d]);
            }
        }
    }
}

// dk and dv of the blocks that no query or more than one item read, and of the keys
// behind a sequence's end: a thread for 8 channels of a key, 16 keys a workgroup, the
// results of four items in flight.  Bound by reading those (8192 tokens: 50 us).  The
// workgroups behind them sum the bias's gradient.
template <class T>
__global__ __launch_bounds__(256) void k_grad_kv_join(AttnShape s, KeyPlan plan, int32_t dp, SideOut dk, SideOut dv, GradPlan sums,
                                                      uint16_t *__restrict__ dtable) {
    const uint32_t joins = (uint32_t)plan.entries * plan.subs * 4;
    if (blockIdx.x >= joins) {
        sum_table<T>(s, sums, blockIdx.x - joins, dtable);
        return;
    }
    const uint32_t e = blockIdx.x / 4 / (uint32_t)plan.subs, head = e / (uint32_t)s.nblocks;
    const int sub = (int)(blockIdx.x / 4 - e * plan.subs);
    const int64_t entry = e;
    const int32_t first = plan.first[entry], items = plan.first[entry + 1] - first;
    const int c = (int)(e - head * s.nblocks), b = head / (uint32_t)s.k_heads, g = head - b * s.k_heads;
    const int n = blockIdx.x % 4 * 16 + threadIdx.x / 16, d = threadIdx.x % 16 * 8, j = c * s.block + sub * 64 + n;
    if (d >= s.dim) return;
    if (j >= s.kl(b)) {
        if (s.clear && j < s.k_len) {
            *reinterpret_cast<s16x8 *>(dk.at(b, j, g) + d) = s16x8{};
            *reinterpret_cast<s16x8 *>(dv.at(b, j, g) + d) = s16x8{};
        }
        return;
    }
    if (items == 1) return;
    const f32x4 *from = reinterpret_cast<const f32x4 *>(plan.part + (((int64_t)plan.slot[entry] * plan.subs + sub) * 2 * 64 + n) * dp + d);
    const int64_t step = (int64_t)plan.subs * 2 * 64 * dp / 4, other = 64 * dp / 4;
    f32x4 x[2] = {}, y[2] = {};
    for (int t0 = 0; t0 < items; t0 += 4) {
        f32x4 z[4][4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const f32x4 *at = from + min(t0 + t, items - 1) * step;
            z[t][0] = at[0];
            z[t][1] = at[1];
            z[t][2] = at[other];
            z[t][3] = at[other + 1];
        }
#pragma unroll
        for (int t = 0; t < 4; ++t)
            if (t0 + t < items) {
                x[0] += z[t][0];
                x[1] += z[t][1];
                y[0] += z[t][2];
                y[1] += z[t][3];
            }
    }
    float u[8], v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        u[i] = x[i / 4][i % 4] * s.scale;
        v[i] = y[i / 4][i % 4];
    }
    *reinterpret_cast<s16x8 *>(dk.at(b, j, g) + d) = Mma<T>::pack(u);
    *reinterpret_cast<s16x8 *>(dv.at(b, j, g) + d) = Mma<T>::pack(v);
}

}  // namespace dev
}  // namespace ias
