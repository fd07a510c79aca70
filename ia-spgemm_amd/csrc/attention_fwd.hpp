// attention_fwd.hpp — block-sparse attention, forward (k_attend, k_attend_join).
//
// A workgroup takes up to ROWS rows of one key head: its query heads for a few
// consecutive queries (row r is query r / span, head r % span), or some of the heads
// of one query where there are more of them than rows.  It walks the union of the blocks
// that these queries chose, each block once: neighbouring queries choose mostly the same
// blocks, and where they do not the walk reads no more than the queries would one by one.
// A row that did not choose a block masks it.  The W waves share nothing while they walk:
// wave w takes every W-th piece of 32 keys and keeps its own running maximum, sum and
// output (softmax in one pass), and they meet once at the end.
//
// Per piece: K and V go from memory through registers (the next piece's loads run
// under this one's work) into the wave's own LDS tiles.  S^T = K Q^T with Q^T
// resident in registers.  In S^T's result a lane holds one row and 2 x 4 keys, which is
// just what the right operand of O^T += V^T P^T asks for, so P never leaves the
// registers; it is rounded to the inputs' type for that product (off by half a
// step relative to each probability, as the values are), everything else is
// fp32.  V^T's fragments need the keys of one channel side by side: transposed
// LDS reads.  The tiles' 32-byte columns are permuted by row, so that the 8 rows
// which half a wave reads lie in 8 different groups of banks.
//
// Prompts are bound by the latency of a piece's chain (load, LDS, scores, exponentials,
// product) with the two waves a SIMD that 256 registers a lane allow (three for heads of
// 64): 8192 tokens, 32/8 heads of 128, 16 blocks of 64 keys a query, random choices: 0.52 to
// 0.55 ms, where a union of 8 queries has 39 blocks.  Of the CUs' cycles the matrix units are
// busy in 26 % (SQ_VALU_MFMA_BUSY_CYCLES), the vector ALUs in 35 % (SQ_ACTIVE_INST_VALU), LDS in
// 48 % (SQ_LDS_IDX_ACTIVE), the vector cache in 54 % (TCP_TOTAL_CACHE_ACCESSES).  Single tokens are bound by the
// read of K and V (16 users, 32 of up to 512 blocks, 8 heads of 128: 134 MB in 28.8 us,
// 4.7 TB/s) and few of them by one workgroup's chain of loads for each key head (13.7 us
// for one user).
#pragma once

#include "attention_kernels.hpp"

namespace ias {
namespace dev {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

template <class T> struct Mma;
template <> struct Mma<Bf16> {
    static __device__ f32x4 run(s16x8 a, s16x8 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
    static __device__ f32x16 run(s16x8 a, s16x8 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
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
    static __device__ f32x16 run(s16x8 a, s16x8 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
    static __device__ s16x8 pack(const float *x) {
        f16x8 y;
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = (_Float16)x[e];
        return __builtin_bit_cast(s16x8, y);
    }
};

// k_attend's probabilities are relative to a maximum that is moved only where exponentials
// would pass 2^SLACK.  fp16 has 11 bits down to 2^-14 only, and 2^18 keys of 2^-24 each are
// worth 1.5 % of one of 1: they are rounded at 2^11 times their size, 2^15 at most, which
// holds 11 bits down to 2^-25.  The exponentials' argument takes the 11.
template <class T> constexpr float SLACK = T::NARROW ? 4.0f : 8.0f;
template <class T> constexpr float RAISE = T::NARROW ? 11.0f : 0.0f;
template <class T> constexpr float LOWER = T::NARROW ? 0x1p-11f : 1.0f;

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

__device__ inline s16x8 load8(const uint16_t *p) { return *reinterpret_cast<const s16x8 *>(p); }

// How the matrix instructions lay out 16 or 32 rows of queries by 32 keys.  The results
// of S^T = K Q^T: a lane holds one row, of the keys 4 PARTS * (e / 4) + 4 * part + e % 4
// for e < N, and PARTS lanes share the row.  The same, in this order and in groups of 8,
// is what the right operand of O^T += V^T P^T asks for.
template <int ROWS> struct Form;
template <> struct Form<16> {
    static constexpr int PARTS = 4, N = 8, K = 32;   // K: terms of one instruction
    typedef f32x4 Acc;
};
template <> struct Form<32> {
    static constexpr int PARTS = 2, N = 16, K = 16;
    typedef f32x16 Acc;
};

// A tile of 32 rows by DP channels (16 bits) in LDS, 32-byte columns permuted by row:
// column c of row r lies at c ^ mix(r), so that the 8 rows which half a wave reads, and
// the 4 rows by 64 bytes of a transposed read, lie in different banks.  Addresses are LDS
// offsets; all of one lane's come from four by xor and constant offsets.
template <int DP, int ROWS = 16> struct Tile {
    typedef __attribute__((address_space(3))) s16x8 lds8;
    typedef __attribute__((address_space(3))) s16x4 lds4;
    static constexpr int ROW = DP * 2, BYTES = 32 * ROW, CH = DP / 8, N = 32 * CH / 64, STEP = 64 / CH;
    static __device__ uint32_t mix(int row) {
        return DP == 128 ? 2 * (row & 3) + (row >> 2 & 1) : (row & 2) + (row >> 2 & 1);
    }
    // 16-byte chunk c of a row
    static __device__ uint32_t chunk(int row, int c) { return row * ROW + ((((uint32_t)c >> 1) ^ mix(row)) * 32) + (c & 1) * 16; }
    static __device__ uint32_t offset(const char *lds) {
        return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char *)lds;
    }
    template <class P> static __device__ P *lds(uint32_t at) { return (P *)(uintptr_t)at; }
    uint32_t even, odd, nat, tr;
    __device__ Tile(const char *lds, int lane) {
        const uint32_t base = offset(lds);
        even = base + chunk(lane / CH, lane % CH);
        odd = base + chunk(STEP + lane / CH, lane % CH);   // mix has a period of 8 rows
        nat = base + chunk(lane % ROWS, lane / ROWS);
        const int r = 4 * (lane / ROWS) + ((lane & 15) >> 2), c = lane % ROWS / 16;
        tr = base + r * ROW + (c ^ mix(r)) * 32 + (lane & 3) * 8;
    }
    // A piece that lies in registers as Piece::load leaves it; `at`: a tile's offset from the lane's.
    __device__ void fill(const s16x8 (&f)[N], int at) const {
#pragma unroll
        for (int n = 0; n < N; ++n) {
            if (STEP == 8) *lds<lds8>(even + at + n * 8 * ROW) = f[n];
            else *lds<lds8>((n % 2 ? odd : even) + at + n / 2 * 8 * ROW) = f[n];
        }
    }
    // Left operand from the tile as it is: row row0 + lane % ROWS, channels K * ks + 8 * (lane / ROWS) + 0..7.
    __device__ s16x8 natural(int at, int row0, int ks) const { return *lds<lds8>((nat ^ (ks * 2 * Form<ROWS>::K)) + at + row0 * ROW); }
    // Operand from the transposed tile: channel ROWS * c + lane % ROWS, rows row0 + 4 * (lane / ROWS) + 0..3
    // and 4 PARTS further.
    __device__ s16x8 transposed(int at, int c, int row0 = 0) const {
        const uint32_t a = (tr ^ (c * 2 * ROWS)) + at + row0 * ROW;
        const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16(lds<lds4>(a));
        const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16(lds<lds4>(a + 4 * Form<ROWS>::PARTS * ROW));
        return __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
    }
};

// x[e] for the N keys of a lane: a tile's 32 keys against the rows whose operands are q.
// AHEAD: all reads before the first product, where there are registers for that; the
// compiler alone keeps one or two under way (k_attend 537 -> 529 us for 8192 tokens; in
// k_grad_q other operands would be spilled, 306 -> 420).
template <class T, int DP, int ROWS, bool AHEAD>
__device__ inline void scores(const Tile<DP, ROWS> &tile, int at, const s16x8 *q, float *x) {
    typedef Form<ROWS> F;
    constexpr int KS = DP / F::K;
    s16x8 f[32 / ROWS * KS];
#pragma unroll
    for (int n = 0; n < 32 / ROWS * KS; ++n) f[n] = tile.natural(at, ROWS * (n / KS), n % KS);
    if (AHEAD) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int sub = 0; sub < 32 / ROWS; ++sub) {
        typename F::Acc acc{};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) acc = Mma<T>::run(f[sub * KS + ks], q[ks], acc);
#pragma unroll
        for (int e = 0; e < F::N * ROWS / 32; ++e) x[sub * (F::N * ROWS / 32) + e] = acc[e];
    }
}
// o[c]: channels ROWS * c + .., += the tile's rows, transposed, times y.
template <class T, int DP, int ROWS>
__device__ inline void products(const Tile<DP, ROWS> &tile, int at, const float *y, typename Form<ROWS>::Acc *o) {
    typedef Form<ROWS> F;
    s16x8 f[F::N / 8];
#pragma unroll
    for (int n = 0; n < F::N / 8; ++n) f[n] = Mma<T>::pack(y + 8 * n);
#pragma unroll
    for (int c = 0; c < DP / ROWS; ++c)
#pragma unroll
        for (int n = 0; n < F::N / 8; ++n) o[c] = Mma<T>::run(tile.transposed(at, c, 16 * n), f[n], o[c]);
}

// Which of `total` parts of the work a workgroup has, -1 if none.  Consecutive ids go to
// the 8 dies in turn; each die gets a contiguous stretch, so that parts that read the same
// K and V meet in one L2.
// (All parts of a call are fewer than 2^31: 32-bit divisions, which take a fraction of the
// instructions.)
__device__ inline int32_t work_of(uint32_t total) {
    const uint32_t per = (total + 7) / 8, n = blockIdx.x / 8, w = blockIdx.x % 8 * per + n;
    return n < per && w < total ? (int32_t)w : -1;
}
// The same for `each` tiles of `heads` key heads, the last tiles of a head first: those of
// a causal call walk furthest, and short walks at the end even it out (8192 tokens 587 ->
// 538 us).  Where fewer heads than dies divide them, a head's tiles go to its dies in turn,
// since a stretch of a head's first ones would be the shorter work.
struct Part {
    int32_t head, tile;   // head -1: none
};
__device__ inline Part tile_of(uint32_t heads, uint32_t each) {
    if (heads < 8 && (heads & (heads - 1)) == 0) {
        const uint32_t shift = 31 - __clz(heads), die = blockIdx.x % 8, n = ((blockIdx.x / 8) << (3 - shift)) + (die >> shift);
        if (n >= each) return {-1, 0};
        return {(int32_t)(die & (heads - 1)), (int32_t)(each - 1 - n)};
    }
    const int32_t w = work_of(heads * each);
    if (w < 0) return {-1, 0};
    const uint32_t head = (uint32_t)w / each;
    return {(int32_t)head, (int32_t)(each - 1 - ((uint32_t)w - head * each))};
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
        const int qi = s.per_keep(e), c = blocks[row0 * s.keep + e];
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
        const int qi = s.per_keep(e), c = blocks[row0 * s.keep + e];
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

// Maximum and sum over the lanes that hold a row's keys (lanes 32, or 32 and 16 apart).
template <int PARTS> __device__ inline float row_max(float x) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    if (PARTS == 2) return x;
    const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
template <int PARTS> __device__ inline float row_sum(float x) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    if (PARTS == 2) return x;
    const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// What a lane knows of its row of queries.
template <int DP, int ROWS> struct Row {
    typedef Form<ROWS> F;
    int part, query, head, pos, end;   // head: of the key head's; end: keys before it may be read
    bool there;
    __device__ Row(int lane, int rows, int per, int h0, int span, int i0, int kl, int ql, bool causal) {
        const int r = lane % ROWS;
        part = lane / ROWS;
        there = r < rows;
        query = there ? per : 0;
        head = h0 + (there ? r - per * span : 0);
        pos = i0 + query + kl - ql;
        end = !there ? 0 : causal ? min(kl, pos + 1) : kl;
    }
    // right operand of the scores; zeros where there is no row or channel
    __device__ void load(s16x8 (&f)[DP / F::K], const uint16_t *row, int dim) const {
#pragma unroll
        for (int ks = 0; ks < DP / F::K; ++ks) {
            const int d = F::K * ks + 8 * part;
            f[ks] = there && d < dim ? load8(row + d) : s16x8{};
        }
    }
    static __device__ int key(int e) { return 4 * F::PARTS * (e / 4) + e % 4; }   // without 4 * part
};

__device__ inline s16x8 negated(s16x8 x) { return x ^ (short)0x8000; }

// A wave's way along the union: pieces of 32 keys, every W-th is its own.
template <int W> struct Walk {
    int step, part, per;   // block of the union, piece of the block, pieces of a block
    __device__ Walk(int start, int per_block) : step(start / per_block), part(start % per_block), per(per_block) {}
    __device__ void on() {
        for (part += W; part >= per; part -= per) ++step;
    }
};

// 32 rows of K or V at the piece j0, 64 consecutive 16-byte chunks of consecutive
// rows at a time.  (A load straight into the matrix instruction's layout, 16 rows of
// 64 bytes, costs the cache one access for each lane instead of one for four, and was
// what bound the walk.)  Whole pieces take a scalar base and one 32-bit offset for
// all loads; at a sequence's end, and for narrower heads, addresses are kept inside
// and what is beyond becomes 0.
template <int DP> struct Piece {
    static constexpr int CH = DP / 8, N = 32 * CH / 64;
    const uint16_t *base;
    int64_t token;
    uint32_t off;          // bytes
    int lane, dim, last;   // last: row that may be read at most
    __device__ Piece(const Side &x, int b, int g, int lane, int dim, int kl)
        : base(x.at(b, 0, g)), token(x.token), lane(lane), dim(dim), last(kl - 1) {
        off = (uint32_t)((lane / CH) * token * 2 + (lane % CH) * 16);
    }
    __device__ void load(s16x8 (&f)[N], int j0, int end) const {
        if (j0 + 32 <= end && dim == DP) {
            const uint16_t *row = base + j0 * token;
#pragma unroll
            for (int n = 0; n < N; ++n, row += token * (64 / CH))
                f[n] = *reinterpret_cast<const s16x8 *>(reinterpret_cast<const char *>(row) + off);
            return;
        }
        int here = lane;
        asm volatile("" : "+v"(here));   // else every row's offset stays in a register all the way
        const int d = here % CH * 8;
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int j = j0 + n * (64 / CH) + here / CH;
            const s16x8 x = load8(base + min(j, last) * token + (d < dim ? d : 0));
            f[n] = j < end && d < dim ? x : s16x8{};
        }
    }
};

struct RowPlan {
    int32_t nq, span, parts;   // queries and heads of a workgroup, workgroups of one query's heads
    uint32_t inverse;          // ceil(2^16 / span)
    int32_t tiles;     // per batch element and key head
    int32_t splits;    // workgroups that share a tile's walk
    int32_t most;      // bound on the blocks of a union
    float *part;       // splits > 1: [tile][split][ROWS][DP] sums
    float *stat;       //             [tile][split][ROWS][2] maximum and sum
    __device__ int per_span(int r) const { return (int)((uint32_t)r * inverse >> 16); }   // r / span, r < 64
};

// LDS of k_attend: the end's sums (the waves' V tiles lie in the same place),
// the lists, the rows' figures, the bias table.
constexpr int walk_area(int dp, int rows, int waves) {
    return waves * (2 * 32 * dp * 2 > rows * (dp + 4) * 4 ? 2 * 32 * dp * 2 : rows * (dp + 4) * 4);
}
inline size_t attend_lds(int dp, int rows, int waves, int nblocks, int most, int table) {
    return walk_area(dp, rows, waves) + 8 * (size_t)((nblocks + 31) / 32) + 8 * (size_t)most + waves * (size_t)rows * 2 * 4 + 16 + 4 * (size_t)table;
}

// Zeros (and lse -inf) for the queries [from, to) of a tile, those behind a sequence's end.
__device__ inline void clear_rows(const AttnShape &s, int b, int g, int h0, int heads, int64_t from, int64_t to, const SideOut &out, float *lse) {
    const int chunks = s.dim / 8, each = heads * chunks;
    for (int64_t e = threadIdx.x; e < (to - from) * each; e += blockDim.x) {
        const int64_t i = from + e / each, h = (int64_t)g * s.group + h0 + e % each / chunks;
        *reinterpret_cast<s16x8 *>(out.at(b, i, h) + e % chunks * 8) = s16x8{};
        if (lse && e % chunks == 0) lse[((int64_t)b * s.q_heads + h) * s.q_len + i] = -INFINITY;
    }
}

template <class T, int DP, int ROWS, int W, bool BIAS>
__global__ __launch_bounds__(64 * W, 2) void k_attend(AttnShape s, RowPlan plan, Side q, Side k, Side v,
                                                      const int32_t *__restrict__ blocks, SideOut out, float *__restrict__ lse) {
    typedef Form<ROWS> F;
    constexpr int VL = Tile<DP>::N, CH = DP / 8, N = F::N;
    constexpr int AREA = walk_area(DP, ROWS, W);
    extern __shared__ __attribute__((aligned(16))) char lds[];
    float *sums = reinterpret_cast<float *>(lds);                       // [W][ROWS][DP + 4]
    float *stat = reinterpret_cast<float *>(lds + AREA);                // [W][ROWS][2]
    int32_t *scratch = reinterpret_cast<int32_t *>(stat + W * ROWS * 2);   // total, flag
    int32_t *ids = scratch + 4;
    uint32_t *masks = reinterpret_cast<uint32_t *>(ids + plan.most);
    uint32_t *words = masks + plan.most;
    float *table = reinterpret_cast<float *>(words + 2 * ((s.nblocks + 31) / 32));

    const Part part = tile_of(s.batch * s.k_heads, plan.tiles * plan.splits);
    if (part.head < 0) return;
    const uint32_t tile_no = (uint32_t)part.tile / (uint32_t)plan.splits, step = tile_no / (uint32_t)plan.parts;
    const int split = part.tile - tile_no * plan.splits;
    const int64_t tile_id = (int64_t)part.head * plan.tiles + tile_no, i0 = (int64_t)step * plan.nq;
    const int h0 = (int)(tile_no - step * plan.parts) * plan.span;   // of the key head's query heads
    const int b = (uint32_t)part.head / (uint32_t)s.k_heads, g = part.head - b * s.k_heads;
    const int ql = s.ql(b), kl = s.kl(b);
    if (s.clear && split == 0 && i0 + plan.nq > ql)
        clear_rows(s, b, g, h0, min(plan.span, s.group - h0), max(i0, (int64_t)ql), min(i0 + plan.nq, s.q_len), out, lse);
    if (i0 >= ql) return;
    const int nq = min(plan.nq, ql - (int)i0), rows = (nq - 1) * plan.span + min(plan.span, s.group - h0);
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / 64), lane = tid % 64;
    const Tile<DP, ROWS> tile(lds + wave * 2 * Tile<DP>::BYTES, lane);   // K, then V
    constexpr int KT = 0, VT = Tile<DP>::BYTES;

    // single tokens search the edges and save the map's launch
    int32_t *edges = reinterpret_cast<int32_t *>(table + s.num_buckets * plan.span);
    if (BIAS && ROWS == 16 && tid < s.num_buckets - 1) edges[tid] = s.edges[tid];
    if (BIAS)
        for (int e = tid; e < s.num_buckets * plan.span; e += 64 * W)
            if (h0 + e % plan.span < s.group) table[e] = T::up(s.table[(e / plan.span) * s.q_heads + g * s.group + h0 + e % plan.span]);
    const int found = __builtin_amdgcn_readfirstlane(block_union(s, blocks, b, g, i0, nq, ql, kl, words, ids, masks, scratch));

    const Row<DP, ROWS> row(lane, rows, plan.per_span(lane % ROWS), h0, plan.span, (int)i0, kl, ql, s.causal);
    s16x8 qf[DP / F::K];
    row.load(qf, q.at(b, i0 + row.query, (int64_t)g * s.group + row.head), s.dim);
    if (s.scale < 0.0f)
#pragma unroll
        for (int ks = 0; ks < DP / F::K; ++ks) qf[ks] = negated(qf[ks]);
    const int per_block = s.block / 32;
    const int share = (found + plan.splits - 1) / plan.splits;
    const int first = min(found, split * share), stop = min(found, (split + 1) * share);
    // scores in units of log 2 where there is no bias; with one in its own units, so
    // that a bias of the type's lowest value stays finite
    const float c = fmaxf(fabsf(BIAS ? s.scale : s.scale * LOG2E), 1e-38f);
    const float unit = BIAS ? LOG2E : 1.0f;
    const int sure = s.causal ? min(kl, (int)i0 + kl - ql + 1) : kl;   // keys that every row may read
    const Piece<DP> kp(k, b, g, lane, s.dim, kl), vp(v, b, g, lane, s.dim, kl);

    // turn 0: all queries together.  Zeros of P times infinities of V make NaN
    // in rows that do not read them: if anything in the result is not finite, each
    // query is done again by itself with the values that it does not read cleared.
    for (int turn = 0; turn <= nq; ++turn) {
        const uint32_t only = turn == 0 ? ~0u : 1u << (turn - 1);
        const int vend = turn == 0 || !s.causal ? kl : min(kl, (int)i0 + turn - 1 + kl - ql + 1);
        typename F::Acc o[DP / ROWS];
        float top = -INFINITY, sum = 0.0f;
#pragma unroll
        for (int t = 0; t < DP / ROWS; ++t) o[t] = typename F::Acc{};
        s16x8 kr[VL], vr[VL];
        Walk<W> at(first * per_block + wave, per_block);
        auto skip = [&]() {   // to the next piece that anyone here reads
            while (turn > 0 && at.step < stop && !(masks[at.step] & only)) at.on();
        };
        skip();
        int j0 = 0;
        uint32_t mask = 0;
        if (at.step < stop) {
            j0 = __builtin_amdgcn_readfirstlane(ids[at.step]) * s.block + at.part * 32;
            mask = __builtin_amdgcn_readfirstlane(masks[at.step]) & only;
            kp.load(kr, j0, kl);
            vp.load(vr, j0, vend);
        }
        while (at.step < stop) {
            at.on();
            skip();
            const bool more = at.step < stop;
            const int id = more ? ids[at.step] : 0;
            const uint32_t chose = more ? masks[at.step] : 0;
            tile.fill(kr, KT);
            float y[N];
            __builtin_amdgcn_s_setprio(1);   // the SIMD's other wave has its turn between the products
            scores<T, DP, ROWS, true>(tile, KT, qf, y);
            __builtin_amdgcn_s_setprio(0);
            tile.fill(vr, VT);
            const int jn = __builtin_amdgcn_readfirstlane(id) * s.block + at.part * 32;
            const uint32_t maskn = __builtin_amdgcn_readfirstlane(chose) & only;
            if (more) {
                kp.load(kr, jn, kl);
                vp.load(vr, jn, vend);
            }
            const bool sel = mask >> row.query & 1u;
            if (BIAS) {
#pragma unroll
                for (int n = 0; n < N; n += 4) {
                    uint32_t bucket;
                    if (ROWS == 16) bucket = four_buckets(j0 + row.key(n) + 4 * row.part - row.pos, edges, s.num_buckets);
                    else __builtin_memcpy(&bucket, s.map + ((int64_t)j0 + row.key(n) + 4 * row.part - row.pos + s.k_len - 1), 4);
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        y[n + e] = __builtin_fmaf(y[n + e], c, table[(bucket >> (8 * e) & 255) * plan.span + row.head - h0]);
                }
            }
            if (j0 + 32 > sure) {
                const int lim = row.end - j0 - 4 * row.part;
#pragma unroll
                for (int e = 0; e < N; ++e) y[e] = row.key(e) < lim ? y[e] : -INFINITY;
            }
            float big = fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3]));
#pragma unroll
            for (int n = 4; n < N; n += 4) big = fmaxf(big, fmaxf(fmaxf(y[n], y[n + 1]), fmaxf(y[n + 2], y[n + 3])));
            big = row_max<F::PARTS>(big);
            if (!BIAS) big *= c;
            big = sel ? big : -INFINITY;
            // the maximum is moved only where it grew by so much that exponentials would
            // get large: that is the first piece and hardly ever another
            if (__any(big > top + SLACK<T> / unit)) {
                const float now = fmaxf(top, big);
                const float f = __builtin_amdgcn_exp2f((top - (now == -INFINITY ? 0.0f : now)) * unit);
                sum *= f;
#pragma unroll
                for (int t = 0; t < DP / ROWS; ++t) o[t] *= f;
                top = now;
            }
            // a row that did not choose the block: exp(x - inf) = 0
            const float shift = !sel ? INFINITY : (top == -INFINITY ? 0.0f : top) - (BIAS ? 0.0f : RAISE<T>);
#pragma unroll
            for (int e = 0; e < N; ++e)
                y[e] = __builtin_amdgcn_exp2f(BIAS ? __builtin_fmaf(y[e] - shift, LOG2E, RAISE<T>) : __builtin_fmaf(y[e], c, -shift));
            // the piece's sum first: beside the first key's 1 single terms of 2^-25 would be lost, 2^16 of them 0.2 %
            float few[N / 4];
#pragma unroll
            for (int n = 0; n < N; n += 4) few[n / 4] = (y[n] + y[n + 1]) + (y[n + 2] + y[n + 3]);
#pragma unroll
            for (int n = 1; n < N / 4; n *= 2)
#pragma unroll
                for (int e = 0; e < N / 4; e += 2 * n) few[e] += few[e + n];
            sum += few[0];
            __builtin_amdgcn_s_setprio(1);
            products<T, DP, ROWS>(tile, VT, y, o);
            __builtin_amdgcn_s_setprio(0);
            j0 = jn;
            mask = maskn;
        }
        // the waves meet
        const int r0 = lane % ROWS;
        sum = row_sum<F::PARTS>(sum) * LOWER<T>;
        if (row.part == 0) {
            stat[(wave * ROWS + r0) * 2] = top;
            stat[(wave * ROWS + r0) * 2 + 1] = sum;
        }
        if (tid == 0) scratch[1] = 0;
        __syncthreads();
        {
            float all = -INFINITY;
            for (int n = 0; n < W; ++n) all = fmaxf(all, stat[(n * ROWS + r0) * 2]);
            const float f = top == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((top - all) * unit) * LOWER<T>;
            const bool none = top == -INFINITY && sum == sum;   // a wave that read nothing for a row adds nothing
#pragma unroll
            for (int t = 0; t < DP / ROWS; ++t)
#pragma unroll
                for (int n = 0; n < (int)(sizeof(typename F::Acc) / 4); n += 4) {
                    f32x4 z;
#pragma unroll
                    for (int e = 0; e < 4; ++e) z[e] = none ? 0.0f : o[t][n + e] * f;
                    *reinterpret_cast<f32x4 *>(sums + (wave * ROWS + r0) * (DP + 4) + ROWS * t + row.key(n) + 4 * row.part) = z;
                }
        }
        __syncthreads();
        bool fine = true;
        for (int e = tid; e < ROWS * CH; e += 64 * W) {
            const int r = e / CH, ch = e % CH;
            if (r >= rows || ch * 8 >= s.dim) continue;
            const int rq = plan.per_span(r);
            if (!(only >> rq & 1u)) continue;
            float all = -INFINITY, l = 0.0f, y[8] = {};
            for (int n = 0; n < W; ++n) all = fmaxf(all, stat[(n * ROWS + r) * 2]);
            for (int n = 0; n < W; ++n) {
                const float m = stat[(n * ROWS + r) * 2], x = stat[(n * ROWS + r) * 2 + 1];
                if (m != -INFINITY || x != x) l += x * __builtin_amdgcn_exp2f((m - all) * unit);
#pragma unroll
                for (int d = 0; d < 8; ++d) y[d] += sums[(n * ROWS + r) * (DP + 4) + ch * 8 + d];
            }
            if (plan.splits > 1) {
                const int64_t at = (tile_id * plan.splits + split) * ROWS + r;
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
                const int64_t h = (int64_t)g * s.group + h0 + r - rq * plan.span;
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

// Joins the splits of a tile: one wave for each row, a lane for each split's figures
// and then for two channels.
template <class T>
__global__ __launch_bounds__(64) void k_attend_join(AttnShape s, RowPlan plan, int32_t dp, int32_t tile_rows, float unit,
                                                    SideOut out, float *__restrict__ lse) {
    __shared__ float weight[64];
    const uint32_t tile_id = blockIdx.x / (uint32_t)(plan.nq * plan.span), head = tile_id / (uint32_t)plan.tiles;
    const uint32_t tile_no = tile_id - head * plan.tiles, at_query = tile_no / (uint32_t)plan.parts;
    const int r = blockIdx.x - tile_id * (plan.nq * plan.span), rq = plan.per_span(r);
    const int64_t i = (int64_t)at_query * plan.nq + rq;
    const int hh = (int)(tile_no - at_query * plan.parts) * plan.span + r - rq * plan.span;
    const int b = head / (uint32_t)s.k_heads, g = head - b * s.k_heads, lane = threadIdx.x;
    const int64_t first = (int64_t)tile_id * plan.splits * tile_rows + r;   // splits: at most 64
    const bool on = lane < plan.splits;
    const float m = on ? plan.stat[(first + (int64_t)lane * tile_rows) * 2] : -INFINITY;
    const float x = on ? plan.stat[(first + (int64_t)lane * tile_rows) * 2 + 1] : 0.0f;
    float y[2] = {};
    const float *from = plan.part + first * dp + 2 * lane;
    const int64_t step = (int64_t)tile_rows * dp;
    float all = m;
    for (int d = 32; d; d >>= 1) all = fmaxf(all, __shfl_xor(all, d));
    // a split that read nothing for the row weighs nothing; NaN goes on
    const float f = m == -INFINITY && x == x ? 0.0f : __builtin_amdgcn_exp2f((m - all) * unit);
    float l = x * f;
    for (int d = 32; d; d >>= 1) l += __shfl_xor(l, d);
    weight[lane] = f;
    __syncthreads();
    if (i >= s.ql(b) || hh >= s.group) return;
    if (2 * lane < s.dim)
        for (int n0 = 0; n0 < plan.splits; n0 += 8) {
            float z[8][2];
#pragma unroll
            for (int n = 0; n < 8; ++n) {
                const float *at = from + min(n0 + n, plan.splits - 1) * step;
                z[n][0] = at[0];
                z[n][1] = at[1];
            }
#pragma unroll
            for (int n = 0; n < 8; ++n)
                if (n0 + n < plan.splits && weight[n0 + n] != 0.0f) {
                    y[0] += z[n][0] * weight[n0 + n];
                    y[1] += z[n][1] * weight[n0 + n];
                }
        }
    const int64_t h = (int64_t)g * s.group + hh;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    if (2 * lane < s.dim) {
        uint16_t *to = out.at(b, i, h) + 2 * lane;
        *reinterpret_cast<uint32_t *>(to) = (uint32_t)T::down(y[0] * inv) | (uint32_t)T::down(y[1] * inv) << 16;
    }
    if (lse && lane == 0)
        lse[((int64_t)b * s.q_heads + h) * s.q_len + i] = l == 0.0f ? -INFINITY : (unit == 1.0f ? all * LN2 : all) + __builtin_amdgcn_logf(l) * LN2;
}

}  // namespace dev
}  // namespace ias
