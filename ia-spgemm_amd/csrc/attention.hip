// attention.hip — block-sparse attention: entry points, argument checks and
// launches (ias_block_* of include/ias.h).  The reference has no counterpart.
#include "ias.h"
#include "ias_internal.hpp"
#include "attention_kernels.hpp"
#include "attention_bwd.hpp"
#include "attention_select.hpp"

#include <hip/hip_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>

namespace ias {
namespace {

ias_status check_attention(const ias_attention *a, bool pattern) {
    if (!a) REFUSE(IAS_ERROR_INVALID_ARGUMENT, "no ias_attention");
    if (a->dtype != IAS_DTYPE_BF16 && a->dtype != IAS_DTYPE_F16)
        REFUSE(IAS_ERROR_UNSUPPORTED, "dtype %d: bf16 and f16 are supported", a->dtype);
    if (a->device < 0) REFUSE(IAS_ERROR_INVALID_ARGUMENT, "device %d", a->device);
    if (a->batch < 0 || a->q_len < 0 || a->k_len < 0 || a->batch > INT32_MAX)
        REFUSE(IAS_ERROR_INVALID_ARGUMENT, "batch %lld, q_len %lld, k_len %lld", (long long)a->batch,
               (long long)a->q_len, (long long)a->k_len);
    if (a->q_heads < 1 || a->k_heads < 1 || a->q_heads % a->k_heads)
        REFUSE(IAS_ERROR_DIMENSION_MISMATCH, "q_heads %d is not a multiple of k_heads %d", a->q_heads, a->k_heads);
    if (a->q_heads / a->k_heads > 64)
        REFUSE(IAS_ERROR_UNSUPPORTED, "%d query heads for a key head: at most 64", a->q_heads / a->k_heads);
    if (a->head_dim < 8 || a->head_dim > 128 || a->head_dim % 8)
        REFUSE(IAS_ERROR_UNSUPPORTED, "head_dim %d: a multiple of 8 up to 128", a->head_dim);
    if (a->block < 64 || a->block > 1024 || a->block % 64)
        REFUSE(IAS_ERROR_UNSUPPORTED, "block %d: a multiple of 64 up to 1024", a->block);
    if (pattern && (a->keep < 1 || a->keep > 256)) REFUSE(IAS_ERROR_UNSUPPORTED, "keep %d: 1 to 256", a->keep);
    if (a->k_len > 16384ll * a->block)   // and not by ceil_div, which passes 64 bits at the largest lengths
        REFUSE(IAS_ERROR_UNSUPPORTED, "k_len %lld: at most 16384 blocks of %d", (long long)a->k_len, a->block);
    if (a->q_len > (1 << 24)) REFUSE(IAS_ERROR_UNSUPPORTED, "q_len %lld: at most 2^24", (long long)a->q_len);
    if (!std::isfinite(a->scale)) REFUSE(IAS_ERROR_INVALID_ARGUMENT, "scale is not finite");
    if (a->table) {
        if (a->num_buckets < 1 || a->num_buckets > 64)
            REFUSE(IAS_ERROR_UNSUPPORTED, "%d buckets: 1 to 64", a->num_buckets);
        if (a->num_buckets > 1 && !a->edges) REFUSE(IAS_ERROR_INVALID_ARGUMENT, "table without edges");
    }
    // workgroups of a launch and the products the kernels form of these
    if (a->batch * (int64_t)a->q_heads > INT32_MAX / std::max<int64_t>(1, a->q_len) ||
        a->batch * (int64_t)a->k_heads > INT32_MAX / std::max<int64_t>(1, a->k_len))
        REFUSE(IAS_ERROR_OVERFLOW, "batch x heads x length beyond 2^31 rows");
    return IAS_SUCCESS;
}

ias_status check_heads(const ias_heads *h, const char *name, int64_t batch, int64_t n, int64_t heads) {
    if (!h) REFUSE(IAS_ERROR_INVALID_ARGUMENT, "no %s", name);
    if (batch == 0 || n == 0) return IAS_SUCCESS;
    if (!h->data) REFUSE(IAS_ERROR_INVALID_ARGUMENT, "%s: no data", name);
    if (((uintptr_t)h->data & 15) || (batch > 1 && h->batch % 8) || (n > 1 && h->token % 8) || (heads > 1 && h->head % 8))
        REFUSE(IAS_ERROR_UNSUPPORTED, "%s: data has to be 16-byte aligned and its strides multiples of 8", name);
    if (n > 1 && (h->token < 0 || h->token > (1 << 24)))   // 32 rows by a 32-bit offset
        REFUSE(IAS_ERROR_UNSUPPORTED, "%s: token stride %lld: 0 to 2^24", name, (long long)h->token);
    return IAS_SUCCESS;
}

// An output's rows may not lie over each other (an expanded tensor's do): some order of its
// axes has each stride at least as long as all of the axes within.
ias_status check_apart(const ias_heads *h, const char *name, int64_t batch, int64_t n, int64_t heads, int32_t dim) {
    if (batch == 0 || n == 0) return IAS_SUCCESS;
    struct { int64_t size, stride; } axis[3] = {{batch, h->batch}, {n, h->token}, {heads, h->head}};
    std::sort(axis, axis + 3, [](const auto &x, const auto &y) { return std::abs((double)x.stride) < std::abs((double)y.stride); });
    double within = dim;   // elements from the first to the last of the axes so far
    for (const auto &x : axis) {
        if (x.size <= 1) continue;
        if (std::abs((double)x.stride) < within)
            REFUSE(IAS_ERROR_INVALID_ARGUMENT, "%s: rows of an output that lie over each other (strides %lld, %lld, %lld)", name, (long long)h->batch, (long long)h->token, (long long)h->head);
        within += std::abs((double)x.stride) * (double)(x.size - 1);
    }
    return IAS_SUCCESS;
}

dev::AttnShape shape_of(const ias_attention *a) {
    dev::AttnShape s{};
    s.q_len = a->q_len; s.k_len = a->k_len;
    s.batch = (int32_t)a->batch; s.q_heads = a->q_heads; s.k_heads = a->k_heads;
    s.group = a->q_heads / a->k_heads;
    s.inverse = (uint32_t)ceil_div(65536, s.group);
    s.inverse_keep = a->keep > 1 ? (uint32_t)ceil_div(1ll << 32, a->keep) : 0;
    s.dim = a->head_dim; s.block = a->block; s.keep = a->keep; s.causal = a->causal != 0;
    s.clear = a->clear != 0;
    s.nblocks = (int32_t)ceil_div(a->k_len, a->block);
    s.scale = a->scale;
    s.q_lens = a->q_lens; s.k_lens = a->k_lens;
    s.table = static_cast<const uint16_t *>(a->table);
    s.edges = a->edges;
    s.num_buckets = a->table ? a->num_buckets : 0;
    return s;
}
dev::Side side(const ias_heads *h) { return {static_cast<const uint16_t *>(h->data), h->batch, h->token, h->head}; }
dev::SideOut side_out(const ias_heads *h) { return {static_cast<uint16_t *>(h->data), h->batch, h->token, h->head}; }

// Parts of a workspace, each on a boundary of 256 bytes.
struct Space {
    int64_t used = 0;
    char *base = nullptr;
    template <class T> T *part(int64_t count) {
        T *p = base ? reinterpret_cast<T *>(base + used) : nullptr;
        used += (count * (int64_t)sizeof(T) + 255) / 256 * 256;
        return p;
    }
};

// every distance from a position to a key, the last block's end included
int64_t map_size(const ias_attention *a) { return 2 * a->k_len + a->q_len + a->block + 8; }

ias_status bucket_map(const ias_attention *a, dev::AttnShape &s, uint8_t *map, int32_t *count = nullptr, int64_t entries = 0) {
    const int64_t n = map_size(a);
    dev::k_bucket_map<<<dim3((unsigned)ceil_div(n, 256)), 256, 0, (hipStream_t)a->stream>>>(a->k_len, n, a->num_buckets, a->edges, map, count, entries);
    s.map = map;
    return launched();
}

// How the walks share out the rows.  16 rows where all fit (single tokens), else 32, so
// that more queries share a walk and a fragment of K and V serves more rows.
//
// 16 rows: 8 waves share a walk, and only where it has more than 64 pieces of 32 keys
// and the workgroups are fewer than CUs is it split, since a split costs a second
// launch (one user, 16 blocks of 64 keys: 38 us a step with 8 splits of 4 waves, 35
// without; 16 users, 32 blocks: 57 and 55).
//
// 32 rows: few are split until about every CU has two workgroups, two blocks of keys
// each at least.  The chip holds two waves a SIMD, 2048, of these kernels: a workgroup
// has as many waves as it takes to fill it, since a walk of one wave has no end where
// waves wait for each other (8192 tokens, 8192 tiles, one block of keys each: 148, 90
// and 65 us with 4, 2 and 1 waves; 16 blocks 406, 343, 324 us; 2048 tiles with their
// gradients: 417, 342, 364 us).
struct Rows {
    int rows, dp, waves;
    dev::RowPlan plan{};
    int64_t tiles, part, stat;   // all tiles; floats of the splits' results
    explicit Rows(const ias_attention *a) {
        const int group = a->q_heads / a->k_heads;
        rows = a->q_len * group <= 16 ? 16 : 32;
        dp = a->head_dim > 64 ? 128 : 64;
        plan.span = std::min(group, rows);
        plan.parts = (int32_t)ceil_div(group, plan.span);
        plan.inverse = (uint32_t)ceil_div(65536, plan.span);
        plan.nq = plan.parts > 1 ? 1 : (int32_t)std::max<int64_t>(1, std::min<int64_t>(rows / group, a->q_len));
        // the union's list takes 8 bytes of LDS an entry
        if (std::min<int64_t>((int64_t)plan.nq * a->keep, ceil_div(a->k_len, a->block)) > 2048) plan.nq = std::max(1, 2048 / a->keep);
        plan.tiles = (int32_t)ceil_div(a->q_len, plan.nq) * plan.parts;
        plan.most = (int32_t)std::max<int64_t>(1, std::min<int64_t>((int64_t)plan.nq * a->keep, ceil_div(a->k_len, a->block)));
        tiles = a->batch * a->k_heads * plan.tiles;
        const int64_t pieces = (int64_t)plan.most * (a->block / 32), few = std::max<int64_t>(1, tiles);
        if (rows == 16) {
            waves = 8;
            plan.splits = (int32_t)std::max<int64_t>(1, std::min<int64_t>({ceil_div(256, few), ceil_div(pieces, 64), 64}));
        } else {
            plan.splits = (int32_t)std::max<int64_t>(1, std::min<int64_t>({ceil_div(512, few), ceil_div(plan.most, 2), 64}));
            waves = plan.splits > 1 || tiles < 512 ? 4 : tiles < 4096 ? 2 : 1;
        }
        part = plan.splits > 1 ? tiles * plan.splits * rows * dp : 0;
        stat = plan.splits > 1 ? tiles * plan.splits * rows * 2 : 0;
    }
};

struct Forward {
    uint8_t *map;
    Rows rows;
    explicit Forward(const ias_attention *a, Space &w) : rows(a) {
        map = a->table ? w.part<uint8_t>(map_size(a)) : nullptr;
        rows.plan.part = rows.part ? w.part<float>(rows.part) : nullptr;
        rows.plan.stat = rows.stat ? w.part<float>(rows.stat) : nullptr;
    }
};
// The backward pass: k_grad_q's rows as the forward's, and the items of k_grad_kv: 256 to 1024 rows each, about
// 1024 items where there are few rows.  An item of a block that many queries chose
// writes 64 KB of f32 results, so small ones cost more to join than they even out
// (8192 tokens, 16/2 heads of 128, both kernels: 421, 382 and 415 us with 768, 1024
// and 2048 rows).  Large calls take longer items, so that all results stay within 1 GiB,
// up to 8192 queries (their list is in LDS): there are enough of them then (4 x 8192 tokens,
// 32/8 heads of 128, 32 blocks a query: 4096 rows, a training step 11.1 ms and a peak of 2.3
// GiB; with 1024 rows 11.3 ms and 5.3 GiB).
struct Backward {
    uint8_t *map;
    Rows rows;
    dev::GradPlan q{};
    dev::KeyPlan k{};
    uint32_t *bits;
    int32_t *count, *first, *slot;
    int64_t items;      // at most
    explicit Backward(const ias_attention *a, Space &w) : rows(a) {
        const int64_t group = a->q_heads / a->k_heads, bh = a->batch * a->k_heads, nblocks = ceil_div(a->k_len, a->block);
        q.nq = rows.plan.nq; q.span = rows.plan.span; q.parts = rows.plan.parts; q.inverse = rows.plan.inverse;
        q.tiles = rows.plan.tiles; q.most = rows.plan.most;
        map = a->table ? w.part<uint8_t>(map_size(a)) : nullptr;
        q.delta = w.part<float>(a->batch * a->q_heads * a->q_len);
        q.shift = a->table ? w.part<float>(a->batch * a->q_heads * a->q_len) : nullptr;
        q.corr = a->table ? w.part<float>(a->batch * a->q_heads * a->q_len) : nullptr;
        q.sums = a->table ? w.part<float>(bh * q.tiles * q.span * a->num_buckets) : nullptr;
        k.nw = (int32_t)ceil_div(a->q_len, 32);
        k.subs = a->block / 64;
        k.entries = bh * nblocks;
        const int64_t chosen = bh * a->q_len * std::min<int64_t>(a->keep, nblocks);   // entries of the pattern, at most
        // a block with two items or more has over `per` queries: at most 2 chosen / per results to join
        const int64_t result = (int64_t)k.subs * 2 * 64 * rows.dp * 4;
        k.per = (int32_t)(std::min<int64_t>(1024, std::max<int64_t>(256, chosen * group / 1024)) / group);
        k.per = (int32_t)std::min<int64_t>(8192, std::max<int64_t>(k.per, ceil_div(2 * chosen * result, 1ll << 30)));
        items = k.entries + chosen / k.per;
        k.bits = bits = w.part<uint32_t>(k.entries * k.nw);
        k.count = count = w.part<int32_t>(k.entries);
        k.first = first = w.part<int32_t>(k.entries + 1);
        k.slot = slot = w.part<int32_t>(k.entries + 1);
        k.delta = q.delta; k.shift = q.shift; k.corr = q.corr;
        k.part = w.part<float>(2 * chosen / k.per * result / 4);
    }
};

ias_status check_workspace(const void *p, int64_t have, int64_t need) {
    if (need == 0) return IAS_SUCCESS;
    if (!p || have < need)
        REFUSE(IAS_ERROR_INSUFFICIENT_CAPACITY, "workspace of %lld bytes: %lld are needed", (long long)(p ? have : 0), (long long)need);
    if ((uintptr_t)p & 255) REFUSE(IAS_ERROR_INVALID_ARGUMENT, "the workspace has to be aligned to 256 bytes");
    return IAS_SUCCESS;
}

// A launch with `lds` bytes of dynamic LDS; more than 64 KB are asked for once a device.
template <auto kernel, class... P>
ias_status launch(int device, int64_t grid, int threads, size_t lds, void *stream, P... args) {
    IAS_TRY(check_grid(grid, threads));
    static std::atomic<bool> asked[64];
    if (lds > 64 * 1024 && !(device < 64 && asked[device].load(std::memory_order_relaxed))) {
        HIPC(hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024));
        if (device < 64) asked[device].store(true, std::memory_order_relaxed);
    }
    kernel<<<dim3((unsigned)grid), threads, lds, (hipStream_t)stream>>>(args...);
    return launched();
}

// Workgroups for tile_of: 8 dies, each with its share of a head's tiles or of all.
int64_t tile_grid(int64_t heads, int64_t each) {
    return 8 * (heads < 8 && 8 % heads == 0 ? ceil_div(each, 8 / heads) : ceil_div(heads * each, 8));
}

// Grids of the calls with more than one launch, which are all looked at before the first.
int64_t attend_grid(const ias_attention *a, const Rows &r) { return tile_grid(a->batch * a->k_heads, (int64_t)r.plan.tiles * r.plan.splits); }
int64_t join_grid(const Rows &r) { return r.plan.splits > 1 ? r.tiles * r.plan.nq * r.plan.span : 0; }
int64_t invert_grid(const ias_attention *a, const Backward &w) { return a->batch * a->k_heads * w.k.nw; }
int64_t grad_kv_grid(const Backward &w) { return ceil_div(w.items * w.k.subs, 8) * 8; }
int64_t grad_kv_join_grid(const ias_attention *a, const Backward &w, bool table) {
    return w.k.entries * w.k.subs * 4 + (table ? (int64_t)a->q_heads * a->num_buckets : 0);
}
int grad_q_waves(const Rows &r) { return r.rows == 16 ? 4 : r.waves; }

ias_status check_grids(const ias_attention *a, const Forward &f) {
    IAS_TRY(check_grid(attend_grid(a, f.rows), 64 * f.rows.waves));
    return check_grid(join_grid(f.rows), 64);
}
ias_status check_grids(const ias_attention *a, const Backward &w, bool table) {
    IAS_TRY(check_grid(tile_grid(a->batch * a->k_heads, w.q.tiles), 64 * grad_q_waves(w.rows)));
    IAS_TRY(check_grid(invert_grid(a, w), 256));
    IAS_TRY(check_grid(grad_kv_grid(w), 256));
    return check_grid(grad_kv_join_grid(a, w, table), 256);
}

template <class T, int DP, int MT>
ias_status select_rows(const ias_attention *a, const dev::AttnShape &s, const dev::SelectPlan &p, int threads, const ias_heads *q,
                       const void *summary, int32_t *blocks) {
    const int64_t grid = tile_grid(a->batch * a->k_heads, p.tiles);
    return launch<dev::k_block_select<T, DP, MT>>(a->device, grid, threads, dev::select_lds(p.nq, p.stride, threads / 64), a->stream, s, p, side(q),
                  static_cast<const uint16_t *>(summary), blocks);
}

// 32 rows to a workgroup (64 only for more than 32 heads), so that a summary is read for
// several queries and four waves pick a few each (4096 tokens: 41.2, 38.7 and 40.8 us with
// 64, 32 and 16 rows), while the queries' keys take at most 64 KB of LDS.  Where there are few workgroups and 16
// rows are enough (single tokens), more waves share the blocks.
template <class T, int DP>
ias_status select(const ias_attention *a, const ias_heads *q, const void *summary, int32_t first, int32_t local, int32_t *blocks) {
    const dev::AttnShape s = shape_of(a);
    dev::SelectPlan p{};
    p.first = first; p.local = local;
    p.stride = std::max(1, s.nblocks);
    p.nq = (int32_t)std::min<int64_t>({std::max(1, 32 / s.group), a->q_len, std::max(1, 16384 / p.stride)});
    p.tiles = (int32_t)ceil_div(a->q_len, p.nq);
    const int rows = p.nq * s.group;
    if (rows <= 16) {
        const int64_t few = a->batch * a->k_heads * p.tiles < 512;
        const int threads = few ? (int)std::min<int64_t>(1024, std::max<int64_t>(256, ceil_div(p.stride, 32) * 64)) : 256;
        return select_rows<T, DP, 1>(a, s, p, threads, q, summary, blocks);
    }
    if (rows <= 32) return select_rows<T, DP, 2>(a, s, p, 256, q, summary, blocks);
    return select_rows<T, DP, 4>(a, s, p, 256, q, summary, blocks);
}

template <class T, int DP, int ROWS, int W>
ias_status attend_waves(const ias_attention *a, const dev::AttnShape &s, const ias_heads *q, const ias_heads *k,
                       const ias_heads *v, const int32_t *blocks, const ias_heads *out, float *lse, const Rows &r) {
    const int64_t grid = attend_grid(a, r);
    const size_t lds = dev::attend_lds(DP, ROWS, W, s.nblocks, r.plan.most, s.num_buckets * (r.plan.span + 1));
    if (a->table)
        IAS_TRY((launch<dev::k_attend<T, DP, ROWS, W, true>>(a->device, grid, 64 * W, lds, a->stream, s, r.plan, side(q), side(k), side(v), blocks, side_out(out), lse)));
    else
        IAS_TRY((launch<dev::k_attend<T, DP, ROWS, W, false>>(a->device, grid, 64 * W, lds, a->stream, s, r.plan, side(q), side(k), side(v), blocks, side_out(out), lse)));
    if (r.plan.splits > 1)
        IAS_TRY((launch<dev::k_attend_join<T>>(a->device, join_grid(r), 64, 0, a->stream, s, r.plan, DP, ROWS,
                       a->table ? dev::LOG2E : 1.0f, side_out(out), lse)));
    return IAS_SUCCESS;
}

template <class T, int DP, int ROWS>
ias_status attend_rows(const ias_attention *a, const dev::AttnShape &s, const ias_heads *q, const ias_heads *k,
                       const ias_heads *v, const int32_t *blocks, const ias_heads *out, float *lse, const Rows &r) {
    if constexpr (ROWS == 16) return attend_waves<T, DP, ROWS, 8>(a, s, q, k, v, blocks, out, lse, r);
    else
        return r.waves == 4   ? attend_waves<T, DP, ROWS, 4>(a, s, q, k, v, blocks, out, lse, r)
               : r.waves == 2 ? attend_waves<T, DP, ROWS, 2>(a, s, q, k, v, blocks, out, lse, r)
                              : attend_waves<T, DP, ROWS, 1>(a, s, q, k, v, blocks, out, lse, r);
}

template <class T>
ias_status attend(const ias_attention *a, const ias_heads *q, const ias_heads *k, const ias_heads *v,
                  const int32_t *blocks, const ias_heads *out, float *lse, const Forward &f) {
    dev::AttnShape s = shape_of(a);
    const Rows &r = f.rows;
    if (a->table && r.rows == 32) IAS_TRY(bucket_map(a, s, f.map));
    if (r.dp == 64)
        return r.rows == 16 ? attend_rows<T, 64, 16>(a, s, q, k, v, blocks, out, lse, r) : attend_rows<T, 64, 32>(a, s, q, k, v, blocks, out, lse, r);
    return r.rows == 16 ? attend_rows<T, 128, 16>(a, s, q, k, v, blocks, out, lse, r) : attend_rows<T, 128, 32>(a, s, q, k, v, blocks, out, lse, r);
}

template <class T, int DP, int ROWS, int W>
ias_status grad_waves(const ias_attention *a, const dev::AttnShape &s, const dev::GradPlan &p, const ias_heads *dout, const ias_heads *q,
                      const ias_heads *k, const ias_heads *v, const ias_heads *out, const float *lse, const int32_t *blocks,
                      const ias_heads *dq) {
    const int64_t grid = tile_grid(a->batch * a->k_heads, p.tiles);
    const int32_t area = dev::grad_q_area(DP, ROWS, W, s.num_buckets, p.sums);
    const size_t lds = dev::grad_q_lds(area, s.nblocks, p.most, p.span, s.num_buckets);
    if (a->table)
        return launch<dev::k_grad_q<T, DP, ROWS, W, true>>(a->device, grid, 64 * W, lds, a->stream, s, p, area, side(dout), side(q), side(k), side(v), side(out), lse,
                      blocks, side_out(dq));
    return launch<dev::k_grad_q<T, DP, ROWS, W, false>>(a->device, grid, 64 * W, lds, a->stream, s, p, area, side(dout), side(q), side(k), side(v), side(out), lse, blocks,
                  side_out(dq));
}

template <class T, int DP, int ROWS>
ias_status grad_rows(const ias_attention *a, const dev::AttnShape &s, const dev::GradPlan &p, int waves, const ias_heads *dout,
                     const ias_heads *q, const ias_heads *k, const ias_heads *v, const ias_heads *out, const float *lse,
                     const int32_t *blocks, const ias_heads *dq) {
    if constexpr (ROWS == 16) return grad_waves<T, DP, ROWS, 4>(a, s, p, dout, q, k, v, out, lse, blocks, dq);
    else
        return waves == 4   ? grad_waves<T, DP, ROWS, 4>(a, s, p, dout, q, k, v, out, lse, blocks, dq)
               : waves == 2 ? grad_waves<T, DP, ROWS, 2>(a, s, p, dout, q, k, v, out, lse, blocks, dq)
                            : grad_waves<T, DP, ROWS, 1>(a, s, p, dout, q, k, v, out, lse, blocks, dq);
}

template <class T, int DP>
ias_status grad_all(const ias_attention *a, const ias_heads *dout, const ias_heads *q, const ias_heads *k, const ias_heads *v,
                    const ias_heads *out, const float *lse, const int32_t *blocks, const ias_heads *dq, const ias_heads *dk,
                    const ias_heads *dv, void *dtable, const Backward &w) {
    dev::AttnShape s = shape_of(a);
    dev::GradPlan p = w.q;
    if (!dtable) p.sums = nullptr;
    if (a->table) IAS_TRY(bucket_map(a, s, w.map, w.count, w.k.entries));   // clears the counts too
    const int64_t bh = a->batch * a->k_heads;
    if (bh > 0 && a->q_len > 0) {
        if (w.rows.rows == 16) IAS_TRY((grad_rows<T, DP, 16>(a, s, p, w.rows.waves, dout, q, k, v, out, lse, blocks, dq)));
        else IAS_TRY((grad_rows<T, DP, 32>(a, s, p, w.rows.waves, dout, q, k, v, out, lse, blocks, dq)));
    }
    if (w.k.entries > 0) {
        if (!a->table) IAS_TRY((launch<dev::k_clear>(a->device, ceil_div(w.k.entries, 256), 256, 0, a->stream, w.k.entries, w.count)));
        if (a->q_len > 0)
            IAS_TRY((launch<dev::k_invert>(a->device, invert_grid(a, w), 256, 4 * (size_t)s.nblocks, a->stream, s, w.k.nw, blocks, w.bits, w.count)));
        IAS_TRY((launch<dev::k_items>(a->device, 1, 1024, 0, a->stream, w.k.entries, w.k.per, w.count, w.first, w.slot)));
        const size_t lds = 4 * 32 * (size_t)DP * 2 + 2 * dev::FIGURES * 32 * 4 + 4 * (size_t)w.k.per + 32 + 4 * (size_t)s.group * s.num_buckets;
        const int64_t grid = grad_kv_grid(w);
        if (a->q_len > 0) {
            if (a->table)
                IAS_TRY((launch<dev::k_grad_kv<T, DP, true>>(a->device, grid, 256, lds, a->stream, s, w.k, side(dout), side(q), side(k), side(v), lse, side_out(dk), side_out(dv))));
            else
                IAS_TRY((launch<dev::k_grad_kv<T, DP, false>>(a->device, grid, 256, lds, a->stream, s, w.k, side(dout), side(q), side(k), side(v), lse, side_out(dk), side_out(dv))));
        }
        IAS_TRY((launch<dev::k_grad_kv_join<T>>(a->device, grad_kv_join_grid(a, w, dtable), 256, 0, a->stream, s, w.k, DP, side_out(dk), side_out(dv), p,
                       static_cast<uint16_t *>(dtable))));
    } else if (dtable)
        IAS_TRY((launch<dev::k_grad_table<T>>(a->device, (int64_t)a->q_heads * a->num_buckets, 256, 0, a->stream, s, p, static_cast<uint16_t *>(dtable))));
    return IAS_SUCCESS;
}

template <class T>
ias_status gradients(const ias_attention *a, const ias_heads *dout, const ias_heads *q, const ias_heads *k,
                     const ias_heads *v, const ias_heads *out, const float *lse, const int32_t *blocks,
                     const ias_heads *dq, const ias_heads *dk, const ias_heads *dv, void *dtable, const Backward &w) {
    return w.rows.dp == 64 ? grad_all<T, 64>(a, dout, q, k, v, out, lse, blocks, dq, dk, dv, dtable, w)
                           : grad_all<T, 128>(a, dout, q, k, v, out, lse, blocks, dq, dk, dv, dtable, w);
}

}  // namespace
}  // namespace ias

using namespace ias;

extern "C" ias_status ias_block_summary(const ias_attention *a, const ias_heads *k, int64_t fresh, void *summary) {
    IAS_TRY(check_attention(a, false));
    IAS_TRY(check_heads(k, "k", a->batch, a->k_len, a->k_heads));
    if (fresh < 0) REFUSE(IAS_ERROR_INVALID_ARGUMENT, "fresh %lld", (long long)fresh);
    if (a->batch == 0 || a->k_len == 0) return IAS_SUCCESS;
    if (!summary) REFUSE(IAS_ERROR_INVALID_ARGUMENT, "no summary");
    OnDevice on;
    HIPC(on.to(a->device));
    const dev::AttnShape s = shape_of(a);
    const int32_t per = fresh > 0 ? (int32_t)std::min<int64_t>(s.nblocks, (std::min(fresh, a->k_len) + a->block - 2) / a->block + 1) : s.nblocks;
    const int64_t grid = a->batch * a->k_heads * per;
    uint16_t *o = static_cast<uint16_t *>(summary);
    return a->dtype == IAS_DTYPE_BF16 ? launch<dev::k_block_summary<dev::Bf16>>(a->device, grid, 256, 0, a->stream, s, side(k), fresh, per, o)
                                      : launch<dev::k_block_summary<dev::Fp16>>(a->device, grid, 256, 0, a->stream, s, side(k), fresh, per, o);
}

extern "C" ias_status ias_block_select(const ias_attention *a, const ias_heads *q, const void *summary, int32_t first,
                                       int32_t local, int32_t *blocks) {
    IAS_TRY(check_attention(a, true));
    IAS_TRY(check_heads(q, "q", a->batch, a->q_len, a->q_heads));
    if (first < 0 || local < 0 || (int64_t)first + local > a->keep)
        REFUSE(IAS_ERROR_INVALID_ARGUMENT, "first %d + local %d of keep %d", first, local, a->keep);
    if (local > 0 && !a->causal) REFUSE(IAS_ERROR_INVALID_ARGUMENT, "local blocks are those of a causal call");
    if (a->batch == 0 || a->q_len == 0) return IAS_SUCCESS;
    if ((!summary && a->k_len > 0) || !blocks) REFUSE(IAS_ERROR_INVALID_ARGUMENT, "no summary or blocks");
    OnDevice on;
    HIPC(on.to(a->device));
    if (a->head_dim <= 64)
        return a->dtype == IAS_DTYPE_BF16 ? select<dev::Bf16, 64>(a, q, summary, first, local, blocks)
                                          : select<dev::Fp16, 64>(a, q, summary, first, local, blocks);
    return a->dtype == IAS_DTYPE_BF16 ? select<dev::Bf16, 128>(a, q, summary, first, local, blocks)
                                      : select<dev::Fp16, 128>(a, q, summary, first, local, blocks);
}

extern "C" ias_status ias_block_attention_workspace(const ias_attention *a, int64_t *forward, int64_t *backward) {
    IAS_TRY(check_attention(a, true));
    Space f, b;
    (void)Forward(a, f);
    (void)Backward(a, b);
    if (forward) *forward = f.used;
    if (backward) *backward = b.used;
    return IAS_SUCCESS;
}

extern "C" ias_status ias_block_attention(const ias_attention *a, const ias_heads *q, const ias_heads *k,
                                          const ias_heads *v, const int32_t *blocks, const ias_heads *out,
                                          float *lse, void *workspace, int64_t workspace_bytes) {
    IAS_TRY(check_attention(a, true));
    IAS_TRY(check_heads(q, "q", a->batch, a->q_len, a->q_heads));
    IAS_TRY(check_heads(k, "k", a->batch, a->k_len, a->k_heads));
    IAS_TRY(check_heads(v, "v", a->batch, a->k_len, a->k_heads));
    IAS_TRY(check_heads(out, "out", a->batch, a->q_len, a->q_heads));
    if (a->batch == 0 || a->q_len == 0) return IAS_SUCCESS;
    if (!blocks) REFUSE(IAS_ERROR_INVALID_ARGUMENT, "no blocks");
    Space need;
    (void)Forward(a, need);
    IAS_TRY(check_workspace(workspace, workspace_bytes, need.used));
    Space w;
    w.base = static_cast<char *>(workspace);
    const Forward f(a, w);
    IAS_TRY(check_grids(a, f));
    IAS_TRY(check_apart(out, "out", a->batch, a->q_len, a->q_heads, a->head_dim));
    OnDevice on;
    HIPC(on.to(a->device));
    return a->dtype == IAS_DTYPE_BF16 ? attend<dev::Bf16>(a, q, k, v, blocks, out, lse, f)
                                      : attend<dev::Fp16>(a, q, k, v, blocks, out, lse, f);
}

extern "C" ias_status ias_block_attention_grad(const ias_attention *a, const ias_heads *dout, const ias_heads *q,
                                               const ias_heads *k, const ias_heads *v, const ias_heads *out,
                                               const float *lse, const int32_t *blocks, const ias_heads *dq,
                                               const ias_heads *dk, const ias_heads *dv, void *dtable, void *workspace,
                                               int64_t workspace_bytes) {
    IAS_TRY(check_attention(a, true));
    IAS_TRY(check_heads(dout, "dout", a->batch, a->q_len, a->q_heads));
    IAS_TRY(check_heads(q, "q", a->batch, a->q_len, a->q_heads));
    IAS_TRY(check_heads(k, "k", a->batch, a->k_len, a->k_heads));
    IAS_TRY(check_heads(v, "v", a->batch, a->k_len, a->k_heads));
    IAS_TRY(check_heads(out, "out", a->batch, a->q_len, a->q_heads));
    IAS_TRY(check_heads(dq, "dq", a->batch, a->q_len, a->q_heads));
    IAS_TRY(check_heads(dk, "dk", a->batch, a->k_len, a->k_heads));
    IAS_TRY(check_heads(dv, "dv", a->batch, a->k_len, a->k_heads));
    if (dtable && !a->table) REFUSE(IAS_ERROR_INVALID_ARGUMENT, "dtable without a table");
    if (a->batch > 0 && a->q_len > 0 && (!blocks || !lse)) REFUSE(IAS_ERROR_INVALID_ARGUMENT, "no blocks or lse");
    Space need;
    (void)Backward(a, need);
    IAS_TRY(check_workspace(workspace, workspace_bytes, need.used));
    Space w;
    w.base = static_cast<char *>(workspace);
    const Backward f(a, w);
    IAS_TRY(check_grids(a, f, dtable));
    IAS_TRY(check_apart(dq, "dq", a->batch, a->q_len, a->q_heads, a->head_dim));
    IAS_TRY(check_apart(dk, "dk", a->batch, a->k_len, a->k_heads, a->head_dim));
    IAS_TRY(check_apart(dv, "dv", a->batch, a->k_len, a->k_heads, a->head_dim));
    OnDevice on;
    HIPC(on.to(a->device));
    return a->dtype == IAS_DTYPE_BF16 ? gradients<dev::Bf16>(a, dout, q, k, v, out, lse, blocks, dq, dk, dv, dtable, f)
                                      : gradients<dev::Fp16>(a, dout, q, k, v, out, lse, blocks, dq, dk, dv, dtable, f);
}
