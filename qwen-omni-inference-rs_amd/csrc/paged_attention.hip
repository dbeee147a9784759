// paged_attention.hip -- attention over a paged key/value cache, with or
// without a prefix that sequences share (gfx950).
#include <algorithm>
#include <cmath>

#include "paged_attn.h"

namespace lq8 {
namespace {

// The row's pieces together: o = sum 2^(m_c - m) o_c / sum 2^(m_c - m) l_c, a
// wave per (row, head), own pieces first.
constexpr int JOIN_WAVES = 4;
template <typename T, int D>
__global__ __launch_bounds__(64 * JOIN_WAVES) void k_join(AttnArgs a) {
    const int lane = threadIdx.x & 63;
    const int64_t item = (int64_t)blockIdx.x * JOIN_WAVES + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int row = (int)(item / a.heads), head = (int)(item - (int64_t)row * a.heads);
    if (row >= a.batch.rows) return;
    // the row's sequence, and its group
    int seq = row;
    if (a.batch.row_begin) {
        seq = -1;
        for (int s0 = 0; s0 < a.batch.batch && seq < 0; s0 += 64) {
            bool mine = false;
            if (s0 + lane < a.batch.batch) {
                const RowRange r = rows_of(a.batch, s0 + lane);
                mine = row >= r.first && row - r.first < r.count;
            }
            const uint64_t b = __ballot(mine);
            if (b) seq = s0 + __ffsll((unsigned long long)b) - 1;
        }
        if (seq < 0) return;  // behind the last sequence
    }
    int group = -1;
    for (int g0 = 0; g0 < a.prefix.groups && group < 0; g0 += 64) {
        const bool mine = g0 + lane < a.prefix.groups && seq >= a.prefix.seq_begin[g0 + lane] && seq < a.prefix.seq_begin[g0 + lane + 1];
        const uint64_t b = __ballot(mine);
        if (b) group = g0 + __ffsll((unsigned long long)b) - 1;
    }
    const Span s = own_span(a, seq);
    const int sees = s.sees(row - s.first), len = piece_len(s.length, a.own);
    const int own = (sees + len - 1) / len;
    int pre = 0;
    if (group >= 0) {
        const int n = held(a.prefix.lengths[group], a.prefix.max_pages, a.kv.page_shift);
        const int plen = piece_len(n, a.pre);
        pre = (n + plen - 1) / plen;
    }
    const size_t step = (size_t)a.batch.rows * a.heads;
    auto at = [&](int c) { return (size_t)(c < own ? c : a.own.pieces + c - own) * step + item; };
    float m = -__builtin_huge_valf();
    for (int c = lane; c < own + pre; c += 64) m = fmaxf(m, a.ml[at(c)].x);
    for (int d = 32; d > 0; d /= 2) m = fmaxf(m, __shfl_xor(m, d));
    const bool none = m == -__builtin_huge_valf();  // no piece saw anything
    const float mu = fmaxf(m, -FLT_MAX);
    float l = 0.0f, o[D / 64];
#pragma unroll
    for (int k = 0; k < D / 64; k++) o[k] = 0.0f;
#pragma unroll 4
    for (int c = 0; c < own + pre; c++) {
        const size_t k = at(c);
        const float2 ml = a.ml[k];
        const float f = __builtin_amdgcn_exp2f(ml.x - mu);
        l = fmaf(f, ml.y, l);
        const float* y = a.part + k * D + (D / 64) * lane;
#pragma unroll
        for (int e = 0; e < D / 64; e++) o[e] = fmaf(f, y[e], o[e]);
    }
    const float inv = 1.0f / l;
    T* out = (T*)a.out + (size_t)row * a.os + (size_t)head * D + (D / 64) * lane;
#pragma unroll
    for (int e = 0; e < D / 64; e++) {
        const float y = none ? 0.0f : o[e] * inv;
        if constexpr (sizeof(T) == 4) out[e] = y;
        else out[e].bits = __builtin_bit_cast(uint16_t, (__bf16)y);
    }
}

lq8_status launch_join(const AttnArgs& a, bool f32, int dim, hipStream_t s) {
    const dim3 grid((unsigned)(((size_t)a.batch.rows * a.heads + JOIN_WAVES - 1) / JOIN_WAVES)), block(64 * JOIN_WAVES);
    if (f32 && dim == 64) hipLaunchKernelGGL((k_join<float, 64>), grid, block, 0, s, a);
    else if (f32) hipLaunchKernelGGL((k_join<float, 128>), grid, block, 0, s, a);
    else if (dim == 64) hipLaunchKernelGGL((k_join<Bf16, 64>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((k_join<Bf16, 128>), grid, block, 0, s, a);
    LQ8_HIP(hipGetLastError());
    return LQ8_OK;
}

// How a call runs: which kernel takes each part, and its cuts.
struct Plan {
    bool own_few = false, pre_few = false;
    int own_blocks = 1, pre_blocks = 1;
    size_t own_tiles = 0, pre_tiles = 0;  // row tiles over all spans, at most
    size_t slots = 0, scratch = 0;        // of partial results; their bytes
};

// Pieces of a part whose positions are at most `most`, in `groups` workgroups
// a piece.  few: its kernel takes spans one by one, so that a long one among
// short ones needs pieces of its own.
Cut cut_of(size_t most, size_t groups, int cus, bool few, bool f32_pages) {
    Cut c;
    if (few) {
        c.unit = f32_pages ? 64 : 128;  // a tile for each of the four waves
        c.shortest = c.unit;
        const size_t fill = 4 * (size_t)cus / groups, longest = (most + 4095) / 4096, cap = 16384 / groups;
        c.pieces = (int)std::max<size_t>(1, std::max(fill, std::min(longest, cap)));
    } else {
        c.unit = f32_pages ? 32 : 64;
        c.shortest = 256;
        c.pieces = (int)std::max<size_t>(1, 2 * (size_t)cus / groups);
    }
    c.pieces = (int)std::min<size_t>(c.pieces, std::max<size_t>(1, (most + c.shortest - 1) / c.shortest));
    return c;
}

Plan plan_of(AttnArgs* a, PagedTypes types, int dim, int cus) {
    Plan p;
    const size_t G = a->group, kvh = a->kv.kv_heads, rows = a->batch.rows, batch = a->batch.batch;
    const bool f32 = types == PT_F32_F32;
    const size_t own = (size_t)a->batch.max_rows * G, each = (own + TILE_PACKED - 1) / TILE_PACKED;
    p.own_few = own <= FEW_MAX_ROWS;
    p.own_blocks = own <= 16 ? 1 : 2;
    p.own_tiles = p.own_few ? batch : std::min(batch * each, rows * G / TILE_PACKED + std::min(batch, rows));
    a->own = cut_of((size_t)a->batch.max_pages << a->kv.page_shift, p.own_tiles * kvh, cus, p.own_few, f32);
    p.slots = a->own.pieces;
    if (a->prefix.groups) {
        const size_t groups = a->prefix.groups;
        p.pre_few = rows * G <= FEW_MAX_ROWS;
        p.pre_blocks = rows * G <= 16 ? 1 : 2;
        p.pre_tiles = p.pre_few ? groups : rows * G / TILE_PACKED + std::min(groups, rows);
        a->pre = cut_of((size_t)a->prefix.max_pages << a->kv.page_shift, p.pre_tiles * kvh, cus, p.pre_few, f32);
        p.slots += a->pre.pieces;
    }
    if (p.slots > 1) p.scratch = p.slots * rows * a->heads * (dim * sizeof(float) + sizeof(float2));
    return p;
}

lq8_status check_prefix(const lq8_shared_prefix* p, uint32_t page_size, uint32_t batch, PrefixDev* out) {
    if (!p) return fail(LQ8_ERR_INVALID_ARG, "prefix: null description");
    if (p->groups == 0) return LQ8_OK;
    if (p->groups > batch) return fail(LQ8_ERR_SHAPE_MISMATCH, "prefix: more groups than sequences");
    if (!p->seq_begin || !p->lengths || !p->pages) return fail(LQ8_ERR_INVALID_ARG, "prefix: null pointer");
    if (p->max_pages == 0 || (uint64_t)p->max_pages * page_size > (uint64_t)INT32_MAX / 2)
        return fail(LQ8_ERR_SHAPE_MISMATCH, "prefix: max_pages is zero or holds more than 2^30 positions");
    *out = {(int)p->groups, (int)p->max_pages, p->seq_begin, p->lengths, p->pages};
    return LQ8_OK;
}

lq8_status check_attention(const lq8_kv_pages* kv, const lq8_paged_batch* batch, bool has_prefix,
                           const lq8_shared_prefix* prefix, const lq8_attn_rows* rows, AttnArgs* a, PagedTypes* types) {
    lq8_status st;
    if ((st = check_pages(kv, &a->kv)) || (st = check_batch(batch, kv->page_size, &a->batch))) return st;
    if (has_prefix && (st = check_prefix(prefix, kv->page_size, batch->batch, &a->prefix))) return st;
    if (!rows) return fail(LQ8_ERR_INVALID_ARG, "attention: null rows");
    if ((st = check_types(rows->dtype, kv->dtype, types))) return st;
    if (rows->num_heads == 0 || rows->num_heads > MAX_HEADS || rows->num_heads % kv->num_kv_heads)
        return fail(LQ8_ERR_SHAPE_MISMATCH, "attention: num_heads must be a multiple of num_kv_heads, up to 16384");
    // (a launch has at most 2^32 threads, a wave of which joins a row's head)
    if ((uint64_t)batch->rows * rows->num_heads > MAX_ROW_HEADS)
        return fail(LQ8_ERR_SHAPE_MISMATCH, "attention: rows * num_heads above 2^25");
    if (!(rows->scale > 0.0f) || !std::isfinite(rows->scale * 1.4426950408889634f))
        return fail(LQ8_ERR_INVALID_ARG, "attention: scale must be positive and finite");
    const size_t es = rows->dtype == LQ8_DTYPE_F32 ? 4 : 2, width = (size_t)rows->num_heads * kv->head_dim;
    a->qs = rows->q_stride, a->os = rows->out_stride;
    if ((st = check_rows("attention q", rows->q, &a->qs, width, es)) || (st = check_rows("attention out", rows->out, &a->os, width, es)))
        return st;
    if (rows->q == rows->out && a->qs != a->os) return fail(LQ8_ERR_SHAPE_MISMATCH, "attention: in place needs one stride");
    a->q = (const char*)rows->q;
    a->out = (char*)rows->out;
    a->heads = (int)rows->num_heads;
    a->group = (int)(rows->num_heads / kv->num_kv_heads);
    a->c = rows->scale * 1.4426950408889634f;
    if (batch->batch == 0 || batch->rows == 0) return LQ8_OK;
    const Plan p = plan_of(a, *types, (int)kv->head_dim, 1);
    if (std::max(p.own_tiles, p.pre_tiles) * kv->num_kv_heads >= ((size_t)1 << 32) / 256)
        return fail(LQ8_ERR_SHAPE_MISMATCH, "attention: sequences times kv heads above 2^24");
    return LQ8_OK;
}

lq8_status attention(lq8_ctx* ctx, const lq8_kv_pages* kv, const lq8_paged_batch* batch, bool has_prefix,
                     const lq8_shared_prefix* prefix, const lq8_attn_rows* rows) {
    AttnArgs a{};
    PagedTypes types;
    lq8_status st = check_attention(kv, batch, has_prefix, prefix, rows, &a, &types);
    if (st) return st;
    if (!registry_has(ctx)) return fail(LQ8_ERR_INVALID_ARG, "invalid or released context handle");
    if (batch->batch == 0 || batch->rows == 0) return LQ8_OK;
    DeviceGuard guard(ctx->device);
    if (guard.status) return guard.status;
    const int dim = (int)kv->head_dim;
    const Plan p = plan_of(&a, types, dim, ctx->num_cus);
    if (p.slots > 1) {
        void* sc = nullptr;
        if ((st = ctx_scratch(ctx, p.scratch, &sc))) return st;
        a.part = (float*)sc;
        a.ml = (float2*)(a.part + p.slots * batch->rows * a.heads * dim);
    }
    if (a.prefix.groups) {
        st = p.pre_few ? launch_few(ctx->stream, a, types, dim, p.pre_blocks, true) : launch_tile(ctx->stream, a, types, dim, p.pre_tiles, true);
        if (st) return st;
    }
    st = p.own_few ? launch_few(ctx->stream, a, types, dim, p.own_blocks, false) : launch_tile(ctx->stream, a, types, dim, p.own_tiles, false);
    if (st || p.slots == 1) return st;
    return launch_join(a, rows->dtype == LQ8_DTYPE_F32, dim, ctx->stream);
}

}  // namespace
}  // namespace lq8

using namespace lq8;

extern "C" {

lq8_status lq8_paged_attention_device(lq8_ctx* ctx, const lq8_kv_pages* kv, const lq8_paged_batch* batch,
                                      const lq8_attn_rows* rows) {
    return attention(ctx, kv, batch, false, nullptr, rows);
}

lq8_status lq8_prefix_attention_device(lq8_ctx* ctx, const lq8_kv_pages* kv, const lq8_paged_batch* batch,
                                       const lq8_shared_prefix* prefix, const lq8_attn_rows* rows) {
    return attention(ctx, kv, batch, true, prefix, rows);
}

lq8_status lq8_paged_plan(const lq8_kv_pages* kv, const lq8_paged_batch* batch, const lq8_shared_prefix* prefix,
                          const lq8_attn_rows* rows, uint32_t num_workgroups, lq8_paged_info* out) {
    AttnArgs a{};
    PagedTypes types;
    if (!out || num_workgroups == 0) return fail(LQ8_ERR_INVALID_ARG, "plan: no workgroups, or out is null");
    const lq8_status st = check_attention(kv, batch, prefix != nullptr, prefix, rows, &a, &types);
    if (st) return st;
    *out = {};
    if (batch->batch == 0 || batch->rows == 0) return LQ8_OK;
    const Plan p = plan_of(&a, types, (int)kv->head_dim, (int)num_workgroups);
    out->own_rows = p.own_few ? 16 * p.own_blocks : TILE_PACKED;
    out->own_splits = a.own.pieces;
    out->own_chunk = a.own.shortest;
    out->workgroups = p.own_tiles * kv->num_kv_heads * a.own.pieces;
    if (a.prefix.groups) {
        out->prefix_rows = p.pre_few ? 16 * p.pre_blocks : TILE_PACKED;
        out->prefix_splits = a.pre.pieces;
        out->prefix_chunk = a.pre.shortest;
        out->workgroups += p.pre_tiles * kv->num_kv_heads * a.pre.pieces;
    }
    out->scratch_bytes = p.scratch;
    return LQ8_OK;
}

}  // extern "C"
