// paged_attention.hip -- attention over a paged key/value cache, with or
// without a prefix that sequences share (gfx950).
#include <algorithm>
#include <cmath>

#include "paged_attn.h"

namespace lq8 {
namespace {

// The row's pieces together: o = sum 2^(m_c - m) o_c / sum 2^(m_c - m) l_c.
// head_dim / 4 lanes take four elements each of a (row, head); SUB such groups
// share its pieces, every SUB-th each, U of them in flight, and meet in LDS.
constexpr int JOIN_THREADS = 256;
template <typename T, int D, int SUB>
__global__ __launch_bounds__(JOIN_THREADS) void k_join(AttnArgs a) {
    constexpr int LANES = D / 4, GROUPS = JOIN_THREADS / LANES, U = SUB == 1 ? 8 : 4;
    const int tid = threadIdx.x, lane = tid % LANES, group = tid / LANES, sub = group % SUB;
    const int64_t item = (int64_t)blockIdx.x * (GROUPS / SUB) + group / SUB;
    const int row = (int)(item / a.heads), head = (int)(item - (int64_t)row * a.heads);
    // The largest i < n with begin[i] <= x (ascending), -1: none.  A search with
    // as many branches as the group has lanes.
    auto last_from = [&](const int32_t* begin, int n, int x) {
        int lo = -1, end = n - 1;  // between them, both included
        while (lo < end) {
            const int step = (end - lo + LANES - 1) / LANES, i = lo + (lane + 1) * step;
            const uint64_t below = (__ballot(i <= end && begin[min(i, end)] <= x) >> (tid & 63 & ~(LANES - 1))) & (~0ull >> (64 - LANES));
            lo += __popcll(below) * step;
            end = min(end, lo + step - 1);
        }
        return lo;
    };
    // the row's sequence, its prefix, and their pieces (none: own = pre = 0)
    int seq = row < a.batch.rows ? row : -1;
    if (a.batch.row_begin && seq >= 0) {
        seq = last_from(a.batch.row_begin, a.batch.batch, row);
        if (seq >= 0) {
            const RowRange r = rows_of(a.batch, seq);
            if (row < r.first || row - r.first >= r.count) seq = -1;
        }
    }
    int prefix = -1;
    if (a.prefix.groups && seq >= 0) {
        prefix = last_from(a.prefix.seq_begin, a.prefix.groups, seq);
        if (prefix >= 0 && seq >= a.prefix.seq_begin[prefix + 1]) prefix = -1;
    }
    int own = 0, pre = 0;
    if (seq >= 0) {
        const Span s = own_span(a, seq);
        const int len = piece_len(s.length, a.own);
        own = (s.sees(row - s.first) + len - 1) / len;
        if (prefix >= 0) {
            const int n = held(a.prefix.lengths[prefix], a.prefix.max_pages, a.kv.page_shift), plen = piece_len(n, a.pre);
            pre = (n + plen - 1) / plen;
        }
    }
    const size_t step = (size_t)a.batch.rows * a.heads;
    float m = -__builtin_huge_valf(), l = 0.0f;
    v4f o = {0, 0, 0, 0};
    for (int c0 = sub; c0 < own + pre; c0 += SUB * U) {
        float2 ml[U];
        v4f y[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int c = min(c0 + u * SUB, own + pre - 1);
            const size_t at = (size_t)(c < own ? c : a.own.pieces + c - own) * step + item;
            ml[u] = a.ml[at];
            y[u] = *(const v4f*)(a.part + at * D + 4 * lane);
        }
        float mn = m;
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (c0 + u * SUB >= own + pre) ml[u].x = -__builtin_huge_valf();
            mn = fmaxf(mn, ml[u].x);
        }
        const float mu = fmaxf(mn, -FLT_MAX), f = __builtin_amdgcn_exp2f(m - mu);
        l *= f;
        o *= f;
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (c0 + u * SUB >= own + pre) continue;
            const float w = __builtin_amdgcn_exp2f(ml[u].x - mu);
            l = fmaf(w, ml[u].y, l);
#pragma unroll
            for (int e = 0; e < 4; e++) o[e] = fmaf(w, y[u][e], o[e]);
        }
        m = mn;
    }
    if constexpr (SUB > 1) {
        __shared__ float2 sml[GROUPS];
        __shared__ v4f so[GROUPS][LANES];
        if (lane == 0) sml[group] = make_float2(m, l);
        so[group][lane] = o;
        __syncthreads();
        if (sub) return;
        float mn = m;
#pragma unroll
        for (int u = 1; u < SUB; u++) mn = fmaxf(mn, sml[group + u].x);
        const float mu = fmaxf(mn, -FLT_MAX), f = __builtin_amdgcn_exp2f(m - mu);
        l *= f;
        o *= f;
#pragma unroll
        for (int u = 1; u < SUB; u++) {
            const float w = __builtin_amdgcn_exp2f(sml[group + u].x - mu);
            l = fmaf(w, sml[group + u].y, l);
#pragma unroll
            for (int e = 0; e < 4; e++) o[e] = fmaf(w, so[group + u][lane][e], o[e]);
        }
        m = mn;
    }
    if (seq < 0) return;  // behind the last sequence
    o = m == -__builtin_huge_valf() ? v4f{0, 0, 0, 0} : o * (1.0f / l);  // (no piece saw anything)
    const size_t at = (size_t)row * a.os + (size_t)head * D + 4 * lane;
    if constexpr (sizeof(T) == 4) *(v4f*)((float*)a.out + at) = o;
    else *(uint2*)((uint16_t*)a.out + at) = make_uint2(pack_bf16(o[0], o[1]), pack_bf16(o[2], o[3]));
}

template <typename T, int D>
void launch_join_sub(const AttnArgs& a, size_t slots, hipStream_t s) {
    // up to eight pieces a group takes at once; more are shared by eight groups
    const size_t items = (size_t)a.batch.rows * a.heads, groups = JOIN_THREADS / (D / 4);
    if (slots <= 8) hipLaunchKernelGGL((k_join<T, D, 1>), dim3((unsigned)((items + groups - 1) / groups)), dim3(JOIN_THREADS), 0, s, a);
    else hipLaunchKernelGGL((k_join<T, D, 8>), dim3((unsigned)((items + groups / 8 - 1) / (groups / 8))), dim3(JOIN_THREADS), 0, s, a);
}
lq8_status launch_join(const AttnArgs& a, bool f32, int dim, size_t slots, hipStream_t s) {
    if (f32 && dim == 64) launch_join_sub<float, 64>(a, slots, s);
    else if (f32) launch_join_sub<float, 128>(a, slots, s);
    else if (dim == 64) launch_join_sub<Bf16, 64>(a, slots, s);
    else launch_join_sub<Bf16, 128>(a, slots, s);
    LQ8_HIP(hipGetLastError());
    return LQ8_OK;
}

// How a call runs.
struct Plan {
    size_t own_blocks = 0, pre_blocks = 0;  // workgroups of each part
    size_t slots = 0, scratch = 0;          // of partial results; their bytes
};

// Workgroups a compute unit that a part is cut into.  Tiles beside own
// positions (PRE_FILL) leave these half the machine, and fewer pieces are less
// to join: 64 rows behind 8192 positions 64, 45, 45, 49 and 59 us at 0.25, 0.5,
// 0.75, 1 and 2.  Tiles alone: a chunk of f32 243, 222 and 233 us at 1, 2 and 4.
// Few rows: FEW_FILL, and more, up to FEW_MORE and 16 pieces, while a piece has
// 512 positions for each row tile that reads them.  At 2, 4, 8 and 16 (bf16, 32
// heads over 8 of 128):
//     1 x 30000            27   30   38   38 us: short pieces, many to join
//     8 x 4000             23   25   28   28
//     24 x 9000            93   93   88   88: the pieces' ends even out
//     64 x 8190           197  197  198  192 (191 with pieces of at least 512)
constexpr float FEW_FILL = 2, FEW_MORE = 16, TILE_FILL = 2, PRE_FILL = 0.5f;

size_t few_unit(bool f32_pages) { return f32_pages ? 64 : 128; }  // a tile for each of the four waves

// Pieces of a part whose positions are at most `most`, in `groups` workgroups
// a piece.  few: its kernel takes spans one by one, so that a long one among
// short ones needs pieces of its own; `tiles` row tiles read a span.
Cut cut_of(size_t most, size_t groups, int cus, bool few, bool f32_pages, float tile_fill, size_t tiles) {
    Cut c;
    size_t pieces;
    if (few) {
        c.unit = few_unit(f32_pages);
        // (tables are often wider than their sequences: 64 of 1000 positions in
        // tables for 131072 take 36 us, 34 in tables that fit; with pieces of a
        // unit each and up to 32768 workgroups 71)
        c.shortest = FEW_FILL * cus >= 8 * groups ? c.unit : 512;
        const size_t longest = (most + 2047) / 2048, cap = 8192 / groups;
        const size_t more = std::min<size_t>({(size_t)(FEW_MORE * cus) / groups, most / (512 * tiles), 16});
        pieces = std::max<size_t>({(size_t)(FEW_FILL * cus) / groups, more, std::min(longest, cap)});
    } else {
        c.unit = f32_pages ? 32 : 64;
        c.shortest = 256;
        pieces = (size_t)(tile_fill * cus) / groups;
    }
    c.shift = __builtin_ctz(c.shortest);
    c.pieces = (int)std::max<size_t>(1, std::min(pieces, (most + c.shortest - 1) / c.shortest));
    return c;
}

// Row tiles of 16 fill their products but read the cache once each; tiles of
// 128 read it once, with a workgroup's waves on 32 rows each (of few rows some
// have none).  us, 16-row tiles / 128-row tiles, 32 heads over 8 of 128, by
// packed rows:
//                  packed        32          48          64          96
//     bf16           8 x  4000   37 /  23    55 /  27    60 /  26    56 /  29
//                   32 x  2000   60 /  37    75 /  43    87 /  45   112 /  49
//     f32 over bf16  8 x  4000   32 /  37    42 /  44    49 /  44    47 /  48
//                   32 x  2000   49 /  64    55 /  85    66 /  85    85 /  90
//                    1 x 30000   33 /  39    42 /  54    49 /  53    73 /  57
//     f32            8 x  4000   59 /  64    94 /  73   103 /  71   128 /  74
//                   32 x  2000   88 / 129   134 / 141   139 / 142   188 / 149
//                    1 x 30000   57 /  71    81 /  79   101 /  82   159 /  94
// Where the blocks of 16 rows by 128 positions are at most two a compute unit,
// latency decides: 1 x 2000 of bf16 12 / 15, 14 / 17, 14 / 16; f32 15 / 35, 18 /
// 38, 19 / 36.
bool takes_few(PagedTypes types, size_t packed, size_t blocks, int cus) {
    return packed <= (types == PT_BF16_BF16 ? 16 : types == PT_F32_BF16 ? 64 : 32) || blocks <= 2 * (size_t)cus;
}

Plan plan_of(AttnArgs* a, PagedTypes types, int dim, int cus) {
    Plan p;
    const size_t G = a->group, kvh = a->kv.kv_heads, rows = a->batch.rows, batch = a->batch.batch;
    const bool f32 = types == PT_F32_F32;
    // row tiles of `spans` spans that have `all` rows together, at most `most` each and `usual` by the rule's reckoning
    auto part = [&](size_t spans, size_t all, size_t most, size_t usual, uint32_t pages, Cut* cut, int* few, bool* one, float tile_fill) {
        const size_t positions = (size_t)pages << a->kv.page_shift, units = (positions + 127) / 128;
        auto tiles_of = [&](size_t rows) {
            return std::min(spans * ((most * G + rows - 1) / rows), (all * G + (rows - 1) * std::min(spans, all)) / rows);
        };
        *one = most * G <= FEW_PACKED;
        size_t tiles = *one ? spans : tiles_of(FEW_PACKED);
        const bool is_few = takes_few(types, usual * G, tiles * kvh * units, cus);
        *few = is_few ? (int)tiles : 0;
        if (!is_few) tiles = tiles_of(TILE_PACKED);
        *cut = cut_of(positions, tiles * kvh, cus, is_few, f32, tile_fill, (usual * G + FEW_PACKED - 1) / FEW_PACKED);
        return tiles * kvh * cut->pieces;
    };
    p.own_blocks = part(batch, rows, a->batch.max_rows, a->batch.max_rows, a->batch.max_pages, &a->own, &a->own_few, &a->own_each, TILE_FILL);
    p.slots = a->own.pieces;
    if (a->prefix.groups) {
        const size_t groups = a->prefix.groups;  // (each may have all rows)
        p.pre_blocks = part(groups, rows, rows, (rows + groups - 1) / groups, a->prefix.max_pages, &a->pre, &a->pre_few, &a->pre_each, a->own_few ? PRE_FILL : TILE_FILL);
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
    if ((uint64_t)batch->rows * rows->num_heads > MAX_ROW_HEADS)
        return fail(LQ8_ERR_SHAPE_MISMATCH, "attention: rows * num_heads above 2^23");
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
    if (p.own_blocks + p.pre_blocks >= ((size_t)1 << 32) / 256 / 2)
        return fail(LQ8_ERR_SHAPE_MISMATCH, "attention: sequences times kv heads above 2^23");
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
    if (a.prefix.groups && a.own_few) {
        st = launch_both(ctx->stream, a, types, dim, p.pre_blocks, p.own_blocks, a.pre_few == 0);
    } else {
        if (a.prefix.groups) st = (a.pre_few ? launch_few : launch_tile)(ctx->stream, a, types, dim, p.pre_blocks, true);
        if (!st) st = (a.own_few ? launch_few : launch_tile)(ctx->stream, a, types, dim, p.own_blocks, false);
    }
    if (st || p.slots == 1) return st;
    return launch_join(a, rows->dtype == LQ8_DTYPE_F32, dim, p.slots, ctx->stream);
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
    out->own_rows = a.own_few ? FEW_PACKED : TILE_PACKED;
    out->own_splits = a.own.pieces;
    out->own_chunk = a.own.shortest;
    out->workgroups = p.own_blocks + p.pre_blocks;
    if (a.prefix.groups) {
        out->prefix_rows = a.pre_few ? FEW_PACKED : TILE_PACKED;
        out->prefix_splits = a.pre.pieces;
        out->prefix_chunk = a.pre.shortest;
    }
    out->scratch_bytes = p.scratch;
    return LQ8_OK;
}

}  // extern "C"
