// paged_attention.hip -- attention over a paged key/value cache, with or
// without a prefix that sequences share (gfx950).
#include <cmath>

#include "lq8_numerics.h"
#include "paged.h"

namespace lq8 {
namespace {

struct PrefixDev {
    int groups = 0, max_pages = 0;
    const int32_t *seq_begin = nullptr, *lengths = nullptr, *pages = nullptr;
};

struct AttnArgs {
    PagesDev kv;
    BatchDev batch;
    PrefixDev prefix;
    const char* q;
    char* out;
    size_t qs, os;  // elements
    int heads;
    float scale;
};

__device__ __forceinline__ float load1(const float* p) { return *p; }
__device__ __forceinline__ float load1(const Bf16* p) { return __uint_as_float((uint32_t)p->bits << 16); }
__device__ __forceinline__ void store1(float* p, float x) { *p = x; }
__device__ __forceinline__ void store1(Bf16* p, float x) { p->bits = __builtin_bit_cast(uint16_t, (__bf16)x); }

// One wave per (row of a sequence, query head).
template <typename T, typename C, int D>
__global__ __launch_bounds__(64) void k_attn(AttnArgs a) {
    __shared__ float qs[D];
    const int lane = threadIdx.x, s = blockIdx.z, h = blockIdx.y;
    const RowRange r = rows_of(a.batch, s);
    const int i = blockIdx.x;
    if (i >= r.count) return;
    const int g = h / (a.heads / a.kv.kv_heads);
    const T* q = (const T*)a.q + (size_t)(r.first + i) * a.qs + (size_t)h * D;
    for (int d = lane; d < D; d += 64) qs[d] = load1(q + d);
    __syncthreads();
    float m = -__builtin_huge_valf(), l = 0.0f, o[D / 64] = {};
    int seen = 0;
    auto part = [&](const int32_t* table, int n) {
        for (int j0 = 0; j0 < n; j0 += 64) {
            const int j = j0 + lane;
            int page = j < n ? table[j >> a.kv.page_shift] : -1;
            if (page >= a.kv.num_pages) page = -1;
            const size_t at = page < 0 ? 0
                                       : page * a.kv.page_stride +
                                             (((size_t)g << a.kv.page_shift) + (j & ((1 << a.kv.page_shift) - 1))) * D;
            float x = 0.0f;
            if (page >= 0)
                for (int d = 0; d < D; d++) x = fmaf(qs[d], load1((const C*)a.kv.k + at + d), x);
            x = page < 0 ? -__builtin_huge_valf() : x * a.scale;
            float mx = x;
            for (int d = 32; d; d /= 2) {
                const float y = __shfl_xor(mx, d);
                mx = y != y || y > mx ? y : mx;
            }
            seen += __popcll(__ballot(page >= 0));
            const float mn = m > mx ? m : mx, base = mn == -__builtin_huge_valf() ? 0.0f : mn;
            const float e = page < 0 ? 0.0f : expf(x - base), c = expf(m - base);
            float sum = e;
            for (int d = 32; d; d /= 2) sum += __shfl_xor(sum, d);
            l = l * c + sum;
            m = mn;
            for (int k = 0; k < D / 64; k++) o[k] *= c;
            for (int t = 0; t < 64; t++) {
                const int p = __shfl(page, t);
                const float w = __shfl(e, t);
                const size_t from = __shfl((unsigned long long)at, t);
                if (p >= 0)
                    for (int k = 0; k < D / 64; k++) o[k] = fmaf(w, load1((const C*)a.kv.v + from + lane + 64 * k), o[k]);
            }
        }
    };
    for (int p = 0; p < a.prefix.groups; p++)
        if (s >= a.prefix.seq_begin[p] && s < a.prefix.seq_begin[p + 1])
            part(a.prefix.pages + (size_t)p * a.prefix.max_pages, held(a.prefix.lengths[p], a.prefix.max_pages, a.kv.page_shift));
    const int64_t last = (int64_t)a.batch.lengths[s] - r.count + i;  // the row's own position
    part(a.batch.pages + (size_t)s * a.batch.max_pages,
         (int)max((int64_t)0, min(last + 1, (int64_t)held(a.batch.lengths[s], a.batch.max_pages, a.kv.page_shift))));
    T* out = (T*)a.out + (size_t)(r.first + i) * a.os + (size_t)h * D;
    for (int k = 0; k < D / 64; k++) store1(out + lane + 64 * k, seen ? o[k] / l : 0.0f);
}

template <typename T, typename C>
lq8_status launch_simple(const AttnArgs& a, int dim, hipStream_t s) {
    const dim3 grid((unsigned)a.batch.max_rows, (unsigned)a.heads, (unsigned)a.batch.batch);
    if (dim == 64) hipLaunchKernelGGL((k_attn<T, C, 64>), grid, dim3(64), 0, s, a);
    else hipLaunchKernelGGL((k_attn<T, C, 128>), grid, dim3(64), 0, s, a);
    LQ8_HIP(hipGetLastError());
    return LQ8_OK;
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
    if (!(rows->scale > 0.0f) || !std::isfinite(rows->scale))
        return fail(LQ8_ERR_INVALID_ARG, "attention: scale must be positive and finite");
    const size_t es = rows->dtype == LQ8_DTYPE_F32 ? 4 : 2, width = (size_t)rows->num_heads * kv->head_dim;
    a->qs = rows->q_stride, a->os = rows->out_stride;
    if ((st = check_rows("attention q", rows->q, &a->qs, width, es)) || (st = check_rows("attention out", rows->out, &a->os, width, es)))
        return st;
    if (rows->q == rows->out && a->qs != a->os) return fail(LQ8_ERR_SHAPE_MISMATCH, "attention: in place needs one stride");
    a->q = (const char*)rows->q;
    a->out = (char*)rows->out;
    a->heads = (int)rows->num_heads;
    a->scale = rows->scale;
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
    if (types == PT_F32_F32) return launch_simple<float, float>(a, dim, ctx->stream);
    if (types == PT_F32_BF16) return launch_simple<float, Bf16>(a, dim, ctx->stream);
    return launch_simple<Bf16, Bf16>(a, dim, ctx->stream);
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
    out->own_rows = out->own_splits = 1;
    out->workgroups = (uint64_t)a.batch.max_rows * a.heads * a.batch.batch;
    return LQ8_OK;
}

}  // extern "C"
