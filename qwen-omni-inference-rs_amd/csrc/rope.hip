// rope.hip -- rotary positions with several axes, and the append to a paged
// key/value cache (gfx950).
//
// A pair (x[p], x[p + half]) turns by the angle position[axis(p)] * f_p.  The
// table holds f_p / 2 pi in double: position * turns has 53 bits, so its
// fraction is good to 2^-22 of a turn even at position 2^31 (a float32 angle
// loses a radian there); the fraction is taken in double, reduced to an eighth
// of a turn and handed to the float32 Taylor sums of sin and cos (the next
// terms are below 3e-8 at pi / 4).
//
// A workgroup takes a few rows: its threads compute the sines of the rows'
// pairs into LDS, once for all heads, and go over the heads.  A thread has 2 V
// elements of a head: V consecutive pairs, V = 16 bytes of elements, or 2 V of
// what passes through; head_dim / (2 V) threads make a head.
//
// Bound: HBM for many rows, the launch for few.  4900 rows of 32 heads of 80,
// two axes, bf16: 9.8 us, 5.1 TB/s read and written; the append of 7200 rows of
// 32 + 2 x 8 heads of 128, bf16, with norms and three axes: 49 us, 4.0 TB/s; a
// row of 24 heads 3.6 us.  (A 4 GiB copy reaches 4.8 TB/s.)
#include <algorithm>
#include <cmath>
#include <new>

#include "lq8_numerics.h"
#include "paged.h"

namespace lq8 {
namespace {

constexpr int RT = 256;  // threads of a workgroup

template <typename T> struct Vec;
template <> struct Vec<float> {
    static constexpr int V = 4;
    static __device__ __forceinline__ void load(const void* p, float (&x)[4]) {
        const float4 t = *(const float4*)p;
        x[0] = t.x, x[1] = t.y, x[2] = t.z, x[3] = t.w;
    }
    static __device__ __forceinline__ void store(void* p, const float (&x)[4]) {
        *(float4*)p = make_float4(x[0], x[1], x[2], x[3]);
    }
};

// float -> bf16 to nearest, ties to even (NaN stays NaN), two to a word
__device__ __forceinline__ uint32_t bf16_pair(float a, float b) {
    return (uint32_t)__builtin_bit_cast(uint16_t, (__bf16)a) | ((uint32_t)__builtin_bit_cast(uint16_t, (__bf16)b) << 16);
}
template <> struct Vec<Bf16> {
    static constexpr int V = 8;
    static __device__ __forceinline__ void load(const void* p, float (&x)[8]) {
        const uint4 t = *(const uint4*)p;
        const uint32_t w[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            x[2 * i] = __uint_as_float(w[i] << 16);
            x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        }
    }
    static __device__ __forceinline__ void store(void* p, const float (&x)[8]) {
        *(uint4*)p = make_uint4(bf16_pair(x[0], x[1]), bf16_pair(x[2], x[3]), bf16_pair(x[4], x[5]), bf16_pair(x[6], x[7]));
    }
};

// V values into a cache row of type C
template <typename C, int V>
__device__ __forceinline__ void store_cache(C* p, const float (&x)[V]) {
    if constexpr (sizeof(C) == 4) {
        *(float4*)p = make_float4(x[0], x[1], x[2], x[3]);
    } else if constexpr (V == 4) {
        *(uint2*)p = make_uint2(bf16_pair(x[0], x[1]), bf16_pair(x[2], x[3]));
    } else {
        Vec<Bf16>::store(p, x);
    }
}

// cos and sin of position * turns full circles
__device__ __forceinline__ void turn(int position, double turns, float* c, float* s) {
    const double t = (double)position * turns;
    const double f = t - rint(t);      // -1/2 .. 1/2
    const double k = rint(4.0 * f);    // the quarter, -2 .. 2
    const float r = (float)((f - 0.25 * k) * 6.283185307179586477);
    const float q = r * r;
    float sn = fmaf(q, 2.7557319e-6f, -1.9841270e-4f);
    sn = fmaf(q, sn, 8.3333333e-3f);
    sn = fmaf(q, sn, -1.6666667e-1f);
    sn = fmaf(r * q, sn, r);
    float cs = fmaf(q, 2.4801587e-5f, -1.3888889e-3f);
    cs = fmaf(q, cs, 4.1666667e-2f);
    cs = fmaf(q, cs, -0.5f);
    cs = fmaf(q, cs, 1.0f);
    const int ki = (int)k;
    const float a = ki & 1 ? sn : cs, b = ki & 1 ? cs : sn;  // |cos|, |sin| of the quarter
    *c = ki == 1 || ki == 2 || ki == -2 ? -a : a;
    *s = ki == -1 || ki == 2 || ki == -2 ? -b : b;
}

// What a thread does of a head: unit u holds pairs u V .. + V - 1 (elements at
// lo and lo + half), or past the rotary part two runs of V elements.
template <int V>
struct Unit {
    int lo, hi;
    bool turns;
    __device__ __forceinline__ Unit(int u, int half) {
        turns = u * V < half;
        lo = turns ? u * V : half + u * V;  // 2 half + (u V - half)
        if (!turns) lo = 2 * half + 2 * (u * V - half);
        hi = turns ? lo + half : lo + V;
    }
};

// cos and sin of `rows` rows from row0 on into sc [row][half], by the whole
// workgroup; at(i, axis): position of row row0 + i.
template <typename F>
__device__ __forceinline__ void sines(const RopePair* table, int half, int rows, float2* sc, F at) {
    for (int x = threadIdx.x; x < rows * half; x += RT) {
        const int i = x / half;
        const RopePair p = table[x - i * half];
        float2 v;
        turn(at(i, p.axis), p.turns, &v.x, &v.y);
        sc[x] = v;
    }
}

template <int V>
__device__ __forceinline__ void rotate(float (&a)[V], float (&b)[V], const float2* sc, float sign) {
#pragma unroll
    for (int i = 0; i < V; i += 2) {
        const float4 s = *(const float4*)(sc + i);
        const float s0 = s.y * sign, s1 = s.w * sign;
        const float x0 = a[i], y0 = b[i], x1 = a[i + 1], y1 = b[i + 1];
        a[i] = fmaf(x0, s.x, -(y0 * s0));
        b[i] = fmaf(y0, s.x, x0 * s0);
        a[i + 1] = fmaf(x1, s.z, -(y1 * s1));
        b[i + 1] = fmaf(y1, s.z, x1 * s1);
    }
}

constexpr int ROWS_MAX = 8;  // rows of a workgroup

struct RopeArgs {
    const RopePair* table;
    const char* x;
    char* y;
    size_t xs, ys;  // bytes
    const int32_t* positions;
    size_t ps;
    int rows, heads, half, units, dim, per;  // per: rows of a workgroup
    float sign;
};

template <typename T>
__global__ __launch_bounds__(RT) void k_rope(RopeArgs a) {
    constexpr int V = Vec<T>::V;
    __shared__ __attribute__((aligned(16))) float2 sc[ROWS_MAX * 128];
    const int row0 = blockIdx.x * a.per, rows = min(a.per, a.rows - row0);
    sines(a.table, a.half, rows, sc, [&](int i, int axis) { return a.positions[axis * a.ps + row0 + i]; });
    __syncthreads();
    const int each = a.heads * a.units, total = rows * each;
    for (int item = blockIdx.y * RT + threadIdx.x; item < total; item += gridDim.y * RT) {
        const int i = item / each, in = item - i * each, h = in / a.units, u = in - h * a.units;
        const Unit<V> w(u, a.half);
        const size_t off = (size_t)h * a.dim * sizeof(T);
        const char* x = a.x + (row0 + i) * a.xs + off;
        char* y = a.y + (row0 + i) * a.ys + off;
        float p[V], q[V];
        Vec<T>::load(x + w.lo * sizeof(T), p);
        Vec<T>::load(x + w.hi * sizeof(T), q);
        if (w.turns) rotate<V>(p, q, sc + i * a.half + u * V, a.sign);
        Vec<T>::store(y + w.lo * sizeof(T), p);
        Vec<T>::store(y + w.hi * sizeof(T), q);
    }
}

struct AppendArgs {
    PagesDev kv;
    BatchDev batch;
    const RopePair* table;  // null: no rotation
    const char *q, *k, *v;  // q null: no queries
    char* q_out;
    size_t qs, ks, vs, qos;  // bytes
    const float *q_norm, *k_norm;
    float eps;
    const int32_t* positions;
    size_t ps;
    int heads, half, per;  // per: rows of a workgroup
};

// Where a row goes: its position in its sequence, and the page and slot of it
// (page -1: none); seq < 0: no sequence has the row.
struct Place {
    int seq, slot, page;
};

// The places of `rows` rows from row0 on, by the whole workgroup.
__device__ __forceinline__ void find_places(const AppendArgs& a, int row0, int rows, Place* places) {
    const BatchDev& b = a.batch;
    if ((int)threadIdx.x < rows) places[threadIdx.x] = {-1, 0, -1};
    __syncthreads();
    auto put = [&](int i, int s, const RowRange& r) {
        const int64_t slot = (int64_t)b.lengths[s] - r.total + (row0 + i - r.first);
        int page = -1;
        if (slot >= 0 && slot < (int64_t)b.max_pages << a.kv.page_shift) page = b.pages[(size_t)s * b.max_pages + (slot >> a.kv.page_shift)];
        places[i] = {s, (int)slot, (unsigned)page < (unsigned)a.kv.num_pages ? page : -1};
    };
    if (!b.row_begin) {
        if ((int)threadIdx.x < rows) put(threadIdx.x, row0 + threadIdx.x, {row0 + (int)threadIdx.x, 1, 1});
    } else {
        for (int s = threadIdx.x; s < b.batch; s += RT) {
            const RowRange r = rows_of(b, s);
            // (an ascending row_begin gives a row one sequence at most)
            for (int i = max(0, r.first - row0); i < min(rows, r.first + r.count - row0); i++) put(i, s, r);
        }
    }
    __syncthreads();
}

// x * rsqrt(mean(x^2) + eps) * w of a head whose LANES threads lie side by
// side, x, w and the result rounded to bf16 (RmsNorm::forward); the squares
// of bf16 values, their sum and the root in double, so that the one rounding
// left is the result's own.
template <int LANES, int V>
__device__ __forceinline__ void norm_head(float (&a)[V], float (&b)[V], const float* w, const Unit<V>& u, float eps) {
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < V; i++) {
        a[i] = (float)(__bf16)a[i], b[i] = (float)(__bf16)b[i];
        sum = fma((double)a[i], (double)a[i], sum);
        sum = fma((double)b[i], (double)b[i], sum);
    }
#pragma unroll
    for (int d = LANES / 2; d > 0; d /= 2) sum += __shfl_xor(sum, d);
    const double inv = 1.0 / sqrt(sum / (double)(2 * V * LANES) + (double)eps);
#pragma unroll
    for (int i = 0; i < V; i++) {
        // (a product of two bf16 is exact in float32)
        a[i] = (float)(__bf16)(float)((double)(a[i] * (float)(__bf16)w[u.lo + i]) * inv);
        b[i] = (float)(__bf16)(float)((double)(b[i] * (float)(__bf16)w[u.hi + i]) * inv);
    }
}

// Rows of the batch: their q heads to q_out, their k and v heads to their slots.
template <typename T, typename C, int D>
__global__ __launch_bounds__(RT) void k_append(AppendArgs a) {
    constexpr int V = Vec<T>::V, UNITS = D / (2 * V);
    static_assert(RT % UNITS == 0 && 64 % UNITS == 0, "a head's threads lie in one wave");
    __shared__ __attribute__((aligned(16))) float2 sc[ROWS_MAX * D / 2];
    __shared__ Place places[ROWS_MAX];
    const int row0 = blockIdx.x * a.per, rows = min(a.per, a.batch.rows - row0);
    find_places(a, row0, rows, places);
    if (a.table) {
        sines(a.table, a.half, rows, sc, [&](int i, int axis) { return a.positions ? a.positions[axis * a.ps + row0 + i] : places[i].slot; });
        __syncthreads();
    }
    const int qh = a.q ? a.heads : 0, each = qh + 2 * a.kv.kv_heads;
    const int u = threadIdx.x % UNITS;
    const Unit<V> w(u, a.half);
    const int step = gridDim.y * (RT / UNITS);
    for (int item = blockIdx.y * (RT / UNITS) + threadIdx.x / UNITS; item < rows * each; item += step) {
        const int i = item / each, h = item - i * each, row = row0 + i;
        const Place at = places[i];
        const bool isq = h < qh, isk = !isq && h < qh + a.kv.kv_heads;
        const int g = isq ? h : isk ? h - qh : h - qh - a.kv.kv_heads;
        if (at.seq < 0 || (!isq && at.page < 0)) continue;
        const char* src = (isq ? a.q + row * a.qs : isk ? a.k + row * a.ks : a.v + row * a.vs) + (size_t)g * D * sizeof(T);
        float p[V], q[V];
        Vec<T>::load(src + w.lo * sizeof(T), p);
        Vec<T>::load(src + w.hi * sizeof(T), q);
        if (isq || isk) {
            const float* nw = isq ? a.q_norm : a.k_norm;
            if (nw) norm_head<UNITS, V>(p, q, nw, w, a.eps);
            if (a.table && w.turns) rotate<V>(p, q, sc + i * a.half + u * V, 1.0f);
        }
        if (isq) {
            char* y = a.q_out + row * a.qos + (size_t)g * D * sizeof(T);
            Vec<T>::store(y + w.lo * sizeof(T), p);
            Vec<T>::store(y + w.hi * sizeof(T), q);
        } else {
            const int in = at.slot & ((1 << a.kv.page_shift) - 1);
            C* y = (C*)(isk ? a.kv.k : a.kv.v) + at.page * a.kv.page_stride + (((size_t)g << a.kv.page_shift) + in) * D;
            store_cache<C, V>(y + w.lo, p);
            store_cache<C, V>(y + w.hi, q);
        }
    }
}

// Rows of a workgroup and workgroups that share them: few rows leave a
// workgroup each, and their heads to several, so that two a CU run; many are
// taken up to eight at a time while eight workgroups a CU are left.
struct RowSplit {
    int per;
    dim3 grid;
};
RowSplit split_rows(size_t rows, size_t items, int cus) {
    const size_t per = std::max<size_t>(1, std::min<size_t>(ROWS_MAX, rows / (8 * (size_t)cus)));
    const size_t groups = (rows + per - 1) / per, most = (per * items + RT - 1) / RT, want = (2 * (size_t)cus + groups - 1) / groups;
    return {(int)per, dim3((unsigned)groups, (unsigned)std::min(want, most))};
}

template <typename T, typename C>
void launch_append(const AppendArgs& a, dim3 grid, int dim, hipStream_t s) {
    if (dim == 64) hipLaunchKernelGGL((k_append<T, C, 64>), grid, dim3(RT), 0, s, a);
    else hipLaunchKernelGGL((k_append<T, C, 128>), grid, dim3(RT), 0, s, a);
}

lq8_status check_rope(const lq8_rope_config* c) {
    if (!c) return fail(LQ8_ERR_INVALID_ARG, "rope: null configuration");
    if (c->head_dim == 0 || c->head_dim % 16 || c->head_dim > 256)
        return fail(LQ8_ERR_SHAPE_MISMATCH, "rope: head_dim must be a multiple of 16 up to 256");
    if (c->rotary_dim == 0 || c->rotary_dim % 16 || c->rotary_dim > c->head_dim)
        return fail(LQ8_ERR_SHAPE_MISMATCH, "rope: rotary_dim must be a multiple of 16 up to head_dim");
    if (c->axes < 1 || c->axes > LQ8_ROPE_MAX_AXES) return fail(LQ8_ERR_INVALID_ARG, "rope: 1 to 4 axes");
    if (c->layout != LQ8_ROPE_SECTIONS && c->layout != LQ8_ROPE_INTERLEAVED)
        return fail(LQ8_ERR_INVALID_ARG, "rope: unknown layout");
    if (!(c->theta > 0.0) || !std::isfinite(c->theta)) return fail(LQ8_ERR_INVALID_ARG, "rope: theta must be positive");
    const uint32_t pairs = c->rotary_dim / 2;
    uint64_t sum = 0;
    for (uint32_t a = 0; a < c->axes; a++) sum += c->sections[a];
    if (!(c->axes == 1 && sum == 0) && sum != pairs)
        return fail(LQ8_ERR_SHAPE_MISMATCH, "rope: the sections must add up to rotary_dim / 2");
    if (c->layout == LQ8_ROPE_INTERLEAVED)
        for (uint32_t a = 1; a < c->axes; a++)
            if (c->sections[a] && (uint64_t)c->axes * (c->sections[a] - 1) + a >= pairs)
                return fail(LQ8_ERR_SHAPE_MISMATCH, "rope: an interleaved section reaches past the last pair");
    return LQ8_OK;
}

int axis_of(const lq8_rope_config& c, uint32_t p) {
    if (c.axes == 1) return 0;
    if (c.layout == LQ8_ROPE_INTERLEAVED) {
        const uint32_t a = p % c.axes;
        return a > 0 && p < (uint64_t)c.axes * c.sections[a] ? (int)a : 0;
    }
    uint32_t end = 0;
    for (uint32_t a = 0; a + 1 < c.axes; a++) {
        end += c.sections[a];
        if (p < end) return (int)a;
    }
    return (int)c.axes - 1;
}

size_t elem_size(int32_t dtype) { return dtype == LQ8_DTYPE_F32 ? 4 : 2; }

}  // namespace

// ---- host checks ------------------------------------------------------------------

static bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

lq8_status check_pages(const lq8_kv_pages* kv, PagesDev* out) {
    if (!kv) return fail(LQ8_ERR_INVALID_ARG, "pages: null description");
    if (!kv->k || !kv->v) return fail(LQ8_ERR_INVALID_ARG, "pages: null pointer");
    if (kv->dtype != LQ8_DTYPE_F32 && kv->dtype != LQ8_DTYPE_BF16)
        return fail(LQ8_ERR_DTYPE_MISMATCH, "pages: F32 or BF16");
    if (kv->head_dim != 64 && kv->head_dim != 128) return fail(LQ8_ERR_SHAPE_MISMATCH, "pages: head_dim must be 64 or 128");
    if (kv->page_size < (uint32_t)PAGE_MIN || kv->page_size > (uint32_t)PAGE_MAX || (kv->page_size & (kv->page_size - 1)))
        return fail(LQ8_ERR_SHAPE_MISMATCH, "pages: page_size must be a power of two from 16 to 1024");
    if (kv->num_kv_heads == 0 || kv->num_kv_heads > MAX_KV_HEADS)
        return fail(LQ8_ERR_SHAPE_MISMATCH, "pages: 1 to 1024 kv heads");
    if (kv->num_pages == 0 || kv->num_pages > (uint32_t)INT32_MAX) return fail(LQ8_ERR_SHAPE_MISMATCH, "pages: no pages, or too many");
    const size_t dense = (size_t)kv->num_kv_heads * kv->page_size * kv->head_dim, es = elem_size(kv->dtype);
    const size_t stride = kv->page_stride ? kv->page_stride : dense;
    if (stride < dense) return fail(LQ8_ERR_SHAPE_MISMATCH, "pages: page_stride is below a page");
    if (stride > ((size_t)1 << 60) / kv->num_pages) return fail(LQ8_ERR_SHAPE_MISMATCH, "pages: page_stride too large");
    if (!aligned16(kv->k) || !aligned16(kv->v) || (stride * es) % 16)
        return fail(LQ8_ERR_INVALID_ARG, "pages: pointers and page_stride must be multiples of 16 bytes");
    out->k = kv->k;
    out->v = kv->v;
    out->num_pages = (int)kv->num_pages;
    out->page_shift = __builtin_ctz(kv->page_size);
    out->kv_heads = (int)kv->num_kv_heads;
    out->page_stride = stride;
    return LQ8_OK;
}

lq8_status check_batch(const lq8_paged_batch* b, uint32_t page_size, BatchDev* out) {
    if (!b) return fail(LQ8_ERR_INVALID_ARG, "batch: null description");
    if (b->batch > MAX_BATCH || b->rows > MAX_ROWS) return fail(LQ8_ERR_SHAPE_MISMATCH, "batch: above 65536 sequences or 2^23 rows");
    if (b->batch && b->rows) {
        if (!b->lengths || !b->pages) return fail(LQ8_ERR_INVALID_ARG, "batch: null pointer");
        if (!b->row_begin && b->rows != b->batch)
            return fail(LQ8_ERR_SHAPE_MISMATCH, "batch: without row_begin every sequence has one row");
        if (b->row_begin && (b->max_rows == 0 || b->max_rows > b->rows))
            return fail(LQ8_ERR_SHAPE_MISMATCH, "batch: max_rows must be from 1 to rows");
        if (b->max_pages == 0 || (uint64_t)b->max_pages * page_size > (uint64_t)INT32_MAX / 2)
            return fail(LQ8_ERR_SHAPE_MISMATCH, "batch: max_pages is zero or holds more than 2^30 positions");
    }
    out->batch = (int)b->batch;
    out->rows = (int)b->rows;
    out->max_rows = b->row_begin ? (int)b->max_rows : 1;
    out->max_pages = (int)b->max_pages;
    out->row_begin = b->row_begin;
    out->lengths = b->lengths;
    out->pages = b->pages;
    return LQ8_OK;
}

lq8_status check_types(int32_t rows, int32_t pages, PagedTypes* out) {
    if (rows == LQ8_DTYPE_F32 && pages == LQ8_DTYPE_F32) *out = PT_F32_F32;
    else if (rows == LQ8_DTYPE_F32 && pages == LQ8_DTYPE_BF16) *out = PT_F32_BF16;
    else if (rows == LQ8_DTYPE_BF16 && pages == LQ8_DTYPE_BF16) *out = PT_BF16_BF16;
    else return fail(LQ8_ERR_DTYPE_MISMATCH, "rows and pages: F32 with F32 or BF16 pages, BF16 with BF16 pages");
    return LQ8_OK;
}

lq8_status check_rows(const char* what, const void* p, size_t* stride, size_t width, size_t elem) {
    if (!p) return fail(LQ8_ERR_INVALID_ARG, std::string(what) + ": null pointer");
    if (*stride == 0) *stride = width;
    if (*stride < width || *stride > (size_t)1 << 32) return fail(LQ8_ERR_SHAPE_MISMATCH, std::string(what) + ": stride below a row, or above 2^32");
    if (!aligned16(p) || (*stride * elem) % 16)
        return fail(LQ8_ERR_INVALID_ARG, std::string(what) + ": pointer and stride must be multiples of 16 bytes");
    return LQ8_OK;
}

}  // namespace lq8

using namespace lq8;

#define CHECK_CTX(ctx) \
    if (!registry_has(ctx)) return fail(LQ8_ERR_INVALID_ARG, "invalid or released context handle")

// positions of every axis lie inside what the strides span
static lq8_status check_positions(const int32_t* p, size_t* stride, size_t rows) {
    if (!p) return LQ8_OK;
    if (*stride == 0) *stride = rows;
    if (*stride < rows || *stride > (size_t)1 << 32) return fail(LQ8_ERR_SHAPE_MISMATCH, "positions: stride below the rows, or above 2^32");
    return LQ8_OK;
}

extern "C" {

lq8_status lq8_rope_axes(const lq8_rope_config* cfg, uint8_t* axis_of_pair) {
    const lq8_status st = check_rope(cfg);
    if (st) return st;
    if (axis_of_pair)
        for (uint32_t p = 0; p < cfg->rotary_dim / 2; p++) axis_of_pair[p] = (uint8_t)axis_of(*cfg, p);
    return LQ8_OK;
}

lq8_status lq8_rope_create(lq8_ctx* ctx, const lq8_rope_config* cfg, lq8_rope** out) {
    lq8_status st = check_rope(cfg);
    if (st) return st;
    CHECK_CTX(ctx);
    if (!out) return fail(LQ8_ERR_INVALID_ARG, "out is null");
    *out = nullptr;
    DeviceGuard guard(ctx->device);
    if (guard.status) return guard.status;
    RopePair host[128];
    const uint32_t pairs = cfg->rotary_dim / 2;
    for (uint32_t p = 0; p < pairs; p++) {
        const double e = -2.0 * (double)(cfg->repeated ? p & ~1u : p) / (double)cfg->rotary_dim;
        host[p] = {std::pow(cfg->theta, e) / 6.283185307179586477, axis_of(*cfg, p), 0};
    }
    lq8_rope* r = new (std::nothrow) lq8_rope();
    if (!r) return fail(LQ8_ERR_OUT_OF_MEMORY, "rope: host memory");
    r->device = ctx->device;
    r->cfg = *cfg;
    hipError_t e = hipMalloc(&r->table, pairs * sizeof(RopePair));
    if (e == hipSuccess) e = hipMemcpyAsync(r->table, host, pairs * sizeof(RopePair), hipMemcpyHostToDevice, ctx->stream);
    if (e == hipSuccess) e = hipStreamSynchronize(ctx->stream);
    if (e != hipSuccess) {
        if (r->table) (void)hipFree(r->table);
        delete r;
        return hip_fail(e, "rope table");
    }
    registry_add(r);
    *out = r;
    return LQ8_OK;
}

lq8_status lq8_rope_free(lq8_rope* rope) {
    if (!registry_has(rope)) return fail(LQ8_ERR_INVALID_ARG, "invalid or released rope handle");
    // (the context may be gone; hipFree waits for the table's readers)
    registry_remove(rope);
    (void)hipFree(rope->table);
    delete rope;
    return LQ8_OK;
}

lq8_status lq8_rope_device(lq8_ctx* ctx, const lq8_rope* rope, const lq8_rope_rows* rows) {
    CHECK_CTX(ctx);
    if (!registry_has(rope)) return fail(LQ8_ERR_INVALID_ARG, "invalid or released rope handle");
    if (!rows) return fail(LQ8_ERR_INVALID_ARG, "rope: null rows");
    if (rope->device != ctx->device) return fail(LQ8_ERR_INVALID_ARG, "rope: the handle is another device's");
    if (rows->dtype != LQ8_DTYPE_F32 && rows->dtype != LQ8_DTYPE_BF16) return fail(LQ8_ERR_DTYPE_MISMATCH, "rope: F32 or BF16 rows");
    if (rows->rows > MAX_ROWS || rows->heads > MAX_HEADS) return fail(LQ8_ERR_SHAPE_MISMATCH, "rope: above 2^23 rows or 16384 heads");
    if (rows->rows == 0 || rows->heads == 0) return LQ8_OK;
    const size_t es = elem_size(rows->dtype), width = (size_t)rows->heads * rope->cfg.head_dim;
    size_t xs = rows->x_stride, ys = rows->y_stride, ps = rows->positions_stride;
    lq8_status st;
    if ((st = check_rows("rope x", rows->x, &xs, width, es)) || (st = check_rows("rope y", rows->y, &ys, width, es))) return st;
    if (rows->x == rows->y && xs != ys) return fail(LQ8_ERR_SHAPE_MISMATCH, "rope: in place needs one stride");
    if (!rows->positions) return fail(LQ8_ERR_INVALID_ARG, "rope: null positions");
    if ((st = check_positions(rows->positions, &ps, rows->rows))) return st;
    DeviceGuard guard(ctx->device);
    if (guard.status) return guard.status;
    const bool f32 = rows->dtype == LQ8_DTYPE_F32;
    const int units = (int)rope->cfg.head_dim / (2 * (f32 ? 4 : 8));
    RopeArgs a{(const RopePair*)rope->table, (const char*)rows->x, (char*)rows->y, xs * es, ys * es, rows->positions, ps,
               (int)rows->rows, (int)rows->heads, (int)rope->cfg.rotary_dim / 2, units, (int)rope->cfg.head_dim, 1,
               rows->inverse ? -1.0f : 1.0f};
    const RowSplit r = split_rows(rows->rows, (size_t)rows->heads * units, ctx->num_cus);
    a.per = r.per;
    if (f32) hipLaunchKernelGGL(k_rope<float>, r.grid, dim3(RT), 0, ctx->stream, a);
    else hipLaunchKernelGGL(k_rope<Bf16>, r.grid, dim3(RT), 0, ctx->stream, a);
    LQ8_HIP(hipGetLastError());
    return LQ8_OK;
}

lq8_status lq8_paged_append_device(lq8_ctx* ctx, const lq8_rope* rope, const lq8_kv_pages* kv,
                                   const lq8_paged_batch* batch, const lq8_qkv_rows* rows) {
    AppendArgs a{};
    PagedTypes types;
    lq8_status st;
    if ((st = check_pages(kv, &a.kv)) || (st = check_batch(batch, kv->page_size, &a.batch))) return st;
    if (!rows) return fail(LQ8_ERR_INVALID_ARG, "append: null rows");
    if ((st = check_types(rows->dtype, kv->dtype, &types))) return st;
    if (!rows->q != !rows->q_out) return fail(LQ8_ERR_INVALID_ARG, "append: q and q_out go together");
    if (rows->q && (rows->num_heads == 0 || rows->num_heads > MAX_HEADS))
        return fail(LQ8_ERR_SHAPE_MISMATCH, "append: 1 to 16384 query heads");
    const size_t es = elem_size(rows->dtype), d = kv->head_dim;
    size_t qs = rows->q_stride, ks = rows->k_stride, vs = rows->v_stride, os = rows->q_out_stride, ps = rows->positions_stride;
    if ((st = check_rows("append k", rows->k, &ks, kv->num_kv_heads * d, es)) ||
        (st = check_rows("append v", rows->v, &vs, kv->num_kv_heads * d, es)))
        return st;
    if (rows->q) {
        if ((st = check_rows("append q", rows->q, &qs, rows->num_heads * d, es)) ||
            (st = check_rows("append q_out", rows->q_out, &os, rows->num_heads * d, es)))
            return st;
        if (rows->q == rows->q_out && qs != os) return fail(LQ8_ERR_SHAPE_MISMATCH, "append: q in place needs one stride");
    }
    if ((rows->q_norm || rows->k_norm) && !(rows->eps >= 0.0f)) return fail(LQ8_ERR_INVALID_ARG, "append: eps must be at least 0");
    if ((st = check_positions(rows->positions, &ps, batch->rows))) return st;
    CHECK_CTX(ctx);
    if (rope) {
        if (!registry_has(rope)) return fail(LQ8_ERR_INVALID_ARG, "invalid or released rope handle");
        if (rope->device != ctx->device) return fail(LQ8_ERR_INVALID_ARG, "append: the rope handle is another device's");
        if (rope->cfg.head_dim != kv->head_dim) return fail(LQ8_ERR_SHAPE_MISMATCH, "append: rope of another head_dim");
    }
    if (batch->batch == 0 || batch->rows == 0) return LQ8_OK;
    DeviceGuard guard(ctx->device);
    if (guard.status) return guard.status;
    a.table = rope ? (const RopePair*)rope->table : nullptr;
    a.half = rope ? (int)rope->cfg.rotary_dim / 2 : (int)d / 2;
    a.q = (const char*)rows->q, a.k = (const char*)rows->k, a.v = (const char*)rows->v, a.q_out = (char*)rows->q_out;
    a.qs = qs * es, a.ks = ks * es, a.vs = vs * es, a.qos = os * es;
    a.q_norm = rows->q_norm, a.k_norm = rows->k_norm, a.eps = rows->eps;
    a.positions = rows->positions, a.ps = ps;
    a.heads = rows->q ? (int)rows->num_heads : 0;
    const size_t units = d / (2 * (rows->dtype == LQ8_DTYPE_F32 ? 4 : 8));
    const RowSplit r = split_rows(batch->rows, (a.heads + 2 * (size_t)kv->num_kv_heads) * units, ctx->num_cus);
    a.per = r.per;
    if (types == PT_F32_F32) launch_append<float, float>(a, r.grid, (int)d, ctx->stream);
    else if (types == PT_F32_BF16) launch_append<float, Bf16>(a, r.grid, (int)d, ctx->stream);
    else launch_append<Bf16, Bf16>(a, r.grid, (int)d, ctx->stream);
    LQ8_HIP(hipGetLastError());
    return LQ8_OK;
}

}  // extern "C"
