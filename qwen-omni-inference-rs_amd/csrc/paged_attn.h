// paged_attn.h -- what the kernels of attention over a paged cache share
// (paged_few.h, paged_tile.h, paged_attention.hip).
//
// Rows.  The queries of a kv head are packed: packed row r of a sequence (or
// of a group's rows) is query head r % G of row r / G, G = num_heads /
// num_kv_heads.  Row i of a sequence sees positions 0 .. base + i - 1.
//
// Pieces.  A long row range of positions is cut into pieces that run on
// different workgroups: piece c holds positions c * len .. of its sequence,
// len from the sequence's own length alone (piece_len), so that a row's bits do
// not depend on its batch.  A piece gives (o, m, l) per row: m the largest
// scaled score in units of log 2, o = sum 2^(s - m) v, l = sum 2^(s - m).
// m = -inf: the row sees nothing of it; m = -FLT_MAX: it does, and every score
// is -inf.  With one piece, and no prefix, the kernel writes o / l itself.
#pragma once

#include <cfloat>

#include "lq8_numerics.h"
#include "paged.h"

namespace lq8 {

struct PrefixDev {
    int groups = 0, max_pages = 0;
    const int32_t *seq_begin = nullptr, *lengths = nullptr, *pages = nullptr;
};

struct Cut {
    int pieces = 1;     // at most
    int shortest = 64;  // positions of the shortest piece, a power of two
    int shift = 6;      // its logarithm
    int unit = 64;      // pieces are multiples of it, a power of two up to `shortest`
};

struct AttnArgs {
    PagesDev kv;
    BatchDev batch;
    PrefixDev prefix;
    const char* q;
    char* out;
    size_t qs, os;  // elements
    int heads, group;
    float c;        // scale * log2(e)
    Cut own, pre;
    int own_few = 0, pre_few = 0;  // row tiles, at most, in launch_few's kernel (0: launch_tile's)
    bool own_each = false, pre_each = false;  // of these tile t is all rows of span t
    float* part;    // [slots][rows][heads][head_dim], own pieces first; null: one piece, results go to out
    float2* ml;     // [slots][rows][heads]
};

__host__ __device__ inline int piece_len(int length, const Cut& c) {
    const int n = (int)(((unsigned)length + c.shortest - 1) >> c.shift);
    if (n <= c.pieces) return c.shortest;
    return (int)(((unsigned)(length + c.pieces - 1) / (unsigned)c.pieces + c.unit - 1) & ~(unsigned)(c.unit - 1));
}

// What one workgroup's rows attend to.
struct Span {
    int first, total, count;  // rows
    const int32_t* table;
    int length;               // positions that exist
    int base;                 // row i sees min(max(base + i, 0), length)
    __device__ __forceinline__ int sees(int i) const { return min(max(base + i, 0), length); }
};
__device__ __forceinline__ Span own_span(const AttnArgs& a, int s) {
    const RowRange r = rows_of(a.batch, s);
    const int raw = max(a.batch.lengths[s], 0);
    return {r.first, r.total, r.count, a.batch.pages + (size_t)s * a.batch.max_pages,
            held(raw, a.batch.max_pages, a.kv.page_shift), raw - r.total + 1};
}
// rows of the sequences of group g, each of which sees the whole prefix
__device__ __forceinline__ Span prefix_span(const AttnArgs& a, int g) {
    const int b = min(max(a.prefix.seq_begin[g], 0), a.batch.batch);
    const int e = min(max(a.prefix.seq_begin[g + 1], b), a.batch.batch);
    const int lo = !a.batch.row_begin ? b : min(max(a.batch.row_begin[b], 0), a.batch.rows);
    const int hi = !a.batch.row_begin ? e : min(max(a.batch.row_begin[e], lo), a.batch.rows);
    return {lo, hi - lo, hi - lo, a.prefix.pages + (size_t)g * a.prefix.max_pages,
            held(a.prefix.lengths[g], a.prefix.max_pages, a.kv.page_shift), 1 << 30};
}

constexpr int THREADS = 256;  // of a workgroup

// The span and the row tile (of PACKED packed rows) of tile number `want` over
// all spans, by all threads; false: there are fewer tiles.
template <int PACKED, bool PREFIX>
__device__ __forceinline__ bool find_tile(const AttnArgs& a, int want, int* span, int* tile) {
    __shared__ int sums[THREADS / 64], found[2];
    const int n = PREFIX ? a.prefix.groups : a.batch.batch, tid = threadIdx.x, lane = tid & 63;
    if (tid == 0) found[0] = -1;
    int before = 0;
    for (int s0 = 0; s0 < n; s0 += THREADS) {
        int t = 0;
        if (s0 + tid < n) {
            const int rows = PREFIX ? prefix_span(a, s0 + tid).count : rows_of(a.batch, s0 + tid).count;
            t = (int)(((int64_t)rows * a.group + PACKED - 1) / PACKED);
        }
        int x = t;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const int y = __shfl_up(x, d);
            if (lane >= d) x += y;
        }
        if (lane == 63) sums[tid >> 6] = x;
        __syncthreads();
        int base = before, all = before;
        for (int w = 0; w < THREADS / 64; w++) {
            if (w < tid >> 6) base += sums[w];
            all += sums[w];
        }
        const int first = base + x - t;
        if (t > 0 && want >= first && want < first + t) found[0] = s0 + tid, found[1] = want - first;
        __syncthreads();
        before = all;
        if (want < all) break;
    }
    *span = __builtin_amdgcn_readfirstlane(found[0]);
    *tile = __builtin_amdgcn_readfirstlane(found[1]);
    return *span >= 0;
}

// The page of position j (the same for the whole wave), -1 where none holds
// it.  The entry is loaded whether j exists or not (that of the last position
// before `end` then, end > 0), by a scalar load.
typedef const int32_t __attribute__((address_space(4))) * ScalarInts;
__device__ __forceinline__ int page_at(const AttnArgs& a, const Span& s, int j, int end) {
    const int at = __builtin_amdgcn_readfirstlane(min(j, end - 1) >> a.kv.page_shift);
    const int p = ((ScalarInts)s.table)[at];
    const bool there = (j < end) & ((unsigned)p < (unsigned)a.kv.num_pages);
    return there ? p : -1;
}
// Element offset of position j (in page p) of kv head g; p < 0: of a slot of page 0, which is there to be read.
__device__ __forceinline__ size_t slot_off(const AttnArgs& a, int p, int g, int j, int dim) {
    return max(p, 0) * a.kv.page_stride + (size_t)(unsigned)(((g << a.kv.page_shift) + (j & ((1 << a.kv.page_shift) - 1))) * dim);
}

typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef __bf16 v8b __attribute__((ext_vector_type(8)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));

// to nearest, ties to even, NaN kept (one instruction for both)
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
    typedef float v2f __attribute__((ext_vector_type(2)));
    typedef __bf16 v2b __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((v2f{a, b}), v2b));
}
__device__ __forceinline__ float low_bf16(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float high_bf16(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }

// x = t[0] + t[1] + t[2] with terms of bf16, exactly: 8 + 8 + 8 bits.  The
// first is cut, not rounded (a rounded one could be infinite); what is not
// finite is its own first term.
__device__ __forceinline__ void three_terms(float x, float (&t)[3]) {
    const uint32_t b = __float_as_uint(x);
    const bool fine = (b & 0x7F800000u) != 0x7F800000u;
    t[0] = fine ? __uint_as_float(b & 0xFFFF0000u) : x;
    const float r = fine ? x - t[0] : 0.0f;
    t[1] = __uint_as_float(__float_as_uint(r) & 0xFFFF0000u);
    t[2] = r - t[1];
}

// both halves of w added to x
__device__ __forceinline__ float add_bf16(uint32_t w, float x) {
    typedef __bf16 v2b __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(v2b, w), v2b{(__bf16)1.0f, (__bf16)1.0f}, x, false);
}
__device__ __forceinline__ v8b join_halves(v4s a, v4s b) {
    return __builtin_bit_cast(v8b, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
}

// A loaded value waited for here: used inside a loop it would otherwise be
// waited for there, and with it, loads returning in order, the loop's own.
template <typename T> __device__ __forceinline__ void arrived(T& x) { asm volatile("" : "+v"(x)); }

// A row's reference m lies this far above its largest scaled score, so that
// sums of up to 2^16 values weighted 2^(s - m) cannot pass float32's range where
// their mean does not (2^8 of it goes to references that lag behind).
constexpr float ABOVE = 24.0f;

// Where the largest scaled score is this large, its rounding (2^-24 of it,
// which s c - m in one fma leaves in the exponent: the same factor for every
// position, but one that can leave the range) is taken off by rounding s c too.
__device__ __forceinline__ bool far_score(float m) { return fabsf(m) > 1e6f && m > -FLT_MAX; }

// Byte offset of 16-byte chunk c of row j of a tile in LDS, ROW bytes a row:
// chunks change places within their 256 bytes so that 4, 8 and 16 neighbouring
// rows' pieces of the same columns lie on different banks.
template <int ROW>
__device__ __forceinline__ int lds_slot(int j, int c) {
    static_assert(ROW == 128 || ROW == 256 || ROW == 512, "row bytes");
    if constexpr (ROW == 128) {
        const int line = j >> 1, f = ((line & 1) << 2) | ((line >> 1) & 3);
        return line * 256 + (((((j & 1) << 3) | c) ^ f) << 4);
    }
    return j * ROW + (((c & ~15) | ((c & 15) ^ (((j & 3) << 2) | ((j >> 2) & 3)))) << 4);
}
// 4 rows of 16 16-bit columns, one column a lane (16 lanes; lane i's address: row i / 4, columns 4 (i % 4) ..)
__device__ __forceinline__ v4s read_transposed(const char* p) {
    typedef v4s __attribute__((address_space(3))) * LP;
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((LP)p);
}

// Sets a sign bit of `bits` where w, two bf16 or a float32, is not finite: an
// exponent of ones carries into it.
template <bool F32>
__device__ __forceinline__ void mark_odd(v4u v, uint32_t& bits) {
#pragma unroll
    for (int e = 0; e < 4; e++) bits |= F32 ? (v[e] & 0x7FFFFFFFu) + 0x00800000u : (v[e] & 0x7FFF7FFFu) + 0x00800080u;
}
template <bool F32>
__device__ __forceinline__ bool is_odd(uint32_t bits) { return (bits & (F32 ? 0x80000000u : 0x80008000u)) != 0; }
// v with zeros in place of what is not finite
template <bool F32>
__device__ __forceinline__ v4u finite_part(v4u v) {
#pragma unroll
    for (int e = 0; e < 4; e++) {
        if ((v[e] & 0x7F800000u) == 0x7F800000u) v[e] &= F32 ? 0u : 0xFFFFu;
        if (!F32 && (v[e] & 0x7F80u) == 0x7F80u) v[e] &= 0xFFFF0000u;
    }
    return v;
}

// Values that are not finite enter the products as zeros (a zero probability
// times one of them would be NaN in rows that do not see it) and meet the rows
// that see them here, after the sums are done: for positions from .. to - 1 in
// runs of `run` every `step`, each(values of the position, whether the lane's
// row sees it, its probability).  The lane's row has its query at q, sees
// positions before `sees` and has reference m.
template <typename T, typename C, int D, typename F>
__device__ __forceinline__ void meet_odd(const AttnArgs& a, const Span& s, int g, int from, int to, int run, int step, int end,
                                         const T* q, int sees, float m, F each) {
    auto value = [](const auto* p) {
        if constexpr (sizeof(*p) == 4) return (float)*(const float*)p;
        else return __uint_as_float((uint32_t) * (const uint16_t*)p << 16);
    };
    for (int j0 = from; j0 < to; j0 += step)
        for (int j = j0; j < min(j0 + run, end); j++) {
            const int page = page_at(a, s, j, end);
            if (page < 0) continue;
            const size_t off = slot_off(a, page, g, j, D);
            each((const C*)a.kv.v + off, j < sees, value, [&]() {
                const C* k = (const C*)a.kv.k + off;
                float x = 0.0f;
                for (int d = 0; d < D; d++) x = fmaf(value(q + d), value(k + d), x);
                const float mu = fmaxf(m, -FLT_MAX);
                return __builtin_amdgcn_exp2f(far_score(mu) ? x * a.c - mu : fmaf(x, a.c, -mu));
            });
        }
}

constexpr int FEW_PACKED = 16;    // packed rows of a launch_few block
constexpr int TILE_PACKED = 128;  // of a launch_tile one
// `blocks` workgroups of the prefix part or of the own one; launch_both: of
// both, the prefix by launch_tile's kernel or launch_few's, the own by launch_few's.
lq8_status launch_few(hipStream_t s, const AttnArgs& a, PagedTypes types, int dim, size_t blocks, bool prefix);
lq8_status launch_tile(hipStream_t s, const AttnArgs& a, PagedTypes types, int dim, size_t blocks, bool prefix);
lq8_status launch_both(hipStream_t s, const AttnArgs& a, PagedTypes types, int dim, size_t pre, size_t own, bool tile);

}  // namespace lq8
