// paged_few.h -- attention over a paged cache for few packed rows a kv head:
// single tokens, and a few drafted ones (gfx950).  Sixteen rows to a workgroup.
//
// Bound: the cache's bytes.  Each of a workgroup's four waves runs its own
// online softmax over tiles of the piece (32 positions of bf16 pages, 16 of
// f32: 16 KiB of K and V at head_dim 128), with no barrier before the end: the
// next tile's K goes out when the scores are done and its V when this one's has
// left its registers, so a wave always has about a tile in flight.  64 sequences
// of up to 8190 bf16 positions, 32 heads over 8 of 128: 191 us, 5.83 TB/s (a
// read-only stream reaches 6.8); f32 rows over 8 x 131072: 400 us, 5.3 TB/s (a
// third workgroup on a compute unit would need its registers).
//
// The packed rows are the columns of every product, S^T = K Q^T and O^T =
// V^T P^T on 16 x 16 tiles.  Lane (r = lane % 16, p = lane / 16) of S^T holds
// row r's scores of positions 4 p .. + 3 of a 16-block, which is the B operand
// that P^T needs (the order of the positions inside a product is free), so the
// probabilities never move between lanes, and the maximum and the rescaling of
// O stay in the row's own lanes.
//   bf16 pages  K straight from the cache as the A operand; V through a
//               wave's own LDS tile, read back transposed (ds_read_tr)
//   f32 pages   16 x 16 x 4: both operands straight from the cache, four
//               products per 16-byte load with d in the order 4 r + component
// f32 rows over bf16 pages: q and p as three bf16 terms each (three_terms),
// every product exact, sums in float32.
#pragma once

#include <type_traits>

#include "paged_attn.h"

namespace lq8 {
namespace {

constexpr int FEW_WAVES = THREADS / 64;

template <int TYPES, int D> struct Tile;
// bf16 pages
template <int D> struct TileB {
    static constexpr int N = 32;            // positions
    static constexpr int KS = D / 32;       // products of a score block
    static constexpr int VI = D / 16;       // 16-byte loads of V per lane
    static constexpr int RPI = 512 / D;     // rows a wave's load covers
    v4u k[2][KS], v[VI];
};
template <int D> struct TileF {
    static constexpr int N = 16;
    static constexpr int KS = D / 16;       // 16-byte loads of K per lane
    static constexpr int VH = D / 64;
    v4f k[KS], v[4][VH];
};
template <int D> struct Tile<PT_BF16_BF16, D> : TileB<D> {};
template <int D> struct Tile<PT_F32_BF16, D> : TileB<D> {};
template <int D> struct Tile<PT_F32_F32, D> : TileF<D> {};

// 16 bytes of the cache.  Past the caches (each is read once) where the
// kernel is bound by the reads: 64 sequences of up to 8190 bf16 positions 198
// us against 211.  The three-term kernel (8 x 131072 positions) takes 437 us
// that way against 402 through them.
template <bool PAST>
__device__ __forceinline__ v4u stream(const uint16_t* p) {
    if constexpr (PAST) return __builtin_nontemporal_load((const v4u*)p);
    else return *(const v4u*)p;
}

// The head dimension of element e of O's tile t in a lane of group p.
template <bool F32C>
__device__ __forceinline__ int few_column(int t, int p, int e) {
    return F32C ? 64 * (t / 4) + 16 * p + 4 * e + t % 4 : 16 * t + 4 * p + e;
}

// LDS of a workgroup: the waves' V tiles, where their sums meet at the end, and
// their maxima and denominators
template <int D> constexpr int few_lds() { return FEW_WAVES * 16 * D * 4 + FEW_WAVES * 16 * (int)sizeof(float2); }

// Workgroup `block` of the launch; sm: few_lds<D>() bytes.
template <int TYPES, int D, bool PREFIX>
__device__ __forceinline__ void few_body(const AttnArgs& a, int block, char* sm) {
    constexpr bool F32C = TYPES == PT_F32_F32, F32Q = TYPES != PT_BF16_BF16;
    constexpr int TERMS = TYPES == PT_F32_BF16 ? 3 : 1;
    typedef Tile<TYPES, D> T;
    constexpr int N = T::N, DT = D / 16, WBYTES = 16 * D * 4;
    static_assert(WBYTES >= 32 * D * 2, "one wave's region");
    float2(*sml)[16] = (float2(*)[16])(sm + FEW_WAVES * WBYTES);
    const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, p = lane >> 4;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    char* own = sm + w * WBYTES;

    // block -> (piece, row tile, kv head), kv head fastest: the blocks of one
    // go to one XCD where their number divides by eight, and the row tiles of a
    // piece read its pages at about the same time
    const Cut& cut = PREFIX ? a.pre : a.own;
    const int G = a.group, kvh = a.kv.kv_heads, tiles = PREFIX ? a.pre_few : a.own_few;
    const int g = block % kvh, piece = block / kvh / tiles;
    int sp = block / kvh % tiles, tile = 0;
    if (!(PREFIX ? a.pre_each : a.own_each) && !find_tile<FEW_PACKED, PREFIX>(a, sp, &sp, &tile)) return;
    const int row0 = tile * FEW_PACKED;
    const Span s = PREFIX ? prefix_span(a, sp) : own_span(a, sp);
    const int packed = min(s.count * G - row0, FEW_PACKED);
    if (packed <= 0) return;
    const int len = piece_len(s.length, cut);
    const int most = s.sees((row0 + packed - 1) / G), least = s.sees(row0 / G);
    const int beg = piece * len, end = min(beg + len, most);
    if (a.part ? beg >= most : piece > 0) return;

    // this lane's row
    const bool valid = r < packed;
    const int i = (row0 + r) / G, row = s.first + (valid ? i : 0), head = g * G + (valid ? row0 + r - i * G : 0);
    const int sees = valid ? s.sees(i) : 0;
    const size_t qat = row * a.qs + (size_t)head * D;
    v4u q[F32C ? 1 : TERMS][F32C ? 1 : D / 32];
    v4f qf[F32C ? D / 16 : 1];
    if constexpr (F32C) {
        const float* qp = (const float*)a.q + qat + 4 * p;
#pragma unroll
        for (int t = 0; t < D / 16; t++) qf[t] = *(const v4f*)(qp + 16 * t);
    } else if constexpr (F32Q) {
        const float* qp = (const float*)a.q + qat + 8 * p;
#pragma unroll
        for (int t = 0; t < D / 32; t++) {
            const v4f y0 = *(const v4f*)(qp + 32 * t), y1 = *(const v4f*)(qp + 32 * t + 4);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                float t0[3], t1[3];
                three_terms(e < 2 ? y0[2 * e] : y1[2 * e - 4], t0);
                three_terms(e < 2 ? y0[2 * e + 1] : y1[2 * e - 3], t1);
#pragma unroll
                for (int z = 0; z < TERMS; z++) q[z][t][e] = pack_bf16(t0[z], t1[z]);
            }
        }
    } else {
        const uint16_t* qp = (const uint16_t*)a.q + qat + 8 * p;
#pragma unroll
        for (int t = 0; t < D / 32; t++) q[0][t] = *(const v4u*)(qp + 32 * t);
    }

    v4f acc[DT];
#pragma unroll
    for (int t = 0; t < DT; t++) acc[t] = v4f{0, 0, 0, 0};
    float m = -__builtin_huge_valf(), l = 0.0f;

    T kv;
    constexpr int BLOCKS = N / 16;
    const char *kc = (const char*)a.kv.k, *vc = (const char*)a.kv.v;
    auto load_k = [&](const size_t (&off)[BLOCKS]) {
        if constexpr (F32C) {
            const float* kp = (const float*)kc + off[0] + r * D + 4 * p;
#pragma unroll
            for (int t = 0; t < T::KS; t++) kv.k[t] = *(const v4f*)(kp + 16 * t);
        } else {
#pragma unroll
            for (int b = 0; b < BLOCKS; b++) {
                const uint16_t* kp = (const uint16_t*)kc + off[b] + r * D + 8 * p;
#pragma unroll
                for (int t = 0; t < T::KS; t++) kv.k[b][t] = stream<TERMS == 1>(kp + 32 * t);
            }
        }
    };
    auto load_v = [&](const size_t (&off)[BLOCKS]) {
        if constexpr (F32C) {
            const float* vp = (const float*)vc + off[0] + 4 * p * D + 4 * r;
#pragma unroll
            for (int v = 0; v < 4; v++)
#pragma unroll
                for (int h = 0; h < T::VH; h++) kv.v[v][h] = *(const v4f*)(vp + v * D + 64 * h);
        } else {
#pragma unroll
            for (int i = 0; i < T::VI; i++) {
                const uint16_t* vp = (const uint16_t*)vc + off[i * T::RPI / 16] + (i * T::RPI % 16) * D + lane * 8;
                kv.v[i] = stream<TERMS == 1>(vp);
            }
        }
    };
    // pages of a tile's blocks, and their offsets
    auto pages_of = [&](int j, int (&pg)[BLOCKS], size_t (&off)[BLOCKS]) {
#pragma unroll
        for (int b = 0; b < BLOCKS; b++) {
            pg[b] = page_at(a, s, j + 16 * b, end);
            off[b] = slot_off(a, pg[b], g, j + 16 * b, D);
        }
    };

    int pg[BLOCKS], pn[BLOCKS];
    size_t off[BLOCKS], on[BLOCKS];
    int j = beg + N * w, odd_lo = INT32_MAX, odd_hi = 0;  // odd: the wave's tiles with values that are not finite
    if (j < end) {
        pages_of(j, pg, off);
        load_k(off);
        load_v(off);
    }
    if constexpr (F32C) {
#pragma unroll
        for (int t = 0; t < D / 16; t++) arrived(qf[t]);
    } else {
#pragma unroll
        for (int z = 0; z < TERMS; z++)
#pragma unroll
            for (int t = 0; t < D / 32; t++) arrived(q[z][t]);
    }
    for (; j < end; j += N * FEW_WAVES) {
        const int jn = j + N * FEW_WAVES;
        pages_of(jn, pn, on);
        // scores: lane (r, p) has block b's positions 4 p + e
        v4f sc[BLOCKS];
#pragma unroll
        for (int b = 0; b < BLOCKS; b++) {
            v4f t = {0, 0, 0, 0};
            if constexpr (F32C) {
#pragma unroll
                for (int i = 0; i < T::KS; i++)
#pragma unroll
                    for (int e = 0; e < 4; e++) t = __builtin_amdgcn_mfma_f32_16x16x4f32(kv.k[i][e], qf[i][e], t, 0, 0, 0);
            } else {
#pragma unroll
                for (int z = TERMS - 1; z >= 0; z--)
#pragma unroll
                    for (int i = 0; i < T::KS; i++)
                        t = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8b, kv.k[b][i]), __builtin_bit_cast(v8b, q[z][i]), t, 0, 0, 0);
            }
            sc[b] = t;
        }
        if (jn < end) load_k(on);
        bool hole = false;
#pragma unroll
        for (int b = 0; b < BLOCKS; b++) hole |= pg[b] < 0;
        const bool masked = hole || j + N > least;
        auto seen = [&](int b, int e) { return pg[b] >= 0 && j + 16 * b + 4 * p + e < sees; };
        if (masked) {
#pragma unroll
            for (int b = 0; b < BLOCKS; b++)
#pragma unroll
                for (int e = 0; e < 4; e++) sc[b][e] = seen(b, e) ? sc[b][e] : -__builtin_huge_valf();
        }
        if constexpr (TERMS > 1) {
            // an infinity times the terms of a q may be inf - inf: such scores again, product by product
            float sum = 0.0f;
#pragma unroll
            for (int b = 0; b < BLOCKS; b++)
#pragma unroll
                for (int e = 0; e < 4; e++) sum += sc[b][e];
            if (__any(sum != sum)) {
#pragma unroll
                for (int b = 0; b < BLOCKS; b++)
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        if (sc[b][e] != sc[b][e]) {
                            const float* qp = (const float*)a.q + qat;
                            const uint16_t* kp = (const uint16_t*)kc + off[b] + (4 * p + e) * D;
                            float t = 0.0f;
                            for (int d = 0; d < D; d++) t = fmaf(qp[d], __uint_as_float((uint32_t)kp[d] << 16), t);
                            sc[b][e] = t;
                        }
            }
        }
        // the running maximum, probabilities and sums
        float mx = masked ? -__builtin_huge_valf() : -FLT_MAX;
#pragma unroll
        for (int b = 0; b < BLOCKS; b++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float y = sc[b][e] * a.c;
                mx = fmaxf(mx, masked && seen(b, e) ? fmaxf(y, -FLT_MAX) : y);
            }
        mx = fmaxf(mx, lane_xor<16>(mx));
        mx = fmaxf(mx, lane_xor<32>(mx));
        const float mn = fmaxf(m, mx + ABOVE), mu = fmaxf(mn, -FLT_MAX);
        if (__any(mn != m)) {
            const float al = __builtin_amdgcn_exp2f(m - mu);
            l *= al;
#pragma unroll
            for (int t = 0; t < DT; t++) acc[t] *= al;
        }
        m = mn;
        const bool far = far_score(mu);
#pragma unroll
        for (int b = 0; b < BLOCKS; b++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float y = __builtin_amdgcn_exp2f(far ? sc[b][e] * a.c - mu : fmaf(sc[b][e], a.c, -mu));
                sc[b][e] = y;
                l += y;
            }
        // values: rows no row sees are zeroed, and so is what is not finite
        // where some row must not meet it (meet_odd)
        bool odd = false;
        if constexpr (F32C) {
            if (masked) {
                uint32_t bits = 0;
#pragma unroll
                for (int v = 0; v < 4; v++) {
                    const bool gone = hole || j + 4 * p + v >= end;
#pragma unroll
                    for (int h = 0; h < T::VH; h++) {
                        if (gone) kv.v[v][h] = v4f{0, 0, 0, 0};
                        mark_odd<true>(__builtin_bit_cast(v4u, kv.v[v][h]), bits);
                    }
                }
                odd = __any(is_odd<true>(bits));
                if (odd) {
#pragma unroll
                    for (int v = 0; v < 4; v++)
#pragma unroll
                        for (int h = 0; h < T::VH; h++)
                            kv.v[v][h] = __builtin_bit_cast(v4f, finite_part<true>(__builtin_bit_cast(v4u, kv.v[v][h])));
                }
            }
#pragma unroll
            for (int v = 0; v < 4; v++)
#pragma unroll
                for (int h = 0; h < T::VH; h++)
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        acc[4 * h + e] = __builtin_amdgcn_mfma_f32_16x16x4f32(kv.v[v][h][e], sc[0][v], acc[4 * h + e], 0, 0, 0);
            if (jn < end) load_v(on);
        } else {
            if (masked) {
#pragma unroll
                for (int i = 0; i < T::VI; i++) {
                    const int row = i * T::RPI + lane / (D / 8);
                    if (pg[i * T::RPI / 16] < 0 || j + row >= end) kv.v[i] = v4u{0, 0, 0, 0};
                }
            }
            if (masked || TERMS > 1) {
                uint32_t bits = 0;
#pragma unroll
                for (int i = 0; i < T::VI; i++) mark_odd<false>(kv.v[i], bits);
                odd = __any(is_odd<false>(bits));
                if (odd) {
#pragma unroll
                    for (int i = 0; i < T::VI; i++) kv.v[i] = finite_part<false>(kv.v[i]);
                }
            }
#pragma unroll
            for (int i = 0; i < T::VI; i++)
                *(v4u*)(own + lds_slot<2 * D>(i * T::RPI + lane / (D / 8), lane % (D / 8))) = kv.v[i];
            if (jn < end) load_v(on);
            __builtin_amdgcn_wave_barrier();
            v4u pb[TERMS];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float y0 = sc[e / 2][2 * (e % 2)], y1 = sc[e / 2][2 * (e % 2) + 1];
                if constexpr (TERMS == 1) {
                    pb[0][e] = pack_bf16(y0, y1);
                } else {
                    float t0[3], t1[3];
                    three_terms(y0, t0);
                    three_terms(y1, t1);
#pragma unroll
                    for (int z = 0; z < TERMS; z++) pb[z][e] = pack_bf16(t0[z], t1[z]);
                }
            }
            // lane -> (row 4 p + r / 4 of each block, 4 of 16 columns)
            const int vrow = 4 * p + (r >> 2), ch = (r >> 1) & 1, in = 8 * (r & 1);
#pragma unroll
            for (int t = 0; t < DT; t++) {
                const v8b va = join_halves(read_transposed(own + lds_slot<2 * D>(vrow, 2 * t + ch) + in),
                                           read_transposed(own + lds_slot<2 * D>(vrow + 16, 2 * t + ch) + in));
#pragma unroll
                for (int z = TERMS - 1; z >= 0; z--)
                    acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(va, __builtin_bit_cast(v8b, pb[z]), acc[t], 0, 0, 0);
            }
            __builtin_amdgcn_wave_barrier();
        }
        if (odd) odd_lo = min(odd_lo, j), odd_hi = j + N;
#pragma unroll
        for (int b = 0; b < BLOCKS; b++) pg[b] = pn[b], off[b] = on[b];
    }

    if (odd_hi) {
        typedef typename std::conditional<F32Q, float, uint16_t>::type TQ;
        typedef typename std::conditional<F32C, float, uint16_t>::type TC;
        meet_odd<TQ, TC, D>(a, s, g, odd_lo, odd_hi, N, N * FEW_WAVES, end, (const TQ*)a.q + qat, sees, m,
                            [&](const TC* v, bool see, auto value, auto probability) {
            bool any = false;
#pragma unroll
            for (int t = 0; t < DT; t++)
#pragma unroll
                for (int e = 0; e < 4; e++) any |= !(fabsf(value(v + few_column<F32C>(t, p, e))) < __builtin_huge_valf());
            if (!any || !see) return;
            const float y = probability();
#pragma unroll
            for (int t = 0; t < DT; t++) {
                v4f add;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float x = value(v + few_column<F32C>(t, p, e));
                    add[e] = fabsf(x) < __builtin_huge_valf() ? 0.0f : y * x;
                }
                acc[t] += add;
            }
        });
    }

    // the waves' parts together
    l += lane_xor<16>(l);
    l += lane_xor<32>(l);
    if (p == 0) sml[w][r] = make_float2(m, l);
    __syncthreads();
    constexpr int F4 = D / 4;  // float4 of a row, at places that differ by row
    float mt = -__builtin_huge_valf();
#pragma unroll
    for (int k = 0; k < FEW_WAVES; k++) mt = fmaxf(mt, sml[k][r].x);
    const float f = __builtin_amdgcn_exp2f(m - fmaxf(mt, -FLT_MAX));
#pragma unroll
    for (int t = 0; t < DT; t++) {
        v4f y = acc[t];
        if constexpr (F32C) y = v4f{acc[t & ~3][t % 4], acc[(t & ~3) + 1][t % 4], acc[(t & ~3) + 2][t % 4], acc[(t & ~3) + 3][t % 4]};
        const int c4 = F32C ? 16 * (t / 4) + 4 * p + t % 4 : 4 * t + p;
        *(v4f*)(own + ((r * F4) + (c4 ^ r)) * 16) = y * f;
    }
    __syncthreads();
    const int rr = tid >> 4;
    if (rr >= packed) return;
    float mr = -__builtin_huge_valf(), lr = 0.0f;
#pragma unroll
    for (int k = 0; k < FEW_WAVES; k++) mr = fmaxf(mr, sml[k][rr].x);
#pragma unroll
    for (int k = 0; k < FEW_WAVES; k++) lr += sml[k][rr].y * __builtin_amdgcn_exp2f(sml[k][rr].x - fmaxf(mr, -FLT_MAX));
    const int ir = (row0 + rr) / G;
    const size_t orow = s.first + ir, ohead = g * G + (row0 + rr - ir * G);
    const bool none = mr == -__builtin_huge_valf();
    const float inv = none ? 0.0f : 1.0f / lr;
    const size_t at = ((size_t)(piece + (PREFIX ? a.own.pieces : 0)) * a.batch.rows + orow) * a.heads + ohead;
    if (a.part && (tid & 15) == 0) a.ml[at] = make_float2(mr, lr);
#pragma unroll
    for (int k = 0; k < F4 / 16; k++) {
        const int c4 = (tid & 15) + 16 * k;
        v4f y = {0, 0, 0, 0};
#pragma unroll
        for (int v = 0; v < FEW_WAVES; v++) y += *(const v4f*)(sm + v * WBYTES + ((rr * F4) + (c4 ^ rr)) * 16);
        if (a.part) {
            *(v4f*)(a.part + at * D + 4 * c4) = y;
            continue;
        }
        y = none ? v4f{0, 0, 0, 0} : y * inv;
        const size_t o = orow * a.os + ohead * D + 4 * c4;
        if constexpr (F32Q) *(v4f*)((float*)a.out + o) = y;
        else *(uint2*)((uint16_t*)a.out + o) = make_uint2(pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3]));
    }
}

}  // namespace
}  // namespace lq8
