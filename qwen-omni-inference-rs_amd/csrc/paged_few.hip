// paged_few.hip -- attention over a paged cache for up to 32 packed rows a kv
// head: single tokens, and a few drafted ones (gfx950).
//
// Bound: the cache's bytes.  Each of a workgroup's four waves runs its own
// online softmax over tiles of the piece (32 positions of bf16 pages, 16 of
// f32: 16 KiB of K and V at head_dim 128), with no barrier before the end: the
// next tile's K goes out when the scores are done and its V when this one's has
// left its registers, so a wave always has about a tile in flight.
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
#include <type_traits>

#include "paged_attn.h"

namespace lq8 {
namespace {

constexpr int WAVES = 4;

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
__device__ __forceinline__ int column(int t, int p, int e) {
    return F32C ? 64 * (t / 4) + 16 * p + 4 * e + t % 4 : 16 * t + 4 * p + e;
}

template <int TYPES, int D, int MB, bool PREFIX>
__global__ __launch_bounds__(64 * WAVES, MB == 1 ? 2 : 1) void k_few(AttnArgs a) {
    constexpr bool F32C = TYPES == PT_F32_F32, F32Q = TYPES != PT_BF16_BF16;
    constexpr int TERMS = TYPES == PT_F32_BF16 ? 3 : 1;
    typedef Tile<TYPES, D> T;
    constexpr int N = T::N, M = 16 * MB, DT = D / 16;
    // a wave's V tile, and its 16 x D sums at the end
    constexpr int WBYTES = 16 * D * 4;
    static_assert(WBYTES >= 32 * D * 2, "one wave's region");
    __shared__ __attribute__((aligned(16))) char sm[WAVES * WBYTES];
    __shared__ float2 sml[WAVES][M];
    const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, p = lane >> 4;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    char* own = sm + w * WBYTES;

    // workgroup -> (piece, span, row tile, kv head), kv head fastest: the
    // workgroups of one go to one XCD where their number divides by eight
    const int G = a.group, kvh = a.kv.kv_heads;
    int x = blockIdx.x;
    const int g = x % kvh;
    x /= kvh;
    const int spans = PREFIX ? a.prefix.groups : a.batch.batch;
    const int sp = x % spans, piece = x / spans;
    const Span s = PREFIX ? prefix_span(a, sp) : own_span(a, sp);
    const int packed = min(s.count * G, M);
    if (packed <= 0) return;
    const int len = piece_len(s.length, PREFIX ? a.pre : a.own);
    const int most = s.sees((packed - 1) / G), least = s.sees(0);
    const int beg = piece * len, end = min(beg + len, most);
    if (a.part ? beg >= most : piece > 0) return;

    // this lane's rows
    int sees[MB];
    size_t at[MB];  // row * heads + head
    bool valid[MB];
    uint32_t q[MB][F32C ? 1 : TERMS][F32C ? 1 : D / 32][4];
    float qf[F32C ? MB : 1][D / 4];
#pragma unroll
    for (int mb = 0; mb < MB; mb++) {
        const int pr = 16 * mb + r, i = pr / G;
        valid[mb] = pr < packed;
        sees[mb] = valid[mb] ? s.sees(i) : 0;
        const int row = s.first + (valid[mb] ? i : 0), head = g * G + (valid[mb] ? pr - i * G : 0);
        at[mb] = (size_t)row * a.heads + head;
        if constexpr (F32C) {
            const float* qp = (const float*)a.q + row * a.qs + (size_t)head * D + 4 * p;
#pragma unroll
            for (int t = 0; t < D / 16; t++) {
                const float4 v = *(const float4*)(qp + 16 * t);
                qf[mb][4 * t] = v.x, qf[mb][4 * t + 1] = v.y, qf[mb][4 * t + 2] = v.z, qf[mb][4 * t + 3] = v.w;
            }
        } else if constexpr (F32Q) {
            const float* qp = (const float*)a.q + row * a.qs + (size_t)head * D + 8 * p;
#pragma unroll
            for (int t = 0; t < D / 32; t++) {
                const float4 y0 = *(const float4*)(qp + 32 * t), y1 = *(const float4*)(qp + 32 * t + 4);
                const float y[8] = {y0.x, y0.y, y0.z, y0.w, y1.x, y1.y, y1.z, y1.w};
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    float t0[3], t1[3];
                    three_terms(y[2 * e], t0);
                    three_terms(y[2 * e + 1], t1);
#pragma unroll
                    for (int z = 0; z < TERMS; z++) q[mb][z][t][e] = pack_bf16(t0[z], t1[z]);
                }
            }
        } else {
            const uint16_t* qp = (const uint16_t*)a.q + row * a.qs + (size_t)head * D + 8 * p;
#pragma unroll
            for (int t = 0; t < D / 32; t++) {
                const v4u v = *(const v4u*)(qp + 32 * t);
                q[mb][0][t][0] = v[0], q[mb][0][t][1] = v[1], q[mb][0][t][2] = v[2], q[mb][0][t][3] = v[3];
            }
        }
    }

    v4f acc[MB][DT];
    float m[MB], l[MB];
#pragma unroll
    for (int mb = 0; mb < MB; mb++) {
        m[mb] = -__builtin_huge_valf(), l[mb] = 0.0f;
#pragma unroll
        for (int t = 0; t < DT; t++) acc[mb][t] = v4f{0, 0, 0, 0};
    }

    T tile;
    constexpr int BLOCKS = N / 16;
    const char *kc = (const char*)a.kv.k, *vc = (const char*)a.kv.v;
    auto load_k = [&](const size_t (&off)[BLOCKS]) {
        if constexpr (F32C) {
            const float* kp = (const float*)kc + off[0] + r * D + 4 * p;
#pragma unroll
            for (int t = 0; t < T::KS; t++) tile.k[t] = *(const v4f*)(kp + 16 * t);
        } else {
#pragma unroll
            for (int b = 0; b < BLOCKS; b++) {
                const uint16_t* kp = (const uint16_t*)kc + off[b] + r * D + 8 * p;
#pragma unroll
                for (int t = 0; t < T::KS; t++) tile.k[b][t] = stream<TERMS == 1>(kp + 32 * t);
            }
        }
    };
    auto load_v = [&](const size_t (&off)[BLOCKS]) {
        if constexpr (F32C) {
            const float* vp = (const float*)vc + off[0] + 4 * p * D + 4 * r;
#pragma unroll
            for (int v = 0; v < 4; v++)
#pragma unroll
                for (int h = 0; h < T::VH; h++) tile.v[v][h] = *(const v4f*)(vp + v * D + 64 * h);
        } else {
#pragma unroll
            for (int i = 0; i < T::VI; i++) {
                const uint16_t* vp = (const uint16_t*)vc + off[i * T::RPI / 16] + (i * T::RPI % 16) * D + lane * 8;
                tile.v[i] = stream<TERMS == 1>(vp);
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
#pragma unroll
    for (int mb = 0; mb < MB; mb++) {
        if constexpr (F32C) {
#pragma unroll
            for (int t = 0; t < D / 4; t++) arrived(qf[mb][t]);
        } else {
#pragma unroll
            for (int z = 0; z < TERMS; z++)
#pragma unroll
                for (int t = 0; t < D / 32; t++)
#pragma unroll
                    for (int e = 0; e < 4; e++) arrived(q[mb][z][t][e]);
        }
    }
    for (; j < end; j += N * WAVES) {
        const int jn = j + N * WAVES;
        pages_of(jn, pn, on);
        // scores: lane (r, p) has block b's positions 4 p + e
        v4f sc[MB][BLOCKS];
#pragma unroll
        for (int mb = 0; mb < MB; mb++)
#pragma unroll
            for (int b = 0; b < BLOCKS; b++) {
                v4f t = {0, 0, 0, 0};
                if constexpr (F32C) {
#pragma unroll
                    for (int i = 0; i < T::KS; i++) {
                        t = __builtin_amdgcn_mfma_f32_16x16x4f32(tile.k[i][0], qf[mb][4 * i], t, 0, 0, 0);
                        t = __builtin_amdgcn_mfma_f32_16x16x4f32(tile.k[i][1], qf[mb][4 * i + 1], t, 0, 0, 0);
                        t = __builtin_amdgcn_mfma_f32_16x16x4f32(tile.k[i][2], qf[mb][4 * i + 2], t, 0, 0, 0);
                        t = __builtin_amdgcn_mfma_f32_16x16x4f32(tile.k[i][3], qf[mb][4 * i + 3], t, 0, 0, 0);
                    }
                } else {
#pragma unroll
                    for (int z = TERMS - 1; z >= 0; z--)
#pragma unroll
                        for (int i = 0; i < T::KS; i++) {
                            const v4u qv = v4u{q[mb][z][i][0], q[mb][z][i][1], q[mb][z][i][2], q[mb][z][i][3]};
                            t = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8b, tile.k[b][i]),
                                                                       __builtin_bit_cast(v8b, qv), t, 0, 0, 0);
                        }
                }
                sc[mb][b] = t;
            }
        if (jn < end) load_k(on);
        bool hole = false;
#pragma unroll
        for (int b = 0; b < BLOCKS; b++) hole |= pg[b] < 0;
        const bool masked = hole || j + N > least;
        auto seen = [&](int mb, int b, int e) { return pg[b] >= 0 && j + 16 * b + 4 * p + e < sees[mb]; };
        if (masked) {
#pragma unroll
            for (int mb = 0; mb < MB; mb++)
#pragma unroll
                for (int b = 0; b < BLOCKS; b++)
#pragma unroll
                    for (int e = 0; e < 4; e++) sc[mb][b][e] = seen(mb, b, e) ? sc[mb][b][e] : -__builtin_huge_valf();
        }
        if constexpr (TERMS > 1) {
            // an infinity times the terms of a q may be inf - inf: such scores again, product by product
            float sum = 0.0f;
#pragma unroll
            for (int mb = 0; mb < MB; mb++)
#pragma unroll
                for (int b = 0; b < BLOCKS; b++)
#pragma unroll
                    for (int e = 0; e < 4; e++) sum += sc[mb][b][e];
            if (__any(sum != sum)) {
#pragma unroll
                for (int mb = 0; mb < MB; mb++)
#pragma unroll
                    for (int b = 0; b < BLOCKS; b++)
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            if (sc[mb][b][e] != sc[mb][b][e]) {
                                const float* qp = (const float*)a.q + (at[mb] / a.heads) * a.qs + (at[mb] % a.heads) * D;
                                const uint16_t* kp = (const uint16_t*)kc + off[b] + (4 * p + e) * D;
                                float t = 0.0f;
                                for (int d = 0; d < D; d++) t = fmaf(qp[d], __uint_as_float((uint32_t)kp[d] << 16), t);
                                sc[mb][b][e] = t;
                            }
            }
        }
        // the running maximum, probabilities and sums
#pragma unroll
        for (int mb = 0; mb < MB; mb++) {
            float mx = masked ? -__builtin_huge_valf() : -FLT_MAX;
#pragma unroll
            for (int b = 0; b < BLOCKS; b++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float y = sc[mb][b][e] * a.c;
                    mx = fmaxf(mx, masked && seen(mb, b, e) ? fmaxf(y, -FLT_MAX) : y);
                }
            mx = fmaxf(mx, lane_xor<16>(mx));
            mx = fmaxf(mx, lane_xor<32>(mx));
            const float mn = fmaxf(m[mb], mx), mu = fmaxf(mn, -FLT_MAX);
            if (__any(mn != m[mb])) {
                const float al = __builtin_amdgcn_exp2f(m[mb] - mu);
                l[mb] *= al;
#pragma unroll
                for (int t = 0; t < DT; t++) acc[mb][t] *= al;
            }
            m[mb] = mn;
            const bool far = __any(far_score(mu));
#pragma unroll
            for (int b = 0; b < BLOCKS; b++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float y = __builtin_amdgcn_exp2f(far ? sc[mb][b][e] * a.c - mu : fmaf(sc[mb][b][e], a.c, -mu));
                    sc[mb][b][e] = y;
                    l[mb] += y;
                }
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
                        if (gone) tile.v[v][h] = v4f{0, 0, 0, 0};
                        mark_odd<true>(__builtin_bit_cast(v4u, tile.v[v][h]), bits);
                    }
                }
                odd = __any(is_odd<true>(bits));
                if (odd) {
#pragma unroll
                    for (int v = 0; v < 4; v++)
#pragma unroll
                        for (int h = 0; h < T::VH; h++)
                            tile.v[v][h] = __builtin_bit_cast(v4f, finite_part<true>(__builtin_bit_cast(v4u, tile.v[v][h])));
                }
            }
#pragma unroll
            for (int mb = 0; mb < MB; mb++)
#pragma unroll
                for (int v = 0; v < 4; v++)
#pragma unroll
                    for (int h = 0; h < T::VH; h++) {
                        const float y = sc[mb][0][v];
                        acc[mb][4 * h] = __builtin_amdgcn_mfma_f32_16x16x4f32(tile.v[v][h][0], y, acc[mb][4 * h], 0, 0, 0);
                        acc[mb][4 * h + 1] = __builtin_amdgcn_mfma_f32_16x16x4f32(tile.v[v][h][1], y, acc[mb][4 * h + 1], 0, 0, 0);
                        acc[mb][4 * h + 2] = __builtin_amdgcn_mfma_f32_16x16x4f32(tile.v[v][h][2], y, acc[mb][4 * h + 2], 0, 0, 0);
                        acc[mb][4 * h + 3] = __builtin_amdgcn_mfma_f32_16x16x4f32(tile.v[v][h][3], y, acc[mb][4 * h + 3], 0, 0, 0);
                    }
            if (jn < end) load_v(on);
        } else {
            if (masked) {
#pragma unroll
                for (int i = 0; i < T::VI; i++) {
                    const int row = i * T::RPI + lane / (D / 8);
                    if (pg[i * T::RPI / 16] < 0 || j + row >= end) tile.v[i] = v4u{0, 0, 0, 0};
                }
            }
            if (masked || TERMS > 1) {
                uint32_t bits = 0;
#pragma unroll
                for (int i = 0; i < T::VI; i++) mark_odd<false>(tile.v[i], bits);
                odd = __any(is_odd<false>(bits));
                if (odd) {
#pragma unroll
                    for (int i = 0; i < T::VI; i++) tile.v[i] = finite_part<false>(tile.v[i]);
                }
            }
#pragma unroll
            for (int i = 0; i < T::VI; i++)
                *(v4u*)(own + lds_slot<2 * D>(i * T::RPI + lane / (D / 8), lane % (D / 8))) = tile.v[i];
            if (jn < end) load_v(on);
            __builtin_amdgcn_wave_barrier();
            uint32_t pb[MB][TERMS][4];
#pragma unroll
            for (int mb = 0; mb < MB; mb++)
#pragma unroll
                for (int b = 0; b < BLOCKS; b++)
#pragma unroll
                    for (int e = 0; e < 4; e += 2) {
                        const float y0 = sc[mb][b][e], y1 = sc[mb][b][e + 1];
                        if constexpr (TERMS == 1) {
                            pb[mb][0][2 * b + e / 2] = pack_bf16(y0, y1);
                        } else {
                            float t0[3], t1[3];
                            three_terms(y0, t0);
                            three_terms(y1, t1);
#pragma unroll
                            for (int z = 0; z < TERMS; z++) pb[mb][z][2 * b + e / 2] = pack_bf16(t0[z], t1[z]);
                        }
                    }
            // lane -> (row 4 p + r / 4 of each block, 4 of 16 columns)
#pragma unroll
            for (int t = 0; t < DT; t++) {
                const int row = 4 * p + (r >> 2), ch = 2 * t + ((r >> 1) & 1), in = 8 * (r & 1);
                const v8b va = join_halves(read_transposed(own + lds_slot<2 * D>(row, ch) + in),
                                           read_transposed(own + lds_slot<2 * D>(row + 16, ch) + in));
#pragma unroll
                for (int mb = 0; mb < MB; mb++)
#pragma unroll
                    for (int z = TERMS - 1; z >= 0; z--) {
                        const v4u pv = v4u{pb[mb][z][0], pb[mb][z][1], pb[mb][z][2], pb[mb][z][3]};
                        acc[mb][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(va, __builtin_bit_cast(v8b, pv), acc[mb][t], 0, 0, 0);
                    }
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
#pragma unroll
        for (int mb = 0; mb < MB; mb++) {
            const TQ* qp = (const TQ*)a.q + (at[mb] / a.heads) * a.qs + (at[mb] % a.heads) * D;
            meet_odd<TQ, TC, D>(a, s, g, odd_lo, odd_hi, N, N * WAVES, end, qp, sees[mb], m[mb], [&](const TC* v, bool seen, auto value, auto probability) {
                bool any = false;
#pragma unroll
                for (int t = 0; t < DT; t++)
#pragma unroll
                    for (int e = 0; e < 4; e++) any |= !(fabsf(value(v + column<F32C>(t, p, e))) < __builtin_huge_valf());
                if (!any || !seen) return;
                const float y = probability();
#pragma unroll
                for (int t = 0; t < DT; t++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const float x = value(v + column<F32C>(t, p, e));
                        if (!(fabsf(x) < __builtin_huge_valf())) acc[mb][t][e] = fmaf(y, x, acc[mb][t][e]);
                    }
            });
        }
    }

    // the waves' parts together
#pragma unroll
    for (int mb = 0; mb < MB; mb++) {
        l[mb] += lane_xor<16>(l[mb]);
        l[mb] += lane_xor<32>(l[mb]);
        if (p == 0) sml[w][16 * mb + r] = make_float2(m[mb], l[mb]);
    }
    __syncthreads();
    constexpr int F4 = D / 4;  // float4 of a row
#pragma unroll
    for (int mb = 0; mb < MB; mb++) {
        if (mb) __syncthreads();
        float mt = -__builtin_huge_valf();
#pragma unroll
        for (int k = 0; k < WAVES; k++) mt = fmaxf(mt, sml[k][16 * mb + r].x);
        const float f = __builtin_amdgcn_exp2f(m[mb] - fmaxf(mt, -FLT_MAX));
#pragma unroll
        for (int t = 0; t < DT; t++) {
            v4f y;
            int c4;  // which float4 of the row
            if constexpr (F32C) {
                const int h = t / 4, e = t % 4;
                y = v4f{acc[mb][4 * h][e], acc[mb][4 * h + 1][e], acc[mb][4 * h + 2][e], acc[mb][4 * h + 3][e]};
                c4 = 16 * h + 4 * p + e;
            } else {
                y = acc[mb][t];
                c4 = 4 * t + p;
            }
            *(v4f*)(own + ((r * F4) + (c4 ^ r)) * 16) = y * f;
        }
        __syncthreads();
        const int rr = tid >> 4, pr = 16 * mb + rr;
        if (pr < packed) {
            float M2 = -__builtin_huge_valf(), L = 0.0f;
#pragma unroll
            for (int k = 0; k < WAVES; k++) M2 = fmaxf(M2, sml[k][pr].x);
#pragma unroll
            for (int k = 0; k < WAVES; k++) L += sml[k][pr].y * __builtin_amdgcn_exp2f(sml[k][pr].x - fmaxf(M2, -FLT_MAX));
            const int i = pr / G;
            const size_t row = s.first + i, head = g * G + (pr - i * G);
            const bool none = M2 == -__builtin_huge_valf();
            const float inv = none ? 0.0f : 1.0f / L;
            float* po = nullptr;
            if (a.part) {
                const size_t slot = piece + (PREFIX ? a.own.pieces : 0), k = (slot * a.batch.rows + row) * a.heads + head;
                if ((tid & 15) == 0) a.ml[k] = make_float2(M2, L);
                po = a.part + k * D;
            }
#pragma unroll
            for (int k = 0; k < F4 / 16; k++) {
                const int c4 = (tid & 15) + 16 * k;
                v4f y = {0, 0, 0, 0};
#pragma unroll
                for (int v = 0; v < WAVES; v++) y += *(const v4f*)(sm + v * WBYTES + ((rr * F4) + (c4 ^ rr)) * 16);
                if (a.part) {
                    *(v4f*)(po + 4 * c4) = y;
                    continue;
                }
                y = none ? v4f{0, 0, 0, 0} : y * inv;
                const size_t o = row * a.os + head * D + 4 * c4;
                if constexpr (F32Q) *(v4f*)((float*)a.out + o) = y;
                else *(uint2*)((uint16_t*)a.out + o) = make_uint2(pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3]));
            }
        }
    }
}

template <int TYPES, int D, int MB>
void launch_one(hipStream_t s, const AttnArgs& a, bool prefix) {
    const Cut& c = prefix ? a.pre : a.own;
    const unsigned n = (unsigned)((size_t)a.kv.kv_heads * (prefix ? a.prefix.groups : a.batch.batch) * c.pieces);
    if (prefix) hipLaunchKernelGGL((k_few<TYPES, D, MB, true>), dim3(n), dim3(64 * WAVES), 0, s, a);
    else hipLaunchKernelGGL((k_few<TYPES, D, MB, false>), dim3(n), dim3(64 * WAVES), 0, s, a);
}
template <int TYPES>
void launch_types(hipStream_t s, const AttnArgs& a, int dim, int blocks, bool prefix) {
    if (dim == 64 && blocks == 1) launch_one<TYPES, 64, 1>(s, a, prefix);
    else if (dim == 64) launch_one<TYPES, 64, 2>(s, a, prefix);
    else if (blocks == 1) launch_one<TYPES, 128, 1>(s, a, prefix);
    else launch_one<TYPES, 128, 2>(s, a, prefix);
}

}  // namespace

// blocks: 16-row blocks of a workgroup (1 or 2); every span has at most 16 blocks packed rows
lq8_status launch_few(hipStream_t s, const AttnArgs& a, PagedTypes types, int dim, int blocks, bool prefix) {
    if (types == PT_F32_F32) launch_types<PT_F32_F32>(s, a, dim, blocks, prefix);
    else if (types == PT_F32_BF16) launch_types<PT_F32_BF16>(s, a, dim, blocks, prefix);
    else launch_types<PT_BF16_BF16>(s, a, dim, blocks, prefix);
    LQ8_HIP(hipGetLastError());
    return LQ8_OK;
}

}  // namespace lq8
