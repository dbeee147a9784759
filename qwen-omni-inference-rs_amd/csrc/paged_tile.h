// paged_tile.h -- attention over a paged cache for many packed rows a kv
// head: prompt chunks, and the rows of a group that share a prefix (gfx950).
//
// A workgroup has 128 packed rows, 32 to a wave, and goes over its piece in
// tiles of 64 positions (bf16 pages: K and V in LDS, two buffers, the next
// tile's loads out while this one is computed) or 32 (f32 pages, one buffer).
// The rows are the columns of the products (32 x 32 tiles): S^T = K Q^T leaves
// lane (row = lane % 32, p = lane / 32) with the scores of positions 8 i + 4 p
// .. + 3 of its row, which is the B operand of O^T = V^T P^T when the 16
// positions of a product are taken in the order (4 p + e, 8 + 4 p + e): the
// probabilities stay where they are, the maximum needs one exchange with lane
// +- 32, and the rescaling of O none.  V is read transposed (ds_read_tr).
// f32 rows: three bf16 terms of q and p each; f32 pages: of K and V too.
//
// Bound: the matrix cores are busy 37 % of the cycles, the vector instructions
// 47 % (a bf16 chunk), and the two waves of a SIMD overlap them only in part.  Chunks of up to 2048 rows of three sequences over up to
// 6100 positions, 32 heads over 8 of 128, bf16: 369 us, 890 TFLOP/s (a large
// library product reaches 1204).  Tiles of 32 positions and three workgroups a
// compute unit: 418 us; scores computed a tile ahead: no change.
#pragma once

#include <type_traits>

#include "paged_attn.h"

namespace lq8 {
namespace {

// A workgroup's rows and positions.
struct Work {
    Span s;
    int g, piece, row0, packed, beg, end;
};
// Block -> (row tile, piece, kv head), kv head fastest (one to an XCD where
// there are eight); a sequence's last rows, which see most, first.  false:
// nothing to do.
template <bool PREFIX>
__device__ __forceinline__ bool find_work(const AttnArgs& a, int block, Work* k) {
    const Cut& cut = PREFIX ? a.pre : a.own;
    const int kvh = a.kv.kv_heads, x = block / kvh;
    k->g = block % kvh;
    k->piece = x % cut.pieces;
    int sp, tile;
    if (!find_tile<TILE_PACKED, PREFIX>(a, x / cut.pieces, &sp, &tile)) return false;
    k->s = PREFIX ? prefix_span(a, sp) : own_span(a, sp);
    const int rows = k->s.count * a.group;
    k->row0 = ((rows + TILE_PACKED - 1) / TILE_PACKED - 1 - tile) * TILE_PACKED;
    k->packed = min(rows - k->row0, TILE_PACKED);
    const int len = piece_len(k->s.length, cut), most = k->s.sees((k->row0 + k->packed - 1) / a.group);
    k->beg = k->piece * len;
    k->end = min(k->beg + len, most);
    return a.part ? k->beg < most : k->piece == 0;
}

// A lane's row, and what it and its wave see.
struct LaneRow {
    bool valid, whole;  // whole: no spare rows in the wave (they are masked throughout)
    int row, head, sees, least, most;
    __device__ __forceinline__ LaneRow(const AttnArgs& a, const Work& k, int w, int r) {
        const int G = a.group, first = k.row0 + 32 * w, pr = first + r, i = pr / G, end = k.row0 + k.packed;
        const int last = min(first + 31, end - 1);
        valid = pr < end;
        whole = last == first + 31;
        row = k.s.first + (valid ? i : 0);
        head = k.g * G + (valid ? pr - i * G : 0);
        sees = valid ? k.s.sees(i) : 0;
        least = k.s.sees(first / G);
        most = last < first ? 0 : k.s.sees(last / G);
    }
};

// Results of a lane: piece's (o, m, l), or o / l.  m = -inf: nothing seen.
template <bool F32, int D, bool PREFIX, typename F>
__device__ __forceinline__ void finish(const AttnArgs& a, const Work& k, const LaneRow& me, int p, float m, float l, F put_all) {
    l += lane_xor<32>(l);
    if (!me.valid) return;
    const bool none = m == -__builtin_huge_valf();
    const size_t oat = me.row * a.os + (size_t)me.head * D;
    if (a.part) {
        const size_t slot = k.piece + (PREFIX ? a.own.pieces : 0), at = (slot * a.batch.rows + me.row) * a.heads + me.head;
        if (p == 0) a.ml[at] = make_float2(m, l);
        float* po = a.part + at * D;
        put_all([&](int d, v4f y) { *(v4f*)(po + d) = none ? v4f{0, 0, 0, 0} : y; });
    } else {
        const float f = 1.0f / l;
        put_all([&](int d, v4f y) {
            y = none ? v4f{0, 0, 0, 0} : y * f;
            if constexpr (F32) *(v4f*)((float*)a.out + oat + d) = y;
            else *(uint2*)((uint16_t*)a.out + oat + d) = make_uint2(pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3]));
        });
    }
}

// meet_odd for a lane's sums; column(t, e): the head dimension of acc[t][e].
template <typename T, typename C, int D, typename F>
__device__ __forceinline__ void meet_odd_tile(const AttnArgs& a, const Work& k, const LaneRow& me, size_t qat, int lo, int hi, float m,
                                              F column, v16f (&acc)[D / 32]) {
    meet_odd<T, C, D>(a, k.s, k.g, lo, hi, hi - lo, hi - lo, min(hi, k.end), (const T*)a.q + qat, me.sees, m,
                      [&](const C* v, bool seen, auto value, auto probability) {
        bool any = false;
#pragma unroll
        for (int t = 0; t < D / 32; t++)
#pragma unroll
            for (int e = 0; e < 16; e++) any |= !(fabsf(value(v + column(t, e))) < __builtin_huge_valf());
        if (!any || !seen) return;
        const float y = probability();
#pragma unroll
        for (int t = 0; t < D / 32; t++) {
            v16f add;
#pragma unroll
            for (int e = 0; e < 16; e++) {
                const float x = value(v + column(t, e));
                add[e] = fabsf(x) < __builtin_huge_valf() ? 0.0f : y * x;
            }
            acc[t] += add;  // (as whole vectors: single elements written here split the sums' registers in the main loop)
        }
    });
}

// The running reference of a row's exponents.  It follows the largest score
// only when that passes it by 2^8: any reference gives
// the same quotients, and the sums are rescaled a few times instead of often.
constexpr float LAG = 8.0f;

// LDS of a workgroup: K and V of two tiles, or of one in three terms, and a few words
template <int TYPES, int D> constexpr int tile_lds() { return (TYPES == PT_F32_F32 ? 32 * 6 : 64 * 4) * 2 * D + 16; }

// Block `block` of the launch; sm: tile_lds bytes, aligned to 256.
template <int TERMS, int D, bool PREFIX>
__device__ __forceinline__ void tile_bf16_body(const AttnArgs& a, int block, char* sm) {
    constexpr bool F32Q = TERMS > 1;
    constexpr int ROW = 2 * D, N = 64, SB = N / 32;
    constexpr int CI = N * ROW / (THREADS * 16);  // 1 KiB loads of a wave, K or V
    constexpr int DT = D / 32, KS = D / 16;
    constexpr int VR = TERMS == 1 ? 5 : 3;                // V operands in registers
    constexpr int TB = N * ROW;  // bytes of a tile's K or V; in LDS K of two tiles, then V of two
    int& odd_lo = *(int*)(sm + 4 * TB);  // positions of tiles with values that are not finite
    int& odd_hi = *(int*)(sm + 4 * TB + 4);
    const int tid = threadIdx.x, lane = tid & 63, r = lane & 31, p = lane >> 5;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    Work wk;
    if (!find_work<PREFIX>(a, block, &wk)) return;
    const Span& s = wk.s;
    const int g = wk.g, beg = wk.beg, end = wk.end;
    if (tid == 0) odd_lo = INT32_MAX, odd_hi = 0;
    const LaneRow me(a, wk, w, r);
    const size_t qat = me.row * a.qs + (size_t)me.head * D;

    v4u q[TERMS][KS];
    if constexpr (F32Q) {
        const float* qp = (const float*)a.q + qat + 8 * p;
#pragma unroll
        for (int t = 0; t < KS; t++) {
            const v4f y0 = *(const v4f*)(qp + 16 * t), y1 = *(const v4f*)(qp + 16 * t + 4);
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
        for (int t = 0; t < KS; t++) q[0][t] = *(const v4u*)(qp + 16 * t);
    }

    v16f acc[DT];
#pragma unroll
    for (int t = 0; t < DT; t++)
#pragma unroll
        for (int e = 0; e < 16; e++) acc[t][e] = 0.0f;
    float m = -__builtin_huge_valf(), l = 0.0f;

    // Tiles go from the cache to LDS without registers (16 bytes a lane, lane
    // order in LDS): the lane loads the chunk that lds_slot puts at its place.
    const char *kc = (const char*)a.kv.k, *vc = (const char*)a.kv.v;
    unsigned lane_src;
    int lane_row;  // byte offset inside its 16-row block; row inside its wave's 1 KiB of the tile
    {
        const int sub = lane >> 4;
        if constexpr (ROW == 256) {
            lane_row = sub;
            lane_src = (4 * w + sub) * ROW + (((lane & 15) ^ ((sub << 2) | w)) << 4);
        } else {
            const int x = (lane & 15) ^ (((sub & 1) << 2) | ((2 * w + (sub >> 1)) & 3));
            lane_row = 2 * sub + (x >> 3);
            lane_src = ((8 * w + lane_row) & 15) * ROW + ((x & 7) << 4);
        }
    }
    constexpr int WROWS = 1024 / ROW;  // rows of a wave's load
    const unsigned long long klane = (unsigned long long)kc + lane_src, vlane = (unsigned long long)vc + lane_src;
    // A tile's pages: lane l looks after block l % 4, whose slots lie `off`
    // bytes into the cache (of page 0 where no page holds them).
    struct Pages {
        int id;
        unsigned long long off;
    };
    const unsigned bytes_in = (unsigned)g << a.kv.page_shift, slots = (1u << a.kv.page_shift) - 1;
    const unsigned long long page_bytes = a.kv.page_stride * 2;
    auto ask = [&](int j) {  // the entry, to be waited for
        return s.table[min(j + 16 * (lane & 3), end - 1) >> a.kv.page_shift];
    };
    auto place = [&](int id, int j) {
        const int jb = j + 16 * (lane & 3);
        Pages t;
        const bool there = (jb < end) & ((unsigned)id < (unsigned)a.kv.num_pages);
        t.id = there ? id : -1;
        t.off = (unsigned long long)(unsigned)max(t.id, 0) * page_bytes + (bytes_in + ((unsigned)jb & slots)) * ROW;
        return t;
    };
    auto block_off = [&](const Pages& t, int b) {
        return (unsigned long long)(unsigned)__builtin_amdgcn_readlane((int)t.off, b) |
               (unsigned long long)(unsigned)__builtin_amdgcn_readlane((int)(t.off >> 32), b) << 32;
    };
    // bit b: no page holds block b
    auto holes_of = [&](const Pages& t) { return (unsigned)__ballot(t.id < 0) & 15u; };
    auto fetch = [&](int buf, const Pages& t) {
        typedef __attribute__((address_space(3))) void* LP;
        typedef const __attribute__((address_space(1))) void* GP;
#pragma unroll
        for (int n = 0; n < CI; n++) {
            const unsigned long long off = block_off(t, ROW == 256 ? n : 2 * n + (w >> 1));
            char* to = sm + buf * TB + (4 * n + w) * 1024;
            __builtin_amdgcn_global_load_lds((GP)(klane + off), (LP)to, 16, 0, 0);
            __builtin_amdgcn_global_load_lds((GP)(vlane + off), (LP)(to + 2 * TB), 16, 0, 0);
        }
    };
    // Values of rows that no row sees become zeros, and so does what is not
    // finite where some row must not meet it (three terms: anywhere); each
    // lane looks after the chunks it has loaded.
    const int least = s.sees(wk.row0 / a.group);
    auto mend = [&](char* V, unsigned holes, int j) {
        const bool part = holes || j + N > least;
        if (!part && TERMS == 1) return;
        uint32_t bits = 0;
        v4u v[CI];
#pragma unroll
        for (int n = 0; n < CI; n++) {
            const int row = (4 * n + w) * WROWS;
            v4u* at = (v4u*)(V + (4 * n + w) * 1024 + 16 * lane);
            v[n] = *at;
            if (part && ((holes >> (row / 16) & 1) || j + row + lane_row >= end)) {
                v[n] = v4u{0, 0, 0, 0};
                *at = v[n];
            }
            mark_odd<false>(v[n], bits);
        }
        if (is_odd<false>(bits)) {
            atomicMin(&odd_lo, j);
            atomicMax(&odd_hi, j + N);
#pragma unroll
            for (int n = 0; n < CI; n++) *(v4u*)(V + (4 * n + w) * 1024 + 16 * lane) = finite_part<false>(v[n]);
        }
    };
    // Scores of a tile, K's operands two steps ahead (left alone, the compiler
    // loads all of them first, and spills).
    auto scores = [&](int K, v16f (&sc)[SB]) {
        // lds_slot(32 b + r, 2 c + p) = (lds_slot(r, p) ^ 32 c) + 32 b ROW, from
        // one register (hoisted out of the loop the places take eight)
        int at = K + lds_slot<ROW>(r, p);
        asm volatile("" : "+v"(at));
        v8b ko[3][SB];
        auto load = [&](int c) {
#pragma unroll
            for (int b = 0; b < SB; b++) ko[c % 3][b] = *(const v8b*)(sm + ((at ^ (c << 5)) + 32 * b * ROW));
        };
        load(0);
        load(1);
#pragma unroll
        for (int b = 0; b < SB; b++)
#pragma unroll
            for (int e = 0; e < 16; e++) sc[b][e] = 0.0f;
#pragma unroll
        for (int c = 0; c < KS; c++) {
            if (c + 2 < KS) load(c + 2);
#pragma unroll
            for (int z = TERMS - 1; z >= 0; z--)
#pragma unroll
                for (int b = 0; b < SB; b++)
                    sc[b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ko[c % 3][b], __builtin_bit_cast(v8b, q[z][c]), sc[b], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    int j = beg, ahead = 0;      // the table entry of the tile after next
    unsigned holes = 0;
    Pages next = {};
    if (j < end) {
        const int e0 = ask(j), e1 = ask(j + N);
        ahead = ask(j + 2 * N);
        const Pages first = place(e0, j);
        next = place(e1, j + N);
        holes = holes_of(first);
        fetch(0, first);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();  // odd_lo, odd_hi are set up
        mend(sm + 2 * TB, holes, j);
        __syncthreads();
    }
#pragma unroll
    for (int z = 0; z < TERMS; z++)
#pragma unroll
        for (int t = 0; t < KS; t++) arrived(q[z][t]);
    float mu = -FLT_MAX;
    bool far = false;
    for (int buf = 0; j < end; buf ^= 1, j += N) {
        const int jn = j + N;
        unsigned next_holes = 0;
        if (jn < end) {
            next_holes = holes_of(next);
            fetch(buf ^ 1, next);
            next = place(ahead, jn + N);
            ahead = ask(jn + 2 * N);
        }
        if (j < me.most) {
            v16f sc[SB];
            // (ahead of the other wave's vector instructions: 369 us against 373)
            __builtin_amdgcn_s_setprio(1);
            scores(buf * TB, sc);
            __builtin_amdgcn_s_setprio(0);
            const bool masked = holes || j + N > me.least || !me.whole;
            // element e of block b: position 32 b + 8 (e / 4) + 4 p + e % 4
            float mx = -FLT_MAX;
            if (masked) {
                mx = -__builtin_huge_valf();
#pragma unroll
                for (int b = 0; b < SB; b++)
#pragma unroll
                    for (int e = 0; e < 16; e++) {
                        const bool seen = !(holes >> (2 * b + e / 8) & 1) && j + 32 * b + 8 * (e / 4) + 4 * p + e % 4 < me.sees;
                        sc[b][e] = seen ? sc[b][e] : -__builtin_huge_valf();
                        mx = seen ? -FLT_MAX : mx;
                    }
            }
            if constexpr (TERMS > 1) {
                // an infinity times the terms of a q may be inf - inf: such scores again, product by product
                float sum = 0.0f;
#pragma unroll
                for (int b = 0; b < SB; b++)
#pragma unroll
                    for (int e = 0; e < 16; e++) sum += sc[b][e];
                if (__any(sum != sum)) {
#pragma unroll
                    for (int b = 0; b < SB; b++)
#pragma unroll
                        for (int e = 0; e < 16; e++)
                            if (sc[b][e] != sc[b][e]) {
                                const float* qp = (const float*)a.q + qat;
                                const uint16_t* kp = (const uint16_t*)kc + slot_off(a, page_at(a, s, j + 32 * b + 16 * (e / 8), end), g, j + 32 * b + 16 * (e / 8), D) +
                                                     (8 * (e / 4 % 2) + 4 * p + e % 4) * D;
                                float t = 0.0f;
                                for (int d = 0; d < D; d++) t = fmaf(qp[d], __uint_as_float((uint32_t)kp[d] << 16), t);
                                sc[b][e] = t;
                            }
                }
            }
            {
                // (c > 0: the largest score scaled is the largest scaled score)
                float y = sc[0][0];
#pragma unroll
                for (int b = 0; b < SB; b++)
#pragma unroll
                    for (int e = 0; e < 16; e++) y = fmaxf(y, sc[b][e]);
                mx = fmaxf(mx, y * a.c);
            }
            mx = fmaxf(mx, lane_xor<32>(mx));
            float al = 1.0f;
            if (__any(mx > m - (ABOVE - LAG))) {
                // (of the rows that need it: a row's result is not to depend on others)
                const float mn = mx > m - (ABOVE - LAG) ? fmaxf(m, mx + ABOVE) : m;
                mu = fmaxf(mn, -FLT_MAX);
                al = __builtin_amdgcn_exp2f(m - mu);
                m = mn;
                far = __any(far_score(mu));
            }
            // (on every tile: behind a branch around it, the compiler keeps the
            // sums in two sets of registers and copies them)
            l *= al;
#pragma unroll
            for (int t = 0; t < DT; t++) acc[t] *= al;
            if (far) {
                const float f = far_score(mu) ? a.c : 1.0f, c = far_score(mu) ? 1.0f : a.c;
#pragma unroll
                for (int b = 0; b < SB; b++)
#pragma unroll
                    for (int e = 0; e < 16; e++) sc[b][e] = __builtin_amdgcn_exp2f(fmaf(sc[b][e] * f, c, -mu));
            } else {
#pragma unroll
                for (int b = 0; b < SB; b++)
#pragma unroll
                    for (int e = 0; e < 16; e++) sc[b][e] = __builtin_amdgcn_exp2f(fmaf(sc[b][e], a.c, -mu));
            }
            // lds_slot(16 ks + 8 h + row, ch + 4 t) = (lds_slot(row, ch) ^ 64 t ^ 32 h) + (16 ks + 8 h) ROW
            int vat = (2 + buf) * TB + lds_slot<ROW>(4 * p + ((lane & 15) >> 2), 2 * ((lane >> 4) & 1) + ((lane >> 1) & 1)) + 8 * (lane & 1);
            asm volatile("" : "+v"(vat));
            v8b vo[VR];
            auto load_v = [&](int i) {
                const int ks = i / DT, t = i % DT;
                const char* at = sm + 16 * ks * ROW;
                vo[i % VR] = join_halves(read_transposed(at + (vat ^ (t << 6))), read_transposed(at + 8 * ROW + (vat ^ (t << 6) ^ 32)));
            };
#pragma unroll
            for (int i = 0; i + 1 < VR; i++) load_v(i);
#pragma unroll
            for (int ks = 0; ks < N / 16; ks++) {
                v4u pb[TERMS];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float y0 = sc[ks / 2][8 * (ks % 2) + 2 * e], y1 = sc[ks / 2][8 * (ks % 2) + 2 * e + 1];
                    if constexpr (TERMS == 1) {
                        // (l sums what the values are weighted with)
                        pb[0][e] = pack_bf16(y0, y1);
                        l = add_bf16(pb[0][e], l);
                    } else {
                        l += y0 + y1;
                        float t0[3], t1[3];
                        three_terms(y0, t0);
                        three_terms(y1, t1);
#pragma unroll
                        for (int z = 0; z < TERMS; z++) pb[z][e] = pack_bf16(t0[z], t1[z]);
                    }
                }
#pragma unroll
                for (int t = 0; t < DT; t++) {
                    const int i = ks * DT + t;
                    if (i + VR - 1 < N / 16 * DT) load_v(i + VR - 1);
#pragma unroll
                    for (int z = TERMS - 1; z >= 0; z--)
                        acc[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vo[i % VR], __builtin_bit_cast(v8b, pb[z]), acc[t], 0, 0, 0);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (the fetches)
        if (jn < end) mend(sm + (2 + (buf ^ 1)) * TB, next_holes, jn);
        __syncthreads();
        holes = next_holes;
    }
    __syncthreads();
    if (odd_hi) meet_odd_tile<typename std::conditional<F32Q, float, uint16_t>::type, uint16_t, D>(a, wk, me, qat, odd_lo, odd_hi, m, [&](int t, int e) { return 32 * t + 8 * (e / 4) + 4 * p + e % 4; }, acc);
    finish<F32Q, D, PREFIX>(a, wk, me, p, m, l, [&](auto put) {
#pragma unroll
        for (int t = 0; t < DT; t++)
#pragma unroll
            for (int e = 0; e < 16; e += 4) put(32 * t + 2 * e + 4 * p, v4f{acc[t][e], acc[t][e + 1], acc[t][e + 2], acc[t][e + 3]});
    });
}

// x = the sum of three bf16 terms, exactly, for eight x: z[k] holds the terms k.
// The first is cut (rounded it could be infinite), the second rounded, so that
// the products of second and third terms, which are left out, have either
// sign: 2^-24 of a product in the mean square.  What is not finite becomes NaN.
__device__ __forceinline__ void split_terms(v4f x0, v4f x1, v4u (&z)[3]) {
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const float a = e < 2 ? x0[2 * e] : x1[2 * e - 4], b = e < 2 ? x0[2 * e + 1] : x1[2 * e - 3];
        const uint32_t w0 = __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
        const float ra = a - low_bf16(w0), rb = b - high_bf16(w0);
        const uint32_t w1 = pack_bf16(ra, rb);
        z[0][e] = w0;
        z[1][e] = w1;
        z[2][e] = pack_bf16(ra - low_bf16(w1), rb - high_bf16(w1));
    }
}

// f32 pages.  The float32 products run at a sixteenth of the bf16 ones' rate,
// so every operand is split into three bf16 terms, K and V on their way into
// LDS, and the six products of terms that count are taken: 129 us for 951 rows
// over 2999 positions, 16 heads over 8 of 128 (19.7 GFLOP), against 222 with
// float32 products (152.8 TFLOP/s at most).  One tile in LDS, so that two
// workgroups share a compute unit and one computes while the other splits.
template <int D, bool PREFIX>
__device__ __forceinline__ void tile_f32_body(const AttnArgs& a, int block, char* sm) {
    constexpr int ROW = 2 * D, N = 32, PB = N * ROW;  // a plane: one term of K or V; K's three, then V's
    constexpr int TPR = D / 8, RPN = THREADS / TPR, CI = N / RPN;  // eight values a thread; rows of a step; steps
    constexpr int DT = D / 32, KS = D / 16;
    int& odd_lo = *(int*)(sm + 6 * PB);  // positions of tiles with values that are not finite
    int& odd_hi = *(int*)(sm + 6 * PB + 4);
    const int tid = threadIdx.x, lane = tid & 63, r = lane & 31, p = lane >> 5;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);

    Work wk;
    if (!find_work<PREFIX>(a, block, &wk)) return;
    const Span& s = wk.s;
    const int g = wk.g, beg = wk.beg, end = wk.end;
    if (tid == 0) odd_lo = INT32_MAX, odd_hi = 0;
    const LaneRow me(a, wk, w, r);
    const size_t qat = me.row * a.qs + (size_t)me.head * D;
    v4u q[KS][3];
    {
        const float* qp = (const float*)a.q + qat + 8 * p;
#pragma unroll
        for (int t = 0; t < KS; t++) split_terms(*(const v4f*)(qp + 16 * t), *(const v4f*)(qp + 16 * t + 4), q[t]);
    }

    v16f acc[DT];
#pragma unroll
    for (int t = 0; t < DT; t++)
#pragma unroll
        for (int e = 0; e < 16; e++) acc[t][e] = 0.0f;
    float m = -__builtin_huge_valf(), l = 0.0f, mu = -FLT_MAX;
    bool far = false;

    // staging: values 8 (tid % TPR) .. of row tid / TPR + RPN n of the tile
    v4f kr[CI][2], vr[CI][2];
    int pg[2], pn[2];  // pages of this tile's blocks and the next's
    auto pages_of = [&](int j, int (&pg)[2]) { pg[0] = page_at(a, s, j, end), pg[1] = page_at(a, s, j + 16, end); };
    const float *kc = (const float*)a.kv.k, *vc = (const float*)a.kv.v;
    auto page_of = [&](const int (&pg)[2], int n) { return RPN == 16 ? pg[n] : w >= 2 ? pg[1] : pg[0]; };
    const int lane_at = (tid / TPR & 15) * D + tid % TPR * 8;
    auto load = [&](const int (&pg)[2], int j) {
#pragma unroll
        for (int n = 0; n < CI; n++) {
            const size_t at = slot_off(a, page_of(pg, n), g, j + 16 * (RPN == 16 ? n : w / 2), D) + lane_at;
            kr[n][0] = *(const v4f*)(kc + at), kr[n][1] = *(const v4f*)(kc + at + 4);
            vr[n][0] = *(const v4f*)(vc + at), vr[n][1] = *(const v4f*)(vc + at + 4);
        }
    };
    // registers -> LDS, the tile at position j.  Values of rows that no row
    // sees become zeros, and so does what is not finite (meet_odd).
    auto store = [&](int j, const int (&pg)[2]) {
        uint32_t bits = 0;
#pragma unroll
        for (int n = 0; n < CI; n++) {
            const bool gone = page_of(pg, n) < 0 || j + n * RPN + tid / TPR >= end;
#pragma unroll
            for (int h = 0; h < 2; h++) {
                if (gone) vr[n][h] = v4f{0, 0, 0, 0};
                mark_odd<true>(__builtin_bit_cast(v4u, vr[n][h]), bits);
            }
        }
        if (is_odd<true>(bits)) {
            atomicMin(&odd_lo, j);
            atomicMax(&odd_hi, j + N);
#pragma unroll
            for (int n = 0; n < CI; n++)
#pragma unroll
                for (int h = 0; h < 2; h++) vr[n][h] = __builtin_bit_cast(v4f, finite_part<true>(__builtin_bit_cast(v4u, vr[n][h])));
        }
#pragma unroll
        for (int n = 0; n < CI; n++) {
            char* at = sm + lds_slot<ROW>(n * RPN + tid / TPR, tid % TPR);
            v4u z[3];
            split_terms(kr[n][0], kr[n][1], z);
#pragma unroll
            for (int y = 0; y < 3; y++) *(v4u*)(at + y * PB) = z[y];
            split_terms(vr[n][0], vr[n][1], z);
#pragma unroll
            for (int y = 0; y < 3; y++) *(v4u*)(at + (3 + y) * PB) = z[y];
        }
    };

    int j = beg;
    if (j < end) {
        pages_of(j, pg);
        pages_of(j + N, pn);
        load(pg, j);
        __syncthreads();  // odd_lo, odd_hi are set up
        store(j, pg);
        __syncthreads();
    }
#pragma unroll
    for (int t = 0; t < KS; t++)
#pragma unroll
        for (int z = 0; z < 3; z++) arrived(q[t][z]);
    for (; j < end; j += N) {
        const int jn = j + N;
        if (jn < end) load(pn, jn);
        int pnn[2];  // a tile ahead of its loads
        pages_of(jn + N, pnn);
        if (j < me.most) {
            // scores, K's operands a step ahead, products in two chains (138 us
            // against 141); lds_slot(r, 2 c + p) = lds_slot(r, p) ^ 32 c
            v16f sc;
            {
                int at = lds_slot<ROW>(r, p);
                asm volatile("" : "+v"(at));
                v8b ko[2][3];
                auto load_k = [&](int c) {
#pragma unroll
                    for (int y = 0; y < 3; y++) ko[c % 2][y] = *(const v8b*)(sm + y * PB + (at ^ (c << 5)));
                };
                __builtin_amdgcn_s_setprio(1);  // (129 us against 138)
                load_k(0);
#pragma unroll
                for (int e = 0; e < 16; e++) sc[e] = 0.0f;
                v16f lo = sc;
#pragma unroll
                for (int c = 0; c < KS; c++) {
                    if (c + 1 < KS) load_k(c + 1);
                    auto mul = [&](v16f& to, int y, int z) { to = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ko[c % 2][y], __builtin_bit_cast(v8b, q[c][z]), to, 0, 0, 0); };
                    mul(lo, 0, 2);
                    mul(sc, 0, 1);
                    mul(lo, 1, 1);
                    mul(sc, 1, 0);
                    mul(lo, 2, 0);
                    mul(sc, 0, 0);
                    __builtin_amdgcn_sched_barrier(0);
                }
                __builtin_amdgcn_s_setprio(0);
                sc += lo;
            }
            const bool masked = pg[0] < 0 || pg[1] < 0 || j + N > me.least || !me.whole;
            // element e: position 8 (e / 4) + 4 p + e % 4
            float mx = -FLT_MAX;
            if (masked) {
                mx = -__builtin_huge_valf();
#pragma unroll
                for (int e = 0; e < 16; e++) {
                    const bool seen = pg[e / 8] >= 0 && j + 8 * (e / 4) + 4 * p + e % 4 < me.sees;
                    sc[e] = seen ? sc[e] : -__builtin_huge_valf();
                    mx = seen ? -FLT_MAX : mx;
                }
            }
            {
                // terms of what is not finite, or infinite products of terms: such scores again, product by product
                float sum = 0.0f;
#pragma unroll
                for (int e = 0; e < 16; e++) sum += sc[e];
                if (__any(sum != sum)) {
#pragma unroll
                    for (int e = 0; e < 16; e++)
                        if (sc[e] != sc[e]) {
                            const float* qp = (const float*)a.q + qat;
                            const float* kp = kc + slot_off(a, pg[e / 8], g, j + 16 * (e / 8), D) + (8 * (e / 4 % 2) + 4 * p + e % 4) * D;
                            float t = 0.0f;
                            for (int d = 0; d < D; d++) t = fmaf(qp[d], kp[d], t);
                            sc[e] = t;
                        }
                }
            }
            {
                // (c > 0: the largest score scaled is the largest scaled score)
                float y = sc[0];
#pragma unroll
                for (int e = 1; e < 16; e++) y = fmaxf(y, sc[e]);
                mx = fmaxf(mx, y * a.c);
            }
            mx = fmaxf(mx, lane_xor<32>(mx));
            float al = 1.0f;
            if (__any(mx > m - (ABOVE - LAG))) {
                // (of the rows that need it: a row's result is not to depend on others)
                const float mn = mx > m - (ABOVE - LAG) ? fmaxf(m, mx + ABOVE) : m;
                mu = fmaxf(mn, -FLT_MAX);
                al = __builtin_amdgcn_exp2f(m - mu);
                m = mn;
                far = __any(far_score(mu));
            }
            l *= al;
#pragma unroll
            for (int t = 0; t < DT; t++) acc[t] *= al;
            if (far) sc *= far_score(mu) ? a.c : 1.0f;
            const float c = far && far_score(mu) ? 1.0f : a.c;
#pragma unroll
            for (int e = 0; e < 16; e++) sc[e] = __builtin_amdgcn_exp2f(fmaf(sc[e], c, -mu));
#pragma unroll
            for (int e = 0; e < 16; e++) l += sc[e];
            // lds_slot(16 ks + 8 h + row, ch + 4 t) = (lds_slot(row, ch) ^ 64 t ^ 32 h) + (16 ks + 8 h) ROW
            int vat = 3 * PB + lds_slot<ROW>(4 * p + ((lane & 15) >> 2), 2 * ((lane >> 4) & 1) + ((lane >> 1) & 1)) + 8 * (lane & 1);
            asm volatile("" : "+v"(vat));
            v8b vo[2][3];
            auto load_v = [&](int i) {
                const int ks = i / DT, t = i % DT;
#pragma unroll
                for (int y = 0; y < 3; y++) {
                    const char* at = sm + y * PB + 16 * ks * ROW;
                    vo[i % 2][y] = join_halves(read_transposed(at + (vat ^ (t << 6))), read_transposed(at + 8 * ROW + (vat ^ (t << 6) ^ 32)));
                }
            };
            load_v(0);
#pragma unroll
            for (int ks = 0; ks < 2; ks++) {
                v4u pb[3];
                split_terms(v4f{sc[8 * ks], sc[8 * ks + 1], sc[8 * ks + 2], sc[8 * ks + 3]}, v4f{sc[8 * ks + 4], sc[8 * ks + 5], sc[8 * ks + 6], sc[8 * ks + 7]}, pb);
#pragma unroll
                for (int t = 0; t < DT; t++) {
                    const int i = ks * DT + t;
                    if (i + 1 < 2 * DT) load_v(i + 1);
#pragma unroll
                    for (int o = 2; o >= 0; o--)
#pragma unroll
                        for (int y = 0; y <= o; y++)
                            acc[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vo[i % 2][y], __builtin_bit_cast(v8b, pb[o - y]), acc[t], 0, 0, 0);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        }
        __syncthreads();
        if (jn < end) store(jn, pn);
        __syncthreads();
        pg[0] = pn[0], pg[1] = pn[1], pn[0] = pnn[0], pn[1] = pnn[1];
    }

    __syncthreads();
    if (odd_hi) meet_odd_tile<float, float, D>(a, wk, me, qat, odd_lo, odd_hi, m, [&](int t, int e) { return 32 * t + 8 * (e / 4) + 4 * p + e % 4; }, acc);
    finish<true, D, PREFIX>(a, wk, me, p, m, l, [&](auto put) {
#pragma unroll
        for (int t = 0; t < DT; t++)
#pragma unroll
            for (int e = 0; e < 16; e += 4) put(32 * t + 2 * e + 4 * p, v4f{acc[t][e], acc[t][e + 1], acc[t][e + 2], acc[t][e + 3]});
    });
}

template <int TYPES, int D, bool PREFIX>
__device__ __forceinline__ void tile_body(const AttnArgs& a, int block, char* sm) {
    if constexpr (TYPES == PT_F32_F32) tile_f32_body<D, PREFIX>(a, block, sm);
    else tile_bf16_body<TYPES == PT_F32_BF16 ? 3 : 1, D, PREFIX>(a, block, sm);
}

}  // namespace
}  // namespace lq8
