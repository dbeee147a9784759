// paged_tile.hip -- attention over a paged cache for many packed rows a kv
// head: prompt chunks, and the rows of a group that share a prefix (gfx950).
//
// A workgroup has 128 packed rows, 32 to a wave, and goes over its piece in
// tiles of 64 positions (bf16 pages) or 32 (f32), K and V in LDS, two buffers:
// the next tile's loads are out while this one is computed, one barrier a tile.
// The rows are the columns of the products (32 x 32 tiles): S^T = K Q^T leaves
// lane (row = lane % 32, p = lane / 32) with the scores of positions 8 i + 4 p
// .. + 3 of its row, which is the B operand of O^T = V^T P^T when the 16
// positions of a product are taken in the order (4 p + e, 8 + 4 p + e): the
// probabilities stay where they are, the maximum needs one exchange with lane
// +- 32, and the rescaling of O none.  V is read transposed (ds_read_tr).
// f32 pages: 32 x 32 x 2 products on float32 operands.  f32 rows over bf16
// pages: three bf16 terms of q and p each, as in paged_few.hip.
#include "paged_attn.h"

namespace lq8 {
namespace {

constexpr int THREADS = 256;

// The span and the row tile of tile number `want` over all spans, by all
// threads; false: there are fewer tiles.
template <bool PREFIX>
__device__ __forceinline__ bool find_tile(const AttnArgs& a, int want, int* span, int* tile) {
    __shared__ int sums[THREADS / 64], found[2];
    const int n = PREFIX ? a.prefix.groups : a.batch.batch, tid = threadIdx.x, lane = tid & 63;
    if (tid == 0) found[0] = -1;
    int before = 0;
    for (int s0 = 0; s0 < n; s0 += THREADS) {
        int t = 0;
        if (s0 + tid < n) {
            const int rows = PREFIX ? prefix_span(a, s0 + tid).count : rows_of(a.batch, s0 + tid).count;
            t = (int)(((int64_t)rows * a.group + TILE_PACKED - 1) / TILE_PACKED);
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

template <int TYPES, int D, bool PREFIX>
__global__ __launch_bounds__(THREADS, 2) void k_tile(AttnArgs a) {
    constexpr bool F32C = TYPES == PT_F32_F32, F32Q = TYPES != PT_BF16_BF16;
    constexpr int TERMS = TYPES == PT_F32_BF16 ? 3 : 1;
    constexpr int ES = F32C ? 4 : 2, ROW = D * ES, N = F32C ? 32 : 64;
    constexpr int BLOCKS = N / 16, SB = N / 32;               // page blocks, score blocks of a tile
    constexpr int CPR = ROW / 16, CI = N * CPR / THREADS;     // 16-byte chunks of a row; of a thread
    constexpr int DT = D / 32, VW = D / 32;
    __shared__ __attribute__((aligned(16))) char sk[2][N * ROW], sv[2][N * ROW];
    __shared__ float scratch[4][16 * 32];
    __shared__ int odd_tile[2];
    const int tid = threadIdx.x, lane = tid & 63, r = lane & 31, p = lane >> 5;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);

    // workgroup -> (row tile, piece, kv head), kv head fastest (one to an XCD
    // where there are eight); a sequence's last rows, which see most, first
    const int G = a.group, kvh = a.kv.kv_heads;
    const Cut& cut = PREFIX ? a.pre : a.own;
    int x = blockIdx.x;
    const int g = x % kvh;
    x /= kvh;
    const int piece = x % cut.pieces, want = x / cut.pieces;
    int sp, tile;
    if (!find_tile<PREFIX>(a, want, &sp, &tile)) return;
    const Span s = PREFIX ? prefix_span(a, sp) : own_span(a, sp);
    tile = (s.count * G + TILE_PACKED - 1) / TILE_PACKED - 1 - tile;
    const int row0 = tile * TILE_PACKED, packed = min(s.count * G - row0, TILE_PACKED);
    const int len = piece_len(s.length, cut);
    const int most = s.sees((row0 + packed - 1) / G);
    const int beg = piece * len, end = min(beg + len, most);
    if (a.part ? beg >= most : piece > 0) return;
    if (tid < 2) odd_tile[tid] = -1;

    // the lane's row
    const int wrow = row0 + 32 * w, pr = wrow + r, i = pr / G;
    const bool valid = pr < row0 + packed;
    const int row = s.first + (valid ? i : 0), head = g * G + (valid ? pr - i * G : 0);
    const int sees = valid ? s.sees(i) : 0;
    const int wleast = s.sees(wrow / G), wlast = min(wrow + 31, row0 + packed - 1);
    const int wmost = wlast < wrow ? 0 : s.sees(wlast / G);
    const bool whole = wlast == wrow + 31;  // (a wave with spare rows masks them throughout)
    const size_t qat = row * a.qs + (size_t)head * D;
    uint32_t q[F32C ? 1 : TERMS][F32C ? 1 : D / 16][4];
    float qf[F32C ? D / 2 : 1];
    if constexpr (F32C) {
        const float* qp = (const float*)a.q + qat + 4 * p;
#pragma unroll
        for (int t = 0; t < D / 8; t++) {
            const float4 v = *(const float4*)(qp + 8 * t);
            qf[4 * t] = v.x, qf[4 * t + 1] = v.y, qf[4 * t + 2] = v.z, qf[4 * t + 3] = v.w;
        }
    } else if constexpr (F32Q) {
        const float* qp = (const float*)a.q + qat + 8 * p;
#pragma unroll
        for (int t = 0; t < D / 16; t++) {
            const float4 y0 = *(const float4*)(qp + 16 * t), y1 = *(const float4*)(qp + 16 * t + 4);
            const float y[8] = {y0.x, y0.y, y0.z, y0.w, y1.x, y1.y, y1.z, y1.w};
#pragma unroll
            for (int e = 0; e < 4; e++) {
                float t0[3], t1[3];
                three_terms(y[2 * e], t0);
                three_terms(y[2 * e + 1], t1);
#pragma unroll
                for (int z = 0; z < TERMS; z++) q[z][t][e] = pack_bf16(t0[z], t1[z]);
            }
        }
    } else {
        const uint16_t* qp = (const uint16_t*)a.q + qat + 8 * p;
#pragma unroll
        for (int t = 0; t < D / 16; t++) {
            const v4u v = *(const v4u*)(qp + 16 * t);
            q[0][t][0] = v[0], q[0][t][1] = v[1], q[0][t][2] = v[2], q[0][t][3] = v[3];
        }
    }

    v16f acc[DT];
#pragma unroll
    for (int t = 0; t < DT; t++)
#pragma unroll
        for (int e = 0; e < 16; e++) acc[t][e] = 0.0f;
    float m = -__builtin_huge_valf(), l = 0.0f;

    // staging: chunk tid + 256 n of the tile; a wave's rows lie in one block
    v4u kr[CI], vr[CI];
    int pg[BLOCKS], pn[BLOCKS];  // of this tile and the next
    const char *kc = (const char*)a.kv.k, *vc = (const char*)a.kv.v;
    auto pages_of = [&](int j, int (&pg)[BLOCKS]) {
#pragma unroll
        for (int b = 0; b < BLOCKS; b++) pg[b] = page_at(a, s, j + 16 * b, end);
    };
    constexpr int RPN = THREADS / CPR;  // rows of a step
    auto page_of = [&](const int (&pg)[BLOCKS], int n) {  // of the wave's rows of step n
        if constexpr (RPN <= 16) return pg[n * RPN / 16];
        else return w >= 2 ? pg[2 * n + 1] : pg[2 * n];
    };
    const int lane_at = (tid / CPR & 15) * ROW + tid % CPR * 16;
    auto load = [&](const int (&pg)[BLOCKS], int j) {
#pragma unroll
        for (int n = 0; n < CI; n++) {
            const int b = RPN <= 16 ? n * RPN / 16 : 2 * n + w / 2;
            const size_t at = slot_off(a, page_of(pg, n), g, j + 16 * b, D) * ES;
            const int o = lane_at + (RPN < 16 ? n * RPN % 16 * ROW : 0);
            kr[n] = *(const v4u*)(kc + at + o);
            vr[n] = *(const v4u*)(vc + at + o);
        }
    };
    // registers -> buffer `buf`, tile number k at position j.  Values of rows
    // that no row sees become zeros, and so does what is not finite where
    // some row must not meet it (fixed up after the products).
    const int least = s.sees(row0 / G);
    auto store = [&](int buf, int k, int j, const int (&pg)[BLOCKS]) {
        bool hole = false;
#pragma unroll
        for (int b = 0; b < BLOCKS; b++) hole |= pg[b] < 0;
        const bool check = TERMS > 1 || hole || j + N > least;
        if (check) {
            uint32_t bits = 0;
#pragma unroll
            for (int n = 0; n < CI; n++) {
                if (page_of(pg, n) < 0 || j + n * RPN + tid / CPR >= end) vr[n] = v4u{0, 0, 0, 0};
                mark_odd<F32C>(vr[n], bits);
            }
            if (is_odd<F32C>(bits)) {
                odd_tile[buf] = k;
#pragma unroll
                for (int n = 0; n < CI; n++) vr[n] = finite_part<F32C>(vr[n]);
            }
        }
#pragma unroll
        for (int n = 0; n < CI; n++) {
            const int at = lds_slot<ROW>(n * RPN + tid / CPR, tid % CPR);
            *(v4u*)(sk[buf] + at) = kr[n];
            *(v4u*)(sv[buf] + at) = vr[n];
        }
    };

    int j = beg;
    if (j < end) {
        pages_of(j, pg);
        pages_of(j + N, pn);
        load(pg, j);
        __syncthreads();  // odd_tile is set up
        store(0, 0, j, pg);
    }
    if constexpr (F32C) {
#pragma unroll
        for (int t = 0; t < D / 2; t++) arrived(qf[t]);
    } else {
#pragma unroll
        for (int z = 0; z < TERMS; z++)
#pragma unroll
            for (int t = 0; t < D / 16; t++)
#pragma unroll
                for (int e = 0; e < 4; e++) arrived(q[z][t][e]);
    }
    for (int k = 0; j < end; k++, j += N) {
        const int buf = k & 1, jn = j + N;
        __syncthreads();
        if (jn < end) load(pn, jn);
        int pnn[BLOCKS];  // a tile ahead of its loads
        pages_of(jn + N, pnn);
        if (j < wmost) {
            const char *K = sk[buf], *V = sv[buf];
            v16f sc[SB];
            v8b ko[F32C ? 1 : SB][F32C ? 1 : D / 16];
            if constexpr (!F32C) {
#pragma unroll
                for (int b = 0; b < SB; b++)
#pragma unroll
                    for (int c = 0; c < D / 16; c++) ko[b][c] = *(const v8b*)(K + lds_slot<ROW>(32 * b + r, 2 * c + p));
            }
#pragma unroll
            for (int b = 0; b < SB; b++) {
                v16f t;
#pragma unroll
                for (int e = 0; e < 16; e++) t[e] = 0.0f;
                if constexpr (F32C) {
#pragma unroll
                    for (int c = 0; c < D / 8; c++) {
                        const v4f kv = *(const v4f*)(K + lds_slot<ROW>(32 * b + r, 2 * c + p));
#pragma unroll
                        for (int e = 0; e < 4; e++) t = __builtin_amdgcn_mfma_f32_32x32x2f32(kv[e], qf[4 * c + e], t, 0, 0, 0);
                    }
                } else {
#pragma unroll
                    for (int c = 0; c < D / 16; c++) {
#pragma unroll
                        for (int z = TERMS - 1; z >= 0; z--) {
                            const v4u qv = v4u{q[z][c][0], q[z][c][1], q[z][c][2], q[z][c][3]};
                            t = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ko[b][c], __builtin_bit_cast(v8b, qv), t, 0, 0, 0);
                        }
                    }
                }
                sc[b] = t;
            }
            bool hole = false;
#pragma unroll
            for (int b = 0; b < BLOCKS; b++) hole |= pg[b] < 0;
            const bool masked = hole || j + N > wleast || !whole;
            // element e of block b: position 32 b + 8 (e / 4) + 4 p + e % 4
            auto seen = [&](int b, int e) { return pg[2 * b + e / 8] >= 0 && j + 32 * b + 8 * (e / 4) + 4 * p + e % 4 < sees; };
            if (masked) {
#pragma unroll
                for (int b = 0; b < SB; b++)
#pragma unroll
                    for (int e = 0; e < 16; e++) sc[b][e] = seen(b, e) ? sc[b][e] : -__builtin_huge_valf();
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
                                const uint16_t* kp = (const uint16_t*)kc + slot_off(a, pg[2 * b + e / 8], g, j + 32 * b + 16 * (e / 8), D) + (8 * (e / 4 % 2) + 4 * p + e % 4) * D;
                                float t = 0.0f;
                                for (int d = 0; d < D; d++) t = fmaf(qp[d], __uint_as_float((uint32_t)kp[d] << 16), t);
                                sc[b][e] = t;
                            }
                }
            }
            float mx = masked ? -__builtin_huge_valf() : -FLT_MAX;
            if (masked) {
#pragma unroll
                for (int b = 0; b < SB; b++)
#pragma unroll
                    for (int e = 0; e < 16; e++) {
                        const float y = sc[b][e] * a.c;
                        mx = fmaxf(mx, seen(b, e) ? fmaxf(y, -FLT_MAX) : y);
                    }
            } else {
                // (c > 0: the largest score scaled is the largest scaled score)
                float y = sc[0][0];
#pragma unroll
                for (int b = 0; b < SB; b++)
#pragma unroll
                    for (int e = 0; e < 16; e++) y = fmaxf(y, sc[b][e]);
                mx = fmaxf(mx, y * a.c);
            }
            mx = fmaxf(mx, lane_xor<32>(mx));
            const float mn = fmaxf(m, mx), mu = fmaxf(mn, -FLT_MAX);
            if (__any(mn != m)) {
                const float al = __builtin_amdgcn_exp2f(m - mu);
                l *= al;
#pragma unroll
                for (int t = 0; t < DT; t++) acc[t] *= al;
            }
            m = mn;
            const bool far = __any(far_score(mu));
            if (far) {
#pragma unroll
                for (int b = 0; b < SB; b++)
#pragma unroll
                    for (int e = 0; e < 16; e++) sc[b][e] = sc[b][e] * a.c - mu;
            } else {
#pragma unroll
                for (int b = 0; b < SB; b++)
#pragma unroll
                    for (int e = 0; e < 16; e++) sc[b][e] = fmaf(sc[b][e], a.c, -mu);
            }
#pragma unroll
            for (int b = 0; b < SB; b++)
#pragma unroll
                for (int e = 0; e < 16; e++) {
                    sc[b][e] = __builtin_amdgcn_exp2f(sc[b][e]);
                    l += sc[b][e];
                }
            if constexpr (F32C) {
#pragma unroll
                for (int e = 0; e < 16; e++) {
                    const int vrow = 8 * (e / 4) + 4 * p + e % 4;
                    v4f v;
                    if constexpr (VW == 4) {
                        v = *(const v4f*)(V + lds_slot<ROW>(vrow, r));
                    } else {
                        const float2 two = *(const float2*)(V + lds_slot<ROW>(vrow, r >> 1) + 8 * (r & 1));
                        v = v4f{two.x, two.y, 0.0f, 0.0f};
                    }
#pragma unroll
                    for (int t = 0; t < DT; t++) acc[t] = __builtin_amdgcn_mfma_f32_32x32x2f32(v[t], sc[0][e], acc[t], 0, 0, 0);
                }
            } else {
#pragma unroll
                for (int ks = 0; ks < N / 16; ks++) {
                    uint32_t pb[TERMS][4];
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const float y0 = sc[ks / 2][8 * (ks % 2) + 2 * e], y1 = sc[ks / 2][8 * (ks % 2) + 2 * e + 1];
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
                    const int i16 = lane & 15, dh = (lane >> 4) & 1;
                    const int vrow = 16 * ks + 4 * p + (i16 >> 2), ch = 2 * dh + ((i16 >> 1) & 1), in = 8 * (i16 & 1);
#pragma unroll
                    for (int t = 0; t < DT; t++) {
                        const v8b va = join_halves(read_transposed(V + lds_slot<ROW>(vrow, ch + 4 * t) + in),
                                                   read_transposed(V + lds_slot<ROW>(vrow + 8, ch + 4 * t) + in));
#pragma unroll
                        for (int z = TERMS - 1; z >= 0; z--) {
                            const v4u pv = v4u{pb[z][0], pb[z][1], pb[z][2], pb[z][3]};
                            acc[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(va, __builtin_bit_cast(v8b, pv), acc[t], 0, 0, 0);
                        }
                    }
                }
            }
            if (odd_tile[buf] == k) {
                // the values that are not finite, for the rows that see them
                float* ps = scratch[w];
#pragma unroll
                for (int b = 0; b < BLOCKS; b++) {
#pragma unroll
                    for (int e = 0; e < 8; e++) ps[(8 * (e / 4) + 4 * p + e % 4) * 32 + r] = sc[b / 2][8 * (b % 2) + e];
                    __builtin_amdgcn_wave_barrier();
                    const size_t from = slot_off(a, pg[b], g, j + 16 * b, D);
                    for (int jj = 0; jj < 16 && pg[b] >= 0 && j + 16 * b + jj < end; jj++) {
                        const float y = ps[jj * 32 + r];
                        const bool see = j + 16 * b + jj < sees;
#pragma unroll
                        for (int t = 0; t < DT; t++)
#pragma unroll
                            for (int e = 0; e < 16; e++) {
                                const int mrow = 8 * (e / 4) + 4 * p + e % 4;
                                float v;
                                if constexpr (F32C) v = ((const float*)vc)[from + jj * D + VW * mrow + t];
                                else v = __uint_as_float((uint32_t)((const uint16_t*)vc)[from + jj * D + 32 * t + mrow] << 16);
                                if (!(fabsf(v) < __builtin_huge_valf()) && see) acc[t][e] = fmaf(y, v, acc[t][e]);
                            }
                    }
                    __builtin_amdgcn_wave_barrier();
                }
            }
        }
        if (jn < end) store(buf ^ 1, k + 1, jn, pn);
#pragma unroll
        for (int b = 0; b < BLOCKS; b++) pg[b] = pn[b], pn[b] = pnn[b];
    }

    l += lane_xor<32>(l);
    if (!valid) return;
    const bool none = m == -__builtin_huge_valf();
    float f = none ? 0.0f : 1.0f / l;
    float* po = nullptr;
    if (a.part) {
        const size_t slot = piece + (PREFIX ? a.own.pieces : 0), k = (slot * a.batch.rows + row) * a.heads + head;
        if (p == 0) a.ml[k] = make_float2(m, l);
        po = a.part + k * D;
        f = 1.0f;
    }
    const size_t oat = row * a.os + (size_t)head * D;
    auto put = [&](int d, v4f y) {
        y = none ? v4f{0, 0, 0, 0} : y * f;
        if (a.part) *(v4f*)(po + d) = y;
        else if constexpr (F32Q) *(v4f*)((float*)a.out + oat + d) = y;
        else *(uint2*)((uint16_t*)a.out + oat + d) = make_uint2(pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3]));
    };
    if constexpr (!F32C) {
#pragma unroll
        for (int t = 0; t < DT; t++)
#pragma unroll
            for (int e = 0; e < 16; e += 4) put(32 * t + 2 * e + 4 * p, v4f{acc[t][e], acc[t][e + 1], acc[t][e + 2], acc[t][e + 3]});
    } else if constexpr (VW == 4) {
#pragma unroll
        for (int e = 0; e < 16; e++)
            put(4 * (8 * (e / 4) + 4 * p + e % 4), v4f{acc[0][e], acc[1 % DT][e], acc[2 % DT][e], acc[3 % DT][e]});
    } else {
#pragma unroll
        for (int e = 0; e < 16; e += 2)
            put(2 * (8 * (e / 4) + 4 * p + e % 4), v4f{acc[0][e], acc[1][e], acc[0][e + 1], acc[1][e + 1]});
    }
}

template <int TYPES>
void launch_types(dim3 grid, hipStream_t s, const AttnArgs& a, int dim, bool prefix) {
    if (dim == 64 && prefix) hipLaunchKernelGGL((k_tile<TYPES, 64, true>), grid, dim3(THREADS), 0, s, a);
    else if (dim == 64) hipLaunchKernelGGL((k_tile<TYPES, 64, false>), grid, dim3(THREADS), 0, s, a);
    else if (prefix) hipLaunchKernelGGL((k_tile<TYPES, 128, true>), grid, dim3(THREADS), 0, s, a);
    else hipLaunchKernelGGL((k_tile<TYPES, 128, false>), grid, dim3(THREADS), 0, s, a);
}

}  // namespace

// tiles: at least the row tiles of all spans together
lq8_status launch_tile(hipStream_t s, const AttnArgs& a, PagedTypes types, int dim, size_t tiles, bool prefix) {
    const dim3 grid((unsigned)(tiles * a.kv.kv_heads * (prefix ? a.pre : a.own).pieces));
    if (types == PT_F32_F32) launch_types<PT_F32_F32>(grid, s, a, dim, prefix);
    else if (types == PT_F32_BF16) launch_types<PT_F32_BF16>(grid, s, a, dim, prefix);
    else launch_types<PT_BF16_BF16>(grid, s, a, dim, prefix);
    LQ8_HIP(hipGetLastError());
    return LQ8_OK;
}

}  // namespace lq8
