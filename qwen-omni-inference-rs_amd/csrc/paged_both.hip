// paged_both.hip -- the shared prefix and the sequences' own positions of a
// batch of few rows in one launch (gfx950).
//
// The prefix's products (paged_tile.h: all rows of a group at once) are bound
// by the matrix cores, the own positions (paged_few.h) by memory: side by side
// on a compute unit they overlap, and one launch goes away.
#include <algorithm>

#include "paged_few.h"
#include "paged_tile.h"

namespace lq8 {
namespace {

// Blocks in units of eight (so that block % 8, the XCD, is that of the part's
// own numbering), the two parts' units in turn: one of the rarer part, then
// `ratio` of the other.
struct Turns {
    int pre, own;  // blocks of each part
    int ratio;
    bool pre_rare;
};

constexpr int cmax(int a, int b) { return a > b ? a : b; }

template <int TYPES, int D, bool TILE>
__global__ __launch_bounds__(THREADS, 2) void k_both(AttnArgs a, Turns t) {
    static_assert(THREADS == 64 * FEW_WAVES, "one workgroup size");
    __shared__ __attribute__((aligned(256))) char sm[TILE ? cmax(tile_lds<TYPES, D>(), few_lds<D>()) : few_lds<D>()];
    const int unit = blockIdx.x / 8, turn = unit / (t.ratio + 1), in = unit - turn * (t.ratio + 1);
    const int block = (in == 0 ? turn : turn * t.ratio + in - 1) * 8 + blockIdx.x % 8;
    if ((in == 0) == t.pre_rare) {
        if (block >= t.pre) return;
        if constexpr (TILE) tile_body<TYPES, D, true>(a, block, sm);
        else few_body<TYPES, D, true>(a, block, sm);
    } else {
        if (block < t.own) few_body<TYPES, D, false>(a, block, sm);
    }
}

template <int TYPES>
void launch_types(dim3 grid, hipStream_t s, const AttnArgs& a, const Turns& t, int dim, bool tile) {
    if (dim == 64 && tile) hipLaunchKernelGGL((k_both<TYPES, 64, true>), grid, dim3(THREADS), 0, s, a, t);
    else if (dim == 64) hipLaunchKernelGGL((k_both<TYPES, 64, false>), grid, dim3(THREADS), 0, s, a, t);
    else if (tile) hipLaunchKernelGGL((k_both<TYPES, 128, true>), grid, dim3(THREADS), 0, s, a, t);
    else hipLaunchKernelGGL((k_both<TYPES, 128, false>), grid, dim3(THREADS), 0, s, a, t);
}

}  // namespace

lq8_status launch_both(hipStream_t s, const AttnArgs& a, PagedTypes types, int dim, size_t pre, size_t own, bool tile) {
    const size_t up = (pre + 7) / 8, uo = (own + 7) / 8;
    const bool rare = up <= uo;
    const size_t few = std::min(up, uo), many = std::max(up, uo), ratio = (many + few - 1) / few;
    const Turns t{(int)pre, (int)own, (int)ratio, rare};
    const dim3 grid((unsigned)(few * (ratio + 1) * 8));
    if (types == PT_F32_F32) launch_types<PT_F32_F32>(grid, s, a, t, dim, tile);
    else if (types == PT_F32_BF16) launch_types<PT_F32_BF16>(grid, s, a, t, dim, tile);
    else launch_types<PT_BF16_BF16>(grid, s, a, t, dim, tile);
    LQ8_HIP(hipGetLastError());
    return LQ8_OK;
}

}  // namespace lq8
