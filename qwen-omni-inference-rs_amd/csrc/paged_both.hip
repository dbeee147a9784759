// paged_both.hip -- the shared prefix and the sequences' own positions of a
// batch of few rows in one launch (gfx950).
//
// The prefix's products (paged_tile.h: all rows of a group at once) are bound
// by the matrix cores, the own positions (paged_few.h) by memory: side by side
// on a compute unit they overlap, and one launch goes away.  64 rows, 32 heads
// over 8 of 128, up to 700 own positions behind 8192: 45 us with the joining of
// the pieces, 61 as two launches; the two parts taken in turn instead of the
// prefix's blocks first: 57.
#include "paged_few.h"
#include "paged_tile.h"

namespace lq8 {
namespace {

constexpr int cmax(int a, int b) { return a > b ? a : b; }

template <int TYPES, int D, bool TILE>
__global__ __launch_bounds__(THREADS, 2) void k_both(AttnArgs a, int pre, int own) {
    __shared__ __attribute__((aligned(256))) char sm[TILE ? cmax(tile_lds<TYPES, D>(), few_lds<D>()) : few_lds<D>()];
    // the prefix's blocks, which take longer, then the own ones from `own` on
    const int block = blockIdx.x;
    if (block >= own) {
        few_body<TYPES, D, false>(a, block - own, sm);
    } else if (block < pre) {
        if constexpr (TILE) tile_body<TYPES, D, true>(a, block, sm);
        else few_body<TYPES, D, true>(a, block, sm);
    }
}

template <int TYPES>
void launch_types(dim3 grid, hipStream_t s, const AttnArgs& a, int pre, int own, int dim, bool tile) {
    if (dim == 64 && tile) hipLaunchKernelGGL((k_both<TYPES, 64, true>), grid, dim3(THREADS), 0, s, a, pre, own);
    else if (dim == 64) hipLaunchKernelGGL((k_both<TYPES, 64, false>), grid, dim3(THREADS), 0, s, a, pre, own);
    else if (tile) hipLaunchKernelGGL((k_both<TYPES, 128, true>), grid, dim3(THREADS), 0, s, a, pre, own);
    else hipLaunchKernelGGL((k_both<TYPES, 128, false>), grid, dim3(THREADS), 0, s, a, pre, own);
}

}  // namespace

lq8_status launch_both(hipStream_t s, const AttnArgs& a, PagedTypes types, int dim, size_t pre, size_t own, bool tile) {
    // (from a multiple of eight: block % 8, the XCD, is that of the part's own numbering)
    const size_t first = (pre + 7) / 8 * 8;
    const dim3 grid((unsigned)(first + own));
    if (types == PT_F32_F32) launch_types<PT_F32_F32>(grid, s, a, (int)pre, (int)first, dim, tile);
    else if (types == PT_F32_BF16) launch_types<PT_F32_BF16>(grid, s, a, (int)pre, (int)first, dim, tile);
    else launch_types<PT_BF16_BF16>(grid, s, a, (int)pre, (int)first, dim, tile);
    LQ8_HIP(hipGetLastError());
    return LQ8_OK;
}

}  // namespace lq8
