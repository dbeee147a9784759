// paged_tile.hip -- launches of attention for many packed rows (paged_tile.h).
#include "paged_tile.h"

namespace lq8 {
namespace {

template <int TYPES, int D, bool PREFIX>
__global__ __launch_bounds__(THREADS, 2) void k_tile(AttnArgs a) {
    __shared__ __attribute__((aligned(256))) char sm[tile_lds<TYPES, D>()];
    tile_body<TYPES, D, PREFIX>(a, blockIdx.x, sm);
}

template <int TYPES>
void launch_types(dim3 grid, hipStream_t s, const AttnArgs& a, int dim, bool prefix) {
    if (dim == 64 && prefix) hipLaunchKernelGGL((k_tile<TYPES, 64, true>), grid, dim3(THREADS), 0, s, a);
    else if (dim == 64) hipLaunchKernelGGL((k_tile<TYPES, 64, false>), grid, dim3(THREADS), 0, s, a);
    else if (prefix) hipLaunchKernelGGL((k_tile<TYPES, 128, true>), grid, dim3(THREADS), 0, s, a);
    else hipLaunchKernelGGL((k_tile<TYPES, 128, false>), grid, dim3(THREADS), 0, s, a);
}

}  // namespace

lq8_status launch_tile(hipStream_t s, const AttnArgs& a, PagedTypes types, int dim, size_t blocks, bool prefix) {
    const dim3 grid((unsigned)blocks);
    if (types == PT_F32_F32) launch_types<PT_F32_F32>(grid, s, a, dim, prefix);
    else if (types == PT_F32_BF16) launch_types<PT_F32_BF16>(grid, s, a, dim, prefix);
    else launch_types<PT_BF16_BF16>(grid, s, a, dim, prefix);
    LQ8_HIP(hipGetLastError());
    return LQ8_OK;
}

}  // namespace lq8
