// paged_few.hip -- launches of attention for few packed rows (paged_few.h).
#include "paged_few.h"

namespace lq8 {
namespace {

template <int TYPES, int D, bool PREFIX>
__global__ __launch_bounds__(THREADS, 2) void k_few(AttnArgs a) {
    __shared__ __attribute__((aligned(16))) char sm[few_lds<D>()];
    few_body<TYPES, D, PREFIX>(a, blockIdx.x, sm);
}

template <int TYPES>
void launch_types(dim3 grid, hipStream_t s, const AttnArgs& a, int dim, bool prefix) {
    const dim3 block(THREADS);
    if (dim == 64 && prefix) hipLaunchKernelGGL((k_few<TYPES, 64, true>), grid, block, 0, s, a);
    else if (dim == 64) hipLaunchKernelGGL((k_few<TYPES, 64, false>), grid, block, 0, s, a);
    else if (prefix) hipLaunchKernelGGL((k_few<TYPES, 128, true>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((k_few<TYPES, 128, false>), grid, block, 0, s, a);
}

}  // namespace

lq8_status launch_few(hipStream_t s, const AttnArgs& a, PagedTypes types, int dim, size_t blocks, bool prefix) {
    const dim3 grid((unsigned)blocks);
    if (types == PT_F32_F32) launch_types<PT_F32_F32>(grid, s, a, dim, prefix);
    else if (types == PT_F32_BF16) launch_types<PT_F32_BF16>(grid, s, a, dim, prefix);
    else launch_types<PT_BF16_BF16>(grid, s, a, dim, prefix);
    LQ8_HIP(hipGetLastError());
    return LQ8_OK;
}

}  // namespace lq8
