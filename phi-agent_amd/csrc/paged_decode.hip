// Attention of a few rows over the paged int8 cache (paged_decode.hpp), launched.
#include "paged_decode.hpp"

namespace phi_dev {

template <int DP, bool F32, bool PAGE16, bool SHARED>
__global__ __launch_bounds__(64 * kWaves, DP <= 128 ? 2 : 1) void paged_decode_kernel(KvCache c, PagedAttn p, AttnPart sp,
                                                                  const int32_t* __restrict__ table) {
    __shared__ DecodeLds<DP> lds;
    paged_decode<DP, F32, PAGE16, SHARED, false>(c, p, sp, table, lds, blockIdx.x, threadIdx.x);
}

template <int DP, bool F32, bool SHARED>
static hipError_t launch_shared(hipStream_t stream, const KvCache& c, const PagedAttn& p, const AttnPart& s) {
    const dim3 grid((unsigned)s.blocks * (unsigned)c.heads), block(64 * kWaves);
    if (tiles_of_16(c)) hipLaunchKernelGGL((paged_decode_kernel<DP, F32, true, SHARED>), grid, block, 0, stream, c, p, s, p.table);
    else hipLaunchKernelGGL((paged_decode_kernel<DP, F32, false, SHARED>), grid, block, 0, stream, c, p, s, p.table);
    return hipGetLastError();
}

template <int DP, bool F32>
static hipError_t launch_dp(hipStream_t stream, const KvCache& c, const PagedAttn& p, const AttnPart& s) {
    return p.groups ? launch_shared<DP, F32, true>(stream, c, p, s) : launch_shared<DP, F32, false>(stream, c, p, s);
}

hipError_t launch_paged_decode(hipStream_t stream, const KvCache& c, const PagedAttn& p, const AttnPart& s) {
    if (c.dim <= 64) return p.bf16 ? launch_dp<64, false>(stream, c, p, s) : launch_dp<64, true>(stream, c, p, s);
    if (c.dim <= 128) return p.bf16 ? launch_dp<128, false>(stream, c, p, s) : launch_dp<128, true>(stream, c, p, s);
    return p.bf16 ? launch_dp<256, false>(stream, c, p, s) : launch_dp<256, true>(stream, c, p, s);
}

}  // namespace phi_dev
