// Attention of chunks of new tokens over the paged int8 cache (paged_chunk.hpp), launched.
#include "paged_chunk.hpp"

namespace phi_dev {

template <int DP, int NW, bool PAGE16, bool SHARED>
__global__ __launch_bounds__(64 * NW, DP <= 128 ? 2 : 1) void paged_chunk_kernel(KvCache c, PagedAttn p, AttnPart sp,
                                                                              const int32_t* __restrict__ table) {
    extern __shared__ __align__(16) uint8_t lds_raw[];
    paged_chunk<DP, NW, PAGE16, SHARED>(c, p, sp, table, *(ChunkLds<DP>*)lds_raw, blockIdx.x);
}

template <int DP, int NW, bool SHARED>
static hipError_t launch_shared(hipStream_t stream, const KvCache& c, const PagedAttn& p, const AttnPart& s) {
    const dim3 grid((unsigned)s.blocks * (unsigned)c.heads), block(64 * NW);
    const bool page16 = tiles_of_16(c);
    const void* f = page16 ? (const void*)paged_chunk_kernel<DP, NW, true, SHARED> : (const void*)paged_chunk_kernel<DP, NW, false, SHARED>;
    const size_t lds = sizeof(ChunkLds<DP>);
    if (lds > 65536) {
        const hipError_t e = hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess) return e;
    }
    if (page16) hipLaunchKernelGGL((paged_chunk_kernel<DP, NW, true, SHARED>), grid, block, lds, stream, c, p, s, p.table);
    else hipLaunchKernelGGL((paged_chunk_kernel<DP, NW, false, SHARED>), grid, block, lds, stream, c, p, s, p.table);
    return hipGetLastError();
}

template <int DP, int NW>
static hipError_t launch_dp(hipStream_t stream, const KvCache& c, const PagedAttn& p, const AttnPart& s) {
    return p.groups ? launch_shared<DP, NW, true>(stream, c, p, s) : launch_shared<DP, NW, false>(stream, c, p, s);
}

hipError_t launch_paged_chunk(hipStream_t stream, const KvCache& c, const PagedAttn& p, const AttnPart& s) {
    if (c.dim <= 64) return launch_dp<64, kChunkRows / 32>(stream, c, p, s);
    if (c.dim <= 128) return launch_dp<128, kChunkRows / 32>(stream, c, p, s);
    return launch_dp<256, kChunkRowsWide / 32>(stream, c, p, s);
}

}  // namespace phi_dev
