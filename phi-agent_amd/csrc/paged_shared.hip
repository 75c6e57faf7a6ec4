// Shared prefixes: one launch for the groups' rows over their prefixes, which the matrix
// cores bound (paged_chunk.hpp), and the sequences' over their own tokens, which memory
// bounds (paged_decode.hpp).  Blocks of eight waves take a unit of the first or, behind
// these, two of the second, so that both kinds run at the same time on different compute
// units (64 sequences behind 8192 tokens with 32 to 1024 of their own, 32 heads over 8: 47 us,
// 71 in two launches).  There the prefix's 88 blocks take 38 us each, 2.6 of them to look
// their work up and 2.3 a tile of 64 tokens; a unit of own tokens takes 20 us while all start, 3.4
// for its lookup, 2.9 for Q, 12 for some four steps a wave, 4 for the join.
#include "paged_chunk.hpp"
#include "paged_decode.hpp"

namespace phi_dev {

template <int DP, bool PAGE16>
__global__ __launch_bounds__(512, 2) void paged_shared_kernel(KvCache c, PagedAttn p, AttnPart many, AttnPart few, const int32_t* __restrict__ table) {
    extern __shared__ __align__(16) uint8_t lds[];
    const int chunks = many.blocks * c.heads, block = blockIdx.x;
    if (block < chunks) {
        paged_chunk<DP, 8, PAGE16, true>(c, p, many, table, *(ChunkLds<DP>*)lds, block);
    } else {
        const int half = __builtin_amdgcn_readfirstlane(threadIdx.x >> 8);
        paged_decode<DP, false, PAGE16, true, true>(c, p, few, table, ((DecodeLds<DP>*)lds)[half], 2 * (block - chunks) + half, threadIdx.x & 255);
    }
}

template <int DP>
static hipError_t launch_dp(hipStream_t stream, const KvCache& c, const PagedAttn& p, const AttnPart& many, const AttnPart& few) {
    const int64_t blocks = (int64_t)many.blocks * c.heads + ((int64_t)few.blocks * c.heads + 1) / 2;
    const bool page16 = tiles_of_16(c);
    const size_t lds = sizeof(ChunkLds<DP>) > 2 * sizeof(DecodeLds<DP>) ? sizeof(ChunkLds<DP>) : 2 * sizeof(DecodeLds<DP>);
    const void* f = page16 ? (const void*)paged_shared_kernel<DP, true> : (const void*)paged_shared_kernel<DP, false>;
    if (lds > 65536) {
        const hipError_t e = hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess) return e;
    }
    if (page16) hipLaunchKernelGGL((paged_shared_kernel<DP, true>), dim3((unsigned)blocks), dim3(512), lds, stream, c, p, many, few, p.table);
    else hipLaunchKernelGGL((paged_shared_kernel<DP, false>), dim3((unsigned)blocks), dim3(512), lds, stream, c, p, many, few, p.table);
    return hipGetLastError();
}

hipError_t launch_paged_shared(hipStream_t stream, const KvCache& c, const PagedAttn& p, const AttnPart& many, const AttnPart& few) {
    return c.dim <= 64 ? launch_dp<64>(stream, c, p, many, few) : launch_dp<128>(stream, c, p, many, few);
}

}  // namespace phi_dev
