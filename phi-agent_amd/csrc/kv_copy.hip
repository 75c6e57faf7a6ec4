// Blocks of the paged cache copied: forked sequences' last pages, compaction.
//
// Bound by memory.  A pair's codes of k, then of v, are pieces of 16 bytes in the order
// in which they lie (tokens within heads, or heads within tokens), one a thread; then both
// scales, a float each.  (Four pieces a thread, loaded before they are stored: 115 us, 113 so,
// for 2048 pages of 64 tokens, 8 heads of 128, 4.8 TB/s.)
#include <algorithm>

#include "device_common.hpp"
#include "serving.hpp"

namespace phi_dev {

namespace {

// n / d as (n * mul) >> shift for 0 <= n < 2^31.
struct Div {
    uint32_t d, mul;
    int shift;
};
Div div_by(uint32_t d) {
    int lg = 0;
    while (1u << lg < d) lg++;
    return {d, (uint32_t)(((uint64_t)1 << (31 + lg)) / d + 1), 31 + lg};
}
__device__ __forceinline__ uint32_t quotient(const Div& d, uint32_t n) { return (uint32_t)(((uint64_t)n * d.mul) >> d.shift); }

}  // namespace

// inner, outer: the smaller stride's and the larger's counts of a page's vectors;
// token_inner: the inner are tokens.
__global__ __launch_bounds__(256, 8) void kv_copy_kernel(KvCopy p, Div vector, Div inner, bool token_inner, bool dense, int code_parts, int scale_parts) {
    const int per = 2 * code_parts + scale_parts;
    const int64_t i = blockIdx.x / per;
    const int part = blockIdx.x - (int)i * per;
    const int from = p.from_blocks[i], to = p.to_blocks[i];
    if (from < 0 || from >= p.from.blocks || to < 0 || to >= p.to.blocks) return;
    const uint32_t take = (uint32_t)min(max(p.tokens ? p.tokens[i] : p.from.page, 0), p.from.page);
    const uint32_t vectors = (uint32_t)p.from.heads * (uint32_t)p.from.page;
    const bool scales = part >= 2 * code_parts;
    const bool v = !scales && part >= code_parts;
    const uint32_t first = (uint32_t)(scales ? part - 2 * code_parts : v ? part - code_parts : part) * 256 + threadIdx.x;
    // Vector n's head and token.
    auto place = [&](uint32_t n, uint32_t& head, uint32_t& token) {
        const uint32_t o = quotient(inner, n), in = n - o * inner.d;
        head = token_inner ? o : in, token = token_inner ? in : o;
    };
    if (scales) {
        uint32_t head, token;
        if (first >= vectors) return;
        place(first, head, token);
        if (token >= take) return;
        const int64_t a = from * p.from.s_block_stride + head * p.from.s_head_stride + token * p.from.s_token_stride;
        const int64_t b = to * p.to.s_block_stride + head * p.to.s_head_stride + token * p.to.s_token_stride;
        p.to.ks[b] = p.from.ks[a];
        p.to.vs[b] = p.from.vs[a];
        return;
    }
    const int8_t* src = (v ? p.from.v : p.from.k) + from * p.from.block_stride;
    int8_t* dst = (v ? p.to.v : p.to.k) + to * p.to.block_stride;
    if (first >= vectors * vector.d) return;
    if (dense && take == (uint32_t)p.from.page) {
        *(v4i*)(dst + 16 * (uint64_t)first) = *(const v4i*)(src + 16 * (uint64_t)first);
        return;
    }
    const uint32_t vec = quotient(vector, first), in = 16 * (first - vec * vector.d);
    uint32_t head, token;
    place(vec, head, token);
    if (token < take)
        *(v4i*)(dst + head * p.to.head_stride + token * p.to.token_stride + in) = *(const v4i*)(src + head * p.from.head_stride + token * p.from.token_stride + in);
}

hipError_t launch_kv_cache_copy(hipStream_t stream, const KvCopy& p) {
    const KvCache& c = p.from;
    const bool token_inner = c.token_stride <= c.head_stride;
    const int64_t inner = token_inner ? c.token_stride : c.head_stride, outer = token_inner ? c.head_stride : c.token_stride;
    const bool dense = inner == c.dim && outer == (token_inner ? c.page : c.heads) * inner && p.to.token_stride == c.token_stride && p.to.head_stride == c.head_stride;
    const int64_t vectors = (int64_t)c.heads * c.page, pieces = vectors * (c.dim / 16), each = 256;
    const int code_parts = (int)((pieces + each - 1) / each), scale_parts = (int)((vectors + each - 1) / each);
    const int64_t per = 2 * (int64_t)code_parts + scale_parts, at_once = kMaxBlocks / per;
    for (int64_t i = 0; i < p.n; i += at_once) {
        KvCopy s = p;
        s.n = std::min(p.n - i, at_once);
        s.from_blocks += i, s.to_blocks += i;
        if (s.tokens) s.tokens += i;
        hipLaunchKernelGGL(kv_copy_kernel, dim3((unsigned)(s.n * per)), dim3(256), 0, stream, s, div_by(c.dim / 16),
                           div_by(token_inner ? c.page : c.heads), token_inner, dense, code_parts, scale_parts);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace phi_dev
