// Attention of new tokens over the paged int8 cache: which kernel takes a call,
// how its tokens are split over blocks, and the join of the splits.
#include <algorithm>

#include "paged_attention.hpp"

namespace phi_dev {

// The splits' partial softmaxes of a row and head joined: a wave a row, a
// quarter of its vector's elements a lane at a time.
__global__ __launch_bounds__(256) void attn_join_kernel(PagedAttn p, AttnSplit s, int page, int D) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, b = blockIdx.y;
    const SeqInfo q = seq_info(p, page, b);
    const int at = blockIdx.x * 4 + wave, i = at / p.q_heads, head = at - i * p.q_heads;
    if (i >= min(q.n, p.max_q)) return;
    const int64_t row = (int64_t)(q.first + i) * p.q_heads + head, rows = p.tokens * p.q_heads;
    const int n = max(1, (q.kv + s.len - 1) / s.len);
    float m = kNoMax, l = 0.0f;
    for (int z = 0; z < n; z++) {
        const float mz = s.ml[2 * (z * rows + row)], lz = s.ml[2 * (z * rows + row) + 1];
        const float m2 = fmaxf(m, mz);
        l = l * __builtin_amdgcn_exp2f(m - m2) + lz * __builtin_amdgcn_exp2f(mz - m2);
        m = m2;
    }
    const float inv = l != 0.0f ? 1.0f / l : 0.0f;
    const int d = 4 * lane;
    if (d >= D) return;
    v4f x = {0, 0, 0, 0};
    for (int z = 0; z < n; z++) {
        const float f = __builtin_amdgcn_exp2f(s.ml[2 * (z * rows + row)] - m) * inv;
        x += *(const v4f*)(s.o + (z * rows + row) * D + d) * f;
    }
    const int64_t to = (int64_t)(q.first + i) * p.out_token + head * p.out_head + d;
    if (!p.bf16) *(v4f*)((float*)p.out + to) = x;
    else *(uint2*)((uint16_t*)p.out + to) = make_uint2(f32x2_to_bf16x2(x[0], x[1]), f32x2_to_bf16x2(x[2], x[3]));
}

namespace {

// Sequences of more rows than this go to the chunk kernel.
constexpr int64_t kFewRows = 128;

struct Plan {
    bool few, many;  // the kernels that run
    int len, count;  // tokens a split, splits
};

Plan attn_plan(int64_t q_heads, int64_t kv_heads, int64_t dim, int64_t batch, int64_t max_q, int64_t max_kv, bool bf16) {
    const int64_t rows = max_q * (q_heads / kv_heads);
    const bool many = bf16 && rows > kFewRows;
    const int64_t tile = !many ? kDecodeRows : dim <= 128 ? kChunkRows : kChunkRowsWide;
    const int64_t units = batch * kv_heads * ((rows + tile - 1) / tile);
    const int64_t step = many ? 256 : 128, target = many ? 512 : 2048;
    const int64_t most = (max_kv + step - 1) / step;
    const int64_t want = std::max<int64_t>(1, std::min<int64_t>(most, target / units));
    const int64_t len = std::max<int64_t>(1, (max_kv + want * step - 1) / (want * step)) * step;
    return {!many || batch > 1, many, (int)len, (int)std::max<int64_t>(1, (max_kv + len - 1) / len)};
}

}  // namespace

size_t paged_attention_workspace(int64_t tokens, int q_heads, int kv_heads, int dim, int batch, int max_q, int max_kv, bool bf16) {
    const Plan a = attn_plan(q_heads, kv_heads, dim, batch, max_q, max_kv, bf16);
    return a.count > 1 ? (size_t)a.count * (size_t)tokens * (size_t)q_heads * (size_t)(dim + 2) * sizeof(float) : 0;
}

hipError_t launch_paged_attention(hipStream_t stream, const KvCache& c, const PagedAttn& p, void* workspace) {
    const Plan a = attn_plan(p.q_heads, c.heads, c.dim, p.batch, p.max_q, p.max_kv, p.bf16);
    const int64_t rows = p.tokens * p.q_heads;
    AttnSplit s{a.len, a.count, nullptr, nullptr};
    if (a.count > 1) {
        s.o = (float*)workspace;
        s.ml = s.o + (int64_t)a.count * rows * c.dim;
    }
    const int64_t few = a.many ? kFewRows : INT32_MAX;
    hipError_t e = a.many ? launch_paged_chunk(stream, c, p, s, few) : hipSuccess;
    if (e == hipSuccess && a.few) e = launch_paged_decode(stream, c, p, s, few);
    if (e != hipSuccess || a.count == 1) return e;
    hipLaunchKernelGGL(attn_join_kernel, dim3((unsigned)(((int64_t)p.max_q * p.q_heads + 3) / 4), (unsigned)p.batch), dim3(256),
                       0, stream, p, s, c.page, c.dim);
    return hipGetLastError();
}

}  // namespace phi_dev
