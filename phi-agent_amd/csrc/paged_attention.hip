// Attention of new tokens over the paged int8 cache: which kernel takes a call,
// how its tokens are split over blocks, and the join of the splits.
#include <algorithm>

#include "paged_attention.hpp"

namespace phi_dev {

// The splits' partial softmaxes of a row and head joined, a wave a row.  Lane z
// has split z's maximum and sum, so that these are one round of loads; then a
// lane sums four of the vector's elements, the weights read from their lanes.
// A part of one split has written its rows itself.
__global__ __launch_bounds__(256) void attn_join_kernel(PagedAttn p, AttnPart few, AttnPart many, int page, int D, int kv_heads) {
    const int lane = threadIdx.x & 63;
    const int64_t at = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int token = (int)(at / p.q_heads), head = (int)(at - (int64_t)token * p.q_heads);
    if (token >= p.tokens) return;
    // The sequence of the token: the last that starts at it or before, and has it.
    int b = -1;
    for (int b0 = 0; b0 < p.batch; b0 += 64) {
        const uint64_t on = __ballot(b0 + lane < p.batch && p.q_start[min(b0 + lane, p.batch - 1)] <= token);
        if (on) b = b0 + 63 - __builtin_clzll(on);
        if (~on) break;
    }
    if (b < 0) return;
    const SeqInfo q = seq_info(p, page, b);
    const int i = token - q.first, rows = min(q.n, p.max_q) * p.group, kh = head / p.group;
    if (i >= min(q.n, p.max_q)) return;
    const bool is_few = rows <= p.few_rows;
    const AttnPart& s = is_few ? few : many;
    if (s.count == 1) return;
    const int64_t row = is_few ? ((int64_t)b * kv_heads + kh) * s.row_pitch + i * p.group + head - kh * p.group : at;
    const int n = max(1, (q.kv + s.len - 1) / s.len), d = 4 * lane < D ? 4 * lane : 0;
    float m = kNoMax, l = 0.0f;
    v4f x = {0, 0, 0, 0};
    for (int z0 = 0; z0 < n; z0 += 64) {
        const int z = z0 + lane;
        const float2 ml = z < n ? *(const float2*)(s.ml + 2 * (z * s.rows + row)) : make_float2(kNoMax, 0.0f);
        const float m2 = fmaxf(m, wave_max(ml.x)), keep = __builtin_amdgcn_exp2f(m - m2);
        const float w = __builtin_amdgcn_exp2f(ml.x - m2);
        float sum = ml.y * w;
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off, 64);
        l = l * keep + sum;
        x *= keep;
        m = m2;
        const int count = min(64, n - z0);
        const float* o = s.o + (z0 * s.rows + row) * D + d;
        int k = 0;
        for (; k + 4 <= count; k += 4) {
            v4f y[4];
#pragma unroll
            for (int u = 0; u < 4; u++) y[u] = *(const v4f*)(o + (k + u) * s.rows * D);
#pragma unroll
            for (int u = 0; u < 4; u++) x += y[u] * __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(w), k + u));
        }
        for (; k < count; k++) x += *(const v4f*)(o + k * s.rows * D) * __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(w), k));
    }
    x *= l != 0.0f ? 1.0f / l : 0.0f;
    if (4 * lane >= D) return;
    const int64_t to = token * p.out_token + head * p.out_head + d;
    if (!p.bf16) *(v4f*)((float*)p.out + to) = x;
    else *(uint2*)((uint16_t*)p.out + to) = make_uint2(f32x2_to_bf16x2(x[0], x[1]), f32x2_to_bf16x2(x[2], x[3]));
}

namespace {

// bf16 sequences of more rows than this go to the chunk kernel.
constexpr int kFewRows = 128;

struct Plan {
    int few_rows;
    AttnPart few, many;  // blocks = 0: does not run
};

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// How many splits of `step` tokens' multiples bring `units` blocks to `target`.
void split(AttnPart& s, int64_t units, int64_t target, int64_t step, int64_t max_kv) {
    const int64_t most = std::max<int64_t>(1, ceil_div(max_kv, step));
    const int64_t want = std::max<int64_t>(1, std::min(most, target / std::max<int64_t>(1, units)));
    s.len = (int)(std::max<int64_t>(1, ceil_div(max_kv, want * step)) * step);
    s.count = (int)std::max<int64_t>(1, ceil_div(max_kv, s.len));
}

Plan attn_plan(int64_t tokens, int64_t q_heads, int64_t kv_heads, int64_t dim, int64_t batch, int64_t max_q, int64_t max_kv, bool bf16) {
    const int64_t group = q_heads / kv_heads, rows = max_q * group;
    Plan a{};
    a.few_rows = bf16 ? kFewRows : INT32_MAX;
    const int64_t few = std::min<int64_t>(rows, a.few_rows);
    if (rows > a.few_rows) {
        const int64_t tile = dim <= 128 ? kChunkRows : kChunkRowsWide;
        const int64_t units = std::min(batch * ceil_div(rows, tile), ceil_div(tokens * group, tile) + batch);
        split(a.many, units * kv_heads, 512, 256, max_kv);
        a.many.rows = tokens * q_heads;
        a.many.blocks = (int)std::min<int64_t>(units * a.many.count, INT32_MAX / kv_heads);
    }
    if (rows <= a.few_rows || batch > 1) {
        const int64_t tiles = ceil_div(few, kDecodeRows);
        const int64_t units = std::min(batch * tiles, ceil_div(tokens * group, kDecodeRows) + batch);
        // Beside chunks most sequences of few rows are single tokens.
        split(a.few, (rows <= a.few_rows ? units : batch) * kv_heads, 2048, 128, max_kv);
        a.few.row_pitch = (int)few;
        a.few.rows = batch * kv_heads * few;
        a.few.blocks = (int)std::min<int64_t>(units * a.few.count, INT32_MAX / kv_heads);
    }
    return a;
}

int64_t part_floats(const AttnPart& s, int64_t dim) { return s.count > 1 ? s.count * s.rows * (dim + 2) : 0; }

}  // namespace

size_t paged_attention_workspace(int64_t tokens, int q_heads, int kv_heads, int dim, int batch, int max_q, int max_kv, bool bf16) {
    const Plan a = attn_plan(tokens, q_heads, kv_heads, dim, batch, max_q, max_kv, bf16);
    return (size_t)(part_floats(a.few, dim) + part_floats(a.many, dim)) * sizeof(float);
}

hipError_t launch_paged_attention(hipStream_t stream, const KvCache& c, const PagedAttn& p0, void* workspace) {
    Plan a = attn_plan(p0.tokens, p0.q_heads, c.heads, c.dim, p0.batch, p0.max_q, p0.max_kv, p0.bf16);
    PagedAttn p = p0;
    p.few_rows = a.few_rows;
    float* ws = (float*)workspace;
    for (AttnPart* s : {&a.few, &a.many}) {
        if (s->count <= 1) continue;
        s->o = ws;
        s->ml = ws + s->count * s->rows * c.dim;
        ws += part_floats(*s, c.dim);
    }
    hipError_t e = hipSuccess;
    if (a.many.blocks) e = launch_paged_chunk(stream, c, p, a.many);
    if (e == hipSuccess && a.few.blocks) e = launch_paged_decode(stream, c, p, a.few);
    if (e != hipSuccess || (a.few.count <= 1 && a.many.count <= 1)) return e;
    hipLaunchKernelGGL(attn_join_kernel, dim3((unsigned)ceil_div(p.tokens * p.q_heads, 4)), dim3(256), 0, stream, p, a.few, a.many,
                       c.page, c.dim, c.heads);
    return hipGetLastError();
}

}  // namespace phi_dev
