// Attention of new tokens over the paged int8 cache: which kernel takes a call,
// how its tokens are split over blocks, and the join of the splits.
#include <algorithm>

#include "paged_attention.hpp"

namespace phi_dev {

// In fp32: one block a (row, query head), its four waves on every fourth tile
// of 64 tokens with a running maximum and sum of their own, joined at the end.
__global__ __launch_bounds__(256) void paged_attn_row_kernel(KvCache c, PagedAttn p) {
    __shared__ float qs[256], ps[4][64], os[4][256], ms[4], ls[4];
    __shared__ int64_t at[4][64];
    const int b = blockIdx.z, head = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int kh = head / p.group, D = c.dim;
    const int64_t first = max(0, p.q_start[b]), end = min(p.tokens, (int64_t)p.q_start[b + 1]);
    const int64_t row = first + blockIdx.x;
    if (row >= end) return;
    const int kv = min(p.kv_len[b], min((int64_t)p.max_kv, (int64_t)p.table_width * c.page));
    const int64_t pos = (int64_t)p.kv_len[b] - (end - first) + blockIdx.x;
    for (int d = threadIdx.x; d < D; d += 256) {
        const int64_t i = row * p.q_token + head * p.q_head + d;
        qs[d] = p.bf16 ? bf16_to_f32(((const uint16_t*)p.q)[i]) : ((const float*)p.q)[i];
    }
    __syncthreads();
    const int hi = p.causal ? (int)min((int64_t)kv, pos + 1) : kv;
    const int lo = p.window > 0 ? (int)max((int64_t)0, pos + 1 - p.window) : 0;
    float m = -INFINITY, l = 0.0f, acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int t0 = lo / 64 * 64 + 64 * wave; t0 < hi; t0 += 256) {
        const int t = t0 + lane;
        float s = -INFINITY, sv = 0.0f;
        int64_t off = -1;
        if (t >= lo && t < hi) {
            const int page = page_of(c, t), in = t - page * c.page;
            const int block = p.table[b * p.table_stride + page];
            if (block >= 0 && block < c.blocks) {
                off = block * c.block_stride + kh * c.head_stride + in * c.token_stride;
                const int64_t so = block * c.s_block_stride + kh * c.s_head_stride + in * c.s_token_stride;
                sv = c.vs[so];
                float sum = 0.0f;
                for (int d = 0; d < D; d += 4) {
                    const char4 k = *(const char4*)(c.k + off + d);
                    sum = fmaf(qs[d], k.x, sum);
                    sum = fmaf(qs[d + 1], k.y, sum);
                    sum = fmaf(qs[d + 2], k.z, sum);
                    sum = fmaf(qs[d + 3], k.w, sum);
                }
                s = sum * c.ks[so] * p.scale;
            }
        }
        const float top = wave_max(s), m2 = fmaxf(m, top);
        const float base = m2 == -INFINITY ? 0.0f : m2, keep = expf(m - base), e = off >= 0 ? expf(s - base) : 0.0f;
        float sum = e;
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
        l = l * keep + sum;
        m = m2;
        ps[wave][lane] = off >= 0 ? e * sv : 0.0f;
        at[wave][lane] = off;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
        for (int i = 0; i < 4; i++) acc[i] *= keep;
        for (int j = 0; j < 64; j++) {
            if (at[wave][j] < 0) continue;
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (64 * i + lane < D) acc[i] = fmaf(ps[wave][j], c.v[at[wave][j] + 64 * i + lane], acc[i]);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
#pragma unroll
    for (int i = 0; i < 4; i++) os[wave][64 * i + lane] = acc[i];
    if (lane == 0) ms[wave] = m, ls[wave] = l;
    __syncthreads();
    const float top = fmaxf(fmaxf(ms[0], ms[1]), fmaxf(ms[2], ms[3])), base = top == -INFINITY ? 0.0f : top;
    float total = 0.0f;
    for (int w = 0; w < 4; w++) total += ls[w] * expf(ms[w] - base);
    for (int d = threadIdx.x; d < D; d += 256) {
        float o = 0.0f;
        for (int w = 0; w < 4; w++) o += os[w][d] * expf(ms[w] - base);
        o = total != 0.0f ? o / total : 0.0f;
        const int64_t i = row * p.out_token + head * p.out_head + d;
        if (p.bf16) ((uint16_t*)p.out)[i] = (uint16_t)f32_to_bf16(o);
        else ((float*)p.out)[i] = o;
    }
}

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

struct Plan {
    bool decode;
    int len, count;  // tokens a split, splits
};

Plan attn_plan(int64_t q_heads, int64_t kv_heads, int64_t batch, int64_t max_q, int64_t max_kv) {
    const int64_t rows = max_q * (q_heads / kv_heads), tiles = (rows + kDecodeRows - 1) / kDecodeRows;
    if (tiles > 1) return {false, 0, 1};
    const int64_t units = batch * kv_heads * tiles, most = (max_kv + 127) / 128;
    const int64_t want = std::max<int64_t>(1, std::min<int64_t>(most, (2048 + units - 1) / units));
    const int64_t len = std::max<int64_t>(1, (max_kv + want * 128 - 1) / (want * 128)) * 128;
    return {true, (int)len, (int)std::max<int64_t>(1, (max_kv + len - 1) / len)};
}

}  // namespace

size_t paged_attention_workspace(int64_t tokens, int q_heads, int kv_heads, int dim, int batch, int max_q, int max_kv, bool) {
    const Plan a = attn_plan(q_heads, kv_heads, batch, max_q, max_kv);
    return a.count > 1 ? (size_t)a.count * (size_t)tokens * (size_t)q_heads * (size_t)(dim + 2) * sizeof(float) : 0;
}

hipError_t launch_paged_attention(hipStream_t stream, const KvCache& c, const PagedAttn& p, void* workspace) {
    const Plan a = attn_plan(p.q_heads, c.heads, p.batch, p.max_q, p.max_kv);
    if (!a.decode) {
        hipLaunchKernelGGL(paged_attn_row_kernel, dim3((unsigned)p.max_q, (unsigned)p.q_heads, (unsigned)p.batch), dim3(256),
                           0, stream, c, p);
        return hipGetLastError();
    }
    const int64_t rows = p.tokens * p.q_heads;
    AttnSplit s{a.len, a.count, nullptr, nullptr};
    if (a.count > 1) {
        s.o = (float*)workspace;
        s.ml = s.o + (int64_t)a.count * rows * c.dim;
    }
    const hipError_t e = launch_paged_decode(stream, c, p, s);
    if (e != hipSuccess || a.count == 1) return e;
    hipLaunchKernelGGL(attn_join_kernel, dim3((unsigned)(((int64_t)p.max_q * p.q_heads + 3) / 4), (unsigned)p.batch), dim3(256),
                       0, stream, p, s, c.page, c.dim);
    return hipGetLastError();
}

}  // namespace phi_dev
