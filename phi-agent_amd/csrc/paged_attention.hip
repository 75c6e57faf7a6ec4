// Attention of new tokens over the paged int8 cache, in fp32: one block a
// (row, query head), its four waves on every fourth tile of 64 tokens with a
// running maximum and sum of their own, joined at the end.
#include "decoder.hpp"
#include "device_common.hpp"

namespace phi_dev {

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

size_t paged_attention_workspace(int64_t, int, int, int, int, int, int, bool) { return 0; }

hipError_t launch_paged_attention(hipStream_t stream, const KvCache& c, const PagedAttn& p, void*) {
    hipLaunchKernelGGL(paged_attn_row_kernel, dim3((unsigned)p.max_q, (unsigned)p.q_heads, (unsigned)p.batch), dim3(256), 0,
                       stream, c, p);
    return hipGetLastError();
}

}  // namespace phi_dev
