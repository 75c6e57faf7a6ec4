// Parameters of the decoder layer's kernels: the norm that gives the linear's
// int8 operand (rms_norm_quant.hip), the paged int8 cache (kv_cache.hip) and
// the attention over it (paged_attention.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace phi_dev {

// One row per token, pitches in elements; null residual, residual_out, weight,
// shift and y are left out.
struct RmsNorm {
    const void* x;
    const void* residual;
    void* residual_out;
    const void* weight;
    const void* shift;
    void* y;
    int8_t* q;
    float* s;
    int64_t ldx, ldr, ldy, ldq, rows;
    int K;
    float eps, qmax;
    bool x_bf16, r_bf16, w_bf16, y_bf16, half_even, rotate;
};
hipError_t launch_rms_norm_quant(hipStream_t stream, const RmsNorm& p);

// The cache, and t / page as (t * page_mul) >> page_shift for 0 <= t < 2^31.
struct KvCache {
    int8_t* k;
    int8_t* v;
    float* ks;
    float* vs;
    int64_t block_stride, head_stride, token_stride;
    int64_t s_block_stride, s_head_stride, s_token_stride;
    int64_t slots;  // blocks * page
    int blocks, heads, page, dim;
    uint32_t page_mul;
    int page_shift;
};

__host__ __device__ __forceinline__ int page_of(const KvCache& c, int t) {
    return (int)(((uint64_t)(uint32_t)t * c.page_mul) >> c.page_shift);
}

struct KvTokens {
    void* k;
    void* v;
    int64_t k_token, k_head, v_token, v_head;  // strides, elements
    const int64_t* slots;
    int64_t tokens;
    bool bf16;
};
hipError_t launch_kv_cache_write(hipStream_t stream, const KvCache& c, const KvTokens& t);
hipError_t launch_kv_cache_read(hipStream_t stream, const KvCache& c, const KvTokens& t);

struct PagedAttn {
    const void* q;
    void* out;
    const int32_t* table;
    const int32_t* q_start;
    const int32_t* kv_len;
    int64_t q_token, q_head, out_token, out_head;  // strides, elements
    int64_t table_stride;
    int64_t tokens;
    int q_heads, group;  // group: query heads a key/value head
    int batch, max_q, max_kv, table_width, window;
    int few_rows;  // see paged_attention.hpp
    float scale;
    bool bf16, causal;
};
hipError_t launch_paged_attention(hipStream_t stream, const KvCache& c, const PagedAttn& p, void* workspace);
size_t paged_attention_workspace(int64_t tokens, int q_heads, int kv_heads, int dim, int batch, int max_q, int max_kv,
                                 bool bf16);

}  // namespace phi_dev
