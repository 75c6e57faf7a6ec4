// The int8 paged key/value cache: new tokens' vectors quantised as they are
// written (one scale a token and head, the linear's quantiser without its
// rotation), and slots read back as values.
#include "decoder.hpp"
#include "device_common.hpp"

namespace phi_dev {

// One wave a (token, head, k or v) vector, one element a lane and step.
__global__ __launch_bounds__(64) void kv_write_kernel(KvCache c, KvTokens t) {
    const int64_t token = blockIdx.x;
    const int head = blockIdx.y, lane = threadIdx.x;
    const bool v = blockIdx.z;
    const int64_t slot = t.slots[token];
    if (slot < 0 || slot >= c.slots) return;
    const int64_t from = token * (v ? t.v_token : t.k_token) + head * (v ? t.v_head : t.k_head);
    const int64_t block = slot / c.page, at = slot - block * c.page;
    const void* src = v ? t.v : t.k;
    float x[4], amax = 0.0f;
    bool fine = true;
    for (int i = 0; i < 4; i++) {
        const int d = 64 * i + lane;
        x[i] = d >= c.dim ? 0.0f : t.bf16 ? bf16_to_f32(((const uint16_t*)src)[from + d]) : ((const float*)src)[from + d];
        amax = fmaxf(amax, fabsf(x[i]));
        fine &= __builtin_isfinite(x[i]);
    }
    amax = wave_max(fine ? amax : INFINITY);
    fine = amax != INFINITY;
    const float scale = amax > 1e-30f ? amax / 127.0f : 1.0f, inv = 1.0f / scale;
    int8_t* dst = (v ? c.v : c.k) + block * c.block_stride + head * c.head_stride + at * c.token_stride;
    for (int i = 0; i < 4; i++)
        if (64 * i + lane < c.dim) dst[64 * i + lane] = fine ? (int8_t)quant_code(x[i], inv, 127.0f, 0) : 0;
    if (lane == 0)
        (v ? c.vs : c.ks)[block * c.s_block_stride + head * c.s_head_stride + at * c.s_token_stride] = fine ? scale : __builtin_nanf("");
}

__global__ __launch_bounds__(64) void kv_read_kernel(KvCache c, KvTokens t) {
    const int64_t token = blockIdx.x;
    const int head = blockIdx.y, lane = threadIdx.x;
    const bool v = blockIdx.z;
    const int64_t slot = t.slots[token];
    const bool live = slot >= 0 && slot < c.slots;
    const int64_t to = token * (v ? t.v_token : t.k_token) + head * (v ? t.v_head : t.k_head);
    const int64_t block = live ? slot / c.page : 0, at = live ? slot - block * c.page : 0;
    const int8_t* src = (v ? c.v : c.k) + block * c.block_stride + head * c.head_stride + at * c.token_stride;
    const float scale = (v ? c.vs : c.ks)[block * c.s_block_stride + head * c.s_head_stride + at * c.s_token_stride];
    void* dst = v ? t.v : t.k;
    for (int d = lane; d < c.dim; d += 64) {
        const float x = live ? (float)src[d] * scale : 0.0f;
        if (t.bf16) ((uint16_t*)dst)[to + d] = (uint16_t)f32_to_bf16(x);
        else ((float*)dst)[to + d] = x;
    }
}

hipError_t launch_kv_cache_write(hipStream_t stream, const KvCache& c, const KvTokens& t) {
    hipLaunchKernelGGL(kv_write_kernel, dim3((unsigned)t.tokens, (unsigned)c.heads, 2), dim3(64), 0, stream, c, t);
    return hipGetLastError();
}

hipError_t launch_kv_cache_read(hipStream_t stream, const KvCache& c, const KvTokens& t) {
    hipLaunchKernelGGL(kv_read_kernel, dim3((unsigned)t.tokens, (unsigned)c.heads, 2), dim3(64), 0, stream, c, t);
    return hipGetLastError();
}

}  // namespace phi_dev
