// C ABI of the serving operators (include/phi_serving.h): argument validation and
// dispatch, under the error contract of capi.hip.
#include "../../include/phi_serving.h"
#include "decoder_checks.hpp"
#include "serving.hpp"

using namespace phi_capi;

namespace {

constexpr int64_t kMaxRotaryDim = 1024;   // a wave has a vector
constexpr int64_t kMaxPageVectors = 1 << 26;  // of at most 16 pieces: counted in 31 bits

// [tokens, heads, dim] vectors that are written: one of the strides holds the other's
// vectors apart.
phi_status check_layout(const char* who, const char* name, int64_t tokens, int64_t token_stride, int64_t heads, int64_t head_stride, int64_t dim) {
    const bool by_token = token_stride >= head_stride;
    const int64_t n = by_token ? heads : tokens, s = by_token ? head_stride : token_stride, big = by_token ? token_stride : head_stride;
    if ((n > 1 && s < dim) || ((by_token ? tokens : heads) > 1 && big < (n - 1) * s + dim)) return fail(PHI_ERR_SHAPE, "%s: %s's vectors overlap", who, name);
    return PHI_OK;
}

phi_status check_strides(const char* who, const char* name, const void* x, int dtype, int64_t token_stride, int64_t head_stride) {
    if (!x) return fail(PHI_ERR_ARG, "%s: null %s", who, name);
    if (token_stride < 0 || head_stride < 0 || token_stride > kMaxPitch || head_stride > kMaxPitch)
        return fail(PHI_ERR_SHAPE, "%s: bad stride of %s", who, name);
    if (!aligned(x, elem(dtype))) return fail(PHI_ERR_ALIGN, "%s: %s is not aligned to its type", who, name);
    return PHI_OK;
}

phi_status check_turns(const char* who, const int64_t* positions, const double* freq, int64_t rot, int64_t dim, float scale) {
    if (rot < 2 || rot % 2 != 0 || rot > dim) return fail(PHI_ERR_SHAPE, "%s: %lld rotated elements of %lld", who, (long long)rot, (long long)dim);
    if (!positions || !freq) return fail(PHI_ERR_ARG, "%s: null pointer", who);
    if (!aligned(positions, 8) || !aligned(freq, 8)) return fail(PHI_ERR_ALIGN, "%s: positions or freq is misaligned", who);
    if (!std::isfinite(scale)) return fail(PHI_ERR_ARG, "%s: scale must be finite", who);
    return PHI_OK;
}

}  // namespace

extern "C" {

phi_status phi_hip_rotary(phi_stream_t stream, const void* x, int dtype, int64_t x_token_stride, int64_t x_head_stride,
                          int64_t tokens, int64_t heads, int64_t dim, const int64_t* positions, const double* freq,
                          int64_t rot, int interleaved, float scale, void* out, int64_t out_token_stride,
                          int64_t out_head_stride) {
    static const char* who = "rotary";
    if (device_lost()) return fail(PHI_ERR_DEVICE_LOST, "%s: device was lost earlier", who);
    if (tokens < 0 || heads < 0) return fail(PHI_ERR_SHAPE, "%s: negative size", who);
    if (dim < 1 || dim > kMaxRotaryDim) return fail(PHI_ERR_SHAPE, "%s: dim=%lld is not from 1 to %lld", who, (long long)dim, (long long)kMaxRotaryDim);
    if (!is_float(dtype)) return fail(PHI_ERR_ARG, "%s: x must be f32 or bf16", who);
    if (tokens == 0 || heads == 0) return ok();
    if (tokens > INT32_MAX || heads > 65535) return fail(PHI_ERR_SHAPE, "%s: tokens=%lld heads=%lld out of range", who, (long long)tokens, (long long)heads);
    phi_status st = check_turns(who, positions, freq, rot, dim, scale);
    if (st == PHI_OK) st = check_strides(who, "x", x, dtype, x_token_stride, x_head_stride);
    if (st == PHI_OK) st = check_strides(who, "out", out, dtype, out_token_stride, out_head_stride);
    if (st == PHI_OK) st = check_layout(who, "out", tokens, out_token_stride, heads, out_head_stride, dim);
    if (st != PHI_OK) return st;
    const Pieces to = vectors_of(out, tokens, out_token_stride, heads, out_head_stride, dim, elem(dtype));
    const bool same = x == out && (tokens == 1 || x_token_stride == out_token_stride) && (heads == 1 || x_head_stride == out_head_stride);
    if (!same && meet(to, vectors_of(x, tokens, x_token_stride, heads, x_head_stride, dim, elem(dtype)))) return fail(PHI_ERR_ARG, "%s: out overlaps x", who);
    if (meet(to, {positions, tokens * 8}) || meet(to, {freq, rot * 4})) return fail(PHI_ERR_ARG, "%s: out overlaps positions or freq", who);
    const phi_dev::Rotary p{{x, out, x_token_stride, x_head_stride, out_token_stride, out_head_stride, (int)heads}, {}, {}, positions,
                            freq, nullptr, tokens, (int)dim, (int)rot, scale, dtype == PHI_BF16, interleaved != 0};
    return check_hip(phi_dev::launch_rotary((hipStream_t)stream, p, phi_dev::KvCache{}), who);
}

phi_status phi_hip_rotary_cache_write(phi_stream_t stream, const phi_kv_cache* cache, const void* q,
                                      int64_t q_token_stride, int64_t q_head_stride, int64_t q_heads, void* q_out,
                                      int64_t q_out_token_stride, int64_t q_out_head_stride, const void* k,
                                      int64_t k_token_stride, int64_t k_head_stride, const void* v,
                                      int64_t v_token_stride, int64_t v_head_stride, int dtype,
                                      const int64_t* positions, const double* freq, int64_t rot, int interleaved,
                                      float scale, const int64_t* slots, int64_t tokens) {
    static const char* who = "rotary_cache_write";
    if (device_lost()) return fail(PHI_ERR_DEVICE_LOST, "%s: device was lost earlier", who);
    phi_dev::KvCache c;
    phi_status st = check_cache(who, cache, &c);
    if (st != PHI_OK) return st;
    if (tokens < 0 || q_heads < 0) return fail(PHI_ERR_SHAPE, "%s: negative size", who);
    if (q_heads > 65535) return fail(PHI_ERR_SHAPE, "%s: q_heads=%lld out of range", who, (long long)q_heads);
    if (tokens == 0) return ok();
    st = check_kv_tokens(who, c, k, k_token_stride, k_head_stride, v, v_token_stride, v_head_stride, dtype, slots, tokens);
    if (st == PHI_OK) st = check_turns(who, positions, freq, rot, c.dim, scale);
    if (st == PHI_OK) st = check_cache_apart(who, c);
    phi_dev::RotaryHeads qs{};
    if (st == PHI_OK && q_heads > 0) {
        st = check_vectors(who, "q", q, dtype, q_token_stride, q_head_stride);
        if (st == PHI_OK) st = check_vectors(who, "q_out", q_out, dtype, q_out_token_stride, q_out_head_stride);
        if (st == PHI_OK) st = check_layout(who, "q_out", tokens, q_out_token_stride, q_heads, q_out_head_stride, c.dim);
        if (st != PHI_OK) return st;
        const int64_t e = elem(dtype);
        const Pieces to = vectors_of(q_out, tokens, q_out_token_stride, q_heads, q_out_head_stride, c.dim, e);
        const bool same = q == q_out && (tokens == 1 || q_token_stride == q_out_token_stride) && (q_heads == 1 || q_head_stride == q_out_head_stride);
        if (!same && meet(to, vectors_of(q, tokens, q_token_stride, q_heads, q_head_stride, c.dim, e))) return fail(PHI_ERR_ARG, "%s: q_out overlaps q", who);
        if (meet(to, vectors_of(k, tokens, k_token_stride, c.heads, k_head_stride, c.dim, e)) ||
            meet(to, vectors_of(v, tokens, v_token_stride, c.heads, v_head_stride, c.dim, e)) || meets_cache(to, c))
            return fail(PHI_ERR_ARG, "%s: q_out overlaps k, v or the cache", who);
        if (meet(to, {positions, tokens * 8}) || meet(to, {slots, tokens * 8}) || meet(to, {freq, rot * 4}))
            return fail(PHI_ERR_ARG, "%s: q_out overlaps positions, slots or freq", who);
        qs = {q, q_out, q_token_stride, q_head_stride, q_out_token_stride, q_out_head_stride, (int)q_heads};
    }
    if (st != PHI_OK) return st;
    const phi_dev::Rotary p{qs, {k, nullptr, k_token_stride, k_head_stride, 0, 0, c.heads}, {v, nullptr, v_token_stride, v_head_stride, 0, 0, c.heads},
                            positions, freq, slots, tokens, c.dim, (int)rot, scale, dtype == PHI_BF16, interleaved != 0};
    return check_hip(phi_dev::launch_rotary((hipStream_t)stream, p, c), who);
}

phi_status phi_hip_kv_cache_copy(phi_stream_t stream, const phi_kv_cache* from, const phi_kv_cache* to,
                                 const int32_t* from_blocks, const int32_t* to_blocks, const int32_t* tokens,
                                 int64_t n) {
    static const char* who = "kv_cache_copy";
    if (device_lost()) return fail(PHI_ERR_DEVICE_LOST, "%s: device was lost earlier", who);
    phi_dev::KvCache a, b;
    phi_status st = check_cache(who, from, &a);
    if (st == PHI_OK) st = check_cache(who, to, &b);
    if (st == PHI_OK) st = check_cache_apart(who, b);
    if (st != PHI_OK) return st;
    if (a.heads != b.heads || a.page != b.page || a.dim != b.dim)
        return fail(PHI_ERR_SHAPE, "%s: caches of %d x %d x %d and %d x %d x %d (heads, page, dim)", who, a.heads, a.page, a.dim, b.heads, b.page, b.dim);
    if ((int64_t)a.heads * a.page > kMaxPageVectors) return fail(PHI_ERR_SHAPE, "%s: a page of %d x %d vectors is too large", who, a.heads, a.page);
    if (n < 0 || n > INT32_MAX) return fail(PHI_ERR_SHAPE, "%s: n=%lld out of range", who, (long long)n);
    if (n == 0) return ok();
    if (!from_blocks || !to_blocks) return fail(PHI_ERR_ARG, "%s: null pointer", who);
    if (!aligned(from_blocks, 4) || !aligned(to_blocks, 4) || !aligned(tokens, 4)) return fail(PHI_ERR_ALIGN, "%s: blocks or tokens are misaligned", who);
    const phi_dev::KvCopy p{a, b, from_blocks, to_blocks, tokens, n};
    return check_hip(phi_dev::launch_kv_cache_copy((hipStream_t)stream, p), who);
}

}  // extern "C"
