// Argument checks that the C entries of the decoder layer's operators share.
#pragma once

#include <cmath>

#include "../../include/phi_decoder.h"
#include "capi.hpp"
#include "decoder.hpp"

namespace phi_capi {

inline bool aligned(const void* p, size_t a) { return ((uintptr_t)p & (a - 1)) == 0; }

inline bool is_float(int dtype) { return dtype == PHI_F32 || dtype == PHI_BF16; }

inline int64_t elem(int dtype) { return dtype == PHI_BF16 ? 2 : 4; }

// n1 x n2 pieces of `bytes` bytes at strides of s1 and s2 bytes (null p: none).
struct Pieces {
    const void* p;
    int64_t bytes, n1 = 1, s1 = 0, n2 = 1, s2 = 0;
    int64_t extent() const { return (n1 - 1) * s1 + (n2 - 1) * s2 + bytes; }
    // All pieces lie in the first `width` bytes of periods of P from p on.
    int64_t width(int64_t P) const { return (s1 % P ? (n1 - 1) * s1 : 0) + (s2 % P ? (n2 - 1) * s2 : 0) + bytes; }
};

// Whether a piece of a may meet one of b: not where the memory they span is apart, nor
// where a common period holds them side by side (columns of one buffer).
inline bool meet(const Pieces& a, const Pieces& b) {
    const uintptr_t pa = (uintptr_t)a.p, pb = (uintptr_t)b.p;
    if (!pa || !pb || pa >= pb + (uintptr_t)b.extent() || pb >= pa + (uintptr_t)a.extent()) return false;
    for (const int64_t P : {a.s1, a.s2, b.s1, b.s2}) {
        if (P <= 0) continue;
        const int64_t wa = a.width(P), wb = b.width(P), d = (int64_t)(pb % (uintptr_t)P) - (int64_t)(pa % (uintptr_t)P), at = d < 0 ? d + P : d;
        if (wa <= at && at + wb <= P) return false;
    }
    return true;
}

// rows of K elements, and [tokens, heads, dim] vectors.
inline Pieces rows_of(const void* p, int64_t rows, int64_t K, int64_t pitch, int64_t elem) { return {p, K * elem, rows, pitch * elem}; }
inline Pieces vectors_of(const void* p, int64_t tokens, int64_t token_stride, int64_t heads, int64_t head_stride, int64_t dim, int64_t elem) {
    return {p, dim * elem, tokens, token_stride * elem, heads, head_stride * elem};
}

constexpr int64_t kMaxKv = 1 << 30;  // a sequence's tokens: positions and steps past them stay 32-bit
constexpr int64_t kMaxRows = 1 << 30;  // a sequence's new tokens x query heads a key/value head, the same
constexpr int64_t kMaxK = 32768;      // columns of a norm's row (held on chip)
constexpr int64_t kMaxPage = 1 << 20;
constexpr int64_t kMaxPitch = (int64_t)1 << 29;    // elements: 2^31 rows of it stay within 63 bits
constexpr int64_t kMaxStride = (int64_t)1 << 40;   // of a cache's blocks, heads and tokens
constexpr int64_t kMaxSpan = (int64_t)1 << 56;     // more than any memory

inline phi_status check_cache(const char* who, const phi_kv_cache* c, phi_dev::KvCache* out) {
    if (!c || !c->k || !c->v || !c->k_scale || !c->v_scale) return fail(PHI_ERR_ARG, "%s: null cache", who);
    if (c->blocks <= 0 || c->heads <= 0 || c->page <= 0) return fail(PHI_ERR_SHAPE, "%s: empty cache (blocks=%lld heads=%lld page=%lld)", who, (long long)c->blocks, (long long)c->heads, (long long)c->page);
    if (c->dim < 16 || c->dim > 256 || c->dim % 16 != 0) return fail(PHI_ERR_SHAPE, "%s: dim=%lld is not a multiple of 16 from 16 to 256", who, (long long)c->dim);
    if (c->blocks > INT32_MAX || c->heads > 65535 || c->page > kMaxPage) return fail(PHI_ERR_SHAPE, "%s: cache dimension too large", who);
    const int64_t st[] = {c->block_stride, c->head_stride, c->token_stride, c->s_block_stride, c->s_head_stride, c->s_token_stride};
    for (int64_t s : st)
        if (s < 0 || s > kMaxStride) return fail(PHI_ERR_SHAPE, "%s: bad cache stride %lld", who, (long long)s);
    if (!aligned(c->k, 16) || !aligned(c->v, 16) || c->block_stride % 16 != 0 || c->head_stride % 16 != 0 || c->token_stride % 16 != 0)
        return fail(PHI_ERR_ALIGN, "%s: the cache's codes must be 16-byte aligned at strides of multiples of 16", who);
    if (!aligned(c->k_scale, 4) || !aligned(c->v_scale, 4)) return fail(PHI_ERR_ALIGN, "%s: cache scales are misaligned", who);
    int lg = 0;
    while ((int64_t)1 << lg < c->page) lg++;
    *out = phi_dev::KvCache{c->k, c->v, c->k_scale, c->v_scale, c->block_stride, c->head_stride, c->token_stride,
                            c->s_block_stride, c->s_head_stride, c->s_token_stride, c->blocks * c->page, (int)c->blocks,
                            (int)c->heads, (int)c->page, (int)c->dim,
                            (uint32_t)(((uint64_t)1 << (31 + lg)) / (uint64_t)c->page + 1), 31 + lg};
    return PHI_OK;
}

// Whether x may share memory with the cache (all that its strides span).
inline bool meets_cache(const Pieces& x, const phi_dev::KvCache& c) {
    auto span = [](int64_t n, int64_t stride) { return n > 1 && stride > kMaxSpan / (n - 1) ? kMaxSpan : (n - 1) * stride; };
    const int64_t codes = span(c.blocks, c.block_stride) + span(c.heads, c.head_stride) + span(c.page, c.token_stride) + c.dim;
    const int64_t scales = (span(c.blocks, c.s_block_stride) + span(c.heads, c.s_head_stride) + span(c.page, c.s_token_stride) + 1) * 4;
    return meet(x, {c.k, codes}) || meet(x, {c.v, codes}) || meet(x, {c.ks, scales}) || meet(x, {c.vs, scales});
}

inline phi_status check_vectors(const char* who, const char* name, const void* x, int dtype, int64_t token_stride, int64_t head_stride) {
    if (!x) return fail(PHI_ERR_ARG, "%s: null %s", who, name);
    if (token_stride < 0 || head_stride < 0 || token_stride > kMaxPitch || head_stride > kMaxPitch)
        return fail(PHI_ERR_SHAPE, "%s: bad stride of %s", who, name);
    if (!aligned(x, 16) || token_stride * elem(dtype) % 16 != 0 || head_stride * elem(dtype) % 16 != 0)
        return fail(PHI_ERR_ALIGN, "%s: %s's vectors must be 16-byte aligned", who, name);
    return PHI_OK;
}

// Outputs: one place for two vectors is no result of either.
inline phi_status check_apart(const char* who, const char* name, int64_t tokens, int64_t token_stride, int64_t heads, int64_t head_stride, int64_t dim) {
    if ((tokens > 1 && token_stride < dim) || (heads > 1 && head_stride < dim)) return fail(PHI_ERR_SHAPE, "%s: %s's vectors overlap", who, name);
    return PHI_OK;
}

// The same of a cache that is written.
inline phi_status check_cache_apart(const char* who, const phi_dev::KvCache& c) {
    phi_status st = check_apart(who, "the cache", c.page, c.token_stride, c.heads, c.head_stride, c.dim);
    if (st == PHI_OK) st = check_apart(who, "the cache", c.blocks, c.block_stride, 1, 0, c.dim);
    if (st == PHI_OK) st = check_apart(who, "the cache", c.page, c.s_token_stride, c.heads, c.s_head_stride, 1);
    if (st == PHI_OK) st = check_apart(who, "the cache", c.blocks, c.s_block_stride, 1, 0, 1);
    return st;
}

inline phi_status check_kv_tokens(const char* who, const phi_dev::KvCache& c, const void* k, int64_t kt, int64_t kh, const void* v,
                           int64_t vt, int64_t vh, int dtype, const int64_t* slots, int64_t tokens) {
    if (!is_float(dtype)) return fail(PHI_ERR_ARG, "%s: k and v must be f32 or bf16", who);
    if (tokens > INT32_MAX) return fail(PHI_ERR_SHAPE, "%s: tokens exceeds 2^31", who);
    phi_status st = check_vectors(who, "k", k, dtype, kt, kh);
    if (st == PHI_OK) st = check_vectors(who, "v", v, dtype, vt, vh);
    if (st != PHI_OK) return st;
    if (!slots) return fail(PHI_ERR_ARG, "%s: null slots", who);
    if (!aligned(slots, 8)) return fail(PHI_ERR_ALIGN, "%s: slots is misaligned", who);
    return PHI_OK;
}

}  // namespace phi_capi
