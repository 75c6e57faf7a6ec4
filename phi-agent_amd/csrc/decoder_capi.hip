// C ABI of the decoder layer's operators (include/phi_decoder.h): argument
// validation and dispatch, under the error contract of capi.hip.
#include <cmath>

#include "../../include/phi_decoder.h"
#include "capi.hpp"
#include "decoder.hpp"

using phi_capi::check_hip;
using phi_capi::fail;
using phi_capi::ok;

namespace {

bool aligned(const void* p, size_t a) { return ((uintptr_t)p & (a - 1)) == 0; }

bool is_float(int dtype) { return dtype == PHI_F32 || dtype == PHI_BF16; }

int64_t elem(int dtype) { return dtype == PHI_BF16 ? 2 : 4; }

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
bool meet(const Pieces& a, const Pieces& b) {
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
Pieces rows_of(const void* p, int64_t rows, int64_t K, int64_t pitch, int64_t elem) { return {p, K * elem, rows, pitch * elem}; }
Pieces vectors_of(const void* p, int64_t tokens, int64_t token_stride, int64_t heads, int64_t head_stride, int64_t dim, int64_t elem) {
    return {p, dim * elem, tokens, token_stride * elem, heads, head_stride * elem};
}

constexpr int64_t kMaxKv = 1 << 30;  // a sequence's tokens: positions and steps past them stay 32-bit
constexpr int64_t kMaxRows = 1 << 30;  // a sequence's new tokens x query heads a key/value head, the same
constexpr int64_t kMaxK = 32768;      // columns of a norm's row (held on chip)
constexpr int64_t kMaxPage = 1 << 20;
constexpr int64_t kMaxPitch = (int64_t)1 << 29;    // elements: 2^31 rows of it stay within 63 bits
constexpr int64_t kMaxStride = (int64_t)1 << 40;   // of a cache's blocks, heads and tokens
constexpr int64_t kMaxSpan = (int64_t)1 << 56;     // more than any memory

phi_status check_cache(const char* who, const phi_kv_cache* c, phi_dev::KvCache* out) {
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

phi_status check_vectors(const char* who, const char* name, const void* x, int dtype, int64_t token_stride, int64_t head_stride) {
    if (!x) return fail(PHI_ERR_ARG, "%s: null %s", who, name);
    if (token_stride < 0 || head_stride < 0 || token_stride > kMaxPitch || head_stride > kMaxPitch)
        return fail(PHI_ERR_SHAPE, "%s: bad stride of %s", who, name);
    if (!aligned(x, 16) || token_stride * elem(dtype) % 16 != 0 || head_stride * elem(dtype) % 16 != 0)
        return fail(PHI_ERR_ALIGN, "%s: %s's vectors must be 16-byte aligned", who, name);
    return PHI_OK;
}

// Outputs: one place for two vectors is no result of either.
phi_status check_apart(const char* who, const char* name, int64_t tokens, int64_t token_stride, int64_t heads, int64_t head_stride, int64_t dim) {
    if ((tokens > 1 && token_stride < dim) || (heads > 1 && head_stride < dim)) return fail(PHI_ERR_SHAPE, "%s: %s's vectors overlap", who, name);
    return PHI_OK;
}

phi_status check_kv_tokens(const char* who, const phi_dev::KvCache& c, const void* k, int64_t kt, int64_t kh, const void* v,
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

}  // namespace

extern "C" {

phi_status phi_hip_rms_norm_quant(phi_stream_t stream, const void* x, int x_dtype, int64_t ldx, const void* residual,
                                  void* residual_out, int res_dtype, int64_t ldr, const void* weight,
                                  const void* shift, int w_dtype, float eps, int64_t rows, int64_t K, void* y,
                                  int y_dtype, int64_t ldy, int8_t* q, int64_t ldq, float* s, float qmax,
                                  int round_mode, int rotate) {
    static const char* who = "rms_norm_quant";
    if (phi_capi::device_lost()) return fail(PHI_ERR_DEVICE_LOST, "%s: device was lost earlier", who);
    if (rows < 0 || K < 0) return fail(PHI_ERR_SHAPE, "%s: negative size", who);
    if (rows == 0) return ok();
    if (K == 0) return fail(PHI_ERR_SHAPE, "%s: empty rows", who);
    if (rotate && K % 256 != 0) return fail(PHI_ERR_SHAPE, "%s: K=%lld is not a multiple of 256 (convrot group size)", who, (long long)K);
    if (K > kMaxK) return fail(PHI_ERR_UNSUPPORTED, "%s: K=%lld exceeds %lld", who, (long long)K, (long long)kMaxK);
    if (rows > INT32_MAX) return fail(PHI_ERR_SHAPE, "%s: rows exceeds 2^31", who);
    if (!x || !q || !s) return fail(PHI_ERR_ARG, "%s: null pointer", who);
    if (residual_out && !residual) return fail(PHI_ERR_ARG, "%s: residual_out without residual", who);
    if (!is_float(x_dtype) || (residual && !is_float(res_dtype)) || ((weight || shift) && !is_float(w_dtype)) || (y && !is_float(y_dtype)))
        return fail(PHI_ERR_ARG, "%s: dtypes must be f32 or bf16", who);
    if (round_mode != PHI_ROUND_HALF_AWAY && round_mode != PHI_ROUND_HALF_EVEN) return fail(PHI_ERR_ARG, "%s: bad round mode", who);
    if (!(qmax >= 1.0f && qmax <= 127.0f) || qmax != (float)(int)qmax) return fail(PHI_ERR_ARG, "%s: qmax must be an integer in [1,127]", who);
    if (!(eps >= 0.0f) || !std::isfinite(eps)) return fail(PHI_ERR_ARG, "%s: eps must be finite and not negative", who);
    if (ldx < K || ldq < K || (residual && ldr < K) || (y && ldy < K)) return fail(PHI_ERR_SHAPE, "%s: leading dimension smaller than K", who);
    if (ldx > kMaxPitch || ldq > kMaxPitch || (residual && ldr > kMaxPitch) || (y && ldy > kMaxPitch)) return fail(PHI_ERR_SHAPE, "%s: leading dimension too large", who);
    if (!aligned(x, elem(x_dtype)) || !aligned(s, 4) || (residual && (!aligned(residual, elem(res_dtype)) || !aligned(residual_out, elem(res_dtype)))) ||
        (weight && !aligned(weight, elem(w_dtype))) || (shift && !aligned(shift, elem(w_dtype))) || (y && !aligned(y, elem(y_dtype))))
        return fail(PHI_ERR_ALIGN, "%s: a pointer is not aligned to its type", who);
    const int64_t re = elem(res_dtype);
    const Pieces in[] = {rows_of(x, rows, K, ldx, elem(x_dtype)), rows_of(residual, rows, K, ldr, re), {weight, K * elem(w_dtype)}, {shift, K * elem(w_dtype)}};
    const Pieces out[] = {rows_of(residual_out, rows, K, ldr, re), rows_of(y, rows, K, ldy, elem(y_dtype)), rows_of(q, rows, K, ldq, 1), {s, rows * 4}};
    for (const auto& o : out) {
        for (const auto& i : in)
            if (meet(o, i) && !(o.p == residual_out && i.p == residual && o.p == i.p))
                return fail(PHI_ERR_ARG, "%s: an output overlaps an input", who);
        for (const auto& o2 : out)
            if (&o < &o2 && meet(o, o2)) return fail(PHI_ERR_ARG, "%s: two outputs overlap", who);
    }
    const phi_dev::RmsNorm p{x, residual, residual_out, weight, shift, y, q, s, ldx, ldr, ldy, ldq, rows, (int)K, eps, qmax,
                             x_dtype == PHI_BF16, res_dtype == PHI_BF16, w_dtype == PHI_BF16, y_dtype == PHI_BF16,
                             round_mode == PHI_ROUND_HALF_EVEN, rotate != 0};
    return check_hip(phi_dev::launch_rms_norm_quant((hipStream_t)stream, p), who);
}

phi_status phi_hip_kv_cache_write(phi_stream_t stream, const phi_kv_cache* cache, const void* k, int64_t k_token_stride,
                                  int64_t k_head_stride, const void* v, int64_t v_token_stride, int64_t v_head_stride,
                                  int dtype, const int64_t* slots, int64_t tokens) {
    static const char* who = "kv_cache_write";
    if (phi_capi::device_lost()) return fail(PHI_ERR_DEVICE_LOST, "%s: device was lost earlier", who);
    phi_dev::KvCache c;
    phi_status st = check_cache(who, cache, &c);
    if (st != PHI_OK) return st;
    if (tokens < 0) return fail(PHI_ERR_SHAPE, "%s: negative size", who);
    if (tokens == 0) return ok();
    st = check_kv_tokens(who, c, k, k_token_stride, k_head_stride, v, v_token_stride, v_head_stride, dtype, slots, tokens);
    if (st == PHI_OK) st = check_apart(who, "the cache", c.page, c.token_stride, c.heads, c.head_stride, c.dim);
    if (st == PHI_OK) st = check_apart(who, "the cache", c.blocks, c.block_stride, 1, 0, c.dim);
    if (st == PHI_OK) st = check_apart(who, "the cache", c.page, c.s_token_stride, c.heads, c.s_head_stride, 1);
    if (st == PHI_OK) st = check_apart(who, "the cache", c.blocks, c.s_block_stride, 1, 0, 1);
    if (st != PHI_OK) return st;
    const phi_dev::KvTokens t{(void*)k, (void*)v, k_token_stride, k_head_stride, v_token_stride, v_head_stride, slots, tokens, dtype == PHI_BF16};
    return check_hip(phi_dev::launch_kv_cache_write((hipStream_t)stream, c, t), who);
}

phi_status phi_hip_kv_cache_read(phi_stream_t stream, const phi_kv_cache* cache, const int64_t* slots, int64_t tokens,
                                 void* k, int64_t k_token_stride, int64_t k_head_stride, void* v,
                                 int64_t v_token_stride, int64_t v_head_stride, int dtype) {
    static const char* who = "kv_cache_read";
    if (phi_capi::device_lost()) return fail(PHI_ERR_DEVICE_LOST, "%s: device was lost earlier", who);
    phi_dev::KvCache c;
    phi_status st = check_cache(who, cache, &c);
    if (st != PHI_OK) return st;
    if (tokens < 0) return fail(PHI_ERR_SHAPE, "%s: negative size", who);
    if (tokens == 0) return ok();
    st = check_kv_tokens(who, c, k, k_token_stride, k_head_stride, v, v_token_stride, v_head_stride, dtype, slots, tokens);
    if (st == PHI_OK) st = check_apart(who, "k", tokens, k_token_stride, c.heads, k_head_stride, c.dim);
    if (st == PHI_OK) st = check_apart(who, "v", tokens, v_token_stride, c.heads, v_head_stride, c.dim);
    if (st != PHI_OK) return st;
    const Pieces to[] = {vectors_of(k, tokens, k_token_stride, c.heads, k_head_stride, c.dim, elem(dtype)),
                         vectors_of(v, tokens, v_token_stride, c.heads, v_head_stride, c.dim, elem(dtype))};
    if (meet(to[0], to[1])) return fail(PHI_ERR_ARG, "%s: k overlaps v", who);
    auto span = [](int64_t n, int64_t stride) { return n > 1 && stride > kMaxSpan / (n - 1) ? kMaxSpan : (n - 1) * stride; };
    const int64_t codes = span(c.blocks, c.block_stride) + span(c.heads, c.head_stride) + span(c.page, c.token_stride) + c.dim;
    const int64_t scales = (span(c.blocks, c.s_block_stride) + span(c.heads, c.s_head_stride) + span(c.page, c.s_token_stride) + 1) * 4;
    for (const Pieces& x : to)
        if (meet(x, {c.k, codes}) || meet(x, {c.v, codes}) || meet(x, {c.ks, scales}) || meet(x, {c.vs, scales}))
            return fail(PHI_ERR_ARG, "%s: k or v overlaps the cache", who);
    const phi_dev::KvTokens t{k, v, k_token_stride, k_head_stride, v_token_stride, v_head_stride, slots, tokens, dtype == PHI_BF16};
    return check_hip(phi_dev::launch_kv_cache_read((hipStream_t)stream, c, t), who);
}

phi_status phi_hip_paged_attention(phi_stream_t stream, const void* q, int dtype, int64_t q_token_stride,
                                   int64_t q_head_stride, int64_t tokens, int64_t q_heads, const phi_kv_cache* cache,
                                   const int32_t* block_table, int64_t table_width, int64_t table_stride,
                                   const int32_t* q_start, const int32_t* kv_len, int64_t batch, int64_t max_q,
                                   int64_t max_kv, float scale, int causal, int64_t window, void* out,
                                   int64_t out_token_stride, int64_t out_head_stride, void* workspace,
                                   size_t ws_bytes) {
    static const char* who = "paged_attention";
    if (phi_capi::device_lost()) return fail(PHI_ERR_DEVICE_LOST, "%s: device was lost earlier", who);
    phi_dev::KvCache c;
    phi_status st = check_cache(who, cache, &c);
    if (st != PHI_OK) return st;
    if (tokens < 0 || batch < 0 || max_q < 0 || max_kv < 0 || table_width < 0) return fail(PHI_ERR_SHAPE, "%s: negative size", who);
    if (!is_float(dtype)) return fail(PHI_ERR_ARG, "%s: q must be f32 or bf16", who);
    if (q_heads <= 0 || q_heads % c.heads != 0 || q_heads > 65535)
        return fail(PHI_ERR_SHAPE, "%s: %lld query heads for %d key/value heads", who, (long long)q_heads, c.heads);
    if (tokens == 0 || batch == 0 || max_q == 0) return ok();
    if (tokens > INT32_MAX || batch > 65535 || max_q > tokens || max_kv > kMaxKv)
        return fail(PHI_ERR_SHAPE, "%s: tokens=%lld batch=%lld max_q=%lld max_kv=%lld out of range", who, (long long)tokens, (long long)batch, (long long)max_q, (long long)max_kv);
    if (max_q * (q_heads / c.heads) > kMaxRows)
        return fail(PHI_ERR_SHAPE, "%s: max_q=%lld at %lld query heads a key/value head is out of range", who, (long long)max_q, (long long)(q_heads / c.heads));
    if (max_kv > 0 && (table_width > INT32_MAX || max_kv > table_width * c.page))
        return fail(PHI_ERR_SHAPE, "%s: max_kv=%lld exceeds the block table's %lld x %d tokens", who, (long long)max_kv, (long long)table_width, c.page);
    if (table_stride < table_width || table_stride > kMaxStride) return fail(PHI_ERR_SHAPE, "%s: block table's stride is smaller than its row", who);
    if (window < 0 || (window > 0 && !causal)) return fail(PHI_ERR_ARG, "%s: a window needs causal attention and a positive size", who);
    if (!std::isfinite(scale)) return fail(PHI_ERR_ARG, "%s: scale must be finite", who);
    st = check_vectors(who, "q", q, dtype, q_token_stride, q_head_stride);
    if (st == PHI_OK) st = check_vectors(who, "out", out, dtype, out_token_stride, out_head_stride);
    if (st == PHI_OK) st = check_apart(who, "out", tokens, out_token_stride, q_heads, out_head_stride, c.dim);
    if (st != PHI_OK) return st;
    if ((max_kv > 0 && !block_table) || !q_start || !kv_len) return fail(PHI_ERR_ARG, "%s: null pointer", who);
    if (!aligned(block_table, 4) || !aligned(q_start, 4) || !aligned(kv_len, 4)) return fail(PHI_ERR_ALIGN, "%s: block_table, q_start or kv_len is misaligned", who);
    const Pieces qs = vectors_of(q, tokens, q_token_stride, q_heads, q_head_stride, c.dim, elem(dtype));
    const Pieces os = vectors_of(out, tokens, out_token_stride, q_heads, out_head_stride, c.dim, elem(dtype));
    if (meet(qs, os)) return fail(PHI_ERR_ARG, "%s: out overlaps q", who);
    const size_t need = phi_hip_paged_attention_workspace_bytes(tokens, q_heads, c.heads, c.dim, batch, max_q, max_kv, dtype);
    if (need > 0 && (!workspace || ws_bytes < need))
        return fail(PHI_ERR_WORKSPACE, "%s: needs %zu bytes of workspace, got %zu", who, need, workspace ? ws_bytes : (size_t)0);
    if (need > 0 && !aligned(workspace, 16)) return fail(PHI_ERR_ALIGN, "%s: the workspace must be 16-byte aligned", who);
    if (need > 0 && (meet({workspace, (int64_t)need}, qs) || meet({workspace, (int64_t)need}, os)))
        return fail(PHI_ERR_ARG, "%s: the workspace overlaps q or out", who);
    const phi_dev::PagedAttn p{q, out, block_table, q_start, kv_len, q_token_stride, q_head_stride, out_token_stride,
                               out_head_stride, table_stride, tokens, (int)q_heads, (int)(q_heads / c.heads), (int)batch,
                               (int)max_q, (int)max_kv, (int)table_width, window > INT32_MAX ? 0 : (int)window, 0, scale,
                               dtype == PHI_BF16, causal != 0};
    return check_hip(phi_dev::launch_paged_attention((hipStream_t)stream, c, p, workspace), who);
}

size_t phi_hip_paged_attention_workspace_bytes(int64_t tokens, int64_t q_heads, int64_t kv_heads, int64_t dim,
                                               int64_t batch, int64_t max_q, int64_t max_kv, int dtype) {
    if (tokens <= 0 || q_heads <= 0 || kv_heads <= 0 || dim <= 0 || batch <= 0 || max_q <= 0 || max_kv <= 0) return 0;
    if (tokens > INT32_MAX || q_heads > 65535 || dim > 256 || batch > 65535 || max_q > tokens || max_kv > kMaxKv) return 0;
    if (q_heads % kv_heads != 0 || max_q * (q_heads / kv_heads) > kMaxRows) return 0;
    return phi_dev::paged_attention_workspace(tokens, (int)q_heads, (int)kv_heads, (int)dim, (int)batch, (int)max_q,
                                              (int)max_kv, dtype == PHI_BF16);
}

}  // extern "C"
