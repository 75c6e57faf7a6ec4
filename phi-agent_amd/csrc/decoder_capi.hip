// C ABI of the decoder layer's operators (include/phi_decoder.h): argument
// validation and dispatch, under the error contract of capi.hip.
#include "decoder_checks.hpp"

using namespace phi_capi;

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
    if (st == PHI_OK) st = check_cache_apart(who, c);
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
    for (const Pieces& x : to)
        if (meets_cache(x, c))
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
