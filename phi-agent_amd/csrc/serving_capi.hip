// C ABI of the serving operators (include/phi_serving.h): argument validation and
// dispatch, under the error contract of capi.hip.
#include "../../include/phi_serving.h"
#include "decoder_checks.hpp"
#include "serving.hpp"

using namespace phi_capi;

namespace {

constexpr int64_t kMaxRotaryDim = 1024;   // a wave has a vector
constexpr int64_t kMaxRank = 256;         // of an adapter: h of 64 rows, as three bf16, is held in LDS
constexpr int64_t kMaxLoraRows = 1 << 24, kMaxLoraK = 1 << 24;  // units and columns counted in 31 bits
constexpr int64_t kMaxHeadRows = 4 * phi_dev::kMaxBlocks;  // of shared prefixes, four a block of their join
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

phi_status phi_hip_paged_attention_shared(phi_stream_t stream, const void* q, int dtype, int64_t q_token_stride,
                                          int64_t q_head_stride, int64_t tokens, int64_t q_heads,
                                          const phi_kv_cache* cache, const int32_t* prefix_table,
                                          int64_t prefix_width, int64_t prefix_stride, const int32_t* prefix_len,
                                          const int32_t* group_start, int64_t groups, int64_t max_prefix,
                                          const int32_t* block_table, int64_t table_width, int64_t table_stride,
                                          const int32_t* q_start, const int32_t* kv_len, int64_t batch, int64_t max_q,
                                          int64_t max_kv, float scale, void* out, int64_t out_token_stride,
                                          int64_t out_head_stride, void* workspace, size_t ws_bytes) {
    static const char* who = "paged_attention_shared";
    if (device_lost()) return fail(PHI_ERR_DEVICE_LOST, "%s: device was lost earlier", who);
    phi_dev::KvCache c;
    phi_status st = check_cache(who, cache, &c);
    if (st != PHI_OK) return st;
    if (tokens < 0 || groups < 0 || batch < 0 || max_q < 0 || max_kv < 0 || max_prefix < 0 || table_width < 0 || prefix_width < 0)
        return fail(PHI_ERR_SHAPE, "%s: negative size", who);
    if (!is_float(dtype)) return fail(PHI_ERR_ARG, "%s: q must be f32 or bf16", who);
    if (q_heads <= 0 || q_heads % c.heads != 0 || q_heads > 65535)
        return fail(PHI_ERR_SHAPE, "%s: %lld query heads for %d key/value heads", who, (long long)q_heads, c.heads);
    if (tokens == 0 || batch == 0 || max_q == 0) return ok();
    if (tokens > INT32_MAX || batch > 65535 || groups > 65535 || max_q > tokens || max_kv > kMaxKv || max_prefix > kMaxKv)
        return fail(PHI_ERR_SHAPE, "%s: tokens=%lld groups=%lld batch=%lld max_prefix=%lld max_q=%lld max_kv=%lld out of range", who, (long long)tokens,
                    (long long)groups, (long long)batch, (long long)max_prefix, (long long)max_q, (long long)max_kv);
    if (tokens * (q_heads / c.heads) > kMaxRows)
        return fail(PHI_ERR_SHAPE, "%s: tokens=%lld at %lld query heads a key/value head is out of range", who, (long long)tokens, (long long)(q_heads / c.heads));
    if (tokens * q_heads > kMaxHeadRows) return fail(PHI_ERR_SHAPE, "%s: tokens=%lld of %lld heads is out of range", who, (long long)tokens, (long long)q_heads);
    if (groups == 0) return fail(PHI_ERR_SHAPE, "%s: no groups", who);
    if (max_kv > 0 && (table_width > INT32_MAX || max_kv > table_width * c.page))
        return fail(PHI_ERR_SHAPE, "%s: max_kv=%lld exceeds the block table's %lld x %d tokens", who, (long long)max_kv, (long long)table_width, c.page);
    if (max_prefix > 0 && (prefix_width > INT32_MAX || max_prefix > prefix_width * c.page))
        return fail(PHI_ERR_SHAPE, "%s: max_prefix=%lld exceeds the prefix table's %lld x %d tokens", who, (long long)max_prefix, (long long)prefix_width, c.page);
    if (table_stride < table_width || table_stride > kMaxStride || prefix_stride < prefix_width || prefix_stride > kMaxStride)
        return fail(PHI_ERR_SHAPE, "%s: a table's stride is smaller than its row", who);
    if (!std::isfinite(scale)) return fail(PHI_ERR_ARG, "%s: scale must be finite", who);
    st = check_vectors(who, "q", q, dtype, q_token_stride, q_head_stride);
    if (st == PHI_OK) st = check_vectors(who, "out", out, dtype, out_token_stride, out_head_stride);
    if (st == PHI_OK) st = check_layout(who, "out", tokens, out_token_stride, q_heads, out_head_stride, c.dim);
    if (st != PHI_OK) return st;
    if ((max_kv > 0 && !block_table) || (max_prefix > 0 && !prefix_table) || !prefix_len || !group_start || !q_start || !kv_len)
        return fail(PHI_ERR_ARG, "%s: null pointer", who);
    if (!aligned(block_table, 4) || !aligned(prefix_table, 4) || !aligned(prefix_len, 4) || !aligned(group_start, 4) || !aligned(q_start, 4) || !aligned(kv_len, 4))
        return fail(PHI_ERR_ALIGN, "%s: a table, lengths or starts are misaligned", who);
    const Pieces qs = vectors_of(q, tokens, q_token_stride, q_heads, q_head_stride, c.dim, elem(dtype));
    const Pieces os = vectors_of(out, tokens, out_token_stride, q_heads, out_head_stride, c.dim, elem(dtype));
    if (meet(qs, os)) return fail(PHI_ERR_ARG, "%s: out overlaps q", who);
    const size_t need = phi_hip_paged_attention_shared_workspace_bytes(tokens, q_heads, c.heads, c.dim, groups, batch, max_prefix, max_q, max_kv, dtype);
    if (need == 0) return fail(PHI_ERR_SHAPE, "%s: groups=%lld and batch=%lld are too many for a launch at %d key/value heads", who, (long long)groups, (long long)batch, c.heads);
    if (!workspace || ws_bytes < need)
        return fail(PHI_ERR_WORKSPACE, "%s: needs %zu bytes of workspace, got %zu", who, need, workspace ? ws_bytes : (size_t)0);
    if (!aligned(workspace, 16)) return fail(PHI_ERR_ALIGN, "%s: the workspace must be 16-byte aligned", who);
    const Pieces ws{workspace, (int64_t)need};
    if (meet(ws, qs) || meet(ws, os) || meets_cache(ws, c)) return fail(PHI_ERR_ARG, "%s: the workspace overlaps q, out or the cache", who);
    if (meets_cache(os, c)) return fail(PHI_ERR_ARG, "%s: out overlaps the cache", who);
    phi_dev::PagedAttn p{q, out, block_table, q_start, kv_len, q_token_stride, q_head_stride, out_token_stride, out_head_stride, table_stride,
                         tokens, (int)q_heads, (int)(q_heads / c.heads), (int)batch, (int)max_q, (int)max_kv, (int)table_width, 0, 0, scale,
                         dtype == PHI_BF16, true, prefix_len, group_start, ((int64_t)(uintptr_t)prefix_table - (int64_t)(uintptr_t)block_table) / 4, prefix_stride, (int)groups,
                         (int)max_prefix, (int)prefix_width, (int)max_q, nullptr, nullptr};
    return check_hip(phi_dev::launch_paged_attention_shared((hipStream_t)stream, c, p, workspace), who);
}

size_t phi_hip_paged_attention_shared_workspace_bytes(int64_t tokens, int64_t q_heads, int64_t kv_heads, int64_t dim,
                                                      int64_t groups, int64_t batch, int64_t max_prefix,
                                                      int64_t max_q, int64_t max_kv, int dtype) {
    if (tokens <= 0 || q_heads <= 0 || kv_heads <= 0 || dim <= 0 || groups <= 0 || batch <= 0 || max_q <= 0 || max_kv < 0 || max_prefix < 0) return 0;
    if (tokens > INT32_MAX || q_heads > 65535 || dim > 256 || groups > 65535 || batch > 65535 || max_q > tokens || max_kv > kMaxKv || max_prefix > kMaxKv) return 0;
    if (q_heads % kv_heads != 0 || tokens * (q_heads / kv_heads) > kMaxRows || tokens * q_heads > kMaxHeadRows) return 0;
    return phi_dev::paged_attention_shared_workspace(tokens, (int)q_heads, (int)kv_heads, (int)dim, (int)groups, (int)batch, (int)max_prefix, (int)max_q,
                                                     (int)max_kv, dtype == PHI_BF16);
}

phi_status phi_hip_lora_batched(phi_stream_t stream, const void* x, int x_dtype, int64_t ldx, int64_t rows, int64_t K,
                                const void* A, int64_t a_adapter_stride, int64_t a_row_stride, const void* B,
                                int64_t b_adapter_stride, int64_t b_row_stride, int w_dtype, int64_t adapters,
                                int64_t R, int64_t N, const int32_t* adapter, const float* scale, const void* base,
                                int64_t ld_base, void* out, int out_dtype, int64_t ldo, void* workspace,
                                size_t ws_bytes) {
    static const char* who = "lora_batched";
    if (device_lost()) return fail(PHI_ERR_DEVICE_LOST, "%s: device was lost earlier", who);
    if (rows < 0 || K < 0 || N < 0 || R < 0 || adapters < 0) return fail(PHI_ERR_SHAPE, "%s: negative size", who);
    if (!is_float(x_dtype) || !is_float(w_dtype) || !is_float(out_dtype)) return fail(PHI_ERR_ARG, "%s: dtypes must be f32 or bf16", who);
    if (rows == 0 || N == 0) return ok();
    if (K == 0 || R == 0 || adapters == 0) return fail(PHI_ERR_SHAPE, "%s: empty factors (K=%lld R=%lld adapters=%lld)", who, (long long)K, (long long)R, (long long)adapters);
    if (R > kMaxRank) return fail(PHI_ERR_UNSUPPORTED, "%s: R=%lld exceeds %lld", who, (long long)R, (long long)kMaxRank);
    if (rows > kMaxLoraRows || K > kMaxLoraK || N > kMaxLoraK || adapters > INT32_MAX)
        return fail(PHI_ERR_SHAPE, "%s: rows=%lld K=%lld N=%lld adapters=%lld out of range", who, (long long)rows, (long long)K, (long long)N, (long long)adapters);
    if (!x || !A || !B || !adapter || !out) return fail(PHI_ERR_ARG, "%s: null pointer", who);
    if (ldx < K || ldo < N || (base && ld_base < N) || a_row_stride < K || b_row_stride < R) return fail(PHI_ERR_SHAPE, "%s: leading dimension smaller than the row", who);
    if (ldx > kMaxPitch || ldo > kMaxPitch || (base && ld_base > kMaxPitch) || a_row_stride > kMaxPitch || b_row_stride > kMaxPitch)
        return fail(PHI_ERR_SHAPE, "%s: leading dimension too large", who);
    for (int64_t s : {a_adapter_stride, b_adapter_stride})
        if (s < 0 || s > kMaxStride / 2 || (adapters > 1 && s > kMaxSpan / (adapters - 1))) return fail(PHI_ERR_SHAPE, "%s: bad adapter stride %lld", who, (long long)s);
    const int64_t xe = elem(x_dtype), we = elem(w_dtype), oe = elem(out_dtype);
    if (!aligned(x, xe) || !aligned(A, we) || !aligned(B, we) || !aligned(adapter, 4) || !aligned(scale, 4) || !aligned(out, oe) || !aligned(base, oe))
        return fail(PHI_ERR_ALIGN, "%s: a pointer is not aligned to its type", who);
    const size_t need = phi_hip_lora_batched_workspace_bytes(rows, K, R);
    if (!workspace || ws_bytes < need) return fail(PHI_ERR_WORKSPACE, "%s: needs %zu bytes of workspace, got %zu", who, need, workspace ? ws_bytes : (size_t)0);
    if (!aligned(workspace, 16)) return fail(PHI_ERR_ALIGN, "%s: the workspace must be 16-byte aligned", who);
    const Pieces to = rows_of(out, rows, N, ldo, oe), from = rows_of(base, rows, N, ld_base, oe), ws{workspace, (int64_t)need};
    const Pieces in[] = {rows_of(x, rows, K, ldx, xe), {A, K * we, R, a_row_stride * we, adapters, a_adapter_stride * we},
                         {B, R * we, N, b_row_stride * we, adapters, b_adapter_stride * we}, {adapter, rows * 4}, {scale, adapters * 4}};
    for (const auto& i : in) {
        if (meet(to, i)) return fail(PHI_ERR_ARG, "%s: out overlaps an input", who);
        if (meet(ws, i)) return fail(PHI_ERR_ARG, "%s: the workspace overlaps an operand", who);
    }
    if (meet(ws, to) || meet(ws, from)) return fail(PHI_ERR_ARG, "%s: the workspace overlaps an operand", who);
    const bool same = base == out && (rows == 1 || ld_base == ldo);
    if (!same && meet(to, from)) return fail(PHI_ERR_ARG, "%s: out overlaps base", who);
    const phi_dev::LoraBatched p{x, A, B, adapter, scale, base, out, (float*)workspace, nullptr, nullptr, nullptr, ldx, a_adapter_stride, a_row_stride, b_adapter_stride,
                                 b_row_stride, ld_base, ldo, (int)rows, (int)K, (int)N, (int)R, (int)adapters, 0, 0,
                                 x_dtype == PHI_BF16, w_dtype == PHI_BF16, out_dtype == PHI_BF16};
    return check_hip(phi_dev::launch_lora_batched((hipStream_t)stream, p), who);
}

size_t phi_hip_lora_batched_workspace_bytes(int64_t rows, int64_t K, int64_t R) {
    if (rows <= 0 || K <= 0 || R <= 0 || rows > kMaxLoraRows || K > kMaxLoraK || R > kMaxRank) return 0;
    return phi_dev::lora_batched_workspace(rows, K, R);
}

}  // extern "C"
