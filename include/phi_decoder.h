/*
 * phi_decoder.h -- the operators between a decoder layer's int8 linears, in
 * the manner of phi_qlinear.h: every entry point enqueues work on the caller's
 * HIP stream and returns a phi_status (message: phi_hip_last_error()), nothing
 * synchronises, nothing allocates device memory.
 *
 *   phi_hip_rms_norm_quant    residual addition, root-mean-square norm and the
 *                             int8 operand of the linear that follows
 *   phi_hip_kv_cache_write    new tokens' keys and values into an int8 paged cache
 *   phi_hip_kv_cache_read     tokens back out of it
 *   phi_hip_paged_attention   attention of new tokens over that cache
 *
 * The reference runs a norm (core/kernels/ops.cpp:95-) and attention
 * (core/kernels/attn.cpp:337-) on fp32 tensors and keeps no quantised cache;
 * these entries have its linear's quantiser (core/host/quant.cpp:134-169) in
 * common with it and are otherwise this library's own.
 */
#ifndef PHI_DECODER_H
#define PHI_DECODER_H

#include "phi_qlinear.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * Per row (token) of x [rows, ldx]:
 *   r = x + residual                      fp32; residual_out = r, rounded to res_dtype
 *   y = r * (1 / sqrt(mean(r^2) + eps)) * weight + shift
 *   q, s = the rotate + quantise of phi_hip_quant_rotate on y (fp32)
 * so that (q, s) are the A operand of phi_hip_i8_gemm.
 *
 *   x             of x_dtype (PHI_F32 or PHI_BF16)
 *   residual      NULL (0), or [rows, ldr] of res_dtype (PHI_F32 or PHI_BF16)
 *   residual_out  NULL, or [rows, ldr] of res_dtype; may be residual itself.
 *                 Needs residual.  The norm is of r as it is in fp32, before
 *                 that rounding.
 *   weight, shift NULL (1 and 0), or [K] of w_dtype (PHI_F32 or PHI_BF16)
 *   y             NULL, or [rows, ldy] of y_dtype (PHI_F32 or PHI_BF16): the
 *                 normalised row itself, for consumers beside the linear
 *                 (phi_hip_lora_tail reads the linear's unquantised input)
 *   q             [rows, ldq] int8, s [rows] fp32
 *   rotate        1: the 256-wide rotation first (K % 256 == 0)
 *   qmax          an integer in 1..127; round_mode a phi_round
 * Any K from 1 to 32768 without the rotation; any pitch of at least K; every
 * pointer aligned to its own type.  residual_out apart, no output may share
 * memory with an input.  A row with an infinity or a NaN in r, or one
 * whose squares sum past fp32, gets y and the scale NaN (codes 0), so that what a
 * linear makes of it is NaN too; the scale is NaN also where, with eps 0, the squares
 * are all 0 in fp32.  rows == 0 is a no-op.
 */
phi_status phi_hip_rms_norm_quant(phi_stream_t stream, const void* x, int x_dtype, int64_t ldx, const void* residual,
                                  void* residual_out, int res_dtype, int64_t ldr, const void* weight,
                                  const void* shift, int w_dtype, float eps, int64_t rows, int64_t K, void* y,
                                  int y_dtype, int64_t ldy, int8_t* q, int64_t ldq, float* s, float qmax,
                                  int round_mode, int rotate);

/*
 * A paged int8 cache of keys and values: `blocks` blocks of `page` tokens, for
 * each of `heads` key/value heads.  A vector of `dim` codes and its fp32 scale
 * stand for code * scale.  Token t of block b, head h:
 *   codes   k + b * block_stride + h * head_stride + t * token_stride   (bytes; v the same)
 *   scales  k_scale + b * s_block_stride + h * s_head_stride + t * s_token_stride  (floats)
 * so both [blocks, heads, page, dim] and [blocks, page, heads, dim] fit.  dim:
 * a multiple of 16 from 16 to 256; any page from 1 to 2^20; code strides multiples of
 * 16, k and v 16-byte aligned.  What was never written may hold anything; the scale
 * of a token that is seen is finite, or NaN, which makes NaN of what sees it.
 */
typedef struct phi_kv_cache {
    int8_t* k;
    int8_t* v;
    float* k_scale;
    float* v_scale;
    int64_t blocks, heads, page, dim;
    int64_t block_stride, head_stride, token_stride;
    int64_t s_block_stride, s_head_stride, s_token_stride;
} phi_kv_cache;

/*
 * Quantise and store `tokens` new tokens.  k, v [tokens, heads, dim] of dtype
 * (PHI_F32 or PHI_BF16), token and head strides in elements (columns of a fused
 * projection's output fit), vectors 16-byte aligned.  One scale a token and
 * head: amax > 1e-30 ? amax / 127 : 1, codes rounded half away from zero; a
 * vector with an infinity or a NaN gets the scale NaN (codes 0).
 * slots [tokens] int64: block * page + place in the block; one that is
 * negative or past the cache skips its token.  Two tokens with one slot in one
 * call leave a mixture there, codes of either and the scale of either.
 */
phi_status phi_hip_kv_cache_write(phi_stream_t stream, const phi_kv_cache* cache, const void* k, int64_t k_token_stride,
                                  int64_t k_head_stride, const void* v, int64_t v_token_stride, int64_t v_head_stride,
                                  int dtype, const int64_t* slots, int64_t tokens);

/* The values of `tokens` slots, k, v [tokens, heads, dim] of dtype (PHI_F32:
 * code * scale; PHI_BF16: that, rounded), strides as for the write; zeros for
 * a slot that is negative or past the cache.  k and v share no memory with each
 * other or the cache. */
phi_status phi_hip_kv_cache_read(phi_stream_t stream, const phi_kv_cache* cache, const int64_t* slots, int64_t tokens,
                                 void* k, int64_t k_token_stride, int64_t k_head_stride, void* v,
                                 int64_t v_token_stride, int64_t v_head_stride, int dtype);

/*
 * Attention of a batch of new tokens over the cache (their own keys and values
 * already written).  Sequence b's new tokens are rows q_start[b] .. q_start[b+1] - 1
 * of q; its kv_len[b] tokens (the new ones among them, last) lie in the blocks
 * block_table[b][0..].  With n = q_start[b+1] - q_start[b], row i is at position
 * pos = kv_len[b] - n + i, and for query head h, over the tokens t it sees,
 *   out = sum_t softmax_t(scale * q . k_t) v_t      key/value head h / (q_heads / cache heads)
 *   seen: t < kv_len[b];  t <= pos if causal;  t > pos - window if window > 0
 * A row that sees nothing gives zeros.
 *
 *   q, out       [tokens, q_heads, dim] of dtype (PHI_BF16 or PHI_F32), token and
 *                head strides in elements, vectors 16-byte aligned; out must not
 *                share memory with q
 *   block_table  [batch, table_stride] int32, `table_width` entries a row; the
 *                tokens of an entry that is no block of the cache are not seen
 *   q_start      [batch + 1] int32, ascending from 0 to at most tokens: rows past the
 *                last sequence's are left as they are
 *   kv_len       [batch] int32
 *   max_q        at least the longest sequence's n, at most tokens, and 2^30 times key/value
 *                heads over query heads: rows past it are left as they are
 *   max_kv       at least the longest kv_len, at most table_width * page and 2^30:
 *                tokens past it are not seen
 *   window       0, or with causal the number of tokens seen, the row's own included
 *   workspace    phi_hip_paged_attention_workspace_bytes() bytes, 16-byte aligned
 *                (NULL when that is 0)
 * q_start, kv_len and block_table are read on the device, so a captured graph
 * serves growing sequences up to max_kv.
 * Arithmetic.  Sums, maxima and the softmax are fp32 or exact integers.  q is
 * held as integers of 16 bits (PHI_BF16) or 24 bits (PHI_F32) relative to the
 * row's largest |q|, k and v as their codes, exactly, and p enters p.v with 16
 * or 24 bits.  PHI_BF16 sequences of more than 128 rows (new tokens x query heads
 * a key/value head; a batch of one: where max_q allows as many) have q exactly
 * (elements below 2^-21 of the row's largest apart), k's elements rounded to 11 bits or
 * an error of 2^-32 of the largest scale of k of 16 tokens, v's scales and v's elements
 * to 11 bits each or an error of 2^-29 of the largest scale of v of 16 tokens (vectors
 * of zeros apart), and p's to 11 bits or an error of 2^-39 of the row's largest p,
 * times the ratio of the largest scale of v, of all 16 tokens that the row sees some of,
 * to that of p's own 16.  16 tokens' largest is that of those which some row of a
 * block of 256 (dim above 128: 128) sees.
 * Sums of p v are fp32 and divided last, with p up to 2^8, so v beyond 2^119 over
 * the number of tokens may pass them.
 * The order of sums, and so a result's last bits, depends on the sizes, the lengths
 * and max_q, max_kv and batch; the same call gives the same bits.
 */
phi_status phi_hip_paged_attention(phi_stream_t stream, const void* q, int dtype, int64_t q_token_stride,
                                   int64_t q_head_stride, int64_t tokens, int64_t q_heads, const phi_kv_cache* cache,
                                   const int32_t* block_table, int64_t table_width, int64_t table_stride,
                                   const int32_t* q_start, const int32_t* kv_len, int64_t batch, int64_t max_q,
                                   int64_t max_kv, float scale, int causal, int64_t window, void* out,
                                   int64_t out_token_stride, int64_t out_head_stride, void* workspace,
                                   size_t ws_bytes);

/* Workspace of phi_hip_paged_attention for these sizes, with a window or without (0
 * when a call does not split its tokens, and for sizes that no call may have). */
size_t phi_hip_paged_attention_workspace_bytes(int64_t tokens, int64_t q_heads, int64_t kv_heads, int64_t dim,
                                               int64_t batch, int64_t max_q, int64_t max_kv, int dtype);

#ifdef __cplusplus
}
#endif

#endif /* PHI_DECODER_H */
