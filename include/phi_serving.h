/*
 * phi_serving.h -- what a server of many requests runs beside phi_decoder.h's
 * operators, in the manner of phi_qlinear.h: every entry point enqueues work on
 * the caller's HIP stream and returns a phi_status (message:
 * phi_hip_last_error()), nothing synchronises, nothing allocates device memory.
 *
 *   phi_hip_rotary               rotary positions of [tokens, heads, dim] vectors
 *   phi_hip_rotary_cache_write   the same of a projection's q and k, with k and v
 *                                quantised into the paged cache
 *   phi_hip_kv_cache_copy        pages of a cache copied (forked sequences, compaction)
 *   phi_hip_paged_attention_shared  attention of sequences that share prefixes
 *   phi_hip_lora_batched         a linear's output plus each row's own low-rank adapter
 *
 * The reference rotates pairs of half a head's distance on fp32 tensors
 * (rope_half, core/kernels/attn.cpp:99-) and adds one adapter to all rows
 * (apply_lora_tail, core/models/model_common.cpp:1667-1700); it has no cache.
 */
#ifndef PHI_SERVING_H
#define PHI_SERVING_H

#include "phi_decoder.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * Rotary positions: of each vector's first `rot` elements, pair j (elements j and
 * j + rot/2, or 2j and 2j + 1 if interleaved) is turned by the angle
 * t = positions[token] * freq[j]:
 *   a' = scale (a cos t - b sin t),   b' = scale (b cos t + a sin t)
 * Elements from rot on are copied.
 *
 *   x, out     [tokens, heads, dim] of dtype (PHI_F32 or PHI_BF16), token and head
 *              strides in elements; any strides of x, vectors of out apart.  out may
 *              be x itself (the same strides), or must not share memory with it.
 *   positions  [tokens] int64, any value: negative ones turn back
 *   freq       [rot / 2] fp64, finite, radians a position: contexts stretched by
 *              any rule are other frequencies (and a scale)
 *   dim        from 1 to 1024; rot even, from 2 to dim
 * The angle is kept as a 64-bit fraction of a turn: freq / 2 pi modulo 1 to 2^-64 (freq
 * to 2^40), its product with the position exactly; scale times its cosine and sine are
 * the nearest fp32 (2^-24 of them and 2^-30), products and sums fp32, rounded once.
 */
phi_status phi_hip_rotary(phi_stream_t stream, const void* x, int dtype, int64_t x_token_stride, int64_t x_head_stride,
                          int64_t tokens, int64_t heads, int64_t dim, const int64_t* positions, const double* freq,
                          int64_t rot, int interleaved, float scale, void* out, int64_t out_token_stride,
                          int64_t out_head_stride);

/*
 * A projection's output on its way to attention, in one launch: q [tokens, q_heads,
 * cache dim] rotated to q_out (which may be q itself), k [tokens, cache heads, dim]
 * rotated and v as it is quantised into the cache at slots [tokens], as
 * phi_hip_kv_cache_write does (k from its fp32 values, not rounded to dtype
 * between).  All of dtype; strides in elements, vectors 16-byte aligned.  q_heads 0:
 * no q.  A token whose slot is skipped has its q rotated all the same.  q_out shares
 * no memory with k, v or the cache.
 */
phi_status phi_hip_rotary_cache_write(phi_stream_t stream, const phi_kv_cache* cache, const void* q,
                                      int64_t q_token_stride, int64_t q_head_stride, int64_t q_heads, void* q_out,
                                      int64_t q_out_token_stride, int64_t q_out_head_stride, const void* k,
                                      int64_t k_token_stride, int64_t k_head_stride, const void* v,
                                      int64_t v_token_stride, int64_t v_head_stride, int dtype,
                                      const int64_t* positions, const double* freq, int64_t rot, int interleaved,
                                      float scale, const int64_t* slots, int64_t tokens);

/*
 * Copy blocks of one cache (codes and scales of k and v, all heads) to blocks of
 * another, or of the same: for i < n the first tokens[i] tokens (NULL: all; fewer
 * than 1: none; more than a page: all) of block from_blocks[i] to block to_blocks[i].  A pair with a
 * block that its cache does not have is skipped.  The caches agree in heads, page and
 * dim; their strides may differ.  Blocks that are written are written once and not
 * read in the same call: else they are left with a mixture.  A page of at most 2^26
 * tokens x heads.
 */
phi_status phi_hip_kv_cache_copy(phi_stream_t stream, const phi_kv_cache* from, const phi_kv_cache* to,
                                 const int32_t* from_blocks, const int32_t* to_blocks, const int32_t* tokens,
                                 int64_t n);

/*
 * phi_hip_paged_attention (causal) for a batch whose sequences share prefixes.  A prefix is
 * read for all rows of its group together: once for every 16 (a row: one query head of a
 * key/value head of one new token), but for every 256 (dim above 128: 128) where the group has
 * more than 128 and q is PHI_BF16.  Group g's prefix, prefix_len[g] tokens in the blocks
 * prefix_table[g][0..], comes before the own tokens of the sequences
 * group_start[g] .. group_start[g+1] - 1: all of their rows see all of it.  A
 * sequence's own tokens, kv_len[b] with the new ones last, lie in the blocks
 * block_table[b][0..], from the first block's first place on; of these its row i sees
 * t <= kv_len[b] - n + i.  With n = q_start[b+1] - q_start[b],
 *   out = sum softmax(scale * q . k) v   over both, one softmax.
 * A row that sees nothing gives zeros.  For single tokens and a few at a time: chunks of many
 * new tokens take less time in phi_hip_paged_attention, with the prefix' blocks first in each
 * sequence's table, and so does a batch that shares nothing.
 *
 *   groups       from 1 to 65535; group_start [groups + 1] int32, ascending from 0 on
 *                to at most batch: sequences before the first group's or past the last's
 *                have no prefix
 *   prefix_table [groups, prefix_stride] int32, `prefix_width` entries a row, as block_table
 *   prefix_len   [groups] int32; max_prefix at least the longest, at most
 *                prefix_width * page and 2^30: tokens past it are not seen
 *   tokens       at most 2^30 times key/value heads over query heads; times q_heads at most 2^26 - 4.
 *                groups + batch times key/value heads past some 2^22 is more than a launch
 *                has blocks for: refused
 *   workspace    phi_hip_paged_attention_shared_workspace_bytes() bytes, 16-byte aligned
 * All else as phi_hip_paged_attention, its arithmetic too, a group's rows over their
 * prefix being one sequence of it: behind a prefix whose group has more than 128 rows,
 * PHI_BF16's p has 11 bits as there, and a row's last bits depend on how many rows its
 * group has.  The parts are joined in fp32.  Lengths, starts and tables are read on the
 * device, so a captured graph serves growing sequences and other groups.
 */
phi_status phi_hip_paged_attention_shared(phi_stream_t stream, const void* q, int dtype, int64_t q_token_stride,
                                          int64_t q_head_stride, int64_t tokens, int64_t q_heads,
                                          const phi_kv_cache* cache, const int32_t* prefix_table,
                                          int64_t prefix_width, int64_t prefix_stride, const int32_t* prefix_len,
                                          const int32_t* group_start, int64_t groups, int64_t max_prefix,
                                          const int32_t* block_table, int64_t table_width, int64_t table_stride,
                                          const int32_t* q_start, const int32_t* kv_len, int64_t batch, int64_t max_q,
                                          int64_t max_kv, float scale, void* out, int64_t out_token_stride,
                                          int64_t out_head_stride, void* workspace, size_t ws_bytes);

/* Workspace of phi_hip_paged_attention_shared (0 for sizes that no call may have). */
size_t phi_hip_paged_attention_shared_workspace_bytes(int64_t tokens, int64_t q_heads, int64_t kv_heads, int64_t dim,
                                                      int64_t groups, int64_t batch, int64_t max_prefix,
                                                      int64_t max_q, int64_t max_kv, int dtype);

/*
 * Low-rank adapters of many requests beside one linear:
 *   out[m] = base[m] + scale[a] B[a] (A[a] x[m]),   a = adapter[m]
 * for rows m in any order of adapters; a row whose adapter is below 0 or not below
 * `adapters` has none: out[m] = base[m].
 *
 *   x        [rows, ldx] of x_dtype, K columns
 *   A, B     [adapters, R, K] and [adapters, N, R] of w_dtype, last dimension
 *            contiguous, the others' strides in elements.  Adapters of fewer ranks
 *            have zeros in the rest.
 *   adapter  [rows] int32; scale [adapters] fp32, or NULL: 1
 *   base     [rows, ld_base] of out_dtype, N columns: the linear's output; NULL: 0
 *   out      [rows, ldo] of out_dtype; may be base, else shares no memory with an input
 *   workspace  phi_hip_lora_batched_workspace_bytes() bytes, 16-byte aligned
 * All dtypes PHI_F32 or PHI_BF16; every pointer aligned to its own type; R to 256, rows,
 * K and N to 2^24.  Products of bf16 by bf16 are exact, the others fp32; all sums and A x
 * itself are fp32, and out is rounded once.  phi_hip_lora_tail has one adapter for
 * all rows and the reference's order of sums; here a sum's order depends on rows, K
 * and R alone, so a row's bits do not depend on its neighbours' adapters.
 */
phi_status phi_hip_lora_batched(phi_stream_t stream, const void* x, int x_dtype, int64_t ldx, int64_t rows, int64_t K,
                                const void* A, int64_t a_adapter_stride, int64_t a_row_stride, const void* B,
                                int64_t b_adapter_stride, int64_t b_row_stride, int w_dtype, int64_t adapters,
                                int64_t R, int64_t N, const int32_t* adapter, const float* scale, const void* base,
                                int64_t ld_base, void* out, int out_dtype, int64_t ldo, void* workspace,
                                size_t ws_bytes);

/* Workspace of phi_hip_lora_batched (0 for sizes that no call may have). */
size_t phi_hip_lora_batched_workspace_bytes(int64_t rows, int64_t K, int64_t R);

#ifdef __cplusplus
}
#endif

#endif /* PHI_SERVING_H */
