// What the attention kernels share: a batch's geometry on the device, the
// query's integer form, and how partial softmaxes are kept and joined.
//
// A row's logits are kept in base 2, x_t = log2(e) scale q.k_t, as
//   x_t = rq * (sk_t * c_t),   c_t = sum_d Q_d K_td  (exact integers)
// with K the cache's codes, sk_t their scale, and Q = round(q' / rq) the
// integer form of q' = log2(e) scale q at 16 bits (bf16 q) or 24 bits (fp32 q)
// relative to the row's largest |q'|.  Q is split into signed bytes, Q = 256 Q1
// + Q0 (or 65536 Q2 + 256 Q1 + Q0), so that q.k runs on the int8 matrix
// instructions, which read K as it lies in the cache at twice the rate of the
// 16-bit ones: two products of half the cost, no conversion of K, and less
// error than q itself has (2^-16 of the row's largest element).
//
// p.v: paged_decode.hip, bound by memory, has V's codes exactly in bf16 against
// p_t sv_t as a sum of two bf16 (16 bits; fp32 q: three, 24 bits), which have
// fp32's whole range.  paged_chunk.hip, bound by the matrix cores, has one
// product of fp16 (11 bits), both factors kept in its range.
#pragma once

#include "decoder.hpp"
#include "device_common.hpp"

namespace phi_dev {

typedef __bf16 b8 __attribute__((ext_vector_type(8)));

// m of a row that has seen nothing: finite, so that exp2(-inf - m) is 0 and
// exp2(m - m) is 1, and below every logit that matters.
constexpr float kNoMax = -1e30f;

// One sequence's new tokens and range, as the device arrays give them, within
// the bounds that the host checked.
struct SeqInfo {
    int first, n;  // its rows of q
    int kv;        // tokens that can be seen
    int pos0;      // position of its first new token (below 0: rows before any token)
};

__device__ __forceinline__ SeqInfo seq_info(const PagedAttn& p, int page, int b) {
    SeqInfo s;
    const int64_t a = p.q_start[b], e = p.q_start[b + 1], T = p.tokens;
    s.first = (int)(a < 0 ? 0 : a > T ? T : a);
    s.n = max(0, (int)(e < 0 ? 0 : e > T ? T : e) - s.first);
    const int kv = max(0, p.kv_len[b]);
    s.kv = (int)min((int64_t)min(kv, p.max_kv), (int64_t)p.table_width * page);
    s.pos0 = kv - s.n;
    return s;
}

// A sequence's rows are the query heads of a key/value head x its new tokens, in
// that order.  Sequences of at most few_rows rows go to paged_decode.hip (AttnPart
// few), those of more to paged_chunk.hip (many; bf16 queries only).
//
// A part's blocks share out the (sequence, row tile, split) triples that there
// are, kv_heads blocks each; the grid is an upper bound of their number and the
// blocks past it end at once.  (A grid over the longest sequence's tiles and
// splits leaves working blocks at a fixed stride among idle ones, which the
// dispatcher deals to the same few compute units: 358 us against 118 for a chunk of
// 512 tokens over 4352 beside seven empty sequences.)
//
// Split z of a sequence has its tokens [z * len, (z + 1) * len).  With count > 1
// each leaves for its rows the undivided sum of p v, o [splits][rows][dim], and
// the maximum and the sum of p, ml [splits][rows][2], for attn_join_kernel.
struct AttnPart {
    int len, count;
    int64_t rows;   // rows of o and ml a split
    int row_pitch;  // few: rows a (sequence, key/value head) in them
    int blocks;     // the grid, over kv_heads
    float* o;
    float* ml;
};

hipError_t launch_paged_decode(hipStream_t stream, const KvCache& c, const PagedAttn& p, const AttnPart& s);
hipError_t launch_paged_chunk(hipStream_t stream, const KvCache& c, const PagedAttn& p, const AttnPart& s);
// Rows of a block's tile.
constexpr int kDecodeRows = 16;
constexpr int kChunkRows = 256, kChunkRowsWide = 128;  // dim to 128, above

// Whether 16 tokens from a multiple of 16 lie in one block, their scales in a
// row at 16-byte alignment, with offsets in the block and strides of blocks
// within 31 bits.
inline bool tiles_of_16(const KvCache& c) {
    const int64_t lim = (int64_t)1 << 31;
    return c.page % 16 == 0 && c.s_token_stride == 1 && c.s_block_stride % 4 == 0 && c.s_head_stride % 4 == 0 &&
           (uintptr_t)c.ks % 16 == 0 && (uintptr_t)c.vs % 16 == 0 && c.page * c.token_stride < lim && c.block_stride < lim &&
           c.s_block_stride < lim;
}

// Triple number `unit` of a part (the same in all lanes): its sequence, row tile
// and split; b < 0: there are fewer.  A sequence's triples: late tiles first
// (they see most tokens), splits inside.  FEW: the sequences of at most few_rows.
struct AttnUnit {
    int b, tile, z;
};

template <bool FEW>
__device__ __forceinline__ AttnUnit attn_unit(const PagedAttn& p, const AttnPart& s, int page, int tile_rows, int unit) {
    const int lane = threadIdx.x & 63;
    for (int b0 = 0; b0 < p.batch; b0 += 64) {
        int tiles = 0, splits = 1;
        if (b0 + lane < p.batch) {
            const SeqInfo q = seq_info(p, page, b0 + lane);
            const int rows = min(q.n, p.max_q) * p.group;
            if ((rows <= p.few_rows) == FEW) tiles = (rows + tile_rows - 1) / tile_rows;
            splits = max(1, (q.kv + s.len - 1) / s.len);
        }
        int end = tiles * splits;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const int x = __shfl_up(end, off, 64);
            end += lane >= off ? x : 0;
        }
        const uint64_t past = __ballot(end > unit);
        if (past) {
            const int at = __builtin_ctzll(past), local = unit - __builtin_amdgcn_readlane(end - tiles * splits, at);
            const int n = __builtin_amdgcn_readlane(splits, at), tile = local / n;
            return {b0 + at, __builtin_amdgcn_readlane(tiles, at) - 1 - tile, local - tile * n};
        }
        unit -= __builtin_amdgcn_readlane(end, 63);
    }
    return {-1, 0, 0};
}

// The maximum over lanes l, l ^ 16, l ^ 32, l ^ 48, and over l, l ^ 32.
__device__ __forceinline__ float max_x32(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float max_x16(float v) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float add_x32(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float add_x16(float v) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Sixteen elements of a query vector at element offset off, as fp32.
template <bool F32>
__device__ __forceinline__ void load_q16(const void* __restrict__ q, int64_t off, float (&x)[16]) {
    if (F32) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float4 t = *(const float4*)((const float*)q + off + 4 * i);
            x[4 * i] = t.x, x[4 * i + 1] = t.y, x[4 * i + 2] = t.z, x[4 * i + 3] = t.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const uint4 t = *(const uint4*)((const uint16_t*)q + off + 8 * i);
            const uint32_t w[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
            for (int j = 0; j < 4; j++) x[8 * i + 2 * j] = bf16_to_f32(w[j] & 0xffffu), x[8 * i + 2 * j + 1] = bf16_to_f32(w[j] >> 16);
        }
    }
}

// The integer form's terms (2 or 3 signed bytes an element) and its largest
// value: 127 (256 + 1) and, a little below 127 (65536 + 256 + 1), 0x7f7f00,
// because the product with the row's largest element may round one up there.
template <bool F32> constexpr int q_terms = F32 ? 3 : 2;
template <bool F32> constexpr float q_steps = F32 ? 8355584.0f : 32639.0f;

// Sixteen elements x * inv as integers, byte-split, term 0 the low one.
template <bool F32>
__device__ __forceinline__ void split_q16(const float (&x)[16], float inv, v4i (&out)[q_terms<F32>]) {
#pragma unroll
    for (int w = 0; w < 4; w++) {
        int b[q_terms<F32>][4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            int r = (int)rintf(x[4 * w + j] * inv);
#pragma unroll
            for (int t = 0; t < q_terms<F32>; t++) {
                b[t][j] = (int)(int8_t)r;
                r = (r - b[t][j]) >> 8;
            }
        }
#pragma unroll
        for (int t = 0; t < q_terms<F32>; t++) out[t][w] = (int)pack4(b[t][0], b[t][1], b[t][2], b[t][3]);
    }
}

// c_t in fp32 (exactly, for bf16 q's two terms at dim <= 256: below 2^31) from
// the terms' products.
template <bool F32>
__device__ __forceinline__ float join_terms(const int (&c)[q_terms<F32>]) {
    if (F32) return fmaf((float)c[q_terms<F32> - 1], 65536.0f, fmaf((float)c[1], 256.0f, (float)c[0]));
    return (float)(c[1] * 256 + c[0]);
}

// How far above the running maximum a logit may lie (as a power of two) before
// that moves: sums are fp32, so p may well exceed 1.
constexpr float kHead = 8.0f;

}  // namespace phi_dev
