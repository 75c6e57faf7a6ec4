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

#include <climits>

#include "attn_row.hpp"
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

// With shared prefixes a group's prefix is a sequence too, the groups' before the
// batch's own: its rows are those of all its sequences, each past all of its tokens.
template <bool SHARED>
__device__ __forceinline__ SeqInfo seq_info(const PagedAttn& p, int page, int b) {
    SeqInfo s;
    if constexpr (!SHARED) {
        const int64_t a = p.q_start[b], e = p.q_start[b + 1], T = p.tokens;
        s.first = (int)(a < 0 ? 0 : a > T ? T : a);
        s.n = max(0, (int)(e < 0 ? 0 : e > T ? T : e) - s.first);
        const int kv = max(0, p.kv_len[b]);
        s.kv = (int)min((int64_t)min(kv, p.max_kv), (int64_t)p.table_width * page);
        s.pos0 = kv - s.n;
        return s;
    }
    const bool prefix = b < p.groups;
    int from = b - p.groups, to = from + 1;
    if (prefix) {
        const int batch = p.batch - p.groups;
        from = min(max(p.group_start[b], 0), batch), to = min(max(p.group_start[b + 1], 0), batch);
    }
    const int64_t a = p.q_start[from], e = p.q_start[to], T = p.tokens;
    s.first = (int)(a < 0 ? 0 : a > T ? T : a);
    s.n = max(0, (int)(e < 0 ? 0 : e > T ? T : e) - s.first);
    const int kv = max(0, prefix ? p.prefix_len[b] : p.kv_len[from]);
    s.kv = (int)min((int64_t)min(kv, prefix ? p.max_prefix : p.max_kv), (int64_t)(prefix ? p.prefix_width : p.table_width) * page);
    s.pos0 = prefix ? s.kv : kv - s.n;
    if (!prefix) s.n = min(s.n, p.own_q);
    return s;
}

// A sequence's row of the block table; prefixes' lie prefix_at further on.
template <bool SHARED>
__device__ __forceinline__ const int32_t* table_row(const PagedAttn& p, const int32_t* __restrict__ table, int b) {
    if constexpr (!SHARED) return table + (int64_t)b * p.table_stride;
    const int64_t at = b < p.groups ? p.prefix_at + b * p.prefix_stride : (b - p.groups) * p.table_stride;
    return table + at;
}

// A sequence's rows are the query heads of a key/value head x its new tokens, in
// that order.  Sequences of at most few_rows rows go to paged_decode.hip (AttnPart
// few), those of more to paged_chunk.hip (many; bf16 queries only).
//
// A part's blocks take the (sequence, row tile, split of the tokens) triples that
// there are, kv_heads blocks each; the grid is an upper bound of their number and
// the blocks past it end at once.  (A grid over the longest sequence's tiles and
// splits leaves working blocks at a fixed stride among idle ones, which the
// dispatcher deals to the same few compute units: 358 us against 118 for a chunk of
// 512 tokens over 4352 beside seven empty sequences.)
//
// A tile of more than one split leaves for its rows, split by split in a slot each,
// the undivided sum of p v, o [kv_heads][slots][tile's rows][dim], and the maximum
// and the sum of p, ml [..][2], for attn_join_kernel.
struct AttnPart {
    int step;     // tokens
    int shares;   // a split has at least 1 / shares of all tiles' steps; 0: no splits
    int slots;    // a key/value head
    int rows;     // a tile
    int blocks;   // the grid, over kv_heads; 0: does not run
    int seqs;     // with shared prefixes, the sequences that may be of this part, from the first on
    float* o;
    float* ml;
};

// Rows of a block's tile.
constexpr int kDecodeRows = 16;
constexpr int kChunkRows = 256, kChunkRowsWide = 128;  // dim to 128, above

hipError_t launch_paged_decode(hipStream_t stream, const KvCache& c, const PagedAttn& p, const AttnPart& s);
hipError_t launch_paged_chunk(hipStream_t stream, const KvCache& c, const PagedAttn& p, const AttnPart& s);
// Both in one launch (bf16, dim to 128).
hipError_t launch_paged_shared(hipStream_t stream, const KvCache& c, const PagedAttn& p, const AttnPart& many, const AttnPart& few);

// Whether 16 tokens from a multiple of 16 lie in one block, their scales in a
// row at 16-byte alignment, with offsets in the block and strides of blocks
// within 31 bits.
inline bool tiles_of_16(const KvCache& c) {
    const int64_t lim = (int64_t)1 << 31;
    return c.page % 16 == 0 && c.s_token_stride == 1 && c.s_block_stride % 4 == 0 && c.s_head_stride % 4 == 0 &&
           (uintptr_t)c.ks % 16 == 0 && (uintptr_t)c.vs % 16 == 0 && c.page * c.token_stride < lim && c.block_stride < lim &&
           c.s_block_stride < lim;
}

// The work of block number `unit` of a part (the same in all lanes): row tile `tile`
// of sequence b, tokens from z0 to z1, to be left in a slot (-1: there is no other
// split, so written out).  b < 0: there are fewer.
// Of its tile's `splits`, those but the last are in slots from `first` on.
struct AttnUnit {
    int b, tile, slot, z0, z1;
    SeqInfo s;
    int first, splits;
    bool last;
};

__device__ __forceinline__ void leave_row(const PagedAttn& p, const AttnUnit& u, int r, int in, bool many) {
    const bool prefix = u.b < p.groups;
    const int i = r / p.group;
    (prefix ? p.prefix_rows : p.own_rows)[(int64_t)(u.s.first + i) * p.group + (r - i * p.group)] =
        {u.first, u.slot, (uint32_t)u.splits | (uint32_t)in << 16 | (many ? 1u << 31 : 0u), prefix ? u.b : u.b - p.groups};
}

__device__ __forceinline__ SeqInfo seq_of_lane(const SeqInfo& q, int at) {
    return {__builtin_amdgcn_readlane(q.first, at), __builtin_amdgcn_readlane(q.n, at), __builtin_amdgcn_readlane(q.kv, at),
            __builtin_amdgcn_readlane(q.pos0, at)};
}

// The sum over lanes up to the own: within rows of 16, then rows 0 and 2's onto the
// next, then the first half's onto the second.
__device__ __forceinline__ int lanes_sum(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);  // row_shr:1
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row_bcast:15
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // row_bcast:31
    return v;
}

// The sequences of a part, 64 at a time, one a lane (FEW: those of at most few_rows
// rows).  How long a split is follows from the steps there are, so that the splits that are not their tile's last, all of one
// length, are at most `shares`.  These come first among the 64 sequences' blocks,
// then the last ones, longer before shorter by quarters of that length, so that the
// work evens out whatever the lengths.
template <bool FEW, bool SHARED> struct AttnScan {
    int b0 = -64, base = 0;  // the first lane's sequence, blocks before its
    int len, total = 0;      // steps a split, 0: being counted; steps in all
    SeqInfo q;
    int tiles, first, n, k;  // n steps from `first` on, k splits a tile
    int full_end = 0, last = 0;  // splits but the last up to the lane's own; its tiles' first last split
    int lasts = 0;               // last splits

    __device__ __forceinline__ explicit AttnScan(const AttnPart& s) : len(s.shares ? 0 : 1 << 30) {}
    __device__ __forceinline__ int fulls() const { return __builtin_amdgcn_readlane(full_end, 63); }
    __device__ __forceinline__ int blocks() const { return fulls() + lasts; }
    // On to the next 64; false: there are none.
    __device__ __forceinline__ bool next(const PagedAttn& p, const AttnPart& s, int page) {
        for (;;) {
            const int seqs = SHARED ? s.seqs : p.batch;
            const bool counted = b0 + 64 >= seqs;
            if (counted) {
                if (len) return false;
                len = max(1, (total + s.shares - 1) / s.shares);
                if (b0 > 0) b0 = -64;
            }
            if (!counted || b0 < 0) {
                base += blocks();
                b0 += 64;
                const int at = b0 + (threadIdx.x & 63);
                q = SeqInfo{}, tiles = 0;
                first = 0, n = 1;
                if (at < seqs) {
                    q = seq_info<SHARED>(p, page, at);
                    const int rows = min(q.n, p.max_q) * p.group;
                    if ((rows <= p.few_rows) == FEW) tiles = (rows + s.rows - 1) / s.rows;
                    // The steps that hold what some row sees.
                    const int hi = p.causal ? min(q.kv, q.pos0 + min(q.n, p.max_q)) : q.kv;
                    if (p.window > 0) first = min(max(0, q.pos0 + 1 - p.window), p.max_kv) / s.step;
                    n = max(1, (hi > 0 ? (hi - 1) / s.step + 1 : 0) - first);
                }
                if (!len) {
                    total += __builtin_amdgcn_readlane(lanes_sum(tiles * n), 63);
                    continue;
                }
            }
            k = (n - 1) / len + 1;
            full_end = lanes_sum(tiles * (k - 1));
            lasts = 0;
            const int quarter = (4 * (n - (k - 1) * len) - 1) / len;
#pragma unroll
            for (int c = 3; c >= 0; c--) {
                const int t = c == 3 ? (quarter >= 3 ? tiles : 0) : quarter == c ? tiles : 0, sum = lanes_sum(t);
                last = t ? lasts + sum - t : last;
                lasts += __builtin_amdgcn_readlane(sum, 63);
            }
            return true;
        }
    }
};

template <bool FEW, bool SHARED>
__device__ __forceinline__ AttnUnit attn_unit(const PagedAttn& p, const AttnPart& s, int page, int unit) {
    AttnScan<FEW, SHARED> f(s);
    while (f.next(p, s, page)) {
        const int local = unit - f.base;
        if (local >= f.blocks()) continue;
        const bool full = local < f.fulls();
        const int full_begin = f.full_end - f.tiles * (f.k - 1);
        const int off = full ? local : local - f.fulls(), begin = full ? full_begin : f.last;
        const int at = __builtin_ctzll(__ballot(begin <= off && off < (full ? f.full_end : begin + f.tiles)));
        const int k = __builtin_amdgcn_readlane(f.k, at), in = off - __builtin_amdgcn_readlane(begin, at);
        const int tile = full ? in / (k - 1) : in, z = full ? in - tile * (k - 1) : k - 1;
        const int z0 = (__builtin_amdgcn_readlane(f.first, at) + z * f.len) * s.step;
        // Late tiles first: they see most tokens.
        return {f.b0 + at, __builtin_amdgcn_readlane(f.tiles, at) - 1 - tile, k > 1 || SHARED ? unit : -1, z0, full ? z0 + f.len * s.step : INT_MAX, seq_of_lane(f.q, at),
                f.base + __builtin_amdgcn_readlane(full_begin, at) + tile * (k - 1), k, !full};
    }
    return {-1, 0, 0, 0, 0, {}, 0, 0, false};
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

// Sixteen elements of a query vector as they lie in memory, and element j.
template <bool F32> struct Q16 {
    uint32_t w[F32 ? 16 : 8];
};
template <bool F32>
__device__ __forceinline__ void load_q16(const void* __restrict__ q, int64_t off, Q16<F32>& x) {
    const uint4* src = F32 ? (const uint4*)((const float*)q + off) : (const uint4*)((const uint16_t*)q + off);
#pragma unroll
    for (int i = 0; i < (F32 ? 4 : 2); i++) {
        const uint4 t = src[i];
        x.w[4 * i] = t.x, x.w[4 * i + 1] = t.y, x.w[4 * i + 2] = t.z, x.w[4 * i + 3] = t.w;
    }
}
template <bool F32>
__device__ __forceinline__ float elem_q16(const Q16<F32>& x, int j) {
    return __uint_as_float(F32 ? x.w[j] : j & 1 ? x.w[j >> 1] & 0xffff0000u : x.w[j >> 1] << 16);
}

// The integer form's terms (2 or 3 signed bytes an element) and its largest
// value: 127 (256 + 1) and, a little below 127 (65536 + 256 + 1), 0x7f7f00,
// because the product with the row's largest element may round one up there.
template <bool F32> constexpr int q_terms = F32 ? 3 : 2;
template <bool F32> constexpr float q_steps = F32 ? 8355584.0f : 32639.0f;

// Sixteen elements x * inv as integers, byte-split, term 0 the low one.  An
// integer with 128 added to each byte but the highest has its terms as bytes, those
// below the highest with their sign bit turned.
template <bool F32>
__device__ __forceinline__ void split_q16(const Q16<F32>& x, float inv, v4i (&out)[q_terms<F32>]) {
#pragma unroll
    for (int w = 0; w < 4; w++) {
        uint32_t r[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const float v = elem_q16<F32>(x, 4 * w + j);
            // 1.5 2^23 + 128: the integer part as the sum's low 16 bits.
            r[j] = F32 ? (uint32_t)((int)rintf(v * inv) + 0x8080) : __float_as_uint(fmaf(v, inv, 12583040.0f));
        }
        const uint32_t a = __builtin_amdgcn_perm(r[1], r[0], 0x05010400u), b = __builtin_amdgcn_perm(r[3], r[2], 0x05010400u);
        out[0][w] = (int)(__builtin_amdgcn_perm(b, a, 0x05040100u) ^ 0x80808080u);
        const uint32_t second = __builtin_amdgcn_perm(b, a, 0x07060302u);
        out[1][w] = (int)(F32 ? second ^ 0x80808080u : second);
        if constexpr (F32) {
            const uint32_t e = __builtin_amdgcn_perm(r[1], r[0], 0x0c0c0602u), f = __builtin_amdgcn_perm(r[3], r[2], 0x0c0c0602u);
            out[2][w] = (int)__builtin_amdgcn_perm(f, e, 0x05040100u);
        }
    }
}

// c_t in fp32, rounded once for bf16 q (its two terms' sum is exact, below 2^31 at
// dim <= 256), three times for fp32 q.
template <bool F32>
__device__ __forceinline__ float join_terms(const int (&c)[q_terms<F32>]) {
    if (F32) return fmaf((float)c[q_terms<F32> - 1], 65536.0f, fmaf((float)c[1], 256.0f, (float)c[0]));
    return (float)(c[1] * 256 + c[0]);
}

// How far above the running maximum a logit may lie (as a power of two) before
// that moves: sums are fp32, so p may well exceed 1.
constexpr float kHead = 8.0f;

}  // namespace phi_dev
