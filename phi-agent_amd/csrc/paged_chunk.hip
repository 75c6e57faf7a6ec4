// Attention of chunks of new tokens over the paged int8 cache (bf16 queries).
//
// Bound by the matrix cores, and next to them by LDS reads and vector work, all
// near each other, so each is kept small and they are made to overlap:
//   - A block holds 32 rows a wave (query heads of one key/value head x new
//     tokens, in that order, so that heads share the cache's tokens) and walks
//     the tokens in tiles of 64.  Q, O and the softmax stay in registers.
//   - K and V are made fp16 once a block: the tile's codes come to registers one
//     tile ahead, become code * scale in the unit of a power of two for every 16
//     tokens (so that all of them use fp16's range), and go to a double buffer in
//     LDS in the order in which the products read them, without bank
//     conflicts.  K: one fp32 product and one rounding to 11 bits a code, at
//     random sides, so that a logit is off by some 2^-13 |s| / sqrt(dim) (q is
//     exact in fp16).  V: the scale has 11 bits too, which makes it two packed
//     instructions for two codes, the first of which makes the codes exact in a unit
//     that leaves the product fp16's range.  (With one, code * scale less the bias, the
//     bias loses its bits: a token of 2^-12 of its 16 tokens' largest scale is off by 0.2 %,
//     to one side, one of 2^-20 by 40 %.  The second costs 0.8 % of the time below, 1.3 % at
//     dim 256; fp32 scales in v_fma_mix, as for K, 3 % and 7 %.)
//     int8 products for q.k, exact, cost the matrix cores the same but the
//     vector unit three more instructions for every logit (join, convert, scale).
//   - S^T = K Q^T and O^T = V^T P^T (v_mfma_f32_32x32x16_f16): the logits' layout
//     is already that of P's operand, as in paged_decode.hip.
//   - The running maximum moves only when a logit exceeds it by a factor of 2^kUp,
//     and masks are looked at only in tiles that a mask or the length cuts.
//   - Waves 0-3 and 4-7 (one of each on a SIMD) run half a tile apart: while one
//     group has its products, the other has its softmax and stages the next
//     tiles, waves 0-3 V's and 4-7 K's.
// 4096 tokens over 16384, 32 heads over 8 of 128: 1.08 ms, 890 TFLOP/s of the 1458 that
// a product of 8192^3 in fp16 reaches; the matrix cores are busy 43 % of the time.  A
// tile takes 5400 clocks, of which the matrix cores need 2048 and the vector unit some
// 3300 (two waves' softmax and staging), and each group's turn waits for the other's.
// A block costs 13 us beside its tiles: the batch's lookup and Q 4, the first tiles 4,
// O's stores 3 to 8.
#include <type_traits>
#include <utility>

#include "paged_attention.hpp"

namespace phi_dev {

namespace {

constexpr int kTile = 64;  // tokens
constexpr int kGroups = kTile / 16;
// p enters fp16 as p 2^kP in the unit of its 16 tokens' V, and may reach 2^kUp
// before the running maximum moves: at most 2^15.  The rest of fp16's range lies
// below, so that weights keep their 11 bits down to 2^-28 of the row's largest
// and an absolute error of 2^-39 of it from there.  V's unit of a row, 2^vexp, is that
// of the groups it has seen some of: one for all rows of a wave lets tokens that only
// some of them see take the others' weights (and saves 0.4 % of the time).
constexpr int kP = 14, kUp = 1;
constexpr int kMinExp = -100;  // of a group's unit: its inverse stays finite
// V's fp16 is code 2^-9 * M, M = scale * 2^(kM - E) below 2^15, both factors in fp16: below
// 2^13, with 11 bits down to 2^-20 of the unit 2^E of its 16 tokens.
constexpr int kM = 14;

typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float v16f __attribute__((ext_vector_type(16)));

// LDS writes and reads of all waves before it are done; loads from memory may
// be under way.
__device__ __forceinline__ void lds_barrier() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// Two codes, biased by 128, that lie alone in the halves of u: code * f as
// fp16, the bias taken off in the same fma (the halves are the subnormals (code +
// 128) 2^-24; f24 = f 2^24, off = -128 f).
__device__ __forceinline__ uint32_t scale_pair(uint32_t u, float f24, float off) {
    uint32_t r;
    asm("v_fma_mixlo_f16 %0, %1, %2, %3 op_sel_hi:[1,0,0]" : "=v"(r) : "v"(u), "v"(f24), "v"(off));
    asm("v_fma_mixhi_f16 %0, %1, %2, %3 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "+v"(r) : "v"(u), "v"(f24), "v"(off));
    return r;
}

template <int N> using int_c = std::integral_constant<int, N>;

// f(0), f(1), .. f(N - 1), each with its number as a type.
template <class F, int... I>
__device__ __forceinline__ void each_of(F f, std::integer_sequence<int, I...>) {
    (f(int_c<I>{}), ...);
}
template <int N, class F>
__device__ __forceinline__ void each(F f) {
    each_of(f, std::make_integer_sequence<int, N>{});
}

// max over 16 lanes of a value >= 0; uniform where every 16 lanes hold the same values.
__device__ __forceinline__ float row_top(float v) {
    uint32_t u = __float_as_uint(v);
    u = max(u, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)u, 0xB1, 0xF, 0xF, false));   // quad_perm 1,0,3,2
    u = max(u, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)u, 0x4E, 0xF, 0xF, false));   // quad_perm 2,3,0,1
    u = max(u, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)u, 0x141, 0xF, 0xF, false));  // row_half_mirror
    u = max(u, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)u, 0x140, 0xF, 0xF, false));  // row_mirror
    return __uint_as_float(__builtin_amdgcn_readfirstlane(u));
}

// E of a group of scales: 2^E <= top < 2^(E+1), within [kMinExp, 127].
__device__ __forceinline__ int exp_of(float top) { return max(kMinExp, (int)(__float_as_uint(top) >> 23) - 127); }

// 2^e, -127 < e < 128.
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

}  // namespace

template <int DP> struct ChunkTile {
    _Float16 k[kTile * DP];  // rows of DP, 16-byte chunk n of row t in slot k_slot(t, n)
    _Float16 v[kTile * DP];  // [2 group + half][slot][8 tokens], slot = (d % 4) DP / 4 + d / 4
};
// Of a tile's 16-token groups: 2^(Ek - 7), Ev, and bit t: token t is there.
struct ChunkMeta {
    float k_unit[kGroups];
    int v_exp[kGroups];
    uint32_t seen[kGroups];
};
template <int DP> struct ChunkLds {
    ChunkTile<DP> tile[2];
    // Of tile n in n % 4, staged with its K.
    ChunkMeta meta[4];
};

template <int DP>
__device__ __forceinline__ int k_slot(int t, int n) {
    return n ^ (DP == 64 ? (t >> 1) & 7 : t & 15);
}

// DP: dim rounded up to 64, 128 or 256; NW waves, 32 rows each; PAGE16 as in
// paged_decode.hip.
template <int DP, int NW, bool PAGE16>
__global__ __launch_bounds__(64 * NW, DP <= 128 ? 2 : 1) void paged_chunk_kernel(KvCache c, PagedAttn p, AttnPart sp,
                                                                              const int32_t* __restrict__ table) {
    constexpr int KS = DP / 16, OT = DP / 32;
    constexpr int NVI = DP == 256 ? 2 : 1, NKI = DP / 64;  // V's and K's items a lane
    extern __shared__ __align__(16) uint8_t lds_raw[];
    ChunkLds<DP>& lds = *(ChunkLds<DP>*)lds_raw;
    ChunkTile<DP>* tile = lds.tile;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 31, h = lane >> 5;
    const int heads = c.heads, D = c.dim;
    const int kh = blockIdx.x % heads;
    const AttnUnit unit_of = attn_unit<false>(p, sp, c.page, blockIdx.x / heads);
    if (unit_of.b < 0) return;
    const int b = unit_of.b, z0 = unit_of.z0;
    const SeqInfo s = unit_of.s;
    const int rows = min(s.n, p.max_q) * p.group, r0 = unit_of.tile * 32 * NW;

    // The lane's row, and the ranges of the wave's rows and of the block's.
    const int w0 = r0 + 32 * wave;
    const int r = min(w0 + col, rows - 1), i = r / p.group, head = kh * p.group + (r - i * p.group);
    const int64_t token = s.first + i;
    const int pos = s.pos0 + i;
    const int row_hi = p.causal ? min(s.kv, pos + 1) : s.kv, row_lo = p.window > 0 ? max(0, pos + 1 - p.window) : 0;
    auto pos_of = [&](int row) { return s.pos0 + min(row, rows - 1) / p.group; };
    auto hi_of = [&](int ps) { return min(p.causal ? min(s.kv, ps + 1) : s.kv, unit_of.z1); };
    auto lo_of = [&](int ps) { return max(p.window > 0 ? max(0, ps + 1 - p.window) : 0, z0); };
    const int hi = hi_of(pos_of(r0 + 32 * NW - 1)), lo = lo_of(pos_of(r0));
    const int all_hi = hi_of(pos_of(w0)), all_lo = lo_of(pos_of(w0 + 31));

    // Q in fp16, exactly but for elements below 2^-21 of the row's largest,
    // scaled to bring that into [2^7, 2^8).
    h8 q[KS];
    float rq;
    {
        uint4 raw[KS];
        float amax = 0.0f, bad = 0.0f;
        const uint16_t* src = (const uint16_t*)p.q + token * p.q_token + head * p.q_head;
#pragma unroll
        for (int ks = 0; ks < KS; ks++) {
            const int d = 16 * ks + 8 * h;
            raw[ks] = d < D ? *(const uint4*)(src + d) : make_uint4(0, 0, 0, 0);
            const uint32_t w[4] = {raw[ks].x, raw[ks].y, raw[ks].z, raw[ks].w};
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float x = bf16_to_f32(j & 1 ? w[j >> 1] >> 16 : w[j >> 1] & 0xffffu);
                amax = fmaxf(amax, fabsf(x));
                bad += x * 0.0f;  // NaN once an infinity or a NaN is met
            }
        }
        amax = max_x32(amax);
        bad = add_x32(bad);
        const int e = exp_of(amax);
        const float f = p.scale * 1.4426950408889634f, unit = pow2(min(e, 127)) * 0.0078125f;
        float mul = pow2(7 - e);
        rq = fabsf(f) * unit;
        if (!(rq > 0x1p-126f)) mul = 0.0f, rq = 1.0f;  // every logit is 0
        if (f < 0.0f) mul = -mul;
        rq += bad;
#pragma unroll
        for (int ks = 0; ks < KS; ks++) {
            const uint32_t w[4] = {raw[ks].x, raw[ks].y, raw[ks].z, raw[ks].w};
#pragma unroll
            for (int j = 0; j < 8; j++) q[ks][j] = (_Float16)(bf16_to_f32(j & 1 ? w[j >> 1] >> 16 : w[j >> 1] & 0xffffu) * mul);
        }
    }

    // ---- the tile's codes: a wave takes 16 tokens, V's or (four waves: and) K's.
    // Lane l finds token l & 15 and has its scales; a token below lo, at hi or past it,
    // or without a block, reads whatever lies there, in the last page or in block 0
    // and counts as scale 0.  Loads run a tile ahead of what is being staged, and the table's
    // entry for them two; nothing loaded is looked at before.
    const int begin = lo & ~(kTile - 1), count = begin < hi ? (hi - begin + kTile - 1) / kTile : 0;
    auto start = [&](int n) { return begin + n * kTile; };
    const int group = wave & 3, n16 = lane & 15;
    const int32_t* trow = table + (int64_t)b * p.table_stride;
    const int last_page = page_of(c, max(hi - 1, 0));
    struct Raw {
        uint32_t w[8 * NVI > 4 * NKI ? 8 * NVI : 4 * NKI];  // V's items' 8 words, K's items' 4
        float vs, ks;
        int ok;   // token l & 15 is there
        int blk;  // the next load's block, fetched one load ahead
    };
    // V's (and, with eight waves, K's in its place), K's: being staged, and loading.
    Raw raw_of[NW == 8 ? 1 : 2], next_of[NW == 8 ? 1 : 2];
    Raw &raw_v = raw_of[0], &raw_k = raw_of[NW == 8 ? 0 : 1], &next_v = next_of[0], &next_k = next_of[NW == 8 ? 0 : 1];
    // A vector load, also where the entry is uniform: a scalar one would have the
    // LDS reads around it wait for each other.
    int lane0 = 0;
    asm("" : "+v"(lane0));
    auto fetch = [&](Raw& raw, int t0) __attribute__((always_inline)) {
        const int t = min(t0 + 16 * group + (PAGE16 ? 0 : n16), hi - 1);
        raw.blk = trow[min(page_of(c, t), last_page) + lane0];
    };
    // V's item of a lane: 4 d of 8 tokens; K's: 16 codes of a token.
    auto v_item = [&](int it) { return (it * 64 + lane) % (DP / 2); };
    auto k_token = [&](int it) { return (it * 64 + lane) / (DP / 16); };
    auto k_chunk = [&](int it) { return (it * 64 + lane) % (DP / 16); };
    auto token_of = [](int ih, int j) { return 8 * (j >> 2) + 4 * ih + (j & 3); };
    const int ts = (int)c.token_stride;
    uint32_t v_off[NVI], k_off[NKI];  // PAGE16: a lane's offset in its group's rows
#pragma unroll
    for (int it = 0; it < NVI; it++) {
        const int dq = v_item(it) % (DP / 4);
        v_off[it] = (PAGE16 ? 4 * (v_item(it) / (DP / 4)) * ts : 0) + (4 * dq < D ? 4 * dq : 0);
    }
#pragma unroll
    for (int it = 0; it < NKI; it++) k_off[it] = (PAGE16 ? k_token(it) * ts : 0) + (16 * k_chunk(it) < D ? 16 * k_chunk(it) : 0);

    // Codes and scales of the group's tokens from t0 on: V's or K's.
    const int64_t s_head = kh * c.s_head_stride;
    auto load = [&](Raw& raw, int t0, bool is_k) __attribute__((always_inline)) {
        const int g0 = t0 + 16 * group;
        const int8_t* codes = (is_k ? c.k : c.v) + kh * c.head_stride;
        const int entry = PAGE16 ? __builtin_amdgcn_readfirstlane(raw.blk) : raw.blk;
        const bool ok = entry >= 0 && entry < c.blocks;
        const int64_t blk = ok ? entry : 0;
        raw.ok = ok && g0 + n16 < hi;
        const int t = min(g0 + (PAGE16 ? 0 : n16), hi - 1), in = (PAGE16 ? t & ~15 : t) - page_of(c, t) * c.page;
        if (PAGE16) {
            // 32-bit strides within a block and of blocks (tiles_of_16); the lane's
            // offsets stay 32-bit beside a scalar base.
            codes += (uint64_t)(uint32_t)blk * (uint32_t)c.block_stride + (uint32_t)in * (uint32_t)ts;
            const int64_t sat = (int64_t)((uint64_t)(uint32_t)blk * (uint32_t)c.s_block_stride) + s_head + in;
            uint32_t at = n16;
            asm("" : "+v"(at));
            raw.vs = (c.vs + sat)[at];
            if (is_k) {
                raw.ks = (c.ks + sat)[at];
#pragma unroll
                for (int it = 0; it < NKI; it++) {
                    uint32_t off = k_off[it];
                    asm("" : "+v"(off));
                    *(v4i*)&raw.w[4 * it] = *(const v4i*)(codes + off);
                }
            } else {
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const int8_t* row = codes + (uint32_t)(token_of(0, j) * ts);
#pragma unroll
                    for (int it = 0; it < NVI; it++) {
                        uint32_t off = v_off[it];
                        asm("" : "+v"(off));
                        raw.w[8 * it + j] = *(const uint32_t*)(row + off);
                    }
                }
            }
        } else {
            const int64_t at = blk * c.block_stride + in * c.token_stride;
            const int64_t sat = blk * c.s_block_stride + s_head + in * c.s_token_stride;
            raw.vs = c.vs[sat];
            if (is_k) {
                raw.ks = c.ks[sat];
#pragma unroll
                for (int it = 0; it < NKI; it++) *(v4i*)&raw.w[4 * it] = *(const v4i*)(codes + __shfl(at, k_token(it), 64) + k_off[it]);
            } else {
#pragma unroll
                for (int it = 0; it < NVI; it++)
#pragma unroll
                    for (int j = 0; j < 8; j++)
                        raw.w[8 * it + j] = *(const uint32_t*)(codes + __shfl(at, token_of(v_item(it) / (DP / 4), j), 64) + v_off[it]);
            }
        }
        fetch(raw, t0 + kTile);
    };
    // E of the group's V scales, the same from V's wave and K's: 2^E <= the largest that
    // is there and finite and no zeros'.  The cache has a vector of zeros at the scale
    // 1, whatever its neighbours' are, so the codes of tokens with that scale are looked
    // at, a quarter of a vector's pieces a lane.  (Rare, so by loads of its own: the
    // branch costs 1 %, 2 % at dim 256, and 20 % where every tenth vector is zeros; a test of
    // all codes as V is staged 5 % to 10 %.)
    auto v_exp_of = [&](const Raw& raw, int tile_n, float& f) __attribute__((always_inline)) {
        f = (raw.ok != 0) & __builtin_isfinite(raw.vs) ? raw.vs : 0.0f;
        if (__any(f == 1.0f)) {
            int codes = 0;
            if (f == 1.0f) {
                const int t = start(tile_n) + 16 * group + n16, page = page_of(c, t);
                const int8_t* row = c.v + kh * c.head_stride + trow[page] * c.block_stride + (t - page * c.page) * c.token_stride;
                for (int d = 16 * (lane >> 4); d < D; d += 64) {
                    const v4i w = *(const v4i*)(row + d);
                    codes |= w[0] | w[1] | w[2] | w[3];
                }
            }
            const uint64_t some = __ballot(codes != 0), half = some | some >> 32;
            f = (half | half >> 16) >> n16 & 1 ? f : f == 1.0f ? 0.0f : f;
        }
        return exp_of(row_top(fabsf(f)));
    };
    // Staging in pieces without a branch (but that) and of a few instructions each, which the
    // turn of products takes one at a time between its own.  Both kinds: take what
    // was loaded, load the tile after, the scales; then an eighth of an item's
    // codes each.
    constexpr int kVPieces = 4 + 8 * NVI, kKPieces = 5 + 8 * NKI;
    int v_e = 0;
    float v_f = 0.0f;
    h2 v_mul[NVI][4];
    h8 v_out;
    auto v_piece = [&](auto index, int tile_n, int next_t0) __attribute__((always_inline)) {
        constexpr int P = decltype(index)::value;
        if constexpr (P == 0) {
            raw_v = next_v;
        } else if constexpr (P == 1) {
            load(next_v, next_t0, false);
        } else if constexpr (P == 2) {
            v_e = v_exp_of(raw_v, tile_n, v_f);
        } else if constexpr (P == 3) {
            // Lane l has the factors of tokens l & 15 and the next, as a pair.
            const float m0 = v_f * pow2(kM - v_e);
            const float m1 = __uint_as_float(__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(m0), 0xF5, 0xF, 0xF, false));  // quad_perm 1,1,3,3
            const int pair = (int)__builtin_bit_cast(uint32_t, h2{(_Float16)m0, (_Float16)m1});
#pragma unroll
            for (int it = 0; it < NVI; it++)
#pragma unroll
                for (int j = 0; j < 4; j++)
                    v_mul[it][j] = __builtin_bit_cast(h2, __builtin_amdgcn_ds_bpermute(4 * token_of(v_item(it) / (DP / 4), 2 * j), pair));
        } else {
            constexpr int it = (P - 4) / 8, e4 = (P - 4) % 8 / 2, half = (P - 4) % 2;
            const uint32_t sel = 0x0c000c00u | (uint32_t)((4 + e4) << 16) | (uint32_t)e4;
#pragma unroll
            for (int j = 2 * half; j < 2 * half + 2; j++) {
                if constexpr (e4 == 0) raw_v.w[8 * it + 2 * j] ^= 0x80808080u, raw_v.w[8 * it + 2 * j + 1] ^= 0x80808080u;
                // The halves (code + 128) 2^-24 to code 2^-9, exactly; a factor a token.
                const h2 u = __builtin_bit_cast(h2, __builtin_amdgcn_perm(raw_v.w[8 * it + 2 * j + 1], raw_v.w[8 * it + 2 * j], sel));
                const h2 y = __builtin_elementwise_fma(u, h2{(_Float16)0x1p15f, (_Float16)0x1p15f}, h2{(_Float16)-0.25f, (_Float16)-0.25f}) * v_mul[it][j];
                v_out[2 * j] = y[0], v_out[2 * j + 1] = y[1];
            }
            if constexpr (half) {
                const int ih = v_item(it) / (DP / 4), dq = v_item(it) % (DP / 4);
                *(h8*)(tile[tile_n & 1].v + (((2 * group + ih) * DP + e4 * (DP / 4) + dq) * 8)) = v_out;
            }
        }
    };
    float k_f = 0.0f, k_mul[NKI];
    int k_e = 0, k_ev = 0;
    uint32_t k_out[4];
    auto k_piece = [&](auto index, int tile_n, int next_t0) __attribute__((always_inline)) {
        constexpr int P = decltype(index)::value;
        if constexpr (P == 0) {
            raw_k = next_k;
        } else if constexpr (P == 1) {
            load(next_k, next_t0, true);
        } else if constexpr (P == 2) {
            float fv;
            k_ev = v_exp_of(raw_k, tile_n, fv);
            // A token whose value is not finite is NaN to the rows that see it.
            const float fk = __builtin_isfinite(raw_k.vs) ? raw_k.ks : __builtin_nanf("");
            k_f = raw_k.ok != 0 ? fk : 0.0f;
            k_e = exp_of(row_top(__builtin_isfinite(k_f) ? fabsf(k_f) : 0.0f));
        } else if constexpr (P == 3) {
            const float own = k_f * pow2(7 - k_e) * 0x1p24f;
#pragma unroll
            for (int it = 0; it < NKI; it++) k_mul[it] = __uint_as_float(__builtin_amdgcn_ds_bpermute(4 * k_token(it), (int)__float_as_uint(own)));
        } else if constexpr (P == 4) {
            ChunkMeta& meta = lds.meta[tile_n & 3];  // the same from all lanes
            meta.k_unit[group] = pow2(k_e - 7), meta.v_exp[group] = k_ev;
            meta.seen[group] = (uint32_t)__ballot(raw_k.ok != 0) & 0xffffu;
        } else {
            constexpr int it = (P - 5) / 8, w = (P - 5) % 8 / 2, half = (P - 5) % 2;
            const float f24 = k_mul[it], off = f24 * -0x1p-17f;
            if constexpr (half == 0) raw_k.w[4 * it + w] ^= 0x80808080u;
            const uint32_t u = raw_k.w[4 * it + w];
            k_out[2 * (w & 1) + half] = scale_pair(__builtin_amdgcn_perm(u, u, half ? 0x0c030c02u : 0x0c010c00u), f24, off);
            if constexpr ((w & 1) && half) {
                const int t = 16 * group + k_token(it);
                *(uint4*)(tile[tile_n & 1].k + t * DP + 8 * k_slot<DP>(t, 2 * k_chunk(it) + (w >> 1))) = make_uint4(k_out[0], k_out[1], k_out[2], k_out[3]);
            }
        }
    };

    v16f o[OT];
#pragma unroll
    for (int n = 0; n < OT; n++)
#pragma unroll
        for (int j = 0; j < 16; j++) o[n][j] = 0.0f;
    float m = kNoMax, l = 0.0f;
    int vexp = kMinExp;

    // Products: P V of a tile (the first kNV) and S of the next.  Each takes 16
    // bytes a lane of LDS.
    constexpr int kNV = kGroups * OT, kNS = 2 * KS;
    v16f x[2];
    h8 ph[kGroups];
    auto operand = [&](auto index, const ChunkTile<DP>& v_of, const ChunkTile<DP>& k_of) __attribute__((always_inline)) {
        constexpr int P = decltype(index)::value;
        if constexpr (P < kNV) {
            return *(const h8*)(v_of.v + ((2 * (P / OT) + h) * DP + 32 * (P % OT) + col) * 8);
        } else {
            constexpr int ks = (P - kNV) / 2, u = (P - kNV) % 2;
            const int t = 32 * u + col;
            return *(const h8*)(k_of.k + t * DP + 8 * k_slot<DP>(t, 2 * ks + h));
        }
    };
    auto product = [&](auto index, h8 a) __attribute__((always_inline)) {
        constexpr int P = decltype(index)::value;
        if constexpr (P < kNV) {
            o[P % OT] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, ph[P / OT], o[P % OT], 0, 0, 0);
        } else {
            constexpr int ks = (P - kNV) / 2, u = (P - kNV) % 2;
            const v16f zero = {0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
            x[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, q[ks], ks == 0 ? zero : x[u], 0, 0, 0);
        }
    };
    // Products FROM .. TO - 1 with their operands read kAhead before, and beside
    // each the piece of other work that beside(product) does.  The scheduling
    // barriers keep that order (left alone, the compiler has the other work
    // first and the operands read one by one: 3150 clocks a turn, against
    // 1024 of the matrix cores).
    auto products = [&](auto from, auto to, const ChunkTile<DP>& v_of, const ChunkTile<DP>& k_of, auto beside) __attribute__((always_inline)) {
        constexpr int F = decltype(from)::value, T = decltype(to)::value, kAhead = 4;
        h8 a[kAhead];
        each<kAhead>([&](auto n) __attribute__((always_inline)) { a[n] = operand(int_c<F + decltype(n)::value>{}, v_of, k_of); });
        each<T - F>([&](auto n) __attribute__((always_inline)) {
            constexpr int P = F + decltype(n)::value, S = decltype(n)::value % kAhead;
            __builtin_amdgcn_sched_barrier(0);
            product(int_c<P>{}, a[S]);
            if constexpr (P + kAhead < T) a[S] = operand(int_c<P + kAhead>{}, v_of, k_of);
            beside(int_c<P>{});
        });
        __builtin_amdgcn_sched_barrier(0);
    };
    auto nothing = [](auto) __attribute__((always_inline)) {};
    ChunkMeta ct;  // the next softmax's tile
    auto read_meta = [&](int tile_n) __attribute__((always_inline)) {
        const ChunkMeta& from = lds.meta[tile_n & 3];
#pragma unroll
        for (int g = 0; g < kGroups; g++) {
            ct.k_unit[g] = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(from.k_unit[g])));
            ct.v_exp[g] = __builtin_amdgcn_readfirstlane(from.v_exp[g]);
            ct.seen[g] = __builtin_amdgcn_readfirstlane(from.seen[g]);
        }
    };
    auto softmax = [&](int t0) __attribute__((always_inline)) {
        float ru[kGroups];
        uint32_t holes = 0;
        int all_e = kMinExp, e;
#pragma unroll
        for (int g = 0; g < kGroups; g++) {
            // Above 0 whatever the units (a row of zeros, 16 tokens that are not there), so
            // that a masked logit stays -inf; 2^-149 more is nothing to the others.
            ru[g] = fmaf(rq, ct.k_unit[g], 0x1p-149f);
            holes |= ct.seen[g] ^ 0xffffu;
            all_e = max(all_e, ct.v_exp[g]);
        }
        e = max(vexp, all_e);
        if (t0 < all_lo || t0 + kTile > all_hi || holes) {
            e = vexp;  // of the groups that the row sees some of
            const int from = max(row_lo, lo) - t0, to = min(row_hi, hi) - t0;
#pragma unroll
            for (int g = 0; g < kGroups; g++) {
                const uint32_t range = (1u << min(max(to - 16 * g, 0), 16)) - (1u << min(max(from - 16 * g, 0), 16));
                e = to > from && (range & ct.seen[g]) ? max(e, ct.v_exp[g]) : e;
            }
            const int a = max(row_lo, lo) - t0 - 4 * h, z = min(row_hi, hi) - t0 - 4 * h;
#pragma unroll
            for (int g = 0; g < kGroups; g++) {
                const uint32_t bits = ct.seen[g] >> (4 * h);
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const int k = 8 * (j >> 2) + (j & 3), tt = 16 * g + k;
                    const bool in = tt >= a && tt < z && (bits >> k & 1);
                    x[g >> 1][8 * (g & 1) + j] = in ? x[g >> 1][8 * (g & 1) + j] : -INFINITY;
                }
            }
        }
        float xm = -INFINITY;
#pragma unroll
        for (int g = 0; g < kGroups; g++) {
            float top = x[g >> 1][8 * (g & 1)];
#pragma unroll
            for (int j = 1; j < 8; j++) top = fmaxf(top, x[g >> 1][8 * (g & 1) + j]);
            xm = fmaxf(xm, top * ru[g]);
        }
        if (__any((xm > m + (float)kUp) | (e != vexp))) {
            const float m2 = fmaxf(m, max_x32(xm)), keep = __builtin_amdgcn_exp2f(m - m2);
            const float ko = keep * (e - vexp > 126 ? 0.0f : pow2(vexp - e));
            m = m2;
            vexp = e;
            l *= keep;
#pragma unroll
            for (int n = 0; n < OT; n++)
#pragma unroll
                for (int j = 0; j < 16; j++) o[n][j] *= ko;
        }
#pragma unroll
        for (int g = 0; g < kGroups; g++) {
            // p in units of 2^-kP and of the group's own power of two for sv (one that
            // the row sees nothing of may lie above its own).
            const int de = min(max(ct.v_exp[g] - vexp, kMinExp), 0);
            const float base = (float)(kP + de) - m;
            float sum = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float pe = __builtin_amdgcn_exp2f(fmaf(x[g >> 1][8 * (g & 1) + j], ru[g], base));
                sum += pe;
                ph[g][j] = (_Float16)pe;
            }
            l = fmaf(sum, pow2(-de), l);
        }
        asm volatile("" : "+v"(l));  // summed here, not beside the products
    };

    // A wave has, in turn, the softmax of tile n, and the products P V of n and S of
    // n + 1 with its staging among them: waves 0-3 V's, 4-7 K's.  Of eight waves
    // the second four are half a tile behind, and then
    //   waves 0-3 have the softmax of n in turn 2n + 1 and the products in 2n + 2,
    //   waves 4-7 in turns 2n + 2 and 2n + 3;
    //   S reads K of n in turns 2n and 2n + 1, P V reads V of n in 2n + 2 and 2n + 3;
    //   turn 2n + 2 stages V of n + 1 over n - 1, read until 2n + 1;
    //   turn 2n + 3 stages K of n + 2 over n, read until 2n + 1, and what belongs to
    //   it over that of n - 2, which the softmax read until 2n - 2;
    // a barrier ends every turn.  Four waves have one turn a tile.  Tiles staged
    // past the last are never read.
    auto walk = [&](auto with_v, auto with_k) __attribute__((always_inline)) {
        constexpr bool V = decltype(with_v)::value, K = decltype(with_k)::value;
        if (V) {
            fetch(next_v, start(0));
            load(next_v, start(0), false);
            next_v.ok &= start(0) + 16 * group + n16 >= lo;  // only the first tile has tokens below lo
            each<kVPieces>([&](auto i) __attribute__((always_inline)) { v_piece(i, 0, start(1)); });
        }
        if (K) {
            fetch(next_k, start(0));
            load(next_k, start(0), true);
            next_k.ok &= start(0) + 16 * group + n16 >= lo;
            for (int n = 0; n < 2; n++)
                each<kKPieces>([&](auto i) __attribute__((always_inline)) { k_piece(i, n, start(n + 1)); });
        }
        lds_barrier();
        if (NW == 8 && K) lds_barrier();
        products(int_c<kNV>{}, int_c<kNV + kNS>{}, tile[0], tile[0], nothing);
        read_meta(0);
        lds_barrier();
        for (int n = 0; n + 1 < count; n++) {
            softmax(start(n));
            if (NW == 8) lds_barrier();
            __builtin_amdgcn_s_setprio(1);  // before the other group's softmax, which takes every slot
            products(int_c<0>{}, int_c<kNV + kNS>{}, tile[n & 1], tile[(n + 1) & 1], [&](auto at) __attribute__((always_inline)) {
                // The pieces evenly over the products.
                constexpr int P = decltype(at)::value, N = kNV + kNS, pieces = (V ? kVPieces : 0) + (K ? kKPieces : 0);
                constexpr int first = (P * pieces + N - 1) / N, end = ((P + 1) * pieces + N - 1) / N;
                static_assert(pieces <= N, "a piece a product");
                if constexpr (end > first) {
                    if constexpr (V && first < kVPieces) v_piece(int_c<first>{}, n + 1, start(n + 2));
                    else k_piece(int_c<first - (V ? kVPieces : 0)>{}, n + 2, start(n + 3));
                }
                if constexpr (P == N - 8) read_meta(n + 1);
            });
            __builtin_amdgcn_s_setprio(0);
            lds_barrier();
        }
        softmax(start(count - 1));
        if (NW == 8 && V) lds_barrier();  // as many as the waves behind
        products(int_c<0>{}, int_c<kNV>{}, tile[(count - 1) & 1], tile[0], nothing);
    };
    if (count > 0) {
        constexpr std::true_type yes;
        constexpr std::false_type no;
        if constexpr (NW == 4) walk(yes, yes);
        else if (wave < 4) walk(yes, no);
        else walk(no, yes);
    }

    l = add_x32(l);
    if (w0 + col >= rows) return;
    const bool split = unit_of.slot >= 0;
    const int64_t at = ((int64_t)kh * sp.slots + unit_of.slot) * (32 * NW) + 32 * wave + col;
    // O holds sum p v in units of 2^(kP + kM - 9 - vexp), l of 2^kP.
    const float unit = pow2(vexp + 9 - kM), share = split ? 1.0f / (1 << kP) : l != 0.0f ? 1.0f / l : 0.0f;
    if (split && h == 0) sp.ml[2 * at] = m, sp.ml[2 * at + 1] = l * (1.0f / (1 << kP));
    // Value n, j is of slot 32 n + 8 (j / 4) + 4 h + j % 4, so d = 4 (slot % (DP/4))
    // + slot / (DP/4): the four d of a slot % (DP/4) together.
#pragma unroll
    for (int k = 0; k < DP / 8; k++) {
        // the lane's k-th quad: dq over its 4 h + ... positions
        constexpr int Q = DP / 4;
        const int jj = k & 3, blk = k >> 2;  // position 8 blk + jj (+ 4 h) below Q
        const int dq = 8 * blk + jj + 4 * h;
        if (4 * dq >= D) continue;
        v4f y;
#pragma unroll
        for (int e4 = 0; e4 < 4; e4++) {
            const int slot = e4 * Q + 8 * blk + jj;  // less 4 h, which the lane's registers carry
            y[e4] = o[slot >> 5][4 * ((slot & 31) >> 3) + (slot & 3)] * share * unit;
        }
        if (split) {
            *(v4f*)(sp.o + at * D + 4 * dq) = y;
        } else {
            *(u2*)((uint16_t*)p.out + token * p.out_token + head * p.out_head + 4 * dq) =
                u2{f32x2_to_bf16x2(y[0], y[1]), f32x2_to_bf16x2(y[2], y[3])};
        }
    }
}

template <int DP, int NW>
static hipError_t launch_dp(hipStream_t stream, const KvCache& c, const PagedAttn& p, const AttnPart& s) {
    const dim3 grid((unsigned)s.blocks * (unsigned)c.heads), block(64 * NW);
    const bool page16 = tiles_of_16(c);
    const void* f = page16 ? (const void*)paged_chunk_kernel<DP, NW, true> : (const void*)paged_chunk_kernel<DP, NW, false>;
    const size_t lds = sizeof(ChunkLds<DP>);
    if (lds > 65536) {
        const hipError_t e = hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess) return e;
    }
    if (page16) hipLaunchKernelGGL((paged_chunk_kernel<DP, NW, true>), grid, block, lds, stream, c, p, s, p.table);
    else hipLaunchKernelGGL((paged_chunk_kernel<DP, NW, false>), grid, block, lds, stream, c, p, s, p.table);
    return hipGetLastError();
}

hipError_t launch_paged_chunk(hipStream_t stream, const KvCache& c, const PagedAttn& p, const AttnPart& s) {
    if (c.dim <= 64) return launch_dp<64, kChunkRows / 32>(stream, c, p, s);
    if (c.dim <= 128) return launch_dp<128, kChunkRows / 32>(stream, c, p, s);
    return launch_dp<256, kChunkRowsWide / 32>(stream, c, p, s);
}

}  // namespace phi_dev
