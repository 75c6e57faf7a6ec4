// Attention of a few rows over the paged int8 cache: single new tokens, or a
// handful, with the query heads that share a key/value head.
//
// Bound by the cache's one read.  A wave takes 32 tokens a step straight from
// memory in the order that the matrix instructions want them, with no LDS and
// no shuffles in the loop:
//   S^T = K Q^T (v_mfma_i32_16x16x64_i8): lane l holds K's token l & 15, bytes
//     16 (l >> 4) .. + 15 of each 64: one 16-byte load of the cache's row.  The
//     result has row l & 15 in the lane and tokens 4 (l >> 4) + i.
//   O^T = V^T P^T (v_mfma_f32_16x16x32_bf16): the sum's order is free, so k
//     index 8 g + j (g = l >> 4) stands for the token the lane's P is of: 4 g + j
//     of the step's first 16 tokens, 4 g + j - 4 of its second.  P is used where
//     it lies.  V^T wants 8 tokens of one d a lane: the lane loads dim/16
//     bytes of each of its 8 tokens' rows (16 lanes read a whole row) and takes
//     byte e of all eight for product e, so d = dim/16 (l & 15) + e.
// The next step's loads are under way while a step is computed, the table's entries
// for those two steps ahead: 32 tokens are 8 KB a wave at dim 128, and the two blocks
// a compute unit holds keep 64 KB in flight.  The four waves of a block take every
// fourth step of its split and join in LDS.
// 64 sequences of 4096 tokens, 32 heads over 8 of 128, pages of 16: 103 us with the
// join, 5.4 TB/s of the 6.2 that reading reaches; one step of one sequence 7.8 us,
// launch, three dependent loads and the join of the waves.  Loads two steps ahead
// are slower (one sequence of 777: 14.4 us against 13.7; 256 of 1024: 118 against 105),
// as are eight waves a block for one step (8.8 against 8.1).
#pragma once

#include "paged_attention.hpp"

namespace phi_dev {

constexpr int kWaves = 4;
constexpr int kStep = 32;  // tokens a wave and step

namespace {

template <int BYTES> struct VWord;
template <> struct VWord<4> { typedef uint32_t type __attribute__((ext_vector_type(1))); };
template <> struct VWord<8> { typedef uint32_t type __attribute__((ext_vector_type(2))); };
template <> struct VWord<16> { typedef uint32_t type __attribute__((ext_vector_type(4))); };

// One step's operands: two tiles of 16 tokens.
template <int DP> struct Step {
    v4i k[2][DP / 64];
    typename VWord<DP / 16>::type v[2][4];
    v4f sk[2], sv[2];
    bool ok[2][4];  // the table has a block for the token (PAGE16: of the tile)
};

// Byte n of w, signed, as fp32: one instruction in this form, two from a cast of a
// byte, which took 64 a step of 280 (one sequence of 777 tokens: 14.5 us to 13.4).
__device__ __forceinline__ float byte_f32(uint32_t w, int n) { return (float)((int32_t)(w << (24 - 8 * n)) >> 24); }

}  // namespace

template <int DP> struct DecodeLds {
    float o[kWaves][kDecodeRows][DP];
    float m[kWaves][kDecodeRows], l[kWaves][kDecodeRows];
};

// DP: dim rounded up to 64, 128 or 256.  F32: fp32 q and out, else bf16.
// PAGE16: tiles_of_16, so that a tile of 16 tokens has one block and its loads
// one scalar base; otherwise every token finds its own.
// Of block number `block`, in threads `tid` of 256.  PAIRED: two of them are one
// block, which has the same barriers whatever they do.
template <int DP, bool F32, bool PAGE16, bool SHARED, bool PAIRED>
__device__ __forceinline__ void paged_decode(KvCache c, PagedAttn p, AttnPart sp, const int32_t* __restrict__ table,
                                             DecodeLds<DP>& lds, int block, int tid) {
    constexpr int KS = DP / 64, EB = DP / 16, NT = q_terms<F32>, NP = F32 ? 3 : 2;
    auto& lo_ = lds.o;
    auto &lm = lds.m, &ll = lds.l;
    const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 15, g = lane >> 4;
    const int kh = block % c.heads;
    const AttnUnit unit = attn_unit<true, SHARED>(p, sp, c.page, block / c.heads);
    if (unit.b < 0) {
        if (PAIRED) __syncthreads(), __syncthreads();
        return;
    }
    const int b = unit.b, slot = unit.slot, z0 = unit.z0;
    const SeqInfo s = unit.s;
    const int rows = min(s.n, p.max_q) * p.group, r0 = unit.tile * kDecodeRows;
    const int D = c.dim;

    // The lane's row of the tile (past the last: the last again, not stored).
    const int r = min(r0 + col, rows - 1), i = r / p.group, head = kh * p.group + (r - i * p.group);
    const int64_t token = s.first + i;
    const int pos = s.pos0 + i;
    const int pos_first = s.pos0 + r0 / p.group, pos_last = s.pos0 + min(r0 + kDecodeRows - 1, rows - 1) / p.group;
    const int row_hi = p.causal ? min(s.kv, pos + 1) : s.kv, row_lo = p.window > 0 ? max(0, pos + 1 - p.window) : 0;
    // Tokens that some row of the tile sees, and that all of them see.
    const int hi = min(p.causal ? min(s.kv, pos_last + 1) : s.kv, unit.z1);
    const int lo = max(p.window > 0 ? max(0, pos_first + 1 - p.window) : 0, z0);
    const int all_hi = p.causal ? min(s.kv, pos_first + 1) : s.kv, all_lo = p.window > 0 ? max(0, pos_last + 1 - p.window) : 0;

    // A lane's bytes past dim read its row's first bytes again: Q is 0 there,
    // and O's columns past dim are not stored.
    const int vd = EB * col < D ? EB * col : 0;
    int kd[KS];
#pragma unroll
    for (int ks = 0; ks < KS; ks++) kd[ks] = 64 * ks + 16 * g < D ? 64 * ks + 16 * g : 0;
    const int32_t* trow = table_row<SHARED>(p, table, b);
    const int last_page = page_of(c, max(hi - 1, 0));

    // The table's entries of a step's tiles (a lane's token's), fetched a step
    // before its loads.
    int entry[2];
    auto fetch = [&](int t0) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < 2; j++) entry[j] = trow[min(page_of(c, min(t0 + 16 * j + (PAGE16 ? 0 : col), hi - 1)), last_page)];
    };
    // A lane's offsets in a tile's rows; kept opaque in the loop, so that they stay
    // 32-bit beside a scalar base.
    const int ts = (int)c.token_stride;
    uint32_t k_off[KS], v_off[4];
#pragma unroll
    for (int ks = 0; ks < KS; ks++) k_off[ks] = (PAGE16 ? col * ts : 0) + kd[ks];
#pragma unroll
    for (int n = 0; n < 4; n++) v_off[n] = (PAGE16 ? (4 * g + n) * ts : 0) + vd;
    // Loads of the step at t0, the next call's being of t0 + kStep * kWaves; tokens
    // at hi and past it read the last page's, or block 0's, whatever these hold.
    const int64_t s_head = kh * c.s_head_stride;
    auto load = [&](Step<DP>& st, int t0) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const int8_t* kb = c.k + kh * c.head_stride;
            const int8_t* vb = c.v + kh * c.head_stride;
            const bool ok = entry[j] >= 0 && entry[j] < c.blocks;
            const int64_t blk = ok ? entry[j] : 0;
            if (PAGE16) {
                const int t = min(t0 + 16 * j, hi - 1), in = (t & ~15) - page_of(c, t) * c.page;
                const uint64_t at = (uint64_t)(uint32_t)blk * (uint32_t)c.block_stride + (uint32_t)in * (uint32_t)ts;
                const int64_t sat = (int64_t)((uint64_t)(uint32_t)blk * (uint32_t)c.s_block_stride) + s_head + in;
                st.ok[j][0] = ok;
#pragma unroll
                for (int ks = 0; ks < KS; ks++) {
                    uint32_t off = k_off[ks];
                    asm("" : "+v"(off));
                    st.k[j][ks] = *(const v4i*)(kb + at + off);
                }
#pragma unroll
                for (int n = 0; n < 4; n++) {
                    uint32_t off = v_off[n];
                    asm("" : "+v"(off));
                    st.v[j][n] = *(const typename VWord<EB>::type*)(vb + at + off);
                }
                uint32_t off = 4 * g;
                asm("" : "+v"(off));
                st.sk[j] = *(const v4f*)(c.ks + sat + off);
                st.sv[j] = *(const v4f*)(c.vs + sat + off);
            } else {
                // Lane l has token l & 15; the others' are read from it.
                const int tk = min(t0 + 16 * j + col, hi - 1), in = tk - page_of(c, tk) * c.page;
                const int64_t at = blk * c.block_stride + in * c.token_stride;
                const int64_t sat = blk * c.s_block_stride + s_head + in * c.s_token_stride;
#pragma unroll
                for (int ks = 0; ks < KS; ks++) st.k[j][ks] = *(const v4i*)(kb + at + k_off[ks]);
#pragma unroll
                for (int n = 0; n < 4; n++) {
                    const int64_t av = __shfl(at, 4 * g + n, 64), as = __shfl(sat, 4 * g + n, 64);
                    st.ok[j][n] = __shfl((int)ok, 4 * g + n, 64);
                    st.v[j][n] = *(const typename VWord<EB>::type*)(vb + av + v_off[n]);
                    st.sk[j][n] = c.ks[as];
                    st.sv[j][n] = c.vs[as];
                }
            }
        }
        fetch(t0 + kStep * kWaves);
    };

    // The first step's loads are under way beside Q's (fp32: Q takes their registers).
    const int begin = (lo & ~(kStep - 1)) + kStep * wave, stride = kStep * kWaves;
    Step<DP> first;
    if (begin < hi) fetch(begin);
    Q16<F32> x[KS];
#pragma unroll
    for (int ks = 0; ks < KS; ks++) {
        const int d = 64 * ks + 16 * g;
        if (d < D) load_q16<F32>(p.q, token * p.q_token + head * p.q_head + d, x[ks]);
        else x[ks] = Q16<F32>{};
    }
    if (!F32 && begin < hi) load(first, begin);

    // Q's integer form in the B operand's order.
    v4i qt[KS][NT];
    float amax = 0.0f, bad = 0.0f;
#pragma unroll
    for (int ks = 0; ks < KS; ks++)
#pragma unroll
        for (int j = 0; j < 16; j++) {
            const float v = elem_q16<F32>(x[ks], j);
            amax = fmaxf(amax, fabsf(v));
            bad = fmaf(v, 0.0f, bad);  // NaN once an infinity or a NaN is met
        }
    amax = max_x16(max_x32(amax));
    bad = add_x16(add_x32(bad));
    const float f = p.scale * 1.4426950408889634f;
    float inv = 0.0f, rq = amax / q_steps<F32> * fabsf(f);
    if (amax > 1e-30f && rq > 0x1p-126f) inv = copysignf(q_steps<F32> / amax, f);
    else rq = 1.0f;  // every logit is 0
    rq += bad;
#pragma unroll
    for (int ks = 0; ks < KS; ks++) split_q16<F32>(x[ks], inv, qt[ks]);
    if (F32 && begin < hi) load(first, begin);

    v4f o[EB];
#pragma unroll
    for (int e = 0; e < EB; e++) o[e] = v4f{0, 0, 0, 0};
    float m = kNoMax, l = 0.0f;

    auto compute = [&](const Step<DP>& st, int t0) __attribute__((always_inline)) {
        float t[8], sv[8];
#pragma unroll
        for (int j = 0; j < 2; j++) {
            v4i acc[NT];
#pragma unroll
            for (int n = 0; n < NT; n++) {
                acc[n] = v4i{0, 0, 0, 0};
#pragma unroll
                for (int ks = 0; ks < KS; ks++) acc[n] = __builtin_amdgcn_mfma_i32_16x16x64_i8(st.k[j][ks], qt[ks][n], acc[n], 0, 0, 0);
            }
#pragma unroll
            for (int n = 0; n < 4; n++) {
                int a[NT];
#pragma unroll
                for (int k = 0; k < NT; k++) a[k] = acc[k][n];
                t[4 * j + n] = join_terms<F32>(a) * st.sk[j][n];
                sv[4 * j + n] = st.sv[j][n];
            }
        }
        bool ok = true;
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
            for (int n = 0; n < (PAGE16 ? 1 : 4); n++) ok &= st.ok[j][n];
        const bool whole = t0 >= all_lo && t0 + kStep <= min(all_hi, hi) && t0 >= lo && (PAGE16 ? ok : __all(ok));
        uint32_t seen = 0xff;
        if (!whole) {
            asm volatile("");  // keeps this a branch: 80 instructions that few steps need
            seen = 0;
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const int tok = t0 + 16 * (k >> 2) + 4 * g + (k & 3);
                const bool in = tok >= max(row_lo, lo) && tok < min(row_hi, hi) && st.ok[k >> 2][PAGE16 ? 0 : k & 3];
                seen |= in ? 1u << k : 0u;
                t[k] = in ? t[k] : -INFINITY;
                sv[k] = in ? sv[k] : 0.0f;
            }
        }
        float top = t[0];
#pragma unroll
        for (int k = 1; k < 8; k++) top = fmaxf(top, t[k]);
        const float xm = top * rq;
        if (__any(xm > m + kHead)) {
            const float m2 = fmaxf(m, max_x16(max_x32(xm)));
            const float keep = __builtin_amdgcn_exp2f(m - m2);
            m = m2;
            l *= keep;
#pragma unroll
            for (int e = 0; e < EB; e++) o[e] *= keep;
        }
        b8 pt[NP];  // p sv, highest bits first
#pragma unroll
        for (int k = 0; k < 8; k++) {
            const float e = __builtin_amdgcn_exp2f(fmaf(t[k], rq, -m));
            l += e;
            float x = whole || (seen >> k & 1) ? e * sv[k] : 0.0f;
#pragma unroll
            for (int n = 0; n < NP; n++) {
                pt[n][k] = (__bf16)x;
                x -= (float)pt[n][k];
            }
        }
        // Byte e of each token's word, as bf16 (a code's 7 bits are exact, so the
        // upper half of its fp32 is it).
#pragma unroll
        for (int e = 0; e < EB; e++) {
            v4i a;
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const float f0 = byte_f32(st.v[k >> 1][2 * (k & 1)][e / 4], e % 4);
                const float f1 = byte_f32(st.v[k >> 1][2 * (k & 1) + 1][e / 4], e % 4);
                a[k] = (int)__builtin_amdgcn_perm(__float_as_uint(f1), __float_as_uint(f0), 0x07060302u);
            }
#pragma unroll
            for (int n = 0; n < NP; n++) o[e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), pt[n], o[e], 0, 0, 0);
        }
    };

    // Two steps in registers, one loading.  Loads run ahead of hi - 1 at most by
    // being clamped to it.
    if (begin < hi) {
        Step<DP> second;
        for (int t0 = begin; t0 < hi; t0 += 2 * stride) {
            load(second, t0 + stride);
            compute(first, t0);
            if (t0 + stride >= hi) break;
            load(first, t0 + 2 * stride);
            compute(second, t0 + stride);
        }
    }

    // Join the four waves.  The largest m of a row decides; a wave without a
    // token has l = 0, o = 0.
    l = add_x16(add_x32(l));
    if (g == 0) lm[wave][col] = m, ll[wave][col] = l;
    __syncthreads();
    float top = lm[0][col];
#pragma unroll
    for (int w = 1; w < kWaves; w++) top = fmaxf(top, lm[w][col]);
    const float share = __builtin_amdgcn_exp2f(m - top);
#pragma unroll
    for (int n = 0; n < 4; n++)
#pragma unroll
        for (int e = 0; e < EB; e += 4)
            *(v4f*)&lo_[wave][col][EB * (4 * g + n) + e] =
                v4f{o[e][n] * share, o[e + 1][n] * share, o[e + 2][n] * share, o[e + 3][n] * share};
    __syncthreads();
    const int row = tid / 16, part = tid & 15;  // a row a team of 16
    if (r0 + row >= rows) return;
    const int ri = (r0 + row) / p.group, rhead = kh * p.group + (r0 + row - ri * p.group);
    const int64_t rtok = s.first + ri;
    float rm = lm[0][row];
#pragma unroll
    for (int w = 1; w < kWaves; w++) rm = fmaxf(rm, lm[w][row]);
    float rl = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; w++) rl = fmaf(ll[w][row], __builtin_amdgcn_exp2f(lm[w][row] - rm), rl);
    const int64_t at = ((int64_t)kh * sp.slots + slot) * kDecodeRows + row;
    const float div = slot >= 0 ? 1.0f : rl != 0.0f ? 1.0f / rl : 0.0f;
    if (slot >= 0 && part == 0) sp.ml[2 * at] = rm, sp.ml[2 * at + 1] = rl;
    if (SHARED && unit.last && kh == 0 && part == 0) leave_row(p, unit, r0 + row, row, false);
#pragma unroll
    for (int q4 = 0; q4 < DP / 64; q4++) {
        const int d = 4 * (part + 16 * q4);
        if (d >= D) break;
        v4f x = *(const v4f*)&lo_[0][row][d];
#pragma unroll
        for (int w = 1; w < kWaves; w++) x += *(const v4f*)&lo_[w][row][d];
        x *= div;
        if (slot >= 0) {
            *(v4f*)(sp.o + at * D + d) = x;
        } else {
            const int64_t to = rtok * p.out_token + rhead * p.out_head + d;
            if (F32) *(v4f*)((float*)p.out + to) = x;
            else *(uint2*)((uint16_t*)p.out + to) = make_uint2(f32x2_to_bf16x2(x[0], x[1]), f32x2_to_bf16x2(x[2], x[3]));
        }
    }
}

}  // namespace phi_dev
