// Attention of chunks of new tokens over the paged int8 cache (bf16 queries).
//
// Bound by the matrix cores, and next by LDS reads and the softmax's vector
// work, all within a factor of 1.3 of each other, so each is kept small:
//   - A block holds 32 rows a wave (query heads of one key/value head x new
//     tokens, in that order, so that heads share the cache's tokens) and walks
//     the tokens in tiles of 64.  Q, O and the softmax stay in registers.
//   - K and V are made fp16 once a block: the tile's codes come to registers one
//     tile ahead, become code * scale * 2^E (E: a power of two for every 16
//     tokens, so that all of them use fp16's range) in one instruction a code,
//     and go to the other half of a double buffer in LDS in the order in
//     which the products read them, without bank conflicts.  A logit so has one
//     rounding to 11 bits for each k_d, at random sides; with q exact in fp16
//     (8 bits, scaled by a power of two) its error is some 2^-13 |s| / sqrt(dim).
//     int8 products, exact, cost the same on the matrix cores but three more
//     vector instructions for every logit (join, convert, scale).
//   - S^T = K Q^T and O^T = V^T P^T (v_mfma_f32_32x32x16_f16): the logits' layout
//     is already that of P's operand, as in paged_decode.hip.
//   - The running maximum moves only when a logit exceeds it by a factor of 2^kUp, and
//     masks are looked at only in tiles that a mask or the length cuts.
#include "paged_attention.hpp"

namespace phi_dev {

namespace {

constexpr int kTile = 64;  // tokens
constexpr int kGroups = kTile / 16;
// p enters fp16 as p 2^kP in the unit of its 16 tokens' V, and may reach 2^kUp
// before the running maximum moves: at most 2^15.  The rest of fp16's range lies
// below, so that weights keep their 11 bits down to 2^-28 of the row's largest
// and an absolute error of 2^-39 of it from there.
constexpr int kP = 14, kUp = 1;
constexpr int kMinExp = -100;  // of a group's unit: its inverse stays finite

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

// Two codes, biased by 128, that lie alone in the halves of u: code * f + 0 as
// fp16, the bias taken off in the same fma (f24 = f 2^24: the halves are
// subnormals (code + 128) 2^-24).
__device__ __forceinline__ h2 scale_pair(uint32_t u, float f24a, float fa, float f24b, float fb) {
    const h2 x = __builtin_bit_cast(h2, u);
    return h2{(_Float16)fmaf((float)x[0], f24a, -128.0f * fa), (_Float16)fmaf((float)x[1], f24b, -128.0f * fb)};
}

// max over a wave's lanes of a value >= 0, uniform.
__device__ __forceinline__ float wave_top(float v) {
#pragma unroll
    for (int off = 8; off > 0; off >>= 1) v = fmaxf(v, __shfl_xor(v, off, 64));
    return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(max_x16(max_x32(v)))));
}

// E of a group of scales: 2^E <= top < 2^(E+1), within [kMinExp, 127].
__device__ __forceinline__ int exp_of(float top) { return max(kMinExp, (int)(__float_as_uint(top) >> 23) - 127); }

// 2^e, |e| < 127.
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

}  // namespace

template <int DP> struct ChunkTile {
    _Float16 k[kTile * DP];  // rows of DP, 16-byte chunk n of row t in slot n ^ swizzle(t)
    _Float16 v[kTile * DP];  // [2 group + half][slot][8 tokens], slot = (d % 4) DP / 4 + d / 4
    float k_unit[kGroups];   // 2^(Ek - 7)
    int v_exp[kGroups];      // Ev
    uint32_t seen[kGroups];  // bit t: token t of the group is there
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
    ChunkTile<DP>* tile = (ChunkTile<DP>*)lds_raw;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 31, h = lane >> 5;
    const int heads = c.heads, D = c.dim;
    const int kh = blockIdx.x % heads;
    const AttnUnit unit_of = attn_unit<false>(p, sp, c.page, 32 * NW, blockIdx.x / heads);
    if (unit_of.b < 0) return;
    const int b = unit_of.b, z = unit_of.z;
    const SeqInfo s = seq_info(p, c.page, b);
    const int rows = min(s.n, p.max_q) * p.group, r0 = unit_of.tile * 32 * NW, z0 = z * sp.len;

    // The lane's row, and the ranges of the wave's rows and of the block's.
    const int w0 = r0 + 32 * wave;
    const int r = min(w0 + col, rows - 1), i = r / p.group, head = kh * p.group + (r - i * p.group);
    const int64_t token = s.first + i;
    const int pos = s.pos0 + i;
    const int row_hi = p.causal ? min(s.kv, pos + 1) : s.kv, row_lo = p.window > 0 ? max(0, pos + 1 - p.window) : 0;
    auto pos_of = [&](int row) { return s.pos0 + min(row, rows - 1) / p.group; };
    auto hi_of = [&](int ps) { return min(p.causal ? min(s.kv, ps + 1) : s.kv, z0 + sp.len); };
    auto lo_of = [&](int ps) { return max(p.window > 0 ? max(0, ps + 1 - p.window) : 0, z0); };
    const int hi = hi_of(pos_of(r0 + 32 * NW - 1)), lo = lo_of(pos_of(r0));
    const int wave_hi = w0 < rows ? hi_of(pos_of(w0 + 31)) : 0, wave_lo = lo_of(pos_of(w0));
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
        const float f = p.scale * 1.4426950408889634f, unit = pow2(min(e, 126)) * 0.0078125f;
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

    // ---- the tile's codes: wave w takes 16 tokens, V's or (four waves: and) K's ----
    const bool does_v = NW == 4 || wave < 4, does_k = NW == 4 || wave >= 4;
    const int group = wave & 3;
    const int32_t* trow = table + (int64_t)b * p.table_stride;
    const int last_page = page_of(c, max(hi - 1, 0));
    uint32_t vraw[NVI][8];
    float vsc[NVI][8];
    v4i kraw[NKI];
    float ksc[NKI], kvs[NKI];
    uint32_t vok = 0, kok = 0;  // bit n: item or token n of the above is there
    uint32_t there = 0;         // K's wave: the group's tokens, a bit each
    auto block_at = [&](int page, bool& ok) {
        const int blk = trow[min(page, last_page)];
        ok = blk >= 0 && blk < c.blocks;
        return (int64_t)(ok ? blk : 0);
    };
    const bool page4 = c.page % 4 == 0;

    // Codes and scales of a tile's group, not looked at before they are staged; a
    // token at hi or past it, or without a block, reads whatever lies in the last
    // page or block 0 and counts as scale 0.
    auto load = [&](int t0) {
        const int g0 = t0 + 16 * group;
        int64_t at = 0, sat = 0;
        bool gok = true;
        if (PAGE16) {
            const int t = min(g0, hi - 1), page = page_of(c, t), in = (t & ~15) - page * c.page;
            const int64_t blk = block_at(page, gok);
            at = blk * c.block_stride + kh * c.head_stride + (int64_t)in * c.token_stride;
            sat = blk * c.s_block_stride + kh * c.s_head_stride + in;
        }
        // Token n (0..15) of the group: its codes' offset, its scales', whether it is there.
        auto find = [&](int n, int64_t& a, int64_t& sa) {
            if (PAGE16) {
                a = at + (uint32_t)(n * (int)c.token_stride);
                sa = sat + n;
                return gok && g0 + n < hi;
            }
            const int t = min(g0 + n, hi - 1), page = page_of(c, t), in = t - page * c.page;
            bool ok;
            const int64_t blk = block_at(page, ok);
            a = blk * c.block_stride + kh * c.head_stride + in * c.token_stride;
            sa = blk * c.s_block_stride + kh * c.s_head_stride + in * c.s_token_stride;
            return ok && g0 + n < hi;
        };
        if (does_v) {
            vok = 0;
#pragma unroll
            for (int it = 0; it < NVI; it++) {
                const int item = (it * 64 + lane) % (DP / 2), ih = item / (DP / 4), dq = item % (DP / 4);
                const int d = 4 * dq < D ? 4 * dq : 0;
#pragma unroll
                for (int half = 0; half < 2; half++) {
                    int64_t a = 0, sa = 0;
                    bool ok = false;
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const int n = 8 * half + 4 * ih + j;
                        if (PAGE16 || !page4 || j == 0) {
                            ok = find(n, a, sa);
                        } else {  // in the block of the first of the four, if before hi
                            const bool on = g0 + n < hi;
                            a += on ? c.token_stride : 0;
                            sa += on ? c.s_token_stride : 0;
                            ok &= on;
                        }
                        vraw[it][4 * half + j] = *(const uint32_t*)(c.v + a + d);
                        vsc[it][4 * half + j] = c.vs[sa];
                        vok |= ok ? 1u << (8 * it + 4 * half + j) : 0u;
                    }
                }
            }
        }
        if (does_k) {
            int64_t a, sa;
            kok = 0;
            there = (uint32_t)__ballot(find(lane & 15, a, sa)) & 0xffffu;
#pragma unroll
            for (int it = 0; it < NKI; it++) {
                const int item = it * 64 + lane, n = item / (DP / 16), ch = item % (DP / 16);
                kok |= find(n, a, sa) ? 1u << it : 0u;
                kraw[it] = *(const v4i*)(c.k + a + (16 * ch < D ? 16 * ch : 0));
                ksc[it] = c.ks[sa];
                kvs[it] = c.vs[sa];
            }
        }
    };
    auto stage_v = [&](ChunkTile<DP>& to) {
        float top = 0.0f;
#pragma unroll
        for (int it = 0; it < NVI; it++)
#pragma unroll
            for (int j = 0; j < 8; j++) {
                vsc[it][j] = (vok >> (8 * it + j) & 1) && __builtin_isfinite(vsc[it][j]) ? vsc[it][j] : 0.0f;
                top = fmaxf(top, fabsf(vsc[it][j]));
            }
        const int e = exp_of(wave_top(top));
        if (lane == 0) to.v_exp[group] = e;
        const float unit = pow2(7 - e);
#pragma unroll
        for (int it = 0; it < NVI; it++) {
            const int item = (it * 64 + lane) % (DP / 2), ih = item / (DP / 4), dq = item % (DP / 4);
            float f[8], f24[8];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                f[j] = vsc[it][j] * unit;
                f24[j] = f[j] * 0x1p24f;
                vraw[it][j] ^= 0x80808080u;
            }
#pragma unroll
            for (int e4 = 0; e4 < 4; e4++) {
                const uint32_t sel = 0x0c000c00u | (uint32_t)((4 + e4) << 16) | (uint32_t)e4;
                h8 x;
#pragma unroll
                for (int j = 0; j < 8; j += 2) {
                    const h2 y = scale_pair(__builtin_amdgcn_perm(vraw[it][j + 1], vraw[it][j], sel), f24[j], f[j], f24[j + 1], f[j + 1]);
                    x[j] = y[0], x[j + 1] = y[1];
                }
                *(h8*)(to.v + (((2 * group + ih) * DP + e4 * (DP / 4) + dq) * 8)) = x;
            }
        }
    };
    auto stage_k = [&](ChunkTile<DP>& to) {
        float top = 0.0f;
#pragma unroll
        for (int it = 0; it < NKI; it++) {
            // A token whose value is not finite is NaN to the rows that see it.
            ksc[it] = !(kok >> it & 1) ? 0.0f : __builtin_isfinite(kvs[it]) ? ksc[it] : __builtin_nanf("");
            top = fmaxf(top, __builtin_isfinite(ksc[it]) ? fabsf(ksc[it]) : 0.0f);
        }
        const int e = exp_of(wave_top(top));
        if (lane == 0) to.k_unit[group] = pow2(e - 7), to.seen[group] = there;
        const float unit = pow2(7 - e);
#pragma unroll
        for (int it = 0; it < NKI; it++) {
            const int item = it * 64 + lane, n = item / (DP / 16), ch = item % (DP / 16), t = 16 * group + n;
            const float f = ksc[it] * unit, f24 = f * 0x1p24f;
            h8 x[2];
#pragma unroll
            for (int w = 0; w < 4; w++) {
                const uint32_t u = (uint32_t)kraw[it][w] ^ 0x80808080u;
                const h2 y0 = scale_pair(__builtin_amdgcn_perm(u, u, 0x0c010c00u), f24, f, f24, f);
                const h2 y1 = scale_pair(__builtin_amdgcn_perm(u, u, 0x0c030c02u), f24, f, f24, f);
                x[w >> 1][4 * (w & 1)] = y0[0], x[w >> 1][4 * (w & 1) + 1] = y0[1];
                x[w >> 1][4 * (w & 1) + 2] = y1[0], x[w >> 1][4 * (w & 1) + 3] = y1[1];
            }
#pragma unroll
            for (int m = 0; m < 2; m++) *(h8*)(to.k + t * DP + 8 * k_slot<DP>(t, 2 * ch + m)) = x[m];
        }
    };

    v16f o[OT];
#pragma unroll
    for (int n = 0; n < OT; n++)
#pragma unroll
        for (int j = 0; j < 16; j++) o[n][j] = 0.0f;
    float m = kNoMax, l = 0.0f;
    int vexp = kMinExp;

    auto compute = [&](const ChunkTile<DP>& ct, int t0) {
        v16f x[2];
#pragma unroll
        for (int u = 0; u < 2; u++) {
#pragma unroll
            for (int j = 0; j < 16; j++) x[u][j] = 0.0f;
            const int t = 32 * u + col;
#pragma unroll
            for (int ks = 0; ks < KS; ks++)
                x[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(*(const h8*)(ct.k + t * DP + 8 * k_slot<DP>(t, 2 * ks + h)), q[ks], x[u], 0, 0, 0);
        }
        float ru[kGroups];
        uint32_t holes = 0;
        int e = vexp;
#pragma unroll
        for (int g = 0; g < kGroups; g++) {
            ru[g] = rq * ct.k_unit[g];
            holes |= ct.seen[g] ^ 0xffffu;
            e = max(e, ct.v_exp[g]);
        }
        e = __builtin_amdgcn_readfirstlane(e);
        if (t0 < all_lo || t0 + kTile > all_hi || __builtin_amdgcn_readfirstlane(holes)) {
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
        if (__any(xm > m + (float)kUp) || e != vexp) {
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
        h8 ph[kGroups];
#pragma unroll
        for (int g = 0; g < kGroups; g++) {
            // p in units of 2^-kP and of the group's own power of two for sv.
            const int de = max(ct.v_exp[g] - vexp, kMinExp);
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
#pragma unroll
        for (int g = 0; g < kGroups; g++)
#pragma unroll
            for (int n = 0; n < OT; n++)
                o[n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(*(const h8*)(ct.v + ((2 * g + h) * DP + 32 * n + col) * 8), ph[g], o[n], 0, 0, 0);
    };

    // Tile n is computed from one buffer while n + 1 goes from registers to the
    // other and n + 2 comes to registers.  V's waves stage before they
    // compute and K's after, so that one kind's vector work lies beside the
    // other's products.
    const int begin = lo & ~(kTile - 1);
    if (begin < hi) {
        load(begin);
        if (does_v) stage_v(tile[0]);
        if (does_k) stage_k(tile[0]);
        if (begin + kTile < hi) load(begin + kTile);
        lds_barrier();
        int cur = 0;
        for (int t0 = begin; t0 < hi; t0 += kTile, cur ^= 1) {
            const bool next = t0 + kTile < hi, more = t0 + 2 * kTile < hi;
            if (next && does_v) stage_v(tile[cur ^ 1]);
            if (NW == 8 && does_v && more) load(t0 + 2 * kTile);
            if (t0 < wave_hi && t0 + kTile > wave_lo) compute(tile[cur], t0);
            if (next && does_k) stage_k(tile[cur ^ 1]);
            if ((NW == 4 || does_k) && more) load(t0 + 2 * kTile);
            lds_barrier();
        }
    }

    l = add_x32(l);
    if (w0 + col >= rows) return;
    const bool split = sp.count > 1;
    const int64_t at = z * sp.rows + token * p.q_heads + head;
    // O holds sum p v in units of 2^-(kP + 7 - vexp), l of 2^-kP.
    const float unit = pow2(max(-126, vexp - 7)) * (split ? 1.0f / (1 << kP) : l != 0.0f ? 1.0f / l : 0.0f);
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
            y[e4] = o[slot >> 5][4 * ((slot & 31) >> 3) + (slot & 3)] * unit;
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
    const size_t lds = 2 * sizeof(ChunkTile<DP>);
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
