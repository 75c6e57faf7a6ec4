// Rotary positions, alone or with the write of k and v into the paged int8 cache.
//
// Bound by memory: every vector is read and written once.  A team of lanes has a
// vector, 8 pairs a lane; a wave's teams have consecutive tokens of one head, so that
// a page's codes and scales are written together (kv_cache.hip); a block's waves have
// neighbouring heads and go over the others with the same tokens, so that a pair's
// cosine and sine are computed once for all of a block's heads.
// 32760 tokens of 40 heads of 128: 118 us, 5.7 TB/s; 4352 tokens of 40 + 2 x 8 heads into
// the cache 27 us, 4 TB/s; 64 tokens 5 us, of which most is the launch and two loads in turn.
//
// The angle position * freq is wanted modulo a turn, to fp32 at any position.  With
// step = freq / 2 pi as a 64-bit fraction of a turn, to its nearest, position * step in 64-bit
// integers drops whole turns by itself and is exact for the step as it is; taken about the
// nearest quarter turn it is an angle within pi/4, for which Taylor's series to x^11 and x^12
// are within 2^-37.  In fp64, so that cosine and sine, scaled, are rounded once; 512 pairs a
// block cost no time that shows.
#include "device_common.hpp"
#include "serving.hpp"

namespace phi_dev {

namespace {

// freq / 2 pi modulo 1 as a 64-bit fraction, to the nearest: the product in two doubles, of
// which the first's whole turns are dropped and then 32 bits taken, all exactly.  (A product of
// one double has its last bit at 2^-53 of the step, and what is cut off goes one way.)
__device__ __forceinline__ uint64_t step_of(double freq) {
    constexpr double k1 = 0x1.45f306dc9c883p-3, k0 = -0x1.6b01ec5417056p-57;  // 1 / 2 pi
    const double hi = freq * k1, lo = fma(freq, k0, fma(freq, k1, -hi)), part = hi - rint(hi);
    const double top = rint((part + lo) * 0x1p32), rest = fma(part, 0x1p32, -top) + lo * 0x1p32;
    return ((uint64_t)(int64_t)top << 32) + (uint64_t)(int64_t)rint(rest * 0x1p32);
}

// scale times cosine and sine of position * freq, the nearest fp32.
__device__ __forceinline__ float2 turn_of(int64_t position, double freq, float scale) {
    const uint64_t at = step_of(freq) * (uint64_t)position + ((uint64_t)1 << 61);
    const double x = (double)((int64_t)(at & (((uint64_t)1 << 62) - 1)) - ((int64_t)1 << 61)) * 0x1.921fb54442d18p-62;  // 2 pi / 2^64
    const double y = x * x;
    double s = fma(y, fma(y, fma(y, fma(y, fma(y, -1.0 / 39916800, 1.0 / 362880), -1.0 / 5040), 1.0 / 120), -1.0 / 6), 1.0);
    s *= x;
    const double c = fma(y, fma(y, fma(y, fma(y, fma(y, fma(y, 1.0 / 479001600, -1.0 / 3628800), 1.0 / 40320), -1.0 / 720), 1.0 / 24), -0.5), 1.0);
    const int quarter = (int)(at >> 62);
    const double a = quarter & 1 ? s : c, b = quarter & 1 ? c : s;
    return make_float2((float)((quarter == 1 || quarter == 2 ? -a : a) * scale), (float)((quarter >= 2 ? -b : b) * scale));
}

// Where piece i of a lane's 8 / W pieces lies: W elements at a, W at b.
struct RotaryPiece {
    int a, b;
    bool turned, has_a, has_b;
};

// A lane's 16 elements as they lie in memory, 2 W of a piece together.
template <bool BF16, int W> constexpr int kRawWords = BF16 && W > 1 ? 8 : 16;

template <bool BF16, int W>
__device__ __forceinline__ void load_run(const void* base, int64_t at, uint32_t* w) {
    if (BF16) {
        const uint16_t* p = (const uint16_t*)base + at;
        if (W == 8) {
            const uint4 t = *(const uint4*)p;
            w[0] = t.x, w[1] = t.y, w[2] = t.z, w[3] = t.w;
        } else if (W == 4) {
            const uint2 t = *(const uint2*)p;
            w[0] = t.x, w[1] = t.y;
        } else {
            w[0] = *p;
        }
    } else {
        const uint32_t* p = (const uint32_t*)base + at;
        if (W == 1) {
            w[0] = *p;
        } else {
#pragma unroll
            for (int i = 0; i < W / 4; i++) {
                const uint4 t = *(const uint4*)(p + 4 * i);
                w[4 * i] = t.x, w[4 * i + 1] = t.y, w[4 * i + 2] = t.z, w[4 * i + 3] = t.w;
            }
        }
    }
}

template <bool BF16, int W>
__device__ __forceinline__ void store_run(void* base, int64_t at, const float* x) {
    if (BF16) {
        uint16_t* p = (uint16_t*)base + at;
        if (W == 8) *(uint4*)p = make_uint4(f32x2_to_bf16x2(x[0], x[1]), f32x2_to_bf16x2(x[2], x[3]), f32x2_to_bf16x2(x[4], x[5]), f32x2_to_bf16x2(x[6], x[7]));
        else if (W == 4) *(uint2*)p = make_uint2(f32x2_to_bf16x2(x[0], x[1]), f32x2_to_bf16x2(x[2], x[3]));
        else *p = (uint16_t)f32_to_bf16(x[0]);
    } else {
        float* p = (float*)base + at;
        if (W == 1) {
            *p = x[0];
        } else {
#pragma unroll
            for (int i = 0; i < W / 4; i++) *(float4*)(p + 4 * i) = make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
        }
    }
}

template <int W>
__device__ __forceinline__ void store_codes(int8_t* p, const float* x, float inv) {
    if (W == 1) {
        *p = (int8_t)quant_code(x[0], inv, 127.0f, 0);
    } else {
#pragma unroll
        for (int i = 0; i < W / 4; i++)
            ((uint32_t*)p)[i] = pack4(quant_code(x[4 * i], inv, 127.0f, 0), quant_code(x[4 * i + 1], inv, 127.0f, 0),
                                      quant_code(x[4 * i + 2], inv, 127.0f, 0), quant_code(x[4 * i + 3], inv, 127.0f, 0));
    }
}

}  // namespace

// W: elements an access (see rotary_width).  A block has the heads from part *
// per_part on of 64 >> lg tokens, `parts` blocks one group of tokens.
template <bool BF16, bool INTER, bool WRITE, int W>
__global__ __launch_bounds__(256) void rotary_kernel(Rotary p, KvCache c, int lg, int parts, int per_part) {
    constexpr int N = 8 / W, RW = kRawWords<BF16, W>;
    __shared__ float2 turns[512];  // [token][pair]: 64 >> lg tokens of at most 8 << lg pairs
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int tokens = 64 >> lg, half = p.rot >> 1;
    const int64_t group = blockIdx.x / parts, first = group * tokens;
    const int part = blockIdx.x - (int)group * parts;

    // At most two a thread, before a cache write side by side (past the last pair and token the
    // last again): 4352 tokens of 56 heads 35.0 us with the read back, one by one 36.3; without it
    // one by one: 32760 tokens of 40 heads 118 us, 122 side by side.
    constexpr int kTogether = WRITE ? 2 : 1;
    const int pairs = tokens * half;
#pragma unroll 1
    for (int i0 = threadIdx.x; i0 < pairs; i0 += 256 * kTogether) {
        int64_t position[kTogether];
        double freq[kTogether];
#pragma unroll
        for (int k = 0; k < kTogether; k++) {
            const int i = min(i0 + 256 * k, pairs - 1), t = i / half;
            position[k] = p.positions[min(first + t, p.tokens - 1)], freq[k] = p.freq[i - t * half];
        }
#pragma unroll
        for (int k = 0; k < kTogether; k++) turns[i0 + 256 * k] = turn_of(position[k], freq[k], p.scale);
    }
    __syncthreads();

    const int mine = lane >> lg, l = lane & ((1 << lg) - 1);
    const int64_t token = first + mine;
    const bool live = token < p.tokens;
    RotaryPiece at[N];
    float2 cs[8];
#pragma unroll
    for (int i = 0; i < N; i++) {
        const int pair = 8 * l + W * i;
        at[i].turned = pair < half;
        at[i].a = at[i].turned && !INTER ? pair : 2 * pair;
        at[i].b = at[i].turned && !INTER ? half + pair : 2 * pair + W;
        at[i].has_a = live && 2 * pair < p.dim;
        at[i].has_b = live && (W > 1 ? 2 * pair : 2 * pair + 1) < p.dim;
#pragma unroll
        for (int j = 0; j < W; j++) cs[W * i + j] = at[i].turned && live ? turns[mine * half + pair + j] : make_float2(1.0f, 0.0f);
    }
    bool keep = false;
    int64_t code = 0, scale_at = 0;
    if (WRITE && live) {
        const int64_t slot = p.slots[token];
        keep = slot >= 0 && slot < c.slots;
        const int64_t use = keep ? slot : 0, block = c.slots <= INT32_MAX ? page_of(c, (int)use) : use / c.page, in = use - block * c.page;
        code = block * c.block_stride + in * c.token_stride;
        scale_at = block * c.s_block_stride + in * c.s_token_stride;
    }

    const int heads = p.q.heads + (WRITE ? 2 * c.heads : 0), end = min(heads, (part + 1) * per_part);
    // U heads of a wave at a time, their loads together.
    constexpr int U = BF16 && W == 8 ? 4 : 2;
    for (int h0 = part * per_part + wave; h0 < end; h0 += 4 * U) {
        uint32_t w[U][RW];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int h = h0 + 4 * u;
            if (h >= end) break;
            const int kind = !WRITE || h < p.q.heads ? 0 : h < p.q.heads + c.heads ? 1 : 2;
            const RotaryHeads& s = kind == 0 ? p.q : kind == 1 ? p.k : p.v;
            const int head = kind == 0 ? h : kind == 1 ? h - p.q.heads : h - p.q.heads - c.heads;
            const int64_t from = token * s.in_token + head * s.in_head;
#pragma unroll
            for (int i = 0; i < N; i++) {
                constexpr int R = RW / N / 2;
                if (at[i].has_a) load_run<BF16, W>(s.in, from + at[i].a, &w[u][2 * R * i]);
                if (at[i].has_b) load_run<BF16, W>(s.in, from + at[i].b, &w[u][2 * R * i + R]);
            }
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int h = h0 + 4 * u;
            if (h >= end) break;
            const int kind = !WRITE || h < p.q.heads ? 0 : h < p.q.heads + c.heads ? 1 : 2;
            const int head = kind == 0 ? h : kind == 1 ? h - p.q.heads : h - p.q.heads - c.heads;
            float x[16];
#pragma unroll
            for (int e = 0; e < 16; e++) {
                if (!BF16) x[e] = __uint_as_float(w[u][e]);
                else if (W == 1) x[e] = bf16_to_f32(w[u][e]);
                else x[e] = bf16_to_f32(e & 1 ? w[u][e / 2 % RW] >> 16 : w[u][e / 2 % RW] & 0xffffu);
            }
            if (kind < 2) {
#pragma unroll
                for (int i = 0; i < N; i++)
#pragma unroll
                    for (int j = 0; j < W; j++) {
                        const int ea = 2 * W * i + (INTER ? 2 * j : j), eb = INTER ? ea + 1 : ea + W;
                        const float a = x[ea], b = x[eb], cos = cs[W * i + j].x, sin = cs[W * i + j].y;
                        x[ea] = at[i].turned ? fmaf(a, cos, -(b * sin)) : a;
                        x[eb] = at[i].turned ? fmaf(b, cos, a * sin) : b;
                    }
            }
            if (kind == 0) {
                const int64_t to = token * p.q.out_token + head * p.q.out_head;
#pragma unroll
                for (int i = 0; i < N; i++) {
                    if (at[i].has_a) store_run<BF16, W>(p.q.out, to + at[i].a, &x[2 * W * i]);
                    if (at[i].has_b) store_run<BF16, W>(p.q.out, to + at[i].b, &x[2 * W * i + W]);
                }
            } else if (WRITE) {
                // As kv_cache.hip quantises.
                float top = 0.0f, bad = 0.0f;
#pragma unroll
                for (int i = 0; i < N; i++)
#pragma unroll
                    for (int j = 0; j < 2 * W; j++) {
                        const float v = (j < W ? at[i].has_a : at[i].has_b) ? x[2 * W * i + j] : 0.0f;
                        top = fmaxf(top, fabsf(v));
                        bad = fmaf(v, 0.0f, bad);  // NaN once an infinity or a NaN is met
                    }
                for (int off = 1; off < 1 << lg; off <<= 1) {
                    top = fmaxf(top, __shfl_xor(top, off, 64));
                    bad += __shfl_xor(bad, off, 64);
                }
                if (!keep) continue;
                const bool fine = bad == 0.0f;
                const float sc = top > 1e-30f ? top / 127.0f : 1.0f, inv = fine ? 1.0f / sc : 0.0f;
                if (!fine) {
#pragma unroll
                    for (int e = 0; e < 16; e++) x[e] = 0.0f;
                }
                int8_t* to = (kind == 1 ? c.k : c.v) + code + head * c.head_stride;
#pragma unroll
                for (int i = 0; i < N; i++) {
                    if (at[i].has_a) store_codes<W>(to + at[i].a, &x[2 * W * i], inv);
                    if (at[i].has_b) store_codes<W>(to + at[i].b, &x[2 * W * i + W], inv);
                }
                if (l == 0) (kind == 1 ? c.ks : c.vs)[scale_at + head * c.s_head_stride] = fine ? sc : __builtin_nanf("");
            }
        }
    }
}

// Elements an access: 8 pairs of a lane are one run of 8 at each side where the
// halves and the rest are whole runs and rows lie at 16 bytes; runs of 4 the same; else
// one by one.
static int rotary_width(const Rotary& p) {
    const int e = p.bf16 ? 2 : 4;
    for (int w : {8, 4}) {
        const int64_t unit = w * e < 16 ? w * e : 16;
        bool ok = p.rot % (2 * w) == 0 && p.dim % (2 * w) == 0;
        for (const RotaryHeads* s : {&p.q, &p.k, &p.v}) {
            if (!s->heads) continue;
            ok = ok && (uintptr_t)s->in % unit == 0 && s->in_token * e % unit == 0 && s->in_head * e % unit == 0 &&
                 (uintptr_t)s->out % unit == 0 && s->out_token * e % unit == 0 && s->out_head * e % unit == 0;
        }
        if (ok) return w;
    }
    return 1;
}

template <bool BF16, bool INTER, bool WRITE>
static hipError_t launch(hipStream_t stream, const Rotary& p, const KvCache& c) {
    int lg = 0;
    while (16 << lg < p.dim) lg++;
    const int64_t groups = (p.tokens + (64 >> lg) - 1) >> (6 - lg);
    const int heads = p.q.heads + (WRITE ? 2 * c.heads : 0), most = (heads + 3) / 4;
    // Enough blocks for every compute unit to have sixteen; beyond, a block's heads share its
    // angles, for the cache all of them (16384 tokens of 56: 111 us, 154 in parts of 4), else 16,
    // a wave's four at a time (32760 tokens of 40: 120 us, 134 in one part, 124 in parts of 4).
    const int64_t want = (4096 + groups - 1) / groups;
    int per_part = 4 * ((most + (int)(want < most ? want : most) - 1) / (int)(want < most ? want : most));
    if (!WRITE && per_part > 16) per_part = 16;
    const int parts = (heads + per_part - 1) / per_part;
    const int64_t at_once = kMaxBlocks / parts << (6 - lg);  // tokens
    const int width = rotary_width(p);
    for (int64_t t = 0; t < p.tokens; t += at_once) {
        Rotary s = p;
        s.tokens = p.tokens - t < at_once ? p.tokens - t : at_once;
        for (RotaryHeads* h : {&s.q, &s.k, &s.v}) {
            h->in = (const char*)h->in + t * h->in_token * (BF16 ? 2 : 4);
            h->out = (char*)h->out + t * h->out_token * (BF16 ? 2 : 4);
        }
        s.positions += t;
        if (WRITE) s.slots += t;
        const dim3 grid((unsigned)(((s.tokens + (64 >> lg) - 1) >> (6 - lg)) * parts)), block(256);
        switch (width) {
            case 8: hipLaunchKernelGGL((rotary_kernel<BF16, INTER, WRITE, 8>), grid, block, 0, stream, s, c, lg, parts, per_part); break;
            case 4: hipLaunchKernelGGL((rotary_kernel<BF16, INTER, WRITE, 4>), grid, block, 0, stream, s, c, lg, parts, per_part); break;
            default: hipLaunchKernelGGL((rotary_kernel<BF16, INTER, WRITE, 1>), grid, block, 0, stream, s, c, lg, parts, per_part);
        }
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

hipError_t launch_rotary(hipStream_t stream, const Rotary& p, const KvCache& c) {
    const bool write = p.k.heads > 0;
    if (p.bf16) {
        if (p.interleaved) return write ? launch<true, true, true>(stream, p, c) : launch<true, true, false>(stream, p, c);
        return write ? launch<true, false, true>(stream, p, c) : launch<true, false, false>(stream, p, c);
    }
    if (p.interleaved) return write ? launch<false, true, true>(stream, p, c) : launch<false, true, false>(stream, p, c);
    return write ? launch<false, false, true>(stream, p, c) : launch<false, false, false>(stream, p, c);
}

}  // namespace phi_dev
