// Residual addition, root-mean-square norm and the linear's int8 operand:
//   r = x + residual,  y = r / sqrt(mean(r^2) + eps) * weight + shift,
//   (q, s) = rotate + quantise of y (quant_rotate.hip).
//
// Bound by memory: 2 to 4 bytes of x, 4 to 8 of the residual stream and 1 of q an
// element, about 25 vector instructions.  So one pass: a lane holds 16 elements of a
// 256-group a round, a wave four groups a round, and the row stays in registers through both of its reductions (the sum of squares, a
// wave's by shuffles and the row's waves' through LDS; the largest |z| the same
// way).  The rotation is that of qr_tiles.hpp, on a 16 x 16 tile of LDS private to
// the group's 16 lanes, and so are the scale and the codes: q and s are to the
// bit what phi_hip_quant_rotate gives for y in fp32.
//
// Rows may start at any element: loads and stores are 16 bytes at the elements'
// own alignment (the hardware takes them unaligned; aligned ones are the same
// instructions).  4352 rows of 5120 in bf16 onto an fp32 stream: 54 us, 4.6 TB/s of
// the 4.9 that a copy reaches; 154 us with the row in LDS, an element a thread.  777 rows
// of 5003 in fp32 without the rotation: 15 us; 19 us with 16 consecutive elements a
// lane, whose four loads each touch every line.
#include "decoder.hpp"
#include "qr_tiles.hpp"

namespace phi_dev {

namespace {

typedef uint32_t u4a1 __attribute__((ext_vector_type(4), aligned(1)));
typedef uint32_t u2a2 __attribute__((ext_vector_type(2), aligned(2)));
typedef uint32_t u1a1 __attribute__((aligned(1)));
typedef uint32_t u4a2 __attribute__((ext_vector_type(4), aligned(2)));
typedef float f4a4 __attribute__((ext_vector_type(4), aligned(4)));

// A lane's 16 elements of a row: e0 .. e0 + 15 (ROT: the rotation wants them together,
// K is a multiple of 16) or, v[4 i + j], e0 + 64 i + j (the 16 lanes' loads are one
// piece; the row's last piece goes one by one).
template <bool ROT> __device__ __forceinline__ int at16(int e0, int j) { return e0 + (ROT ? j : 64 * (j / 4) + j % 4); }

// Of p's row at element offset `row`; 0 from K on.
template <bool ROT, bool BF16>
__device__ __forceinline__ void load_row16(const void* __restrict__ p, int64_t row, int e0, int K, float (&v)[16]) {
    const uint16_t* h = (const uint16_t*)p + row;
    const float* f = (const float*)p + row;
#pragma unroll
    for (int j = 0; j < 16; j++) v[j] = 0.0f;
    if (BF16 && ROT) {
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const u4a2 t = e0 < K ? *(const u4a2*)(h + e0 + 8 * i) : u4a2{0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < 4; j++) v[8 * i + 2 * j] = __uint_as_float(t[j] << 16), v[8 * i + 2 * j + 1] = __uint_as_float(t[j] & 0xffff0000u);
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int e = at16<ROT>(e0, 4 * i);
        if (ROT ? e0 < K : e + 4 <= K) {
            if (BF16) {
                const u2a2 t = *(const u2a2*)(h + e);
#pragma unroll
                for (int j = 0; j < 2; j++) v[4 * i + 2 * j] = __uint_as_float(t[j] << 16), v[4 * i + 2 * j + 1] = __uint_as_float(t[j] & 0xffff0000u);
            } else {
                const f4a4 t = *(const f4a4*)(f + e);
#pragma unroll
                for (int j = 0; j < 4; j++) v[4 * i + j] = t[j];
            }
        } else if (!ROT) {
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (e + j < K) v[4 * i + j] = BF16 ? bf16_to_f32(h[e + j]) : f[e + j];
        }
    }
}

template <bool ROT>
__device__ __forceinline__ void store_row16(void* p, bool bf16, int64_t row, int e0, int K, const float (&v)[16]) {
    uint16_t* h = (uint16_t*)p + row;
    float* f = (float*)p + row;
    if (bf16 && ROT) {
#pragma unroll
        for (int i = 0; i < 2; i++)
            if (e0 < K)
                *(u4a2*)(h + e0 + 8 * i) = u4a2{f32x2_to_bf16x2(v[8 * i], v[8 * i + 1]), f32x2_to_bf16x2(v[8 * i + 2], v[8 * i + 3]),
                                                f32x2_to_bf16x2(v[8 * i + 4], v[8 * i + 5]), f32x2_to_bf16x2(v[8 * i + 6], v[8 * i + 7])};
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int e = at16<ROT>(e0, 4 * i);
        if (ROT ? e0 < K : e + 4 <= K) {
            if (bf16) *(u2a2*)(h + e) = u2a2{f32x2_to_bf16x2(v[4 * i], v[4 * i + 1]), f32x2_to_bf16x2(v[4 * i + 2], v[4 * i + 3])};
            else *(f4a4*)(f + e) = f4a4{v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]};
        } else if (!ROT) {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if (e + j < K && bf16) h[e + j] = (uint16_t)f32_to_bf16(v[4 * i + j]);
                if (e + j < K && !bf16) f[e + j] = v[4 * i + j];
            }
        }
    }
}

enum ResKind { RES_NONE = 0, RES_BF16 = 1, RES_F32 = 2 };

}  // namespace

// R rounds of four groups a wave; a block has blockDim.y rows of blockDim.x / 64
// waves each.
template <bool XB, int RES, bool ROT, int R>
__global__ __launch_bounds__(1024) void rms_norm_quant_kernel(RmsNorm p) {
    extern __shared__ __align__(16) float lds[];
    const int lane = threadIdx.x & 63, wpr = blockDim.x >> 6;
    const int wr = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), ty = __builtin_amdgcn_readfirstlane(threadIdx.y);
    const int wave = ty * wpr + wr, waves = blockDim.y * wpr;
    float* sums = lds;                               // a wave's sum of squares
    uint32_t* tops = (uint32_t*)(lds + 16);          // a wave's largest |z|, bit 31: something is not finite
    const int team = lane >> 4, tl = lane & 15, sw = tl >> 2;
    float* T = lds + 32 + (ROT ? wave * QT_WAVE + team * QT_TILE : 0);
    float* trow = T + tl * 16;
    const int K = p.K;
    const int64_t row = (int64_t)blockIdx.x * blockDim.y + ty, rr = min(row, p.rows - 1);
    const bool live = row < p.rows;
    auto e0_of = [&](int r) { return (wr * 4 * R + team + 4 * r) * 256 + tl * (ROT ? 16 : 4); };

    float v[R][16], sum = 0.0f;
#pragma unroll
    for (int r = 0; r < R; r++) load_row16<ROT, XB>(p.x, rr * p.ldx, e0_of(r), K, v[r]);
    if (RES != RES_NONE) {
#pragma unroll
        for (int r = 0; r < R; r++) {
            float t[16];
            load_row16<ROT, RES == RES_BF16>(p.residual, rr * p.ldr, e0_of(r), K, t);
#pragma unroll
            for (int j = 0; j < 16; j++) v[r][j] += t[j];
        }
    }
#pragma unroll
    for (int r = 0; r < R; r++)
#pragma unroll
        for (int j = 0; j < 16; j++) sum = fmaf(v[r][j], v[r][j], sum);
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off, 64);
    if (wpr > 1) {
        if (lane == 0) sums[wave] = sum;
        __syncthreads();
        sum = 0.0f;
        for (int w = 0; w < wpr; w++) sum += sums[ty * wpr + w];
    }
    if (RES != RES_NONE && p.residual_out && live) {
#pragma unroll
        for (int r = 0; r < R; r++) store_row16<ROT>(p.residual_out, RES == RES_BF16, row * p.ldr, e0_of(r), K, v[r]);
    }
    // Past fp32 (or not a number): no norm, so that y is none either.
    const float rstd = __builtin_isfinite(sum) ? 1.0f / sqrtf(sum / (float)K + p.eps) : __builtin_nanf("");
    bool fine = __builtin_isfinite(sum) && __builtin_isfinite(rstd);
    uint32_t top = 0;
#pragma unroll
    for (int r = 0; r < R; r++) {
        const int e0 = e0_of(r);
#pragma unroll
        for (int j = 0; j < 16; j++) v[r][j] *= rstd;
        if (p.weight) {
            float t[16];
            if (p.w_bf16) load_row16<ROT, true>(p.weight, 0, e0, K, t);
            else load_row16<ROT, false>(p.weight, 0, e0, K, t);
#pragma unroll
            for (int j = 0; j < 16; j++) v[r][j] *= t[j];
        }
        if (p.shift) {
            float t[16];
            if (p.w_bf16) load_row16<ROT, true>(p.shift, 0, e0, K, t);
            else load_row16<ROT, false>(p.shift, 0, e0, K, t);
#pragma unroll
            for (int j = 0; j < 16; j++) v[r][j] += t[j];
        }
        if (p.y && live) store_row16<ROT>(p.y, p.y_bf16, row * p.ldy, e0, K, v[r]);
        float bad = 0.0f;
#pragma unroll
        for (int j = 0; j < 16; j++) bad = fmaf(v[r][j], 0.0f, bad);  // NaN once an infinity or a NaN is met
        if (ROT) {
            // Passes over the index's digits 0 and 1, the transpose, digits 2 and 3:
            // then v[r][j] is element 16 j + tl, before the final 1/16.
            bfly16f<1>(v[r]);
            bfly16f<4>(v[r]);
#pragma unroll
            for (int c = 0; c < 4; c++)
                *(float4*)(trow + 4 * (c ^ sw)) = make_float4(v[r][4 * c], v[r][4 * c + 1], v[r][4 * c + 2], v[r][4 * c + 3]);
            wave_lds_fence();
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const float* col = T + 64 * k + 4 * (sw ^ k) + (tl & 3);
#pragma unroll
                for (int i = 0; i < 4; i++) v[r][4 * k + i] = col[16 * i];
            }
            wave_lds_fence();
            bfly16f<1>(v[r]);
            bad += bfly16f_last(v[r]) * 0.0f;
        }
        fine &= __builtin_isfinite(bad);
        top = max(top, qt_amax16(v[r]));
    }
    top = wave_max_bits(top);
    top |= __all(fine) ? 0u : 0x80000000u;
    if (wpr > 1) {
        if (lane == 0) tops[wave] = top;
        __syncthreads();
        // Lane l reads wave l's word (at most 16 waves a block).
        const uint32_t e = tops[min(lane, waves - 1)];
        const bool mine = lane >= ty * wpr && lane < (ty + 1) * wpr;
        top = wave_max_bits(mine ? e & 0x7fffffffu : 0u);
        if (__builtin_amdgcn_ballot_w64(mine && e >> 31)) top |= 0x80000000u;
    }
    if (!live) return;
    const bool nan = top >> 31;
    if (wr == 0 && lane == 0 && nan) p.s[row] = __builtin_nanf("");
    // Fast where the fused butterflies are exact and no code needs a clamp
    // (qr_tiles.hpp); rows of 2^122 and more take the form with a clamp.
    const bool fast = ROT && __builtin_amdgcn_readfirstlane(top) < 0x7e800000u;
    const QtScale c = fast ? qt_scale_fast(top, p.qmax, 1.0f / p.qmax) : qt_scale(top & 0x7fffffffu, p.qmax, ROT);
    if (wr == 0 && lane == 0 && !nan) p.s[row] = c.scale;
#pragma unroll
    for (int r = 0; r < R; r++) {
        const int e0 = e0_of(r);
        float u[16];
        if (ROT) {
#pragma unroll
            for (int k = 0; k < 4; k++) {
                float* col = T + 64 * k + 4 * (sw ^ k) + (tl & 3);
#pragma unroll
                for (int i = 0; i < 4; i++) col[16 * i] = v[r][4 * k + i];
            }
            wave_lds_fence();
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const float4 t = *(const float4*)(trow + 4 * (k ^ sw));
                u[4 * k] = t.x, u[4 * k + 1] = t.y, u[4 * k + 2] = t.z, u[4 * k + 3] = t.w;
            }
            wave_lds_fence();
        } else {
#pragma unroll
            for (int j = 0; j < 16; j++) u[j] = v[r][j];
        }
        uint32_t packed[4] = {0, 0, 0, 0};
        if (!nan) {
#pragma unroll
            for (int k = 0; k < 4; k++) {
                float d[4];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float x = fast ? u[4 * k + j] : u[4 * k + j] * c.pre;
                    if (p.half_even) d[j] = fast ? pre_half_even_nc(x, c.post) : pre_half_even(x, c.post, p.qmax);
                    else d[j] = fast ? pre_half_away_nc(x, c.post) : pre_half_away(x, c.post, p.qmax);
                }
                packed[k] = cvt_pack4(d[0], d[1], d[2], d[3]);
            }
        }
        int8_t* dst = p.q + row * p.ldq;
        if (ROT) {
            if (e0 < K) *(u4a1*)(dst + e0) = u4a1{packed[0], packed[1], packed[2], packed[3]};
            continue;
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int e = at16<ROT>(e0, 4 * i);
            if (e + 4 <= K) *(u1a1*)(dst + e) = packed[i];
            else
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (e + j < K) dst[e + j] = (int8_t)(packed[i] >> 8 * j);
        }
    }
}

template <bool XB, int RES, bool ROT, int R>
static hipError_t launch_r(hipStream_t stream, const RmsNorm& p) {
    const int G = (p.K + 255) / 256, wpr = (G + 4 * R - 1) / (4 * R), rpb = wpr >= 4 ? 1 : 4 / wpr;
    const size_t lds = (32 + (ROT ? (size_t)rpb * wpr * QT_WAVE : 0)) * sizeof(float);
    if (lds > 65536) {
        const hipError_t e = hipFuncSetAttribute((const void*)rms_norm_quant_kernel<XB, RES, ROT, R>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess) return e;
    }
    hipLaunchKernelGGL((rms_norm_quant_kernel<XB, RES, ROT, R>), dim3((unsigned)((p.rows + rpb - 1) / rpb)),
                       dim3((unsigned)(64 * wpr), (unsigned)rpb), lds, stream, p);
    return hipGetLastError();
}

// Two rounds a wave only where one is more than a block's sixteen waves.
template <bool XB, int RES, bool ROT>
static hipError_t launch_k(hipStream_t stream, const RmsNorm& p) {
    return p.K <= 16384 ? launch_r<XB, RES, ROT, 1>(stream, p) : launch_r<XB, RES, ROT, 2>(stream, p);
}

template <bool XB, int RES>
static hipError_t launch_rot(hipStream_t stream, const RmsNorm& p) {
    return p.rotate ? launch_k<XB, RES, true>(stream, p) : launch_k<XB, RES, false>(stream, p);
}

template <bool XB>
static hipError_t launch_res(hipStream_t stream, const RmsNorm& p) {
    if (!p.residual) return launch_rot<XB, RES_NONE>(stream, p);
    return p.r_bf16 ? launch_rot<XB, RES_BF16>(stream, p) : launch_rot<XB, RES_F32>(stream, p);
}

hipError_t launch_rms_norm_quant(hipStream_t stream, const RmsNorm& p) {
    return p.x_bf16 ? launch_res<true>(stream, p) : launch_res<false>(stream, p);
}

}  // namespace phi_dev
