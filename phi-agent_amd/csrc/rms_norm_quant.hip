// Residual addition, root-mean-square norm and the linear's int8 operand:
//   r = x + residual,  y = r / sqrt(mean(r^2) + eps) * weight + shift,
//   (q, s) = rotate + quantise of y (quant_rotate.hip).
// One row a block, the row in LDS.
#include "decoder.hpp"
#include "device_common.hpp"

namespace phi_dev {

__device__ __forceinline__ float load_elem(const void* p, bool bf16, int64_t i) {
    return bf16 ? bf16_to_f32(((const uint16_t*)p)[i]) : ((const float*)p)[i];
}

__device__ __forceinline__ void store_elem(void* p, bool bf16, int64_t i, float v) {
    if (bf16) ((uint16_t*)p)[i] = (uint16_t)f32_to_bf16(v);
    else ((float*)p)[i] = v;
}

__global__ __launch_bounds__(256) void rms_norm_row_kernel(RmsNorm p) {
    extern __shared__ float row[];
    __shared__ float red[8];
    const int tid = threadIdx.x;
    const int64_t m = blockIdx.x;
    float sum = 0.0f;
    for (int k = tid; k < p.K; k += 256) {
        float r = load_elem(p.x, p.x_bf16, m * p.ldx + k);
        if (p.residual) r += load_elem(p.residual, p.r_bf16, m * p.ldr + k);
        if (p.residual_out) store_elem(p.residual_out, p.r_bf16, m * p.ldr + k, r);
        row[k] = r;
        sum = fmaf(r, r, sum);
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off, 64);
    if ((tid & 63) == 0) red[tid >> 6] = sum;
    __syncthreads();
    sum = (red[0] + red[1]) + (red[2] + red[3]);
    const float rstd = 1.0f / sqrtf(sum / (float)p.K + p.eps);
    for (int k = tid; k < p.K; k += 256) {
        float y = row[k] * rstd;
        if (p.weight) y *= load_elem(p.weight, p.w_bf16, k);
        if (p.shift) y += load_elem(p.shift, p.w_bf16, k);
        if (p.y) store_elem(p.y, p.y_bf16, m * p.ldy + k, y);
        row[k] = y;
    }
    if (p.rotate) {
        for (int st = 1; st < 256; st *= 4) {
            __syncthreads();
            for (int i = tid; i < p.K / 4; i += 256) {
                float* e = row + (i / 64) * 256 + ((i % 64) / st) * 4 * st + i % st;
                const float x0 = e[0], x1 = e[st], x2 = e[2 * st], x3 = e[3 * st];
                const float all = ((x0 + x1) + x2) + x3;
                e[0] = all - 2.0f * x3;
                e[st] = all - 2.0f * x2;
                e[2 * st] = all - 2.0f * x1;
                e[3 * st] = all - 2.0f * x0;
            }
        }
        __syncthreads();
        for (int k = tid; k < p.K; k += 256) row[k] *= 1.0f / 16.0f;
    }
    float amax = 0.0f;
    bool fine = __builtin_isfinite(rstd) && __builtin_isfinite(sum);
    for (int k = tid; k < p.K; k += 256) {
        amax = fmaxf(amax, fabsf(row[k]));
        fine &= __builtin_isfinite(row[k]);
    }
    amax = wave_max(fine ? amax : INFINITY);
    if ((tid & 63) == 0) red[4 + (tid >> 6)] = amax;
    __syncthreads();
    amax = fmaxf(fmaxf(red[4], red[5]), fmaxf(red[6], red[7]));
    fine = amax != INFINITY;
    const float scale = amax > 1e-30f ? amax / p.qmax : 1.0f, inv = 1.0f / scale;
    for (int k = tid; k < p.K; k += 256)
        p.q[m * p.ldq + k] = fine ? (int8_t)quant_code(row[k], inv, p.qmax, p.half_even) : 0;
    if (tid == 0) p.s[m] = fine ? scale : __builtin_nanf("");
}

hipError_t launch_rms_norm_quant(hipStream_t stream, const RmsNorm& p) {
    const size_t lds = (size_t)p.K * sizeof(float);
    const hipError_t e = hipFuncSetAttribute((const void*)rms_norm_row_kernel, hipFuncAttributeMaxDynamicSharedMemorySize,
                                             32768 * (int)sizeof(float));
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(rms_norm_row_kernel, dim3((unsigned)p.rows), dim3(256), lds, stream, p);
    return hipGetLastError();
}

}  // namespace phi_dev
