// Low-rank adapters of many requests beside one linear:
//   out[m] = base[m] + scale[a] B[a] (A[a] x[m]),   a = adapter[m].
//
// Two passes, h = A[a] x[m] and the update.  A tile of 64 rows has its rows sorted
// into classes, those of one adapter; a block takes up to 32 rows of a class as the
// columns of its products, so that an adapter's factors are read once for all of a
// class's rows however they are mixed, and a row's values meet no other adapter's.
// Both operands come straight from memory in the order of the matrix instructions: a
// lane has 8 consecutive k of a row, which are one v_mfma_f32_16x16x32_bf16 or, in
// fp32, eight v_mfma_f32_16x16x4_f32 (k 8 g + e in the e-th, g = lane / 16, on both
// sides).
// h is fp32 throughout: against bf16 factors it enters the second product as three
// bf16, all of its 24 bits.
#include <algorithm>

#include "device_common.hpp"
#include "serving.hpp"

namespace phi_dev {

namespace {

typedef __bf16 b8 __attribute__((ext_vector_type(8)));

constexpr int kCols = 32;  // rows of x a block, two tiles of columns
constexpr int kSplits = 8;

// Unit u of a tile of 64 rows: up to kCols rows of one class, from the skip-th on.
struct LoraUnit {
    int adapter;  // below 0: none
    uint64_t rows;
    int skip, n;
};

__device__ __forceinline__ bool lora_unit(const LoraBatched& p, int tile, int u, LoraUnit& got) {
    const int row = tile * 64 + (threadIdx.x & 63);
    int a = row < p.rows ? p.adapter[row] : 0;
    a = a >= 0 && a < p.adapters ? a : -1;
    uint64_t left = __ballot(row < p.rows);
    while (left) {
        const int one = __builtin_amdgcn_readlane(a, __builtin_ctzll(left));
        const uint64_t mine = __ballot(a == one) & left;
        const int n = __popcll(mine), groups = (n + kCols - 1) / kCols;
        if (u < groups) {
            got = {one, mine, kCols * u, min(n - kCols * u, kCols)};
            return true;
        }
        u -= groups;
        left &= ~mine;
    }
    return false;
}

// The unit's rows, in LDS; every wave writes the same.
__device__ __forceinline__ void unit_rows(const LoraUnit& u, int tile, int* rows) {
    const int lane = threadIdx.x & 63;
    const int at = __popcll(u.rows & (((uint64_t)1 << lane) - 1)) - u.skip;
    if ((u.rows >> lane & 1) && at >= 0 && at < kCols) rows[at] = tile * 64 + lane;
}

// Eight elements k.. of a row of K, zeros past its end.  VEC: K % 8 == 0 and rows at
// 16 bytes.
template <bool B16> struct Eight {
    uint32_t w[B16 ? 4 : 8];
};
template <bool B16, bool VEC>
__device__ __forceinline__ Eight<B16> load_eight(const char* row, int k, int K) {
    Eight<B16> e;
    if (VEC) {
        const uint4* p = (const uint4*)(row + (size_t)(k < K ? k : 0) * (B16 ? 2 : 4));
#pragma unroll
        for (int i = 0; i < (B16 ? 1 : 2); i++) {
            const uint4 t = p[i];
            e.w[4 * i] = k < K ? t.x : 0, e.w[4 * i + 1] = k < K ? t.y : 0, e.w[4 * i + 2] = k < K ? t.z : 0, e.w[4 * i + 3] = k < K ? t.w : 0;
        }
        return e;
    }
    uint32_t t[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int at = k + i < K ? k + i : 0;
        const uint32_t v = B16 ? ((const uint16_t*)row)[at] : ((const uint32_t*)row)[at];
        t[i] = k + i < K ? v : 0;
    }
#pragma unroll
    for (int i = 0; i < (B16 ? 4 : 8); i++) e.w[i] = B16 ? t[2 * i] | t[2 * i + 1] << 16 : t[i];
    return e;
}
template <bool B16>
__device__ __forceinline__ float value(const Eight<B16>& e, int i) {
    return __uint_as_float(B16 ? i & 1 ? e.w[i >> 1] & 0xffff0000u : e.w[i >> 1] << 16 : e.w[i]);
}

template <bool AB, bool BB>
__device__ __forceinline__ v4f product(const Eight<AB>& a, const Eight<BB>& b, v4f c) {
    if constexpr (AB && BB) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(value(a, i), value(b, i), c, 0, 0, 0);
        return c;
    }
}

}  // namespace

// RT tiles of 16 ranks from 16 RT blockIdx.z on.
template <bool XB, bool WB, bool VEC, int RT>
__global__ __launch_bounds__(256) void lora_batched_down_kernel(LoraBatched p, int tiles) {
    constexpr int P = 16 * RT + 4;
    __shared__ int rows[kCols];
    __shared__ float part[4][kCols][P];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int tile = blockIdx.x % tiles, split = blockIdx.y, r0 = 16 * RT * blockIdx.z;
    LoraUnit u;
    if (!lora_unit(p, tile, blockIdx.x / tiles, u) || u.adapter < 0) return;
    unit_rows(u, tile, rows);
    __syncthreads();
    const int col = lane & 15, g = lane >> 4;
    const char* xs[2];
    const char* as[RT];
#pragma unroll
    for (int c = 0; c < 2; c++) xs[c] = (const char*)p.x + (int64_t)rows[min(16 * c + col, u.n - 1)] * p.ldx * (XB ? 2 : 4);
#pragma unroll
    for (int r = 0; r < RT; r++)
        as[r] = (const char*)p.A + (u.adapter * p.a_adapter + min(r0 + 16 * r + col, p.R - 1) * p.a_row) * (WB ? 2 : 4);
    const int steps = (p.K + 31) / 32, parts = 4 * p.splits, me = 4 * split + wave;
    const int s0 = (int)((int64_t)steps * me / parts), s1 = (int)((int64_t)steps * (me + 1) / parts);
    const bool two = u.n > 16;
    v4f acc[2][RT];
#pragma unroll
    for (int c = 0; c < 2; c++)
#pragma unroll
        for (int r = 0; r < RT; r++) acc[c][r] = v4f{0, 0, 0, 0};
    for (int s = s0; s < s1; s++) {
        const int k = 32 * s + 8 * g;
        Eight<XB> x[2];
        Eight<WB> a[RT];
        x[0] = load_eight<XB, VEC>(xs[0], k, p.K);
        if (two) x[1] = load_eight<XB, VEC>(xs[1], k, p.K);
#pragma unroll
        for (int r = 0; r < RT; r++) a[r] = load_eight<WB, VEC>(as[r], k, p.K);
#pragma unroll
        for (int r = 0; r < RT; r++) acc[0][r] = product(a[r], x[0], acc[0][r]);
        if (two) {
#pragma unroll
            for (int r = 0; r < RT; r++) acc[1][r] = product(a[r], x[1], acc[1][r]);
        }
    }
#pragma unroll
    for (int c = 0; c < 2; c++)
#pragma unroll
        for (int r = 0; r < RT; r++) *(v4f*)&part[wave][16 * c + col][16 * r + 4 * g] = acc[c][r];
    __syncthreads();
    for (int i = threadIdx.x; i < u.n * 4 * RT; i += 256) {
        const int c = i / (4 * RT), r = 4 * (i % (4 * RT));
        if (r0 + r >= p.rank_pitch) continue;
        v4f sum = *(const v4f*)&part[0][c][r];
#pragma unroll
        for (int w = 1; w < 4; w++) sum += *(const v4f*)&part[w][c][r];
        *(v4f*)(p.h + ((int64_t)split * p.rows + rows[c]) * p.rank_pitch + r0 + r) = sum;
    }
}

// A wave has 64 columns n of out, as four tiles of the matrix instruction whose rows
// are so chosen that a lane's results are 16 consecutive n: row r of tile t stands
// for n = 16 (r / 4) + 4 t + r % 4.  A block has 256 `chunks` columns.
template <bool WB, bool OB, bool VECB, bool VECO>
__global__ __launch_bounds__(256) void lora_batched_up_kernel(LoraBatched p, int tiles, int chunks) {
    constexpr int T = WB ? 3 : 1;  // terms of h
    __shared__ int rows[kCols];
    extern __shared__ __align__(16) uint8_t lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int tile = blockIdx.x % tiles;
    LoraUnit u;
    if (!lora_unit(p, tile, blockIdx.x / tiles, u)) return;
    const bool some = u.adapter >= 0;
    if (!some && p.out == p.base) return;
    unit_rows(u, tile, rows);
    __syncthreads();
    const int ranks = (p.R + 31) / 32 * 32, pitch = ranks + (WB ? 8 : 4);
    uint16_t* hb = (uint16_t*)lds;  // [term][column][pitch]
    float* hf = (float*)lds;        // [column][pitch]
    const int col = lane & 15, g = lane >> 4;
    if (some) {
        const float scale = p.scale ? p.scale[u.adapter] : 1.0f;
        for (int i = threadIdx.x; i < kCols * ranks / 4; i += 256) {
            const int c = i / (ranks / 4), r = 4 * (i - c * (ranks / 4));
            v4f sum = {0, 0, 0, 0};
            if (c < u.n && r < p.R) {
                const float* from = p.h + (int64_t)rows[c] * p.rank_pitch + r;
                for (int s = 0; s < p.splits; s++) sum += *(const v4f*)(from + (int64_t)s * p.rows * p.rank_pitch);
#pragma unroll
                for (int e = 0; e < 4; e++) sum[e] = r + e < p.R ? sum[e] * scale : 0.0f;
            }
            if constexpr (WB) {
#pragma unroll
                for (int t = 0; t < T; t++) {
                    const uint32_t lo = f32x2_to_bf16x2(sum[0], sum[1]), hi = f32x2_to_bf16x2(sum[2], sum[3]);
                    *(uint2*)(hb + (t * kCols + c) * pitch + r) = make_uint2(lo, hi);
                    // What an infinity leaves is 0, not NaN.
                    const float y[4] = {bf16_to_f32(lo & 0xffffu), bf16_to_f32(lo >> 16), bf16_to_f32(hi & 0xffffu), bf16_to_f32(hi >> 16)};
#pragma unroll
                    for (int e = 0; e < 4; e++) sum[e] = __builtin_isfinite(y[e]) ? sum[e] - y[e] : 0.0f;
                }
            } else {
                *(v4f*)(hf + c * pitch + r) = sum;
            }
        }
        __syncthreads();
    }
    const int tiles_n = u.n > 16 ? 2 : 1;
    for (int chunk = 0; chunk < chunks; chunk++) {
        const int n0 = (blockIdx.y * chunks + chunk) * 256 + 64 * wave;
        if (n0 >= p.N) break;
        v4f acc[2][4];
#pragma unroll
        for (int c = 0; c < 2; c++)
#pragma unroll
            for (int t = 0; t < 4; t++) acc[c][t] = v4f{0, 0, 0, 0};
        if (some) {
            const char* bs[4];
#pragma unroll
            for (int t = 0; t < 4; t++)
                bs[t] = (const char*)p.B + (u.adapter * p.b_adapter + min(n0 + 16 * (col >> 2) + 4 * t + (col & 3), p.N - 1) * p.b_row) * (WB ? 2 : 4);
            for (int k0 = 0; k0 < ranks; k0 += 32) {
                const int k = k0 + 8 * g;
                Eight<WB> b[4];
#pragma unroll
                for (int t = 0; t < 4; t++) b[t] = load_eight<WB, VECB>(bs[t], k, p.R);
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    if (c >= tiles_n) break;
#pragma unroll
                    for (int term = T - 1; term >= 0; term--) {
                        Eight<WB> h;
                        if (WB) {
                            *(uint4*)h.w = *(const uint4*)(hb + (term * kCols + 16 * c + col) * pitch + k);
                        } else {
                            *(v4f*)h.w = *(const v4f*)(hf + (16 * c + col) * pitch + k);
                            *(v4f*)(h.w + (WB ? 0 : 4)) = *(const v4f*)(hf + (16 * c + col) * pitch + k + 4);
                        }
#pragma unroll
                        for (int t = 0; t < 4; t++) acc[c][t] = product(b[t], h, acc[c][t]);
                    }
                }
            }
        }
#pragma unroll
        for (int c = 0; c < 2; c++) {
            if (16 * c + col >= u.n) continue;
            const int64_t row = rows[16 * c + col];
            const int n = n0 + 16 * g;
            if (n >= p.N) continue;
            const int64_t to = row * p.ldo + n, from = row * p.ld_base + n;
            float y[16];
#pragma unroll
            for (int j = 0; j < 16; j++) y[j] = acc[c][j >> 2][j & 3];
            if (VECO) {
                if (p.base) {
                    const uint4* b = OB ? (const uint4*)((const uint16_t*)p.base + from) : (const uint4*)((const float*)p.base + from);
#pragma unroll
                    for (int i = 0; i < (OB ? 2 : 4); i++) {
                        const uint4 v = b[i];
                        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            if (OB) y[8 * i + 2 * j] += bf16_to_f32(w[j] & 0xffffu), y[8 * i + 2 * j + 1] += bf16_to_f32(w[j] >> 16);
                            else y[4 * i + j] += __uint_as_float(w[j]);
                        }
                    }
                }
#pragma unroll
                for (int i = 0; i < (OB ? 2 : 4); i++) {
                    if (OB) *((uint4*)((uint16_t*)p.out + to) + i) = make_uint4(f32x2_to_bf16x2(y[8 * i], y[8 * i + 1]), f32x2_to_bf16x2(y[8 * i + 2], y[8 * i + 3]), f32x2_to_bf16x2(y[8 * i + 4], y[8 * i + 5]), f32x2_to_bf16x2(y[8 * i + 6], y[8 * i + 7]));
                    else *(float4*)((float*)p.out + to + 4 * i) = make_float4(y[4 * i], y[4 * i + 1], y[4 * i + 2], y[4 * i + 3]);
                }
            } else {
#pragma unroll
                for (int j = 0; j < 16; j++) {
                    if (n + j >= p.N) break;
                    if (p.base) y[j] += OB ? bf16_to_f32(((const uint16_t*)p.base)[from + j]) : ((const float*)p.base)[from + j];
                    if (OB) ((uint16_t*)p.out)[to + j] = (uint16_t)f32_to_bf16(y[j]);
                    else ((float*)p.out)[to + j] = y[j];
                }
            }
        }
    }
}

namespace {

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

int rank_pitch(int64_t R) { return (int)(16 * ceil_div(R, 16)); }

// Parts of K: enough blocks where there are few rows, a part no shorter than 16 steps of 32.
int splits_of(int64_t rows, int64_t K) {
    return (int)std::clamp<int64_t>(512 / ceil_div(rows, kCols), 1, std::min<int64_t>(kSplits, ceil_div(K, 512)));
}

bool at16(const void* p, int64_t bytes1, int64_t bytes2 = 0) { return (uintptr_t)p % 16 == 0 && bytes1 % 16 == 0 && bytes2 % 16 == 0; }

template <bool XB, bool WB, bool VEC>
void down(hipStream_t stream, const LoraBatched& p, int tiles, int units) {
    const int rt = (p.R + 15) / 16;
    const dim3 block(256);
    auto grid = [&](int RT) { return dim3((unsigned)(tiles * units), (unsigned)p.splits, (unsigned)((rt + RT - 1) / RT)); };
    if (rt == 1) hipLaunchKernelGGL((lora_batched_down_kernel<XB, WB, VEC, 1>), grid(1), block, 0, stream, p, tiles);
    else if (rt == 2) hipLaunchKernelGGL((lora_batched_down_kernel<XB, WB, VEC, 2>), grid(2), block, 0, stream, p, tiles);
    else hipLaunchKernelGGL((lora_batched_down_kernel<XB, WB, VEC, 4>), grid(4), block, 0, stream, p, tiles);
}

template <bool WB, bool OB>
void up(hipStream_t stream, const LoraBatched& p, int tiles, int units, bool vec_b, bool vec_o) {
    const int ranks = (p.R + 31) / 32 * 32, all = (p.N + 255) / 256;
    const size_t lds = WB ? 3 * kCols * (ranks + 8) * 2 : kCols * (ranks + 4) * 4;
    const int want = (int)std::max<int64_t>(1, 2048 / ceil_div(p.rows, kCols));
    const int chunks = (all + std::min(want, all) - 1) / std::min(want, all);
    const dim3 grid((unsigned)(tiles * units), (unsigned)((all + chunks - 1) / chunks)), block(256);
    if (vec_b && vec_o) hipLaunchKernelGGL((lora_batched_up_kernel<WB, OB, true, true>), grid, block, lds, stream, p, tiles, chunks);
    else if (vec_b) hipLaunchKernelGGL((lora_batched_up_kernel<WB, OB, true, false>), grid, block, lds, stream, p, tiles, chunks);
    else if (vec_o) hipLaunchKernelGGL((lora_batched_up_kernel<WB, OB, false, true>), grid, block, lds, stream, p, tiles, chunks);
    else hipLaunchKernelGGL((lora_batched_up_kernel<WB, OB, false, false>), grid, block, lds, stream, p, tiles, chunks);
}

}  // namespace

size_t lora_batched_workspace(int64_t rows, int64_t K, int64_t R) {
    return (size_t)splits_of(rows, K) * rows * rank_pitch(R) * sizeof(float);
}

hipError_t launch_lora_batched(hipStream_t stream, LoraBatched p) {
    p.splits = splits_of(p.rows, p.K);
    p.rank_pitch = rank_pitch(p.R);
    const int tiles = (p.rows + 63) / 64;
    // Units of a tile, at most: a class each, and one more where a class has more than kCols rows.
    const int units = std::min(std::min(64, p.adapters + 1) + 1, 64);
    const int xe = p.x_bf16 ? 2 : 4, we = p.w_bf16 ? 2 : 4, oe = p.out_bf16 ? 2 : 4;
    const bool vec = p.K % 8 == 0 && at16(p.x, p.ldx * xe) && at16(p.A, p.a_row * we, p.a_adapter * we);
    if (p.x_bf16 && p.w_bf16) vec ? down<true, true, true>(stream, p, tiles, units) : down<true, true, false>(stream, p, tiles, units);
    else if (p.x_bf16) vec ? down<true, false, true>(stream, p, tiles, units) : down<true, false, false>(stream, p, tiles, units);
    else if (p.w_bf16) vec ? down<false, true, true>(stream, p, tiles, units) : down<false, true, false>(stream, p, tiles, units);
    else vec ? down<false, false, true>(stream, p, tiles, units) : down<false, false, false>(stream, p, tiles, units);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const bool vec_b = p.R % 8 == 0 && at16(p.B, p.b_row * we, p.b_adapter * we);
    const bool vec_o = p.N % 16 == 0 && at16(p.out, p.ldo * oe) && (!p.base || at16(p.base, p.ld_base * oe));
    if (p.w_bf16) p.out_bf16 ? up<true, true>(stream, p, tiles, units, vec_b, vec_o) : up<true, false>(stream, p, tiles, units, vec_b, vec_o);
    else p.out_bf16 ? up<false, true>(stream, p, tiles, units, vec_b, vec_o) : up<false, false>(stream, p, tiles, units, vec_b, vec_o);
    return hipGetLastError();
}

}  // namespace phi_dev
