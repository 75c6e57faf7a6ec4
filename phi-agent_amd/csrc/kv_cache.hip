// The int8 paged key/value cache: new tokens' vectors quantised as they are
// written (one scale a token and head, the linear's quantiser without its
// rotation), and slots read back as values.
//
// Bound by memory.  A team of lanes has a vector, 16 elements a lane in pieces of 16
// bytes, each piece of all lanes together; the largest |x| by shuffles within the
// team.  A wave's teams have consecutive tokens of a head, whose codes and scales lie
// together in a page; consecutive waves have the heads of k, then of v, whose
// elements lie together in the projection's output.  32760 tokens of 8 heads of 128 in
// bf16: 49 us for the write (4.1 TB/s, of 4.9 that a copy reaches) and 37 for the read
// (5.5).  With a token's k and v in one team, 56 and 37; with all tokens of one head
// before the next head's, so that elements are read in pieces of 256 bytes, 64 and 34;
// with an element a lane and a wave a vector, 189 and 139.
#include "decoder.hpp"
#include "device_common.hpp"

namespace phi_dev {

namespace {

// What a lane works on: `lanes` (a power of two) lanes a vector, the first
// dim / 16 of them with 16 elements each.
struct KvLane {
    bool live, has;  // the slot is one of the cache; the lane has elements
    bool v;
    int lane;        // of the team
    int64_t elem;    // offset of the vector's elements
    int64_t code, scale;  // offsets of its codes and of its scale
};

// Where piece i of a lane's N / 4 pieces (four elements each, N together) lies in the vector.
template <int N> __device__ __forceinline__ int piece(const KvCache& c, int l, int i) {
    return N * l + (4 * i) % N + (4 * i) / N * (c.dim * N / 16);
}

__device__ __forceinline__ bool kv_lane(const KvCache& c, const KvTokens& t, int lg, KvLane& l) {
    const int64_t wave = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), group = wave / (2 * c.heads);
    const int which = (int)(wave - group * 2 * c.heads), head = which % c.heads;
    const int64_t at = (group << (6 - lg)) + ((threadIdx.x & 63) >> lg);
    if (at >= t.tokens) return false;
    l.v = which >= c.heads;
    l.lane = threadIdx.x & ((1 << lg) - 1);
    l.has = 16 * l.lane < c.dim;
    const int64_t slot = t.slots[at];
    l.live = slot >= 0 && slot < c.slots;
    l.elem = at * (l.v ? t.v_token : t.k_token) + head * (l.v ? t.v_head : t.k_head);
    const int64_t use = l.live ? slot : 0;
    const int64_t block = c.slots <= INT32_MAX ? page_of(c, (int)use) : use / c.page, in = use - block * c.page;
    l.code = block * c.block_stride + head * c.head_stride + in * c.token_stride;
    l.scale = block * c.s_block_stride + head * c.s_head_stride + in * c.s_token_stride;
    return true;
}

}  // namespace

template <bool BF16>
__global__ __launch_bounds__(256) void kv_write_kernel(KvCache c, KvTokens t, int lg) {
    KvLane l;
    if (!kv_lane(c, t, lg, l)) return;
    float x[16], top = 0.0f, bad = 0.0f;
    const void* src = l.v ? t.v : t.k;
    if (l.has && l.live) {
        if (BF16) {
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const uint4 a = *(const uint4*)((const uint16_t*)src + l.elem + piece<8>(c, l.lane, 2 * i));
                const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
                for (int j = 0; j < 4; j++) x[8 * i + 2 * j] = bf16_to_f32(w[j] & 0xffffu), x[8 * i + 2 * j + 1] = bf16_to_f32(w[j] >> 16);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float4 a = *(const float4*)((const float*)src + l.elem + piece<4>(c, l.lane, i));
                x[4 * i] = a.x, x[4 * i + 1] = a.y, x[4 * i + 2] = a.z, x[4 * i + 3] = a.w;
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < 16; j++) x[j] = 0.0f;
    }
#pragma unroll
    for (int j = 0; j < 16; j++) {
        top = fmaxf(top, fabsf(x[j]));
        bad = fmaf(x[j], 0.0f, bad);  // NaN once an infinity or a NaN is met
    }
    for (int off = 1; off < 1 << lg; off <<= 1) {
        top = fmaxf(top, __shfl_xor(top, off, 64));
        bad += __shfl_xor(bad, off, 64);
    }
    if (!l.live || !l.has) return;
    const bool fine = bad == 0.0f;
    const float scale = top > 1e-30f ? top / 127.0f : 1.0f, inv = 1.0f / scale;
    uint32_t w[4] = {0, 0, 0, 0};
    if (fine) {
#pragma unroll
        for (int i = 0; i < 4; i++)
            w[i] = pack4(quant_code(x[4 * i], inv, 127.0f, 0), quant_code(x[4 * i + 1], inv, 127.0f, 0),
                         quant_code(x[4 * i + 2], inv, 127.0f, 0), quant_code(x[4 * i + 3], inv, 127.0f, 0));
    }
    int8_t* dst = (l.v ? c.v : c.k) + l.code;
    if (BF16) {
#pragma unroll
        for (int i = 0; i < 2; i++) *(uint2*)(dst + piece<8>(c, l.lane, 2 * i)) = make_uint2(w[2 * i], w[2 * i + 1]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) *(uint32_t*)(dst + piece<4>(c, l.lane, i)) = w[i];
    }
    if (l.lane == 0) (l.v ? c.vs : c.ks)[l.scale] = fine ? scale : __builtin_nanf("");
}

template <bool BF16>
__global__ __launch_bounds__(256) void kv_read_kernel(KvCache c, KvTokens t, int lg) {
    KvLane l;
    if (!kv_lane(c, t, lg, l) || !l.has) return;
    float x[16];
    if (l.live) {
        const int8_t* from = (l.v ? c.v : c.k) + l.code;
        const float scale = (l.v ? c.vs : c.ks)[l.scale];
        uint32_t w[4];
        if (BF16) {
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const uint2 a = *(const uint2*)(from + piece<8>(c, l.lane, 2 * i));
                w[2 * i] = a.x, w[2 * i + 1] = a.y;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) w[i] = *(const uint32_t*)(from + piece<4>(c, l.lane, i));
        }
#pragma unroll
        for (int j = 0; j < 16; j++) x[j] = (float)(int8_t)(w[j / 4] >> 8 * (j % 4)) * scale;
    } else {
#pragma unroll
        for (int j = 0; j < 16; j++) x[j] = 0.0f;
    }
    void* dst = l.v ? t.v : t.k;
    if (BF16) {
#pragma unroll
        for (int i = 0; i < 2; i++)
            *(uint4*)((uint16_t*)dst + l.elem + piece<8>(c, l.lane, 2 * i)) =
                make_uint4(f32x2_to_bf16x2(x[8 * i], x[8 * i + 1]), f32x2_to_bf16x2(x[8 * i + 2], x[8 * i + 3]),
                           f32x2_to_bf16x2(x[8 * i + 4], x[8 * i + 5]), f32x2_to_bf16x2(x[8 * i + 6], x[8 * i + 7]));
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++)
            *(float4*)((float*)dst + l.elem + piece<4>(c, l.lane, i)) = make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
    }
}

// log2 of the lanes a vector, and the blocks (four waves each); 0 where that is
// more than a grid has.
static int kv_shape(const KvCache& c, const KvTokens& t, unsigned* blocks) {
    int lg = 0;
    while (16 << lg < c.dim) lg++;
    const int64_t groups = (t.tokens + (64 >> lg) - 1) >> (6 - lg), n = (groups * 2 * c.heads + 3) / 4;
    *blocks = n <= INT32_MAX ? (unsigned)n : 0;
    return lg;
}

hipError_t launch_kv_cache_write(hipStream_t stream, const KvCache& c, const KvTokens& t) {
    unsigned grid;
    const int lg = kv_shape(c, t, &grid);
    if (!grid) return hipErrorInvalidConfiguration;
    if (t.bf16) hipLaunchKernelGGL(kv_write_kernel<true>, dim3(grid), dim3(256), 0, stream, c, t, lg);
    else hipLaunchKernelGGL(kv_write_kernel<false>, dim3(grid), dim3(256), 0, stream, c, t, lg);
    return hipGetLastError();
}

hipError_t launch_kv_cache_read(hipStream_t stream, const KvCache& c, const KvTokens& t) {
    unsigned grid;
    const int lg = kv_shape(c, t, &grid);
    if (!grid) return hipErrorInvalidConfiguration;
    if (t.bf16) hipLaunchKernelGGL(kv_read_kernel<true>, dim3(grid), dim3(256), 0, stream, c, t, lg);
    else hipLaunchKernelGGL(kv_read_kernel<false>, dim3(grid), dim3(256), 0, stream, c, t, lg);
    return hipGetLastError();
}

}  // namespace phi_dev
