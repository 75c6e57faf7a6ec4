// Attention of new tokens over the paged int8 cache: which kernel takes a call,
// how its tokens are split over blocks, and the join of the splits.
#include <algorithm>
#include <climits>

#include "paged_attention.hpp"

namespace phi_dev {

// The splits' partial softmaxes of a row and head joined, W waves a row, each for
// every W-th split.  Lane k has split W k's maximum and sum, so that these are one
// round of loads; then a lane sums four of the vector's elements over eight splits
// a round, the weights read from their lanes.  A tile of one split has written its
// rows itself.
template <int W>
__global__ __launch_bounds__(256) void attn_join_kernel(PagedAttn p, AttnPart few, AttnPart many, int page, int D) {
    __shared__ float4 lx[W][64];
    __shared__ float2 lml[W];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), w = wave % W;
    const int64_t at = (int64_t)blockIdx.x * (4 / W) + wave / W;
    const int token = (int)(at / p.q_heads), head = (int)(at - (int64_t)token * p.q_heads);
    if (token >= p.tokens) return;
    // The sequence of the token: the last that starts at it or before, and has it.
    int b = -1;
    for (int b0 = 0; b0 < p.batch; b0 += 64) {
        const uint64_t on = __ballot(b0 + lane < p.batch && p.q_start[min(b0 + lane, p.batch - 1)] <= token);
        if (on) b = b0 + 63 - __builtin_clzll(on);
        if (~on) break;
    }
    if (b < 0) return;
    const SeqInfo q = seq_info(p, page, b);
    const int i = token - q.first, rows = min(q.n, p.max_q) * p.group, kh = head / p.group;
    if (i >= min(q.n, p.max_q)) return;
    const bool is_few = rows <= p.few_rows;
    const AttnPart& s = is_few ? few : many;
    // The row's first split and its last in o and ml, and the way between others.
    int64_t row = at, last = 0, pitch = s.rows;
    int n;
    if (is_few) {
        if (!s.shares) return;
        FewScan f(s);
        while (f.next(p, s, page) && b >= f.b0 + 64) {}
        const int r = i * p.group + head - kh * p.group, tile = r / kDecodeRows, k = b - f.b0;
        const int tiles = __builtin_amdgcn_readlane(f.tiles, k);
        n = __builtin_amdgcn_readlane(f.k, k);
        if (n == 1) return;
        const int first = f.base + __builtin_amdgcn_readlane(f.full_end, k) - (tiles - tile) * (n - 1);
        const int end = f.base + f.fulls() + __builtin_amdgcn_readlane(f.last, k) + tile;
        if (min(first, end) < 0 || max(first + n - 2, end) >= s.rows) return;  // q_start does not ascend to tokens
        row = (kh * s.rows + first) * kDecodeRows + r - tile * kDecodeRows;
        last = (kh * s.rows + end) * kDecodeRows + r - tile * kDecodeRows;
        pitch = kDecodeRows;
    } else {
        if (s.count == 1) return;
        n = splits_of(p, s, q).n;
        last = row + (n - 1) * pitch;
    }
    const int d = 4 * lane < D ? 4 * lane : 0;
    auto row_of = [&](int z) { return z < n - 1 ? row + z * pitch : last; };
    float m = kNoMax, l = 0.0f;
    v4f x = {0, 0, 0, 0};
    for (int k0 = w; k0 < n; k0 += 64 * W) {
        v4f y[8];
        auto load = [&](int k) {
#pragma unroll
            for (int u = 0; u < 8; u++) y[u] = *(const v4f*)(s.o + row_of(k + W * u) * D + d);
        };
        load(k0);
        const int z = k0 + W * lane;
        const float2 ml = z < n ? *(const float2*)(s.ml + 2 * row_of(z)) : make_float2(kNoMax, 0.0f);
        const float m2 = fmaxf(m, wave_max(ml.x)), keep = __builtin_amdgcn_exp2f(m - m2);
        const float share = z < n ? __builtin_amdgcn_exp2f(ml.x - m2) : 0.0f;
        float sum = ml.y * share;
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off, 64);
        l = l * keep + sum;
        x *= keep;
        m = m2;
        for (int k = 0;;) {
#pragma unroll
            for (int u = 0; u < 8; u++) x += y[u] * __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(share), k + u));
            k += 8;
            if (k >= 64 || k0 + W * k >= n) break;
            load(k0 + W * k);
        }
    }
    if (W > 1) {
        lx[w][lane] = make_float4(x[0], x[1], x[2], x[3]);
        if (lane == 0) lml[w] = make_float2(m, l);
        __syncthreads();
        if (w) return;
#pragma unroll
        for (int k = 1; k < W; k++) m = fmaxf(m, lml[k].x);
        x = v4f{0, 0, 0, 0}, l = 0.0f;
#pragma unroll
        for (int k = 0; k < W; k++) {
            const float4 t = lx[k][lane];
            const float share = __builtin_amdgcn_exp2f(lml[k].x - m);
            x += v4f{t.x, t.y, t.z, t.w} * share;
            l = fmaf(lml[k].y, share, l);
        }
    }
    x *= l != 0.0f ? 1.0f / l : 0.0f;
    if (4 * lane >= D) return;
    const int64_t to = token * p.out_token + head * p.out_head + d;
    if (!p.bf16) *(v4f*)((float*)p.out + to) = x;
    else *(uint2*)((uint16_t*)p.out + to) = make_uint2(f32x2_to_bf16x2(x[0], x[1]), f32x2_to_bf16x2(x[2], x[3]));
}

namespace {

// bf16 sequences of more rows than this go to the chunk kernel.
constexpr int kFewRows = 128;

// Sequences of few rows are split so that about kShares blocks have work, the two
// that a compute unit holds (half at dim 256).  64 sequences of random lengths to
// 8192 (32 heads over 8, dim 128): 123 us, 146 with the shorter splits in the batch's
// order, 128 with 2048 splits of one length; all of 4096: 105 (115 with 2048).  One of
// 32768: 24 us with 512 blocks, 31 with 1024.
constexpr int kShares = 512;
// Not where there are enough blocks without: from kSplitTiles on for tiles of several
// a sequence (16 sequences of 8 tokens over 2000: 256 blocks in 26 us, 31 split;
// chunks of fp32: 550 in 33 and 39), kSplitBlocks for one, whose lengths differ more
// (128 sequences to 8192, 1024 blocks: 222 us, whole 242; 256 of them: 421, whole
// 416).
constexpr int kSplitTiles = 256, kSplitBlocks = 2048;
// Nor up to kWhole tokens: a second launch for the join costs the host 4 us, and the
// GPU gains 1.9 at 1024 tokens (14.8 to 12.9), 1 at 777 and loses 2.4 at 512.
constexpr int kWhole = 1024;

// Up to this many rows x heads, a row's join takes four waves (one sequence of 32768:
// 24 us, 28 with one wave; 10 thousand rows: 50, 39 with one).
constexpr int kJoinWide = 1024;

struct Plan {
    int few_rows;
    AttnPart few, many;  // blocks = 0: does not run
};

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Splits of `step` tokens' multiples that bring `units` blocks to `target`, for
// max_kv tokens.  A window's `span` of them lies in one split more than its length
// makes, wherever it begins, and takes no more room.
void split(AttnPart& s, int64_t units, int64_t target, int64_t step, int64_t max_kv, int64_t span) {
    const int64_t want = std::max<int64_t>(1, std::min(ceil_div(max_kv, step), target / std::max<int64_t>(1, units)));
    s.len = (int)(std::max<int64_t>(1, ceil_div(max_kv, want * step)) * step);
    s.count = (int)std::max<int64_t>(1, ceil_div(max_kv, s.len));
    if (span >= max_kv || s.count == 1) return;
    const int64_t len = ceil_div(span, std::min<int64_t>(s.count - 1, ceil_div(span, step)) * step) * step;
    if (len < s.len) s.len = (int)len, s.count = (int)ceil_div(span, len) + 1;
}

Plan attn_plan(int64_t tokens, int64_t q_heads, int64_t kv_heads, int64_t dim, int64_t batch, int64_t max_q, int64_t max_kv,
               int64_t window, bool bf16) {
    const int64_t group = q_heads / kv_heads, rows = max_q * group, span = window > 0 ? std::min(max_kv, window + max_q - 1) : max_kv;
    Plan a{};
    a.few_rows = bf16 ? kFewRows : INT32_MAX;
    const int64_t few = std::min<int64_t>(rows, a.few_rows);
    if (rows > a.few_rows) {
        const int64_t tile = dim <= 128 ? kChunkRows : kChunkRowsWide;
        const int64_t units = std::min(batch * ceil_div(rows, tile), ceil_div(tokens * group, tile) + batch);
        split(a.many, units * kv_heads, 512, 256, max_kv, span);
        a.many.rows = tokens * q_heads;
        a.many.blocks = (int)std::min<int64_t>(units * a.many.count, INT32_MAX / kv_heads);
    }
    if (rows <= a.few_rows || batch > 1) {
        const int64_t units = std::min(batch * ceil_div(few, kDecodeRows), ceil_div(tokens * group, kDecodeRows) + batch);
        const int64_t blocks = units * kv_heads;
        AttnPart& s = a.few;
        s.len = 1 << 30, s.count = INT_MAX;
        if (blocks < (rows > kDecodeRows ? kSplitTiles : kSplitBlocks) && span > kWhole) {
            s.len = 128 * (int)ceil_div(max_kv * units, (int64_t)128 << 30);  // steps of all tiles in 32 bits
            s.shares = (int)std::max<int64_t>(1, (dim <= 128 ? kShares : kShares / 2) / kv_heads);
            s.rows = s.shares + units;
        }
        s.blocks = (int)std::min<int64_t>(s.shares + units, INT32_MAX / kv_heads);
    }
    return a;
}

// Rows of a part's o and ml.
int64_t many_rows(const AttnPart& s) { return s.count > 1 ? s.count * s.rows : 0; }
int64_t few_rows(const AttnPart& s, int64_t kv_heads) { return kv_heads * s.rows * kDecodeRows; }

}  // namespace

size_t paged_attention_workspace(int64_t tokens, int q_heads, int kv_heads, int dim, int batch, int max_q, int max_kv, bool bf16) {
    const Plan a = attn_plan(tokens, q_heads, kv_heads, dim, batch, max_q, max_kv, 0, bf16);
    return (size_t)((many_rows(a.many) + few_rows(a.few, kv_heads)) * (dim + 2)) * sizeof(float);
}

hipError_t launch_paged_attention(hipStream_t stream, const KvCache& c, const PagedAttn& p0, void* workspace) {
    Plan a = attn_plan(p0.tokens, p0.q_heads, c.heads, c.dim, p0.batch, p0.max_q, p0.max_kv, p0.window, p0.bf16);
    PagedAttn p = p0;
    p.few_rows = a.few_rows;
    float* ws = (float*)workspace;
    const int64_t many = many_rows(a.many), few = few_rows(a.few, c.heads);
    a.many.o = ws, a.many.ml = ws + many * c.dim;
    a.few.o = ws + many * (c.dim + 2), a.few.ml = a.few.o + few * c.dim;
    hipError_t e = hipSuccess;
    if (a.many.blocks) e = launch_paged_chunk(stream, c, p, a.many);
    if (e == hipSuccess && a.few.blocks) e = launch_paged_decode(stream, c, p, a.few);
    if (e != hipSuccess || (!a.few.shares && a.many.count <= 1)) return e;
    const int64_t heads = p.tokens * p.q_heads;
    if (heads <= kJoinWide)
        hipLaunchKernelGGL(attn_join_kernel<4>, dim3((unsigned)heads), dim3(256), 0, stream, p, a.few, a.many, c.page, c.dim);
    else
        hipLaunchKernelGGL(attn_join_kernel<1>, dim3((unsigned)ceil_div(heads, 4)), dim3(256), 0, stream, p, a.few, a.many, c.page, c.dim);
    return hipGetLastError();
}

}  // namespace phi_dev
