// Attention of new tokens over the paged int8 cache: which kernel takes a call,
// how its tokens are split over blocks, and the join of the splits.
#include <algorithm>
#include <climits>

#include "paged_attention.hpp"

namespace phi_dev {

// What a block of the join works on: a tile's splits, n of them, the last in a slot
// away from the others.  n <= 1: nothing (the tile's rows are written).
struct TileSplits {
    SeqInfo s;
    int tile, n;
    int64_t first, last;  // slots
};

template <bool FEW>
__device__ __forceinline__ TileSplits tile_splits(const PagedAttn& p, const AttnPart& s, int page, int kh, int unit) {
    AttnScan<FEW> f(s);
    int tiles = 0;
    while (f.next(p, s, page)) {
        const int off = unit - tiles;
        tiles += f.lasts;
        if (off >= f.lasts) continue;
        const int at = __builtin_ctzll(__ballot(f.last <= off && off < f.last + f.tiles)), in = off - __builtin_amdgcn_readlane(f.last, at);
        const int n = __builtin_amdgcn_readlane(f.k, at);
        const int first = f.base + __builtin_amdgcn_readlane(f.full_end - f.tiles * (f.k - 1), at) + in * (n - 1), last = f.base + f.fulls() + off;
        if (first + n - 2 >= s.slots || last >= s.slots) break;  // q_start does not ascend to tokens
        return {seq_of_lane(f.q, at), __builtin_amdgcn_readlane(f.tiles, at) - 1 - in, n, (int64_t)kh * s.slots + first, (int64_t)kh * s.slots + last};
    }
    return {{}, 0, 0, 0, 0};
}

// The splits' partial softmaxes of rows joined, 16 rows of a tile a block and a wave
// a row, or one row a block and a wave for every fourth split (W = 4).  Lane k has its
// wave's split k's maximum and sum, so that these are one round of loads; then a lane
// sums four of the vector's elements over eight splits a round, the weights read
// from their lanes.
template <int W>
__global__ __launch_bounds__(256) void attn_join_kernel(PagedAttn p, AttnPart few, AttnPart many, int few_blocks, int page, int D, int kv_heads) {
    constexpr int kRows = W == 1 ? 16 : 1;
    __shared__ float4 lx[W][64];
    __shared__ float2 lml[W];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), w = wave % W;
    const bool is_few = (int)blockIdx.x < few_blocks;
    const AttnPart& s = is_few ? few : many;
    const int idx = blockIdx.x - (is_few ? 0 : few_blocks), kh = idx % kv_heads, groups = s.rows / kRows, at = idx / kv_heads;
    const int unit = at / groups, r0 = (at - unit * groups) * kRows;
    const TileSplits f = is_few ? tile_splits<true>(p, few, page, kh, unit) : tile_splits<false>(p, many, page, kh, unit);
    const int n = f.n, rows = min(f.s.n, p.max_q) * p.group, d = 4 * lane < D ? 4 * lane : 0;
    if (n <= 1) return;
    for (int in = r0 + wave / W; in < r0 + kRows; in += 4) {
        const int r = f.tile * s.rows + in;
        if (r >= rows) return;
        const int i = r / p.group, head = kh * p.group + (r - i * p.group);
        const int64_t token = f.s.first + i;
        auto row_of = [&](int z) { return (z < n - 1 ? f.first + z : f.last) * s.rows + in; };
        float m = kNoMax, l = 0.0f;
        v4f x = {0, 0, 0, 0};
        for (int k0 = w; k0 < n; k0 += 64 * W) {
            v4f y[8];
            auto load = [&](int k) {
#pragma unroll
                for (int u = 0; u < 8; u++) y[u] = k + W * u < n ? *(const v4f*)(s.o + row_of(k + W * u) * D + d) : v4f{0, 0, 0, 0};
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
        if (4 * lane >= D) continue;
        const int64_t to = token * p.out_token + head * p.out_head + d;
        if (!p.bf16) *(v4f*)((float*)p.out + to) = x;
        else *(uint2*)((uint16_t*)p.out + to) = make_uint2(f32x2_to_bf16x2(x[0], x[1]), f32x2_to_bf16x2(x[2], x[3]));
    }
}

namespace {

// bf16 sequences of more rows than this go to the chunk kernel (8 sequences over 8192:
// 64 rows take 77 us and 128 rows 130 here, 136 rows 110 there).
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
// Chunks: a block fills a compute unit and costs 13 us beside its tiles' 2.3 each, so
// splits only where there are fewer blocks than units (512 tokens over 4096, 64
// blocks: 69 us with 256 shares, 85 with 512; 2048 over 2048, 256: 77 whole, 88 with
// 256 shares).
constexpr int kSplitChunks = 256, kSharesChunks = 256;
// Nor up to kWhole tokens: a second launch for the join costs the host 4 us, and the
// GPU gains 1.5 us for one sequence of 1024 (14.2 to 12.7), 1 at 777, loses 0.8 at 600,
// and 2.5 for eight of 1024.
constexpr int kWhole = 1024;

// Up to this many rows x heads, a row's join takes four waves (one sequence of 32768,
// 32 rows: 25 us, 30 with one wave; 64 sequences of 4096, 2048 rows: 121, 107 with one).
constexpr int kJoinWide = 1024;

struct Plan {
    int few_rows;
    AttnPart few, many;  // blocks = 0: does not run
};

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Splits of a part of at most `units` tiles.
void split(AttnPart& s, int64_t units, int64_t shares, int64_t max_kv) {
    s.step = 128 * (int)ceil_div(max_kv * units, (int64_t)128 << 30);  // all tiles' steps in 32 bits
    s.shares = (int)std::max<int64_t>(1, shares);
    s.slots = s.shares + (int)units;
}

Plan attn_plan(int64_t tokens, int64_t q_heads, int64_t kv_heads, int64_t dim, int64_t batch, int64_t max_q, int64_t max_kv,
               int64_t window, bool bf16) {
    const int64_t group = q_heads / kv_heads, rows = max_q * group, span = window > 0 ? std::min(max_kv, window + max_q - 1) : max_kv;
    Plan a{};
    // A lone sequence takes one kernel, whose launch has to serve all its lengths to max_q.
    a.few_rows = !bf16 ? INT32_MAX : batch == 1 && rows > kFewRows ? 0 : kFewRows;
    for (AttnPart* s : {&a.few, &a.many}) {
        const bool few = s == &a.few;
        if (few ? rows > a.few_rows && batch == 1 : rows <= a.few_rows) continue;
        s->rows = few ? kDecodeRows : dim <= 128 ? kChunkRows : kChunkRowsWide;
        s->step = 1 << 30;
        // Tiles, at most.
        const int64_t units = std::min(batch * ceil_div(few ? std::min<int64_t>(rows, a.few_rows) : rows, s->rows), ceil_div(tokens * group, s->rows) + batch);
        // Beside chunks most sequences of few rows are single tokens.
        const int64_t blocks = (few && rows > a.few_rows ? batch : units) * kv_heads;
        if (span > kWhole && blocks < (!few ? kSplitChunks : rows > kDecodeRows ? kSplitTiles : kSplitBlocks))
            split(*s, units, (few ? dim <= 128 ? kShares : kShares / 2 : kSharesChunks) / kv_heads, max_kv);
        s->blocks = (int)std::min<int64_t>(s->shares + units, INT32_MAX / kv_heads);
    }
    return a;
}

int64_t part_rows(const AttnPart& s, int64_t kv_heads) { return kv_heads * s.slots * s.rows; }

}  // namespace

size_t paged_attention_workspace(int64_t tokens, int q_heads, int kv_heads, int dim, int batch, int max_q, int max_kv, bool bf16) {
    const Plan a = attn_plan(tokens, q_heads, kv_heads, dim, batch, max_q, max_kv, 0, bf16);
    return (size_t)((part_rows(a.many, kv_heads) + part_rows(a.few, kv_heads)) * (dim + 2)) * sizeof(float);
}

hipError_t launch_paged_attention(hipStream_t stream, const KvCache& c, const PagedAttn& p0, void* workspace) {
    Plan a = attn_plan(p0.tokens, p0.q_heads, c.heads, c.dim, p0.batch, p0.max_q, p0.max_kv, p0.window, p0.bf16);
    PagedAttn p = p0;
    p.few_rows = a.few_rows;
    float* ws = (float*)workspace;
    for (AttnPart* s : {&a.many, &a.few}) {
        const int64_t rows = part_rows(*s, c.heads);
        s->o = ws, s->ml = ws + rows * c.dim;
        ws += rows * (c.dim + 2);
    }
    hipError_t e = hipSuccess;
    if (a.many.blocks) e = launch_paged_chunk(stream, c, p, a.many);
    if (e == hipSuccess && a.few.blocks) e = launch_paged_decode(stream, c, p, a.few);
    if (e != hipSuccess || (!a.few.shares && !a.many.shares)) return e;
    const bool wide = p.tokens * p.q_heads <= kJoinWide;
    int64_t blocks[2];  // few, many
    for (int k = 0; k < 2; k++) {
        const AttnPart& s = k ? a.many : a.few;
        blocks[k] = (int64_t)(s.slots - s.shares) * c.heads * (wide ? s.rows : s.rows / 16);
    }
    const dim3 grid((unsigned)(blocks[0] + blocks[1]));
    hipLaunchKernelGGL(wide ? attn_join_kernel<4> : attn_join_kernel<1>, grid, dim3(256), 0, stream, p, a.few, a.many, (int)blocks[0], c.page,
                       c.dim, c.heads);
    return hipGetLastError();
}

}  // namespace phi_dev
