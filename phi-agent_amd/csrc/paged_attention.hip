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
    AttnScan<FEW, false> f(s);
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

// One row's part: its splits' slots, and where their row and dim start.
struct RowPart {
    AttnPart s;
    int n, first, last, in;
    __device__ __forceinline__ int64_t row(int kh, int z) const { return ((int64_t)kh * s.slots + (z < n - 1 ? first + z : last)) * s.rows + in; }
};

// A prefix's and the own tokens' partial softmaxes of rows joined, a wave a row of q (token x
// head), or a block a row and a wave every fourth split (W = 4).  As attn_join_kernel, over the
// splits of both in a row, of which SUB parts of a wave, wide enough for dim each, take turns.
template <int W, int SUB>
__global__ __launch_bounds__(256) void shared_join_kernel(PagedAttn p, AttnPart few, AttnPart many, int D) {
    constexpr int kAhead = 8;
    __shared__ float4 lx[W][64];
    __shared__ float2 lml[W];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), w = wave % W;
    const int sub = lane / (64 / SUB), dl = 4 * (lane % (64 / SUB)), batch = p.batch - p.groups, d = dl < D ? dl : 0;
    const int64_t r = (int64_t)blockIdx.x * (4 / W) + wave / W;
    const int token = (int)(r / p.q_heads), head = (int)(r - (int64_t)token * p.q_heads), kh = head / p.group;
    if (token >= p.tokens) return;  // W = 4: never
    const int64_t at = (int64_t)token * p.group + (head - kh * p.group);
    RowPart part[2];  // prefix, own
    bool mine = false;
#pragma unroll
    for (int k = 0; k < 2; k++) {
        const AttnRow a = (k ? p.own_rows : p.prefix_rows)[at];
        RowPart& x = part[k];
        x.s = a.many() ? many : few;
        x.in = a.in(), x.first = a.first, x.last = a.last;
        // Left by this call only if the row is of that group or sequence.
        int from = a.id, to = a.id + 1;
        bool is = a.id >= 0 && a.id < (k ? batch : p.groups);
        if (k == 0 && is) from = min(max(p.group_start[a.id], 0), batch), to = min(max(p.group_start[a.id + 1], 0), batch);
        if (is) {
            const int first = p.q_start[from];
            is = token >= first && token < p.q_start[to] && (k == 0 || token - first < p.own_q);
        }
        is = is && a.inside(x.s.slots, x.s.rows);
        x.n = is ? a.splits() : 0;
        mine = k ? is : mine;
    }
    if (!mine) return;  // W = 4: the same in all waves
    const int n0 = part[0].n, n = n0 + part[1].n;
    auto ml_of = [&](int z) { const RowPart& x = part[z < n0 ? 0 : 1]; return x.s.ml + 2 * x.row(kh, z < n0 ? z : z - n0); };
    auto o_of = [&](int z) { const RowPart& x = part[z < n0 ? 0 : 1]; return x.s.o + x.row(kh, z < n0 ? z : z - n0) * D; };
    float m = kNoMax, l = 0.0f;
    v4f x = {0, 0, 0, 0};
    // 64 of the wave's splits at a time: w + W i in lane i, the sub-th of every SUB a part's.
    for (int k0 = w; k0 < n; k0 += 64 * W) {
        v4f y[kAhead];
        auto load = [&](int i) {
#pragma unroll
            for (int u = 0; u < kAhead; u++) {
                const int z = k0 + W * (i + SUB * u + sub);
                y[u] = z < n ? *(const v4f*)(o_of(z) + d) : v4f{0, 0, 0, 0};
            }
        };
        load(0);
        const int z = k0 + W * lane;
        const float2 ml = z < n ? *(const float2*)ml_of(z) : make_float2(kNoMax, 0.0f);
        const float m2 = fmaxf(m, wave_max(ml.x)), keep = __builtin_amdgcn_exp2f(m - m2);
        const float share = z < n ? __builtin_amdgcn_exp2f(ml.x - m2) : 0.0f;
        float sum = ml.y * share;
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off, 64);
        l = l * keep + sum;
        x *= keep;
        m = m2;
        for (int i = 0;;) {
#pragma unroll
            for (int u = 0; u < kAhead; u++) x += y[u] * __shfl(share, i + SUB * u + sub, 64);
            i += SUB * kAhead;
            if (i >= 64 || k0 + W * i >= n) break;
            load(i);
        }
    }
#pragma unroll
    for (int off = 64 / SUB; off < 64; off <<= 1)
#pragma unroll
        for (int e = 0; e < 4; e++) x[e] += __shfl_xor(x[e], off, 64);
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
    if (sub || dl >= D) return;
    const int64_t to = (int64_t)token * p.out_token + head * p.out_head + d;
    if (!p.bf16) *(v4f*)((float*)p.out + to) = x;
    else *(uint2*)((uint16_t*)p.out + to) = make_uint2(f32x2_to_bf16x2(x[0], x[1]), f32x2_to_bf16x2(x[2], x[3]));
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

// With shared prefixes every tile leaves its results in slots, for there is a join
// anyhow, and is split by the work there is.
Plan shared_plan(int64_t tokens, int64_t q_heads, int64_t kv_heads, int64_t dim, int64_t groups, int64_t batch, int64_t max_prefix,
                 int64_t max_q, int64_t max_kv, bool bf16) {
    const int64_t group = q_heads / kv_heads, all = tokens * group, own = max_q * group, longest = std::max(max_prefix, max_kv);
    Plan a{};
    a.few_rows = bf16 ? kFewRows : INT32_MAX;
    for (AttnPart* s : {&a.few, &a.many}) {
        const bool few = s == &a.few;
        if (!few && all <= a.few_rows) continue;
        s->rows = few ? kDecodeRows : dim <= 128 ? kChunkRows : kChunkRowsWide;
        // Tiles, at most, of the groups and of the sequences.
        const int64_t most = ceil_div(all, s->rows), cap = ceil_div(few ? a.few_rows : all, s->rows);
        int64_t units = std::min(groups * cap, most + groups);
        s->seqs = (int)groups;
        if (few || own > a.few_rows) s->seqs += (int)batch, units += std::min(batch * ceil_div(few ? std::min<int64_t>(own, a.few_rows) : own, s->rows), most + batch);
        int64_t shares = (few ? dim <= 128 ? kShares : kShares / 2 : kSharesChunks) / kv_heads;
        // Where the sequences fill the compute units, splits only even out their lengths: a
        // unit costs 10 us beside its tokens (64 sequences behind 8192: 47.9 us, 50.1 without).
        if (few && batch * kv_heads >= kShares) shares = (shares + 1) / 2;
        if (!few && dim <= 128) {
            // In one launch with the own tokens' part a prefix's splits take as many compute
            // units as are its share of the work, so that both end together: microseconds a
            // unit, of a block's tile of 64 tokens 2.3 beside 9, of 256 own tokens 2 beside 5.
            // (64 sequences behind 8192 tokens: 49 us with 12 splits a head, 53 with 10, 58 with
            // 24; 96 behind three documents to 32760: 230 with 24, 268 with 18, 241 with 28.)
            // Sequences of chunks, as many as `tokens` holds, have their own tokens here too (64 of
            // 64 query heads over 4096, behind 64: 56 us, 154 unsplit; 1024 of 32 over 8192 behind
            // nothing: 198, 316; paged_attention 44 and 182).
            const int64_t chunks = own > a.few_rows ? std::min(batch, tokens / max_q) : 0;
            const double tiles = most * ceil_div(max_prefix, 64) + chunks * ceil_div(own, s->rows) * ceil_div(max_kv, 64);
            const double here = 2.3 * tiles, rest = (batch - chunks) * (5 + max_kv * 0.008), all_units = std::max<double>(1, 256.0 / kv_heads);
            const double each = std::max((here + rest) / all_units - 9, 7.0);
            shares = (int64_t)std::min(here / each, all_units) + 1;
        }
        split(*s, units, shares, std::max<int64_t>(longest, 1));
        s->blocks = (int)std::min<int64_t>(s->slots, INT32_MAX / kv_heads);
    }
    return a;
}

// Whether a launch can have the plan's blocks: its threads are counted in 32 bits.
bool shared_fits(const Plan& a, int64_t kv_heads, int64_t dim) {
    const int64_t most = (int64_t)1 << 32, many = a.many.blocks * kv_heads, few = a.few.blocks * kv_heads;
    if (many && dim <= 128) return (many + (few + 1) / 2) * 512 < most;  // in one
    return many * 256 < most && few * 256 < most;
}

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

size_t paged_attention_shared_workspace(int64_t tokens, int q_heads, int kv_heads, int dim, int groups, int batch, int max_prefix, int max_q,
                                        int max_kv, bool bf16) {
    const Plan a = shared_plan(tokens, q_heads, kv_heads, dim, groups, batch, max_prefix, max_q, max_kv, bf16);
    if (!shared_fits(a, kv_heads, dim)) return 0;
    return (size_t)((part_rows(a.many, kv_heads) + part_rows(a.few, kv_heads)) * (dim + 2)) * sizeof(float) +
           (size_t)tokens * (q_heads / kv_heads) * 2 * sizeof(AttnRow);
}

hipError_t launch_paged_attention_shared(hipStream_t stream, const KvCache& c, const PagedAttn& p0, void* workspace) {
    Plan a = shared_plan(p0.tokens, p0.q_heads, c.heads, c.dim, p0.groups, p0.batch, p0.max_prefix, p0.max_q, p0.max_kv, p0.bf16);
    PagedAttn p = p0;
    p.few_rows = a.few_rows;
    p.causal = true, p.window = 0;
    p.own_q = p0.max_q, p.max_q = (int)p0.tokens, p.batch = p0.groups + p0.batch;
    float* ws = (float*)workspace;
    for (AttnPart* s : {&a.many, &a.few}) {
        const int64_t rows = part_rows(*s, c.heads);
        s->o = ws, s->ml = ws + rows * c.dim;
        ws += rows * (c.dim + 2);
    }
    p.prefix_rows = (AttnRow*)ws;
    p.own_rows = p.prefix_rows + p.tokens * p.group;
    hipError_t e = hipSuccess;
    if (a.many.blocks && c.dim <= 128) {
        e = launch_paged_shared(stream, c, p, a.many, a.few);
    } else {
        if (a.many.blocks) e = launch_paged_chunk(stream, c, p, a.many);
        if (e == hipSuccess) e = launch_paged_decode(stream, c, p, a.few);
    }
    if (e != hipSuccess) return e;
    const int64_t rows = p.tokens * p.q_heads;
    const bool wide = rows <= kJoinWide;
    const dim3 grid((unsigned)(wide ? rows : ceil_div(rows, 4))), block(256);
    auto join = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, block, 0, stream, p, a.few, a.many, c.dim); };
    if (c.dim <= 64) wide ? join(shared_join_kernel<4, 4>) : join(shared_join_kernel<1, 4>);
    else if (c.dim <= 128) wide ? join(shared_join_kernel<4, 2>) : join(shared_join_kernel<1, 2>);
    else wide ? join(shared_join_kernel<4, 1>) : join(shared_join_kernel<1, 1>);
    return hipGetLastError();
}

}  // namespace phi_dev
