// Low-rank adapters of many requests beside one linear:
//   out[m] = base[m] + scale[a] B[a] (A[a] x[m]),   a = adapter[m].
//
// Two passes, h = A[a] x[m] and the update.  A tile of 128 rows has its rows sorted
// into classes, those of one adapter; a block takes rows of one class as the
// columns of its products, so that an adapter's factors are read for a tile's rows of it
// together however these are mixed (A once for 32 of them, or 128; B's first 32 ranks, or 64,
// once, further ones for every 16), and a row's values meet no other adapter's.  The
// first pass leaves the classes for the second.
// An operand of a matrix instruction is 16 rows of 32 k, 8 consecutive k of row l % 16 in
// lane l: one v_mfma_f32_16x16x32_bf16 or, in fp32, eight v_mfma_f32_16x16x4_f32 (k 8 g + e
// in the e-th, g = l / 16, on both sides).
// h is fp32 throughout: against bf16 factors it enters the second product as three
// bf16, all of its 24 bits; of a result that is not finite, infinite factors meet the first only.
// Bound by memory: x once, base and out once, each tile's factors from L2.  64 rows of
// 4096 on 16 ranks to 6144, 32 adapters at random: 6 + 8 us, latency (counts, classes, rows and
// factors are loads that wait for each other); eight prompts of 4352 rows of 5120 on 64 ranks
// to 5120: 20 + 5 + 33 us, x at 2.3 TB/s, base and out at 2.7.
#include <algorithm>
#include <type_traits>

#include "device_common.hpp"
#include "serving.hpp"

namespace phi_dev {

constexpr int kLoraTile = 128;  // rows

// A tile's classes as the first pass leaves them for the second.
struct LoraClass {
    uint64_t rows[2];
    int adapter, pad[3];
};

namespace {

typedef __bf16 b8 __attribute__((ext_vector_type(8)));

constexpr int kSplits = 8;
constexpr int kSpread = 128;  // places, from which on each XCD has neighbours (4352 rows on 64 ranks: 56 us, 60 never)
constexpr int kUpTiles = 4;   // of 16 columns a wave

// Up to `most` rows of one class, from the skip-th on.
struct LoraUnit {
    int adapter;  // below 0: none
    int index;    // of the class; where there is no unit, the number of classes
    int skip, n;  // n 0: there is none
    uint64_t rows[2];
};

// A tile's classes, as one wave finds them: two rows a lane, the first row of each class by
// the lowest number in a table of adapters (those that fall on one place of it in turns).
// (Class by class from the first row left, 0.2 us each: 7.7 us to the last of 28.)
constexpr int kPlaces = 1024;
struct LoraTable {
    int place[kPlaces], key[kLoraTile], count[kLoraTile];
};
struct LoraClasses {
    int a[2], count[2];  // a row's adapter and, of a class's first row, its rows
    uint64_t some[2], first[2];

    __device__ __forceinline__ void find(const LoraBatched& p, int tile, LoraTable& t) {
        const int lane = threadIdx.x & 63;
        bool left[2], mine[2] = {false, false};
#pragma unroll
        for (int i = 0; i < kPlaces / 256; i++) *(int4*)(t.place + 4 * (lane + 64 * i)) = make_int4(kLoraTile, kLoraTile, kLoraTile, kLoraTile);
        int at[2];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int row = tile * kLoraTile + 64 * h + lane;
            left[h] = row < p.rows;
            some[h] = __ballot(left[h]);
            a[h] = left[h] ? p.adapter[row] : 0;
            a[h] = a[h] >= 0 && a[h] < p.adapters ? a[h] : -1;
            at[h] = (a[h] + 1) & (kPlaces - 1);
            t.key[64 * h + lane] = a[h], t.count[64 * h + lane] = 0;
        }
        // A wave's LDS accesses are done in order; the fences keep the compiler's.
        auto fence = [] {
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup", "local");
        };
        do {
            fence();
#pragma unroll
            for (int h = 0; h < 2; h++)
                if (left[h]) atomicMin(&t.place[at[h]], 64 * h + lane);
            fence();
            int won[2];
#pragma unroll
            for (int h = 0; h < 2; h++) won[h] = t.place[at[h]];
#pragma unroll
            for (int h = 0; h < 2; h++) {
                if (!left[h] || t.key[won[h]] != a[h]) continue;
                mine[h] = won[h] == 64 * h + lane;
                atomicAdd(&t.count[won[h]], 1);
                left[h] = false;
            }
            fence();
            // For the next turn, those that are left begin anew.
#pragma unroll
            for (int h = 0; h < 2; h++)
                if (left[h]) t.place[at[h]] = kLoraTile;
        } while (__any(left[0] || left[1]));
        fence();
#pragma unroll
        for (int h = 0; h < 2; h++) first[h] = __ballot(mine[h]), count[h] = t.count[64 * h + lane];
    }
    // Unit u: all classes' first `most` rows, then the next of those that have more, and so on.
    __device__ __forceinline__ LoraUnit unit(int u, int most) const {
        const uint64_t below = ((uint64_t)1 << (threadIdx.x & 63)) - 1;
        const int classes = __popcll(first[0]) + __popcll(first[1]);
#pragma unroll 1
        for (int skip = 0; skip < kLoraTile; skip += most) {
            const uint64_t of[2] = {__ballot(count[0] > skip) & first[0], __ballot(count[1] > skip) & first[1]};
            const int n0 = __popcll(of[0]), n = n0 + __popcll(of[1]);
            if (u >= n) {
                u -= n;
                continue;
            }
            const int h = u >= n0;
            const uint64_t mask = of[h], got = __ballot((mask & ~below & (below + 1)) && (int)__popcll(mask & below) == u - (h ? n0 : 0));
            const int lane = __builtin_ctzll(got), one = __builtin_amdgcn_readlane(a[h], lane), all = __builtin_amdgcn_readlane(count[h], lane);
            const uint64_t before = ((uint64_t)1 << lane) - 1;
            return {one, (int)(h ? __popcll(first[0]) + __popcll(first[1] & before) : __popcll(first[0] & before)), skip, min(all - skip, most),
                    {__ballot(a[0] == one) & some[0], __ballot(a[1] == one) & some[1]}};
        }
        return {0, classes, 0, 0, {0, 0}};
    }
};

// Block number `id` of `around` as a place (tile x across): where these are 8 ceil(places /
// 8), neighbours, which often have one adapter, on one XCD, whose L2 keeps its factors
// (blocks go round the eight).
__device__ __forceinline__ int lora_place(int id, int around) { return around >= kSpread ? (id & 7) * (around >> 3) + (id >> 3) : id; }

// Rows of a class from the skip-th on, `most` of them, in LDS; every wave writes the same.
__device__ __forceinline__ void class_rows(const uint64_t (&mask)[2], int tile, int skip, int most, int* rows) {
    const int lane = threadIdx.x & 63;
    const uint64_t below = ((uint64_t)1 << lane) - 1;
    const int at[2] = {(int)__popcll(mask[0] & below), (int)(__popcll(mask[0]) + __popcll(mask[1] & below))};
#pragma unroll
    for (int h = 0; h < 2; h++)
        if ((mask[h] >> lane & 1) && at[h] >= skip && at[h] < skip + most) rows[at[h] - skip] = tile * kLoraTile + 64 * h + lane;
}

// Rows may lie at any of their elements: loads are of 16 bytes all the same, which the
// memory path takes at any address.
typedef uint32_t any4 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t any2 __attribute__((ext_vector_type(2), aligned(2)));

template <bool B16> struct Eight {
    uint32_t w[B16 ? 4 : 8];
};
template <bool B16>
__device__ __forceinline__ Eight<B16> load_eight(const char* row, int k) {
    Eight<B16> e;
    const char* p = row + (size_t)(uint32_t)k * (B16 ? 2 : 4);
#pragma unroll
    for (int i = 0; i < (B16 ? 1 : 2); i++) {
        const any4 t = *(const any4*)(p + 16 * i);
        e.w[4 * i] = t[0], e.w[4 * i + 1] = t[1], e.w[4 * i + 2] = t[2], e.w[4 * i + 3] = t[3];
    }
    return e;
}
// The same from k on in a row of K, zeros past its end.  What lies behind the row is read
// with it and dropped, but not from `end`, the operand's, on: there one by one, in a loop
// that costs few registers.
template <bool B16>
__device__ __forceinline__ Eight<B16> load_masked(const char* row, int k, int K, const char* end) {
    constexpr int E = B16 ? 2 : 4;
    Eight<B16> e{};
    const char* p = row + (size_t)(uint32_t)k * E;
    if (__any(k < K && p + 8 * E > end)) {
#pragma unroll 1
        for (int i = 0; i < 8; i++) {
            const int at = min(k + i, K - 1);
            const uint32_t v = B16 ? ((const uint16_t*)row)[at] : ((const uint32_t*)row)[at], x = k + i < K ? v : 0;
#pragma unroll
            for (int j = 0; j < (B16 ? 4 : 8); j++) {
                const uint32_t above = j + 1 < (B16 ? 4 : 8) ? e.w[(j + 1) % (B16 ? 4 : 8)] : x;
                e.w[j] = B16 ? __builtin_amdgcn_alignbit(above, e.w[j], 16) : above;
            }
        }
    } else if (k < K) {
        e = load_eight<B16>(row, k);
#pragma unroll
        for (int j = 0; j < (B16 ? 4 : 8); j++) {
            if (B16) e.w[j] &= (k + 2 * j < K ? 0xffffu : 0u) | (k + 2 * j + 1 < K ? 0xffff0000u : 0u);
            else e.w[j] = k + j < K ? e.w[j] : 0;
        }
    }
    return e;
}

// 16 rows of 32 H k on their way through LDS: loaded with a row's lanes side by side
// (16 lanes that meet 16 rows are taken one by one by the address path).
template <bool B16, int H> struct Rows {
    static constexpr int kLanes = (B16 ? 4 : 8) * H, kLoads = kLanes / 4, kPitch = 16 * kLanes + 16, kBytes = 16 * kPitch;
    any4 w[kLoads];
    static __device__ __forceinline__ int row(int i) { return (threadIdx.x & 63) / kLanes + 64 / kLanes * i; }
    static __device__ __forceinline__ int k() { return (threadIdx.x & (kLanes - 1)) * (B16 ? 8 : 4); }
    // rows[i]: row(i)'s.
    __device__ __forceinline__ void load(const char* const (&rows)[kLoads], int k0) {
#pragma unroll
        for (int i = 0; i < kLoads; i++) w[i] = *(const any4*)(rows[i] + (size_t)(uint32_t)(k0 + k()) * (B16 ? 2 : 4));
    }
    __device__ __forceinline__ void to(uint8_t* lds) const {
#pragma unroll
        for (int i = 0; i < kLoads; i++) *(uint4*)(lds + row(i) * kPitch + 16 * (threadIdx.x & (kLanes - 1))) = make_uint4(w[i][0], w[i][1], w[i][2], w[i][3]);
    }
    // The operand of k from 32 h on.
    static __device__ __forceinline__ Eight<B16> from(const uint8_t* lds, int h) {
        const int lane = threadIdx.x & 63, n = B16 ? 1 : 2;
        Eight<B16> e;
#pragma unroll
        for (int i = 0; i < n; i++) *(uint4*)(e.w + 4 * i) = *(const uint4*)(lds + (lane & 15) * kPitch + 64 * n * h + 16 * n * (lane >> 4) + 16 * i);
        return e;
    }
};
template <bool B16>
__device__ __forceinline__ float value(const Eight<B16>& e, int i) {
    return __uint_as_float(B16 ? i & 1 ? e.w[i >> 1] & 0xffff0000u : e.w[i >> 1] << 16 : e.w[i]);
}

// Eight bf16 with zeros for those that are not finite.
__device__ __forceinline__ Eight<true> finite_of(Eight<true> e) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t f = ((e.w[i] & 0x7f807f80u) + 0x00800080u) & 0x80008000u;
        e.w[i] &= ~(f | (f - (f >> 15)));
    }
    return e;
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

// h of few rows: RT tiles of 16 ranks from 16 RT blockIdx.z on for up to 32 rows of a class,
// every `parts`-th unit of a tile a block.  Each wave has a stretch of K, U steps of 32 at
// a time straight from memory.
constexpr int kFewCols = 32;

template <bool XB, bool WB, int RT>
__global__ __launch_bounds__(256, 2) void lora_batched_down_kernel(LoraBatched p, int tiles, int around, int parts) {
    constexpr int P = 16 * RT + 4, U = XB && WB ? 4 : 2;
    __shared__ int rows[kFewCols];
    __shared__ float part[4][kFewCols][P];
    __shared__ LoraTable table;
    __shared__ LoraUnit found;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int at = lora_place(blockIdx.x % around, around), tile = at / p.splits, split = at - tile * p.splits, r0 = 16 * RT * blockIdx.z;
    if (tile >= tiles) return;
    const int col = lane & 15, g = lane >> 4;
    const int steps = (p.K + 31) / 32, waves = 4 * p.splits, me = 4 * split + wave;
    const int s0 = (int)((int64_t)steps * me / waves), s1 = (int)((int64_t)steps * (me + 1) / waves), whole = min(s1, p.K / 32);
    const bool tells = split == 0 && blockIdx.z == 0 && threadIdx.x == 0;
    LoraClasses classes;
    if (wave == 0) classes.find(p, tile, table);
#pragma unroll 1
    for (int unit = blockIdx.x / around;; unit += parts) {
        if (wave == 0) {
            const LoraUnit u = classes.unit(unit, kFewCols);
            if (lane == 0) found = u;
        }
        __syncthreads();
        const LoraUnit u = found;
        if (!u.n) {
            if (tells) p.counts[tile] = u.index;
            return;
        }
        if (tells && u.skip == 0) p.classes[(int64_t)tile * kLoraTile + u.index] = {{u.rows[0], u.rows[1]}, u.adapter, {}};
        if (u.adapter < 0) {
            __syncthreads();
            continue;
        }
        class_rows(u.rows, tile, u.skip, kFewCols, rows);
        __syncthreads();
        const bool two = u.n > 16;
        const char* xs[2];
        const char* as[RT];
#pragma unroll
        for (int c = 0; c < 2; c++) xs[c] = (const char*)p.x + (int64_t)rows[min(16 * c + col, u.n - 1)] * p.ldx * (XB ? 2 : 4);
#pragma unroll
        for (int r = 0; r < RT; r++)
            as[r] = (const char*)p.A + (u.adapter * p.a_adapter + min(r0 + 16 * r + col, p.R - 1) * p.a_row) * (WB ? 2 : 4);
        v4f acc[2][RT];
#pragma unroll
        for (int c = 0; c < 2; c++)
#pragma unroll
            for (int r = 0; r < RT; r++) acc[c][r] = v4f{0, 0, 0, 0};
        auto multiply = [&](const Eight<XB> (&x)[2], const Eight<WB> (&a)[RT]) __attribute__((always_inline)) {
#pragma unroll
            for (int r = 0; r < RT; r++) acc[0][r] = product(a[r], x[0], acc[0][r]);
            if (two) {
#pragma unroll
                for (int r = 0; r < RT; r++) acc[1][r] = product(a[r], x[1], acc[1][r]);
            }
        };
#pragma unroll 1
        for (int s = s0; s < whole; s += U) {
            Eight<XB> x[U][2];
            Eight<WB> a[U][RT];
#pragma unroll
            for (int i = 0; i < U; i++) {
                const int k = 32 * min(s + i, whole - 1) + 8 * g;  // past the last: unused
                x[i][0] = load_eight<XB>(xs[0], k);
                if (two) x[i][1] = load_eight<XB>(xs[1], k);
#pragma unroll
                for (int r = 0; r < RT; r++) a[i][r] = load_eight<WB>(as[r], k);
            }
#pragma unroll
            for (int i = 0; i < U; i++)
                if (s + i < whole) multiply(x[i], a[i]);
        }
        if (whole < s1) {  // the last of K
            const int k = 32 * whole + 8 * g;
            Eight<XB> x[2];
            Eight<WB> a[RT];
#pragma unroll
            for (int c = 0; c < 2; c++) x[c] = load_masked<XB>(xs[c], k, p.K, p.x_end);
#pragma unroll
            for (int r = 0; r < RT; r++) a[r] = load_masked<WB>(as[r], k, p.K, p.a_end);
            multiply(x, a);
        }
#pragma unroll
        for (int c = 0; c < 2; c++)
#pragma unroll
            for (int r = 0; r < RT; r++) *(v4f*)&part[wave][16 * c + col][16 * r + 4 * g] = acc[c][r];
        __syncthreads();
#pragma unroll 1
        for (int i = threadIdx.x; i < u.n * 4 * RT; i += 256) {
            const int c = i / (4 * RT), r = 4 * (i % (4 * RT));
            if (r0 + r >= p.rank_pitch) continue;
            v4f sum = *(const v4f*)&part[0][c][r];
#pragma unroll
            for (int w = 1; w < 4; w++) sum += *(const v4f*)&part[w][c][r];
            *(v4f*)(p.h + ((int64_t)split * p.rows + rows[c]) * p.rank_pitch + r0 + r) = sum;
        }
        __syncthreads();
    }
}

// h of many rows, up to a tile's 128 of a class a block, so that A is read a fourth as often:
// blocks of one adapter meet in L2, where A's second reading cost more than x from memory
// (4352 rows of 5120 on 64 ranks: 35 us in units of 32 rows, 15 with A from a few lines).
// Waves 0-3 have 32 rows each of the first half of the block's stretch of K, waves 4-7 of the
// second; a half's four waves share A's step of H 32 k in LDS, two steps' in turn, and
// load two steps ahead.
template <bool XB, bool WB>
__global__ __launch_bounds__(512, 2) void lora_batched_down_wide_kernel(LoraBatched p, int tiles, int around, int parts) {
    constexpr int RT = 4, H = XB && WB ? 2 : 1, kStep = 32 * H, P = 16 * RT + 4;
    typedef Rows<XB, H> RX;
    typedef Rows<WB, H> RA;
    constexpr int kA = RT * RA::kBytes, kX = 2 * RX::kBytes, kStage = 2 * 2 * kA + 8 * kX, kJoin = kLoraTile * P * 4;
    constexpr int kMine = RA::kLoads;  // of A's: a tile a wave
    __shared__ int rows[kLoraTile];
    __shared__ __align__(16) uint8_t lds[kStage > kJoin ? kStage : kJoin];
    __shared__ LoraTable table;
    __shared__ LoraUnit found;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = wave >> 2, w = wave & 3;
    const int at = lora_place(blockIdx.x % around, around), tile = at / p.splits, split = at - tile * p.splits, r0 = 16 * RT * blockIdx.z;
    if (tile >= tiles) return;
    const int col = lane & 15, g = lane >> 4;
    const int steps = (p.K + kStep - 1) / kStep, ranges = 2 * p.splits, me = 2 * split + half;
    const int s0 = (int)((int64_t)steps * me / ranges), s1 = (int)((int64_t)steps * (me + 1) / ranges);
    // Both halves go round as often.
    const int turns = max(s1 - s0, (int)((int64_t)steps * (2 * split + 2 - half) / ranges) - (int)((int64_t)steps * (2 * split + 1 - half) / ranges));
    const bool tells = split == 0 && blockIdx.z == 0 && threadIdx.x == 0;
    uint8_t* const lds_x = lds + 4 * kA + wave * kX;
    LoraClasses classes;
    if (wave == 0) classes.find(p, tile, table);
#pragma unroll 1
    for (int unit = blockIdx.x / around;; unit += parts) {
        if (wave == 0) {
            const LoraUnit u = classes.unit(unit, kLoraTile);
            if (lane == 0) found = u;
        }
        __syncthreads();
        const LoraUnit u = found;
        if (!u.n) {
            if (tells) p.counts[tile] = u.index;
            return;
        }
        if (tells && u.skip == 0) p.classes[(int64_t)tile * kLoraTile + u.index] = {{u.rows[0], u.rows[1]}, u.adapter, {}};
        if (u.adapter < 0) {
            __syncthreads();
            continue;
        }
        class_rows(u.rows, tile, 0, kLoraTile, rows);
        __syncthreads();
        const bool mine = 32 * w < u.n;
        const char* xs[2][RX::kLoads];
        const char* as[kMine];
#pragma unroll
        for (int c = 0; c < 2; c++)
#pragma unroll
            for (int i = 0; i < RX::kLoads; i++) xs[c][i] = (const char*)p.x + (int64_t)rows[min(32 * w + 16 * c + RX::row(i), u.n - 1)] * p.ldx * (XB ? 2 : 4);
        auto a_load = [&](int j) { return w * kMine + j; };
#pragma unroll
        for (int j = 0; j < kMine; j++) {
            const int row = 64 / RA::kLanes * a_load(j) + lane / RA::kLanes;
            as[j] = (const char*)p.A + (u.adapter * p.a_adapter + min(r0 + row, p.R - 1) * p.a_row) * (WB ? 2 : 4);
        }
        v4f acc[2][RT];
#pragma unroll
        for (int c = 0; c < 2; c++)
#pragma unroll
            for (int r = 0; r < RT; r++) acc[c][r] = v4f{0, 0, 0, 0};
        struct Step {
            RX x[2];
            any4 a[kMine];
        };
        // Without a branch (what loads meet a branch is waited for with all that came after
        // it): past the last whole step the last again, for rows behind the last the last's.
        const int last = max(min(s1, p.K / kStep) - 1, 0);
        auto load = [&](Step& t, int s) __attribute__((always_inline)) {
            const int k = kStep * min(s, last);
            t.x[0].load(xs[0], k), t.x[1].load(xs[1], k);
#pragma unroll
            for (int j = 0; j < kMine; j++) t.a[j] = *(const any4*)(as[j] + (size_t)(uint32_t)(k + RA::k()) * (WB ? 2 : 4));
        };
        // The last of K, zeros past its end, one by one and straight to LDS.
        auto rest = [&](uint8_t* lds_a) {
            const int k0 = p.K / kStep * kStep;
#pragma unroll 1
            for (int i = lane; i < 32 * kStep; i += 64) {
                const int r = i / kStep, k = i % kStep, at = min(k0 + k, p.K - 1);
                const char* from = (const char*)p.x + (rows[min(32 * w + r, u.n - 1)] * p.ldx + at) * (XB ? 2 : 4);
                uint8_t* to = lds_x + r / 16 * RX::kBytes + r % 16 * RX::kPitch + k * (XB ? 2 : 4);
                if (XB) *(uint16_t*)to = k0 + k < p.K ? *(const uint16_t*)from : 0;
                else *(uint32_t*)to = k0 + k < p.K ? *(const uint32_t*)from : 0;
            }
#pragma unroll 1
            for (int i = 64 * w + lane; i < 16 * RT * kStep; i += 256) {
                const int r = i / kStep, k = i % kStep, at = min(k0 + k, p.K - 1);
                const char* from = (const char*)p.A + (u.adapter * p.a_adapter + min(r0 + r, p.R - 1) * p.a_row + at) * (WB ? 2 : 4);
                uint8_t* to = lds_a + r / 16 * RA::kBytes + r % 16 * RA::kPitch + k * (WB ? 2 : 4);
                if (WB) *(uint16_t*)to = k0 + k < p.K ? *(const uint16_t*)from : 0;
                else *(uint32_t*)to = k0 + k < p.K ? *(const uint32_t*)from : 0;
            }
        };
        auto turn = [&](Step& t, int n) __attribute__((always_inline)) {
            const int s = s0 + n;
            uint8_t* const lds_a = lds + (2 * half + (n & 1)) * kA;
            if (s < s1 && s < p.K / kStep) {
#pragma unroll
                for (int j = 0; j < kMine; j++) {
                    const int at = a_load(j);
                    *(uint4*)(lds_a + (64 / RA::kLanes * at + lane / RA::kLanes) * RA::kPitch + 16 * (lane % RA::kLanes)) = make_uint4(t.a[j][0], t.a[j][1], t.a[j][2], t.a[j][3]);
                }
                if (mine) t.x[0].to(lds_x), t.x[1].to(lds_x + RX::kBytes);
            } else if (s < s1) {
                rest(lds_a);
            }
            load(t, s + 2);
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
            __builtin_amdgcn_s_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
            if (s < s1 && mine) {
#pragma unroll
                for (int h = 0; h < H; h++) {
                    const Eight<XB> x0 = RX::from(lds_x, h), x1 = RX::from(lds_x + RX::kBytes, h);
#pragma unroll
                    for (int r = 0; r < RT; r++) {
                        const Eight<WB> a = RA::from(lds_a + r * RA::kBytes, h);
                        acc[0][r] = product(a, x0, acc[0][r]);
                        acc[1][r] = product(a, x1, acc[1][r]);
                    }
                }
            }
        };
        Step even, odd;
        load(even, s0);
        load(odd, s0 + 1);
#pragma unroll 1
        for (int n = 0; n < turns; n += 2) {
            turn(even, n);
            turn(odd, n + 1);
        }
        // The second half's sums onto the first's.
        float(*join)[P] = (float(*)[P])lds;
        __syncthreads();
#pragma unroll
        for (int c = 0; c < 2; c++)
#pragma unroll
            for (int r = 0; r < RT; r++)
                if (half) *(v4f*)&join[32 * w + 16 * c + col][16 * r + 4 * g] = acc[c][r];
        __syncthreads();
#pragma unroll
        for (int c = 0; c < 2; c++)
#pragma unroll
            for (int r = 0; r < RT; r++) {
                const int at = 32 * w + 16 * c + col, rank = r0 + 16 * r + 4 * g;
                if (half || at >= u.n || rank >= p.rank_pitch) continue;
                *(v4f*)(p.h + ((int64_t)split * p.rows + rows[at]) * p.rank_pitch + rank) = acc[c][r] + *(const v4f*)&join[at][16 * r + 4 * g];
            }
        __syncthreads();
    }
}

// h as the second product takes it: the parts of K summed and scaled, against bf16 factors
// as three bf16, [row][term][ranks], zeros behind R.
template <bool WB>
__device__ __forceinline__ v4f h_of(const LoraBatched& p, int64_t row, int r, float scale) {
    const float* from = p.h + row * p.rank_pitch + r;
    const int64_t step = (int64_t)p.rows * p.rank_pitch;
    v4f sum = {0, 0, 0, 0};
    if (r >= p.R) return sum;
#pragma unroll 1
    for (int s = 0; s < p.splits; s += 4) {
        v4f x[4];
#pragma unroll
        for (int e = 0; e < 4; e++) x[e] = *(const v4f*)(from + min(s + e, p.splits - 1) * step);
        sum += x[0];
#pragma unroll
        for (int e = 1; e < 4; e++)
            if (s + e < p.splits) sum += x[e];
    }
#pragma unroll
    for (int e = 0; e < 4; e++) sum[e] = r + e < p.R ? sum[e] * scale : 0.0f;
    return sum;
}
template <bool WB>
__device__ __forceinline__ void store_h(v4f sum, void* to, int term) {
    if constexpr (WB) {
#pragma unroll
        for (int t = 0; t < 3; t++) {
            // What bf16 would round to infinity has its largest value first.
            constexpr float kTop = 0x1.fep127f;
            float x[4];
#pragma unroll
            for (int e = 0; e < 4; e++) x[e] = t == 0 && __builtin_isfinite(sum[e]) ? fminf(fmaxf(sum[e], -kTop), kTop) : sum[e];
            const uint32_t lo = f32x2_to_bf16x2(x[0], x[1]), hi = f32x2_to_bf16x2(x[2], x[3]);
            *(uint2*)((uint16_t*)to + t * term) = make_uint2(lo, hi);
            // What an infinity leaves is 0, not NaN.
            const float y[4] = {bf16_to_f32(lo & 0xffffu), bf16_to_f32(lo >> 16), bf16_to_f32(hi & 0xffffu), bf16_to_f32(hi >> 16)};
#pragma unroll
            for (int e = 0; e < 4; e++) sum[e] = __builtin_isfinite(y[e]) ? sum[e] - y[e] : 0.0f;
        }
    } else {
        *(v4f*)to = sum;
    }
}

// The same once for all, where many blocks want it (4352 rows on 64 ranks, six parts: each
// block of the update took 14 us to sum them).
template <bool WB>
__global__ __launch_bounds__(256) void lora_batched_join_kernel(LoraBatched p, int ranks) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, row = i / (ranks / 4);
    if (row >= p.rows) return;
    const int a = p.adapter[row], r = 4 * (int)(i - row * (ranks / 4));
    if (a < 0 || a >= p.adapters) return;
    store_h<WB>(h_of<WB>(p, row, r, p.scale ? p.scale[a] : 1.0f), (char*)p.joined + (row * ranks * (WB ? 3 : 1) + r) * (WB ? 2 : 4), ranks);
}

// The update.  A wave has 16 NT columns n of out: lane l's are the NT from NT (l % 16) on, column
// l % 16 of each of NT tiles of the matrix instruction, in rows 4 (l / 16) + i, so that
// 16 lanes read and write 128 bytes of a row together, 256 in fp32.  A block has 4 waves'
// columns `chunks` times for all
// rows of every `parts`-th class of its tile, `most` rows' h in LDS and 16 rows at a time, the
// base of the four times 16 after them loading meanwhile.  B's first KS steps of 32 ranks stay in
// registers, further ones are read again for each 16 rows.
template <bool WB, bool OB, int KS, bool WIDE>
__global__ __launch_bounds__(256, 2) void lora_batched_up_kernel(LoraBatched p, int tiles, int across, int around, int parts, int chunks, int most) {
    constexpr int T = WB ? 3 : 1;  // terms of h
    constexpr int O = OB ? 2 : 4;  // bytes of an element
    constexpr int A = !WIDE ? 1 : OB ? 4 : 2;  // bases ahead
    constexpr int NT = kUpTiles, kWave = 16 * NT, kBlock = 4 * kWave;
    typedef std::conditional_t<NT * O == 8, any2, any4> Run;
    __shared__ int rows[kLoraTile];
    extern __shared__ __align__(16) uint8_t lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int at = lora_place(blockIdx.x % around, around), tile = at / across, col = lane & 15, g = lane >> 4;
    if (tile >= tiles) return;
    const int ranks = (p.R + 31) / 32 * 32, pitch = ranks + (WB ? 8 : 4);
    uint16_t* hb = (uint16_t*)lds;  // [row][term][pitch]
    float* hf = (float*)lds;        // [row][pitch]
    const int first = (at - tile * across) * chunks * kBlock + kWave * wave;
    const int classes = p.counts[tile];
#pragma unroll 1
    for (int i = blockIdx.x / around; i < classes; i += parts) {
        const LoraClass cls = p.classes[(int64_t)tile * kLoraTile + i];
        const bool some = cls.adapter >= 0;
        const int all = __popcll(cls.rows[0]) + __popcll(cls.rows[1]);
        if (!some && p.out == p.base) continue;
#pragma unroll 1
        for (int skip = 0; skip < all; skip += most) {
            const int n = min(all - skip, most), cols = (n + 15) / 16;
            class_rows(cls.rows, tile, skip, most, rows);
            __syncthreads();
            // B's rows of a chunk, 32 ranks.
            auto load_b = [&](int n0, int k0, Eight<WB> (&b)[NT]) __attribute__((always_inline)) {
                const int k = k0 + 8 * g;
                const char* from[NT];
#pragma unroll
                for (int t = 0; t < NT; t++) from[t] = (const char*)p.B + (cls.adapter * p.b_adapter + min(n0 + NT * col + t, p.N - 1) * p.b_row) * (WB ? 2 : 4);
                if (p.R % 8 == 0) {
#pragma unroll
                    for (int t = 0; t < NT; t++) b[t] = load_eight<WB>(from[t], k < p.R ? k : 0);
#pragma unroll
                    for (int t = 0; t < NT; t++)
#pragma unroll
                        for (int i = 0; i < (WB ? 4 : 8); i++) b[t].w[i] = k < p.R ? b[t].w[i] : 0;
                } else {
#pragma unroll
                    for (int t = 0; t < NT; t++) b[t] = load_masked<WB>(from[t], k, p.R, p.b_end);
                }
            };
            // The base of 16 rows' columns (rows behind the last: the last again, and of no base
            // whatever out holds, unused).  No branch: what loads meet a branch is waited for
            // with all that came after it.
            Run base[A][4] = {};
            const char* const was = (const char*)(p.base ? p.base : p.out);
            const int64_t ld_was = p.base ? p.ld_base : p.ldo;
            auto load_base = [&](int n0, int c, Run (&base)[4]) __attribute__((always_inline)) {
#pragma unroll
                for (int i = 0; i < 4; i++) base[i] = __builtin_nontemporal_load((const Run*)(was + (rows[min(16 * c + 4 * g + i, n - 1)] * ld_was + n0 + NT * col) * O));
            };
            const int ahead = cols / A * A;  // tiles whose bases are loaded ahead
#pragma unroll 1
            for (int chunk = 0; chunk < chunks; chunk++) {
                const int n0 = first + kBlock * chunk;
                Eight<WB> b[KS][NT];
                if (some && n0 < p.N) {
#pragma unroll
                    for (int k = 0; k < KS; k++) load_b(n0, 32 * k, b[k]);
                }
                if (chunk == 0) {
                    if (ahead && first + kWave <= p.N) {
#pragma unroll
                        for (int j = 0; j < A; j++) load_base(first, j, base[j]);
                    }
                    if (some && WIDE) {  // also by a wave without columns
                        const int pieces = ranks * T * (WB ? 2 : 4) / 16, each = ranks * (WB ? 2 : 4) / 16;
                        constexpr int kMore = 6;
#pragma unroll 1
                        for (int j = threadIdx.x; j < n * pieces; j += 256 * kMore) {
                            uint4 v[kMore];
                            int c[kMore], e[kMore];
#pragma unroll
                            for (int i = 0; i < kMore; i++) {  // past the last: the last again
                                const int at = min(j + 256 * i, n * pieces - 1);
                                c[i] = at / pieces, e[i] = at - c[i] * pieces;
                                v[i] = *(const uint4*)((const char*)p.joined + ((int64_t)rows[c[i]] * pieces + e[i]) * 16);
                            }
#pragma unroll
                            for (int i = 0; i < kMore; i++) *(uint4*)(lds + (c[i] * T + e[i] / each) * pitch * (WB ? 2 : 4) + e[i] % each * 16) = v[i];
                        }
                        __syncthreads();
                    } else if (some) {
                        const float scale = p.scale ? p.scale[cls.adapter] : 1.0f;
#pragma unroll 1
                        for (int j = threadIdx.x; j < n * ranks / 4; j += 256) {
                            const int c = j / (ranks / 4), r = 4 * (j - c * (ranks / 4));
                            store_h<WB>(h_of<WB>(p, rows[c], r, scale), lds + (c * T * pitch + r) * (WB ? 2 : 4), pitch);
                        }
                        __syncthreads();
                    }
                }
                if (n0 >= p.N) break;
                const bool inside = n0 + kWave <= p.N;
                auto turn = [&](int c, Run (&base)[4], bool inside) __attribute__((always_inline)) {
                    // Without an adapter -0, which leaves the base's own zeros their signs.
                    const float none = some || !p.base ? 0.0f : -0.0f;
                    v4f acc[NT];
#pragma unroll
                    for (int t = 0; t < NT; t++) acc[t] = v4f{none, none, none, none};
                    // (Rows behind the last are the last again.)
                    auto load_h = [&](int c, int k0, int term) __attribute__((always_inline)) {
                        Eight<WB> h;
                        if constexpr (WB) {
                            *(uint4*)h.w = *(const uint4*)(hb + (min(16 * c + col, n - 1) * T + term) * pitch + k0 + 8 * g);
                        } else {
                            *(v4f*)h.w = *(const v4f*)(hf + min(16 * c + col, n - 1) * pitch + k0 + 8 * g);
                            *(v4f*)(h.w + 4) = *(const v4f*)(hf + min(16 * c + col, n - 1) * pitch + k0 + 8 * g + 4);
                        }
                        return h;
                    };
                    auto multiply = [&](int k0, const Eight<WB> (&b)[NT]) __attribute__((always_inline)) {
#pragma unroll
                        for (int term = T - 1; term >= 0; term--) {
                            const Eight<WB> h = load_h(c, k0, term);
#pragma unroll
                            for (int t = 0; t < NT; t++) acc[t] = product(h, b[t], acc[t]);
                        }
                    };
                    if (some) {
#pragma unroll
                        for (int k = 0; k < KS; k++) multiply(32 * k, b[k]);
#pragma unroll 1
                        for (int k0 = 32 * KS; k0 < ranks; k0 += 32) {
                            Eight<WB> rest[NT];
                            load_b(n0, k0, rest);
                            multiply(k0, rest);
                        }
                        if constexpr (WB) {
                            // h's lower terms may be 0 or of another sign, which an infinite factor
                            // makes NaN of: where something is not finite, once more, such factors
                            // with the first term only.
                            float bad = 0.0f;
#pragma unroll
                            for (int t = 0; t < NT; t++)
#pragma unroll
                                for (int i = 0; i < 4; i++) bad = fmaf(acc[t][i], 0.0f, bad);
                            if (__builtin_expect(__any(bad != 0.0f), 0)) {
#pragma unroll
                                for (int t = 0; t < NT; t++) acc[t] = v4f{0, 0, 0, 0};
#pragma unroll 1
                                for (int k0 = 0; k0 < ranks; k0 += 32) {
                                    Eight<WB> all[NT];
                                    load_b(n0, k0, all);
#pragma unroll 1
                                    for (int term = T - 1; term >= 0; term--) {
                                        const Eight<WB> h = load_h(c, k0, term);
#pragma unroll
                                        for (int t = 0; t < NT; t++) acc[t] = product(h, term ? finite_of(all[t]) : all[t], acc[t]);
                                    }
                                }
                            }
                        }
                    }
                    if (inside) {
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            // A row behind the last writes the last's values once more.
                            char* to = (char*)p.out + (rows[min(16 * c + 4 * g + i, n - 1)] * p.ldo + n0 + NT * col) * O;
                            float y[NT];
#pragma unroll
                            for (int t = 0; t < NT; t++) {
                                const uint32_t w = base[i][OB ? t >> 1 : t];
                                const float before = OB ? bf16_to_f32(t & 1 ? w >> 16 : w & 0xffffu) : __uint_as_float(w);
                                y[t] = p.base ? acc[t][i] + before : acc[t][i];
                            }
                            Run w;
#pragma unroll
                            for (int t = 0; t < NT * O / 4; t++) w[t] = OB ? f32x2_to_bf16x2(y[2 * t % NT], y[(2 * t + 1) % NT]) : __float_as_uint(y[t]);
                            *(Run*)to = w;
                        }
                    } else {
                        // Element by element: all are loaded (behind the last: the last again)
                        // before one is used.
                        float was[4][NT] = {};
                        if (p.base) {
#pragma unroll
                            for (int i = 0; i < 4; i++) {
                                const int64_t from = rows[min(16 * c + 4 * g + i, n - 1)] * p.ld_base;
#pragma unroll
                                for (int t = 0; t < NT; t++) {
                                    const int64_t at = from + min(n0 + NT * col + t, p.N - 1);
                                    was[i][t] = OB ? bf16_to_f32(((const uint16_t*)p.base)[at]) : ((const float*)p.base)[at];
                                }
                            }
                        }
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            if (16 * c + 4 * g + i >= n) continue;
                            const int64_t to = rows[16 * c + 4 * g + i] * p.ldo;
#pragma unroll
                            for (int t = 0; t < NT; t++) {
                                const int at = n0 + NT * col + t;
                                if (at >= p.N) continue;
                                const float y = p.base ? acc[t][i] + was[i][t] : acc[t][i];
                                if (OB) ((uint16_t*)p.out)[to + at] = (uint16_t)f32_to_bf16(y);
                                else ((float*)p.out)[to + at] = y;
                            }
                        }
                    }
                };
                if (inside) {
                    // After its last tile a base is that of the next chunk's, if there is one.
                    const int next = chunk + 1 < chunks && n0 + kBlock + kWave <= p.N ? n0 + kBlock : n0;
#pragma unroll 1
                    for (int c = 0; c < ahead; c += A) {
                        const bool end = c + A >= ahead;
#pragma unroll
                        for (int j = 0; j < A; j++) {
                            turn(c + j, base[j], true);
                            load_base(end ? next : n0, end ? j : c + j + A, base[j]);
                        }
                    }
#pragma unroll 1
                    for (int c = ahead; c < cols; c++) {
                        Run one[4];
                        load_base(n0, c, one);
                        turn(c, one, true);
                    }
                } else {
#pragma unroll 1
                    for (int c = 0; c < cols; c++) turn(c, base[0], false);
                }
            }
            __syncthreads();
        }
    }
}

namespace {

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

int rank_pitch(int64_t R) { return (int)(16 * ceil_div(R, 16)); }

constexpr size_t kMaxLds = 159 << 10;  // a compute unit's 160 KB, less the rows' numbers

// Blocks that share a tile's classes are so many that there are about kParts: where rows are
// mixed each has few classes, elsewhere most end at once (4352 rows of eight adapters at random, on
// 16 ranks 60 us, on 64 104; with a fourth of the blocks 69 and 110; runs of rows 37 and 53, 41 and
// 53; but 2048 rows in runs on 32 ranks 29, 27).  Not the wide ones of the first pass, of which
// one fills a compute unit (at random on 64 ranks 112 us, 110 with 256).
constexpr int64_t kParts = 4096;

// Whether blocks take whole tiles' rows (whose loads are whole steps of K): what that saves
// are readings of A, so it is for many ranks.  Microseconds for eight adapters of 4096 x 4096,
// a run of rows each and at random: 4352 rows on 64 ranks 53 and 104, not wide 70 and 100;
// 1024 rows 32 and 41, 39 and 36; 512 rows 24 and 29, 26 and 25; 4352 rows on 16 ranks 42 and
// 82, 37 and 60.
bool is_wide(int64_t rows, int64_t K, int64_t R) { return rows >= 1024 && K >= 512 && R > 32; }

// Parts of K: enough blocks where there are few rows, a part no shorter than 512; of wide
// blocks no more than fit the compute units at once, with room for tiles of two classes.
// (64 rows of 4096: 15.9 us with eight at most, 16.9 with four, 16.3 with 16.)
int splits_of(int64_t rows, int64_t K, int64_t R) {
    const int64_t want = is_wide(rows, K, R) ? 256 / (ceil_div(rows, kLoraTile) * 5 / 4) : 512 / ceil_div(rows, kFewCols);
    return (int)std::clamp<int64_t>(want, 1, std::min<int64_t>(kSplits, ceil_div(K, 512)));
}

int places(int n) { return n >= kSpread ? (n + 7) / 8 * 8 : n; }

template <bool XB, bool WB, int RT>
void down_ranks(hipStream_t stream, const LoraBatched& p, int tiles, int classes, int groups) {
    const int around = places(tiles * p.splits);
    if (RT == 4 && p.joined) {
        const int parts = (int)std::clamp<int64_t>(256 / ((int64_t)tiles * p.splits * groups), 1, classes);
        hipLaunchKernelGGL((lora_batched_down_wide_kernel<XB, WB>), dim3((unsigned)(around * parts), 1, (unsigned)groups), dim3(512), 0, stream,
                           p, tiles, around, parts);
        return;
    }
    // A tile's units are more than its classes by those of more than kFewCols rows.
    const int units = std::min(classes + kLoraTile / kFewCols - 1, kLoraTile);
    const int parts = (int)std::clamp<int64_t>(kParts / ((int64_t)tiles * p.splits * groups), 1, units);
    hipLaunchKernelGGL((lora_batched_down_kernel<XB, WB, RT>), dim3((unsigned)(around * parts), 1, (unsigned)groups), dim3(256), 0, stream, p, tiles,
                       around, parts);
}

template <bool XB, bool WB>
void down(hipStream_t stream, const LoraBatched& p, int tiles, int classes) {
    const int rt = (p.R + 15) / 16;
    if (rt == 1) down_ranks<XB, WB, 1>(stream, p, tiles, classes, 1);
    else if (rt == 2) down_ranks<XB, WB, 2>(stream, p, tiles, classes, 1);
    else down_ranks<XB, WB, 4>(stream, p, tiles, classes, (rt + 3) / 4);
}

template <bool WB, bool OB, int KS, bool WIDE>
hipError_t up_ranks(hipStream_t stream, const LoraBatched& p, int tiles, int classes) {
    const int ranks = (p.R + 31) / 32 * 32, block_n = 64 * kUpTiles, all = (p.N + block_n - 1) / block_n;
    const size_t row = WB ? 3 * (ranks + 8) * 2 : (ranks + 4) * 4;
    const int most = row * kLoraTile <= kMaxLds ? kLoraTile : kLoraTile / 2;
    const size_t lds = row * std::min(most, (p.rows + 15) / 16 * 16);
    if (lds > 65536) {
        const hipError_t e = hipFuncSetAttribute((const void*)lora_batched_up_kernel<WB, OB, KS, WIDE>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess) return e;
    }
    // A block's first loads take 10 us whatever it has to do with them.  Two fit a compute unit:
    // of many rows no more than run at once, a fifth of them for tiles of two classes
    // (4352 rows of 5120 columns in 34 tiles of 10 blocks: 31 us; in 34 of 20, the last of which
    // begin when the first have ended, 42; of 5, 44).
    const int want = (int)std::max<int64_t>(1, (WIDE ? 410 : 1024) / tiles);
    const int chunks = (all + std::min(want, all) - 1) / std::min(want, all), across = (all + chunks - 1) / chunks;
    const int parts = (int)std::clamp<int64_t>(kParts / ((int64_t)tiles * across), 1, classes);
    const int around = places(tiles * across);
    const dim3 grid((unsigned)(around * parts)), block(256);
    if (WIDE) {
        const int64_t pieces = (int64_t)p.rows * (ranks / 4);
        hipLaunchKernelGGL(lora_batched_join_kernel<WB>, dim3((unsigned)ceil_div(pieces, 256)), block, 0, stream, p, ranks);
    }
    hipLaunchKernelGGL((lora_batched_up_kernel<WB, OB, KS, WIDE>), grid, block, lds, stream, p, tiles, across, around, parts, chunks, most);
    return hipGetLastError();
}

template <bool WB, bool OB>
hipError_t up(hipStream_t stream, const LoraBatched& p, int tiles, int classes) {
    return p.joined ? up_ranks<WB, OB, 2, true>(stream, p, tiles, classes) : up_ranks<WB, OB, 1, false>(stream, p, tiles, classes);
}

// h, the tiles' classes and how many they are.
size_t h_bytes(int64_t rows, int64_t K, int64_t R) { return (size_t)splits_of(rows, K, R) * rows * rank_pitch(R) * sizeof(float); }

}  // namespace

size_t lora_batched_workspace(int64_t rows, int64_t K, int64_t R) {
    const size_t joined = is_wide(rows, K, R) ? (size_t)rows * (32 * ceil_div(R, 32)) * 6 : 0;  // three bf16, or fp32
    return h_bytes(rows, K, R) + (size_t)ceil_div(rows, kLoraTile) * (kLoraTile * sizeof(LoraClass) + 16) + joined;
}

hipError_t launch_lora_batched(hipStream_t stream, LoraBatched p) {
    p.splits = splits_of(p.rows, p.K, p.R);
    p.rank_pitch = rank_pitch(p.R);
    const int tiles = (p.rows + kLoraTile - 1) / kLoraTile;
    auto end = [](const void* from, int64_t elements, bool b16) { return (const char*)from + elements * (b16 ? 2 : 4); };
    p.x_end = end(p.x, (p.rows - 1) * p.ldx + p.K, p.x_bf16);
    p.a_end = end(p.A, (p.adapters - 1) * p.a_adapter + (p.R - 1) * p.a_row + p.K, p.w_bf16);
    p.b_end = end(p.B, (p.adapters - 1) * p.b_adapter + (p.N - 1) * p.b_row + p.R, p.w_bf16);
    p.classes = (LoraClass*)((char*)p.h + h_bytes(p.rows, p.K, p.R));
    p.counts = (int*)(p.classes + (int64_t)tiles * kLoraTile);
    p.joined = is_wide(p.rows, p.K, p.R) ? (void*)((char*)p.counts + (int64_t)tiles * 16) : nullptr;
    const int classes = std::min({kLoraTile - 1, p.adapters, p.rows}) + 1;  // of a tile, at most
    if (p.x_bf16) p.w_bf16 ? down<true, true>(stream, p, tiles, classes) : down<true, false>(stream, p, tiles, classes);
    else p.w_bf16 ? down<false, true>(stream, p, tiles, classes) : down<false, false>(stream, p, tiles, classes);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    if (p.w_bf16) return p.out_bf16 ? up<true, true>(stream, p, tiles, classes) : up<true, false>(stream, p, tiles, classes);
    return p.out_bf16 ? up<false, true>(stream, p, tiles, classes) : up<false, false>(stream, p, tiles, classes);
}

}  // namespace phi_dev
