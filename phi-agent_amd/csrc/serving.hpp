// Parameters of the kernels behind include/phi_serving.h.
#pragma once

#include "decoder.hpp"

namespace phi_dev {

// A launch's threads are counted in 32 bits: blocks of 256, at most.
constexpr int64_t kMaxBlocks = (1 << 24) - 1;

// [tokens, heads, dim] vectors, strides in elements.
struct RotaryHeads {
    const void* in;
    void* out;
    int64_t in_token, in_head, out_token, out_head;
    int heads;
};

// q rotated; k and v, of c.heads each, into the cache (heads 0: none).
struct Rotary {
    RotaryHeads q, k, v;
    const int64_t* positions;
    const double* freq;
    const int64_t* slots;
    int64_t tokens;
    int dim, rot;
    float scale;
    bool bf16, interleaved;
};
hipError_t launch_rotary(hipStream_t stream, const Rotary& p, const KvCache& c);

struct KvCopy {
    KvCache from, to;
    const int32_t* from_blocks;
    const int32_t* to_blocks;
    const int32_t* tokens;
    int64_t n;
};
hipError_t launch_kv_cache_copy(hipStream_t stream, const KvCopy& p);

// out = base + scale[a] B[a] (A[a] x), a = adapter of the row; strides in elements.
struct LoraBatched {
    const void* x;
    const void* A;   // [adapters, R, K]
    const void* B;   // [adapters, N, R]
    const int32_t* adapter;
    const float* scale;  // null: 1
    const void* base;    // null: 0
    void* out;
    float* h;        // [splits][rows][rank_pitch]: parts of A x
    struct LoraClass* classes;  // [tiles][128]
    int* counts;                // [tiles]
    void* joined;               // h as the second product takes it; null: from its parts
    int64_t ldx, a_adapter, a_row, b_adapter, b_row, ld_base, ldo;
    int rows, K, N, R, adapters, splits, rank_pitch;
    bool x_bf16, w_bf16, out_bf16;
    const char *x_end, *a_end, *b_end;  // of the operands' memory
};
hipError_t launch_lora_batched(hipStream_t stream, LoraBatched p);
size_t lora_batched_workspace(int64_t rows, int64_t K, int64_t R);

}  // namespace phi_dev
