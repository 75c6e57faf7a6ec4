// Parameters of the kernels behind include/phi_serving.h.
#pragma once

#include "decoder.hpp"

namespace phi_dev {

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

}  // namespace phi_dev
