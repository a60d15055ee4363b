// kvq_chunk.hpp -- launch arguments of chunk attention (kvq_chunk.hip);
// kvq_share_capi.cpp validates and fills them.
#pragma once

#include "kvq_internal.hpp"

namespace kvq {

struct ChunkArgs {
    PageMap pages;
    const int32_t* offsets;
    const int32_t* lengths;
    const int32_t* granted;  // or null
    const void* q;
    void* out;
    const int8_t* k;
    const int8_t* v;
    const float* ks;
    const float* vs;
    int64_t q_stride, out_stride;  // elements from a token to the next
    int B, Hq, Hkv, G, d, T, max_len;
    bool bf16, causal;
    float scale_log2;  // softmax scale * log2 e
};
// vec_ok: 16-byte aligned q and out rows and caches.
hipError_t launch_chunk(const ChunkArgs& a, bool vec_ok, void* workspace, hipStream_t stream);

}  // namespace kvq
