// kvq_chunk.hpp -- launch arguments of chunk attention (kvq_chunk.hip,
// kvq_chunk_mfma.hpp); kvq_share_capi.cpp validates and fills them.
#pragma once

#include "kvq_internal.hpp"

namespace kvq {

struct ChunkArgs {
    PageMap pages;
    FastDiv page;            // division by the page size
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
    // Matrix-core kernel.
    FastDiv heads, group;    // divisions by Hkv and G
    int tile_tokens;         // new tokens of a query tile
    int slots;               // items that a launch aims for where keys are split
    int max_splits;          // most splits of a sequence's keys
    int max_tiles;           // query tiles that the launch has room for
    int* counters;           // [units] arrivals of a split tile's workgroups; left at 0
    float* part_acc;         // [items, rows of a tile, D] partial records of split tiles
    float* part_ml;          // [items, rows of a tile, 2]
};

constexpr int kChunkKeys = 64;   // keys of a tile

struct ChunkPlan {
    bool mfma;       // the matrix-core kernel
    int D, rows;     // its padded head dim and a tile's query rows
    int tile_tokens, slots, max_splits, max_tiles;
    unsigned items;  // workgroups
    size_t records;  // partial records (0: nothing is split)
    size_t bytes;    // workspace
};
// vec_ok: rows and caches are aligned as the matrix-core kernel loads them.
ChunkPlan chunk_plan(const ChunkArgs& a, bool vec_ok);
hipError_t launch_chunk(ChunkArgs a, const ChunkPlan& p, void* workspace, hipStream_t stream);

}  // namespace kvq
