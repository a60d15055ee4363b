// kvq_pages.hpp -- launch arguments of the operators around a paged cache
// (kvq_pages.hip, kvq_select.hip); kvq_pages_capi.cpp validates and fills them.
#pragma once

#include "kvq_internal.hpp"

namespace kvq {

struct PageMapArgs {
    const int32_t* new_tokens;
    const int32_t* lengths;
    int32_t* table;
    int32_t* free_pages;
    const int32_t* free_count;
    int32_t* new_lengths;
    int32_t* new_free_count;
    int32_t* granted;
    int32_t* offsets;
    int32_t* slot_map;
    int32_t* token_seq;
    int32_t* token_pos;
    int* arrivals;  // workgroups that are done (null: one workgroup); left at 0
    int B, max_pages, num_pages, T;
    int cap;  // tokens a sequence can hold, max_pages * page size
    FastDiv page;
};
int page_map_groups(const PageMapArgs& a);  // workgroups of the launch
hipError_t launch_page_map(const PageMapArgs& a, hipStream_t stream);

struct SlotArgs {
    const int32_t* slots;
    int8_t* k;
    int8_t* v;
    float* ks;
    float* vs;
    void* k_rows;  // the packed rows: read by slot_write, written by slot_read
    void* v_rows;
    int64_t k_stride, v_stride;  // elements from a token's rows to the next token's
    int64_t head_stride;         // elements from a row to the next head's
    int T, Hkv, d;
    int slots_in_pool;  // num_pages * page size
    FastDiv page, heads;
};
// vec_ok: rows 16-byte aligned at every token and head, caches 8-byte aligned.
hipError_t launch_slot_write(const SlotArgs& a, bool bf16, bool vec_ok, hipStream_t stream);
hipError_t launch_slot_read(const SlotArgs& a, bool bf16, bool vec_ok, hipStream_t stream);

struct BoundsArgs {
    PageMap pages;
    const int32_t* start;    // or null: 0
    const int32_t* lengths;  // or null: max_len
    const int8_t* k;
    const float* ks;
    int8_t* bounds;
    float* scale;
    int B, Hkv, d, max_len;
    FastDiv heads;  // division by Hkv
};
hipError_t launch_page_bounds(const BoundsArgs& a, bool vec_ok, hipStream_t stream);

struct SelectArgs {
    BoundsArgs b;  // start unused
    const float* q;
    int G;
    int keep_first, keep_last, max_selected;
    int32_t* selected;
    int32_t* selected_lengths;
    unsigned* keys;  // [B * Hkv, key_stride] ranks of the scored pages, or null: kept in LDS
    int key_stride;
    int* counters;   // [B * Hkv] arrivals of a unit's workgroups (splits > 1); left at 0
    int splits;      // workgroups per (sequence, kv head)
};
struct SelectPlan {
    int splits;
    int lds_keys;  // ranks a workgroup keeps in LDS, 0: none
    int key_stride;
    size_t key_bytes;
};
// Workgroups per unit and where the ranks go, for sequences of up to max_pages pages.
// vec_ok: 16-byte aligned q, keys and bounds.
SelectPlan select_plan(int units, int G, int d, bool vec_ok, int max_pages, int max_selected);
hipError_t launch_select(const SelectArgs& a, const SelectPlan& p, bool vec_ok, hipStream_t stream);

}  // namespace kvq
