// kvq_share.hpp -- launch arguments of the operators on shared pages
// (kvq_share.hip); kvq_share_capi.cpp validates and fills them.
#pragma once

#include "kvq_internal.hpp"

namespace kvq {

struct ForkArgs {
    const int32_t* parents;
    const int32_t* keep;  // or null: all
    const int32_t* lengths;
    const int32_t* table;
    const int32_t* shares;
    int32_t* free_pages;
    const int32_t* free_count;
    int32_t* new_lengths;
    int32_t* new_table;
    int32_t* new_shares;
    int32_t* new_free_count;
    int32_t* copy_src;
    int32_t* copy_dst;
    int B, max_pages, num_pages;
    int cap;  // tokens a row can hold
    FastDiv page;
    // Workspace, all zero between calls.
    int* delta;    // [num_pages] holders that a page gains (loses: negative)
    int* writers;  // [num_pages] rows that end inside the page
    int* first;    // [num_pages] B - the first of them
    int* freed;    // [num_pages] pages that have become free, ascending
    int* want;     // [B] tokens that a row keeps
    int* stage;    // [B, max_pages] new rows
};
size_t fork_workspace(const ForkArgs& a);
void fork_place(ForkArgs& a, void* workspace);
hipError_t launch_page_fork(const ForkArgs& a, hipStream_t stream);

struct CopyArgs {
    const int32_t* src;
    const int32_t* dst;
    int n, layers, num_pages;
    static constexpr int kArrays = 6;
    char* base[kArrays];     // K, V, their scales, bounds and theirs (or null)
    size_t bytes[kArrays];   // of a page
    size_t begin[kArrays];   // first piece of each, of a page's in all arrays
    size_t pieces;
    FastDiv pairs;           // division by n
};
hipError_t launch_page_copy(const CopyArgs& a, hipStream_t stream);

struct CompactArgs {
    const int32_t* lengths;
    const int32_t* table;
    const int32_t* shares;  // or null with new_shares
    const int32_t* free_pages;
    const int32_t* free_count;
    int32_t* new_table;
    int32_t* new_shares;
    int32_t* new_free_pages;
    int32_t* copy_src;
    int32_t* copy_dst;
    int32_t* moved;
    int B, max_pages, num_pages, max_moves;
    int cap;
    FastDiv page;
    // Workspace of pools of up to 2^18 pages: free pages before and after as bits,
    // and counts a word; nothing of it is read before it is written.
    unsigned* before;
    unsigned* after;
    int* place;  // [words] where a word's first free page goes in the stack
    int* hole;   // [words] pages below the word that could be moved to
    int* high;   // [words] pages above the word that could move
    // Of larger ones, cleared at the start.
    int* state;  // [num_pages] -1: free, 0: in use, otherwise where the page moves to, + 1
    int* taken;  // [num_pages] 1: a free page that another moves to
};
size_t compact_workspace(const CompactArgs& a);
void compact_place(CompactArgs& a, void* workspace);
hipError_t launch_page_compact(const CompactArgs& a, hipStream_t stream);

}  // namespace kvq
