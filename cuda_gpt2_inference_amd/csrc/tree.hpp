// tree.hpp -- the call that kvattn.hip hands over to tree.hip, and what the kernels for trees of drafted
// tokens share.
#pragma once
#include <stddef.h>

#include "kvattn.h"

namespace kvattn_internal {
constexpr int kMaxMaskWords = 4;                    // 64-bit words of a token's mask
constexpr int kMaxTree = 64 * kMaxMaskWords;        // tokens of a sequence's tree

// Attention of a tree's tokens over a paged cache, of any type; arguments checked but for the plan's.
struct AttendTree {
    void* out;
    const void* qkv;
    const void* kv;
    const float* scale;
    const int* table;
    const int* start;
    const int* lens;
    const unsigned long long* masks;
    int mask_words, max_pages, page_rows, num_pages;
    int B, NH, maxT, num_tokens, max_new, S, kv_dtype;
    void* ws;
    size_t ws_bytes;
    void* stream;
};
__attribute__((visibility("hidden"))) int attend_tree(const AttendTree& c);

void set_last_hip_error(int e);   // kvattn.hip: read back by kvattn_last_hip_error
int merge_poll_limit();           // kvattn.hip: kvattn_set_merge_poll_limit's bound
}  // namespace kvattn_internal
