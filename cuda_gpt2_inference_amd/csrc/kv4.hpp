// kv4.hpp -- the 4-bit cache types shared by the kernels that read and write such caches, and the
// calls that kvattn.hip hands over for them.
//
// A row of 64 channels is 32 bytes of codes (channel 2i in the low half of byte i, 2i+1 in the high
// half) and one float scale; a value is code * scale.
//   INT4      scale = amax * (1/7), the nibble holds round(x / scale) + 8 (1 .. 15; 8 is zero)
//   FP4_E2M1  scale = amax * (1/6), sign bit and one of 0 0.5 1 1.5 2 3 4 6, ties to the even code
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "kvattn.h"

namespace kvattn_internal {
inline bool is_4bit(int dt) { return dt == KVATTN_KV_INT4 || dt == KVATTN_KV_FP4_E2M1; }

// One attention call over a 4-bit cache.  table != nullptr: paged (R = page_rows), else one slot of
// maxT rows per sequence.  start != nullptr: sequence b's queries are the token rows
// start[b] .. start[b+1]-1 of qkv and out, and lens holds positions; else one token a sequence and
// lens holds the current token's position (lens == nullptr: the library's own).
struct Attend4 {
    void* out;
    const void* qkv;
    const void* kv;
    const float* scale;
    const int* table;
    const int* start;
    const int* lens;
    int max_pages, page_rows, num_pages;
    int B, NH, maxT, num_tokens, max_new, lens_per_seq, len_hint, S, kv_dtype;
    void* ws;
    size_t ws_bytes;
    void* stream;
};
__attribute__((visibility("hidden"))) int attend4(const Attend4& c, bool launch);   // launch false: the checks alone

// The launch shape attend4 takes: segments per head, and the least tiles of 64 positions of one.
struct Plan4 {
    int waves, S, seg_tiles;
};
__attribute__((visibility("hidden"))) int plan4(int heads, int queries, int maxT, int len_hint, bool ragged, int S,
                                                 Plan4& p);

// The append into a 4-bit cache: K and V of one token a sequence (pages.hip).
__attribute__((visibility("hidden"))) int append4(void* kv, float* scale, const void* qkv, int B, int NH, int maxT,
                                                  const int* cur_len, int lens_per_seq, const int* table,
                                                  int max_pages, int page_rows, int num_pages, int kv_dtype,
                                                  void* stream);

void set_last_hip_error(int e);   // kvattn.hip: read back by kvattn_last_hip_error
}  // namespace kvattn_internal
