// Interface between the host code of the cache's operators (cache_shim.cpp) and
// their kernels (cache_rows.hip, cache_few.hip, cache_many.hip, cache_prompt.hip).  Nothing here is part of the C-ABI.
#pragma once

#include "cache_plan.hpp"
#include "q8_cache.h"
#include "q8_internal.hpp"

namespace q8 {

// n / d for n < 2^31 as a product's upper half and a shift; d >= 1.
struct Divisor {
    uint32_t d, mul, shift;
};
inline Divisor divisor(uint32_t d) {
    uint32_t s = 0;
    while (s < 31 && (1ull << s) < d) ++s;
    // mul = ceil(2^(31 + s) / d) < 2^32, off by less than 2^s of 2^(31 + s): exact for 31 bits
    return Divisor{d, (uint32_t)(((1ull << (31 + s)) + d - 1) / d), s};
}

struct Rotary {
    const void* x;
    const int32_t* positions;
    const float* freq;
    void* y;
    uint32_t ldx, ldp, ldy, tokens, heads;
    int inverse;
    q8_rotation form;
};
Q8_INTERNAL hipError_t launch_rotary(int dtype, const Rotary& p, hipStream_t stream);

// The cache and the sequences, as kernels take them.
struct Paged {
    int8_t* k;
    int8_t* v;
    float* k_scale;
    float* v_scale;
    uint32_t pages, page_tokens, heads, dim, pitch;
    const int32_t* starts;
    const int32_t* lengths;
    const int32_t* table;
    uint32_t seqs, tokens, width, table_ld;
    Divisor page;               // by page_tokens
};

struct CacheRows {
    Paged at;
    void* k;
    void* v;
    uint32_t ldk, ldv;
};
Q8_INTERNAL hipError_t launch_cache_write(int dtype, const CacheRows& p, hipStream_t stream);
Q8_INTERNAL hipError_t launch_cache_read(int dtype, const CacheRows& p, hipStream_t stream);

struct Attention {
    Paged at;
    const void* q;
    void* out;
    float* lse;                 // may be null
    uint32_t ldq, ldo, heads, group, window;
    float scale;
};
// One launch of it: the sequences of more than `least` and at most `most` rows (new tokens times the heads that share
// one of the cache's), in tiles that `slots` are no fewer than, each one's keys in pieces of `piece`.
struct AttentionArgs {
    Attention a;
    Divisor by_group;
    uint32_t slots, least, most, piece;
    float* sums;        // pieces x tokens x heads x held dim
    float* stats;       // pieces x tokens x heads: R, l
    uint32_t* tickets;  // of each tile: the pieces that are done; 0 before and after a launch
    char* images;       // null: none; image_bytes() for each sequence, head of the cache and 64 keys
    uint32_t images_each;   // of a sequence and head
};
Q8_INTERNAL hipError_t launch_few(int dtype, const AttentionArgs& g, uint32_t pieces, hipStream_t stream);
Q8_INTERNAL hipError_t launch_many(int dtype, const AttentionArgs& g, uint32_t pieces, hipStream_t stream);
Q8_INTERNAL hipError_t launch_prompt(int dtype, const AttentionArgs& g, uint32_t pieces, hipStream_t stream);

}  // namespace q8
