// Device helpers of the cache's operators: where a token's rows lie.
#pragma once

#include "cache_internal.hpp"
#include "q8_device.hpp"

namespace q8 {

__device__ __forceinline__ uint32_t divide(uint32_t n, const Divisor& by) {      // n < 2^31
    return (uint32_t)((uint64_t)n * by.mul >> (31 + by.shift));
}

// Rows of sequence b's chunk, cut to the rows there are.
__device__ __forceinline__ int chunk_begin(const Paged& c, uint32_t b) { return min(max(c.starts[b], 0), (int)c.tokens); }
__device__ __forceinline__ int chunk_end(const Paged& c, uint32_t b) { return min(max(c.starts[b + 1], 0), (int)c.tokens); }

// Row of head 0 for position p of sequence b, or -1 (p may be anything).
__device__ __forceinline__ int64_t row_at(const Paged& c, uint32_t b, int64_t p) {
    if (p < 0 || p >= 0x7fffffff) return -1;
    const uint32_t index = divide((uint32_t)p, c.page);
    if (index >= c.width) return -1;
    const int page = c.table[(uint64_t)b * c.table_ld + index];
    return (uint32_t)page >= c.pages ? -1 : (int64_t)page * c.heads * c.page_tokens + ((uint32_t)p - index * c.page_tokens);
}

}  // namespace q8
