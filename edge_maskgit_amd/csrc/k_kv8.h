// k_kv8.h — where things lie in the 8-bit key / value cache (include/mgh.h has the layout)
#pragma once
#include "mgh_common.h"
#include "mgh_kernels.h"

namespace mgh {

// tokens of sequence b before and after a call's new ones; false: numbers that the cache cannot hold
__device__ __forceinline__ bool spans(const Kv8& c, const int32_t* lens, const int32_t* fresh, int S, int b, int& len,
                                      int& total) {
    len = lens[b];
    const int n = fresh ? fresh[b] : S;
    const int64_t t = (int64_t)len + n;
    total = (int)t;
    return len >= 0 && n >= 0 && n <= S && t <= (int64_t)c.max_blocks * kKvBlock;
}

// the page of a sequence's block, or -1
__device__ __forceinline__ int64_t page_of(const Kv8& c, int b, int block) {
    const int64_t p = c.table[b * c.table_stride + block];
    return p >= 0 && p < c.pages ? p : -1;
}

// V's codes of a block: the 8 tokens of a matrix instruction's operand of one feature side by side, two
// features in 16 bytes
__device__ __forceinline__ int v_at(int t, int d) { return ((d >> 1) * 4 + (t >> 3)) * 16 + (d & 1) * 8 + (t & 7); }

}  // namespace mgh
