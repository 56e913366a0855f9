// qdc_cache.hpp -- what the kernels of the paged cache share.
#pragma once

#include "qdc_common.hpp"
#include "qdc_hip_cache.h"

namespace qdc {

// log2 of a page size that the cache takes, -1 for any other.
static inline int page_shift(int64_t page_size) {
    for (int s = 4; s <= 8; ++s)
        if (page_size == (int64_t)1 << s) return s;
    return -1;
}

__device__ __forceinline__ void raise_flag(int32_t *error_flag) {
    if (error_flag) atomicOr(error_flag, 1);
}

// Inclusive prefix sum over each row of 16 lanes, and over the wavefront: lane moves of
// the vector unit, a few cycles each where a move through LDS takes a hundred.
__device__ __forceinline__ int row_scan(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);  // from 1, 2, 4, 8 below
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
    return v;
}
__device__ __forceinline__ int wave_scan(int v) {
    v = row_scan(v);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row 0 into 1, 2 into 3
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // rows 0, 1 into 2, 3
    return v;
}

// A device range an entry point reads or writes.
struct Range {
    const void *p;
    int64_t bytes;
};

// Whether an output overlaps an input or another output.
static inline bool any_alias(const Range *outs, int n_outs, const Range *ins, int n_ins) {
    for (int i = 0; i < n_outs; ++i) {
        for (int j = 0; j < n_ins; ++j)
            if (overlaps(outs[i].p, outs[i].bytes, ins[j].p, ins[j].bytes)) return true;
        for (int j = 0; j < i; ++j)
            if (overlaps(outs[i].p, outs[i].bytes, outs[j].p, outs[j].bytes)) return true;
    }
    return false;
}

// Bytes that a [tokens, heads] grid of rows of `dim` elements spans.
static inline int64_t grid_span(int64_t tokens, int64_t heads, int64_t tok, int64_t head,
                                int64_t dim, int64_t es) {
    return tokens > 0 ? ((tokens - 1) * tok + (heads - 1) * head + dim) * es : 0;
}

}  // namespace qdc
