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
