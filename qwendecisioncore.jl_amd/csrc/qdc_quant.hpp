// qdc_quant.hpp -- what the kernels on 4-bit weights and 8-bit rows share.
#pragma once

#include "qdc_common.hpp"
#include "qdc_hip_quant.h"

namespace qdc {

constexpr int kQ8Group = 128;   // columns of an 8-bit row that share a scale
constexpr int kW4Outputs = 16;  // of a block of 4-bit weights: a matrix instruction's rows,
constexpr int kW4Inputs = 128;  // and as many inputs as make it 16 bytes a lane
constexpr int kW4Words = 256;
constexpr int64_t kW4RowBytes = (int64_t)1 << 26;  // of x, from a row to the next, at most

// |v| as an integer that orders like it, NaN above infinity.
__device__ __forceinline__ uint32_t size_bits(float v) {
    return __float_as_uint(v) & 0x7fffffffu;
}
template <int CTRL> __device__ __forceinline__ uint32_t dpp_max(uint32_t v) {
    return max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, CTRL, 0xf, 0xf, true));
}
// The maximum over aligned groups of N lanes (as group_sum's sum).
template <int N> __device__ __forceinline__ uint32_t group_max(uint32_t v) {
    if constexpr (N >= 2) v = dpp_max<0xB1>(v);
    if constexpr (N >= 4) v = dpp_max<0x4E>(v);
    if constexpr (N >= 8) v = dpp_max<0x141>(v);
    if constexpr (N >= 16) v = dpp_max<0x140>(v);
    if constexpr (N >= 32) {
        const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        v = max(r[0], r[1]);
    }
    if constexpr (N >= 64) {
        const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        v = max(r[0], r[1]);
    }
    return v;
}

__device__ __forceinline__ uint32_t pack_bytes(int a, int b, int c, int d) {
    return (uint32_t)(a & 255) | (uint32_t)(b & 255) << 8 | (uint32_t)(c & 255) << 16 |
           (uint32_t)d << 24;
}

// The scale of a group of 8-bit values whose largest size is `most`, and values under it: the
// nearest whole numbers of v / scale, of two the even one.  Of bf16 values one in 400 is
// a half (127 times a quotient of 8 bits), of fp32 ones one in 14000 next to it: looked at they
// take rows of 16384 x 1024 from 12.6 to 14.0 us, and none (14.3 to 14.1; the norm 33.8 both).
struct Q8Scale {
    float scale, inverse;
    bool plain;  // whether there is an inverse

    __device__ explicit Q8Scale(uint32_t most) {
        scale = __uint_as_float(most) / 127.0f;
        // below 2^-100 the inverse may overflow; infinities and NaN: every value is 0
        plain = most >= 0x0d800000u && most < 0x7f800000u;
        inverse = plain ? 1.0f / scale : 0.0f;
    }
    // The nearest to v / s, which `near` is or the one beside it: what is left, v - near s, is
    // exact with FMA (24 bits from the last of v or of half of s), so its side of a half is
    // known.  q goes on where more than half of s is left, or half of it and q is odd.
    static __device__ __forceinline__ int settle(float near, float v, float s) {
        const float rest = __builtin_fmaf(-near, s, v);
        const int q = (int)near;
        const bool on = size_bits(rest + rest) + (uint32_t)(q & 1) > __float_as_uint(s);
        return q + (on ? (rest < 0.0f ? -1 : 1) : 0);
    }
    // Of a scale without an inverse: 2^64 times both, which is exact, as is half of such a scale.
    __device__ __forceinline__ int small(float v) const {
        if (!(scale > 0.0f && scale < __builtin_inff())) return 0;
        const float s = scale * 0x1p64f, w = v * 0x1p64f;
        // (one of few bits may be less than 1/127 of the largest value)
        return min(max(settle(__builtin_rintf(w / s), w, s), -127), 127);
    }
    // 4 values.  A product with the inverse is within 2^-16 of the quotient (127, twice rounded),
    // so only next to a half is there more to do.
    __device__ __forceinline__ uint32_t word(const float (&v)[4]) const {
        if (!plain) return pack_bytes(small(v[0]), small(v[1]), small(v[2]), small(v[3]));
        float q[4], off = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float near = v[i] * inverse;
            q[i] = __builtin_rintf(near);
            off = fmaxf(off, __builtin_fabsf(near - q[i]));
        }
        if (off < 0.5f - 0x1p-15f) return pack_bytes((int)q[0], (int)q[1], (int)q[2], (int)q[3]);
        return pack_bytes(settle(q[0], v[0], scale), settle(q[1], v[1], scale),
                          settle(q[2], v[2], scale), settle(q[3], v[3], scale));
    }
};

static inline bool w4_group(int64_t group) { return group == 32 || group == 64 || group == 128; }
// Blocks of outputs and of inputs.
static inline int64_t w4_rows(int64_t out, int32_t gated) {
    return gated ? 2 * ceil_div(out / 2, (int64_t)kW4Outputs) : ceil_div(out, (int64_t)kW4Outputs);
}
static inline int64_t w4_cols(int64_t inner) { return ceil_div(inner, (int64_t)kW4Inputs); }

// A weight's sizes: within 2^24 outputs and inputs, 2^31 words.
static inline bool w4_shape(int64_t out, int64_t inner, int64_t group, int32_t gated) {
    const int64_t lim = (int64_t)1 << 24;
    return out > 0 && inner > 0 && out < lim && inner < lim && inner % 8 == 0 && w4_group(group) &&
           (!gated || out % 2 == 0) &&
           w4_rows(out, gated) * w4_cols(inner) < ((int64_t)1 << 31) / kW4Words;
}
static inline int64_t w4_bytes(int64_t out, int64_t inner, int32_t gated) {
    return w4_rows(out, gated) * w4_cols(inner) * kW4Words * 4;
}
static inline int64_t w4_scale_bytes(int64_t out, int64_t inner, int64_t group, int32_t gated) {
    return w4_rows(out, gated) * w4_cols(inner) * (kW4Inputs / group) * kW4Outputs * 2;
}
static inline int64_t q8_groups(int64_t width) { return ceil_div(width, (int64_t)kQ8Group); }

// Whether the product of these rows and blocks of outputs is a small one: tiles of 32 rows by 4
// blocks are no more than the chip's 256 units, or wider ones mostly empty.
static inline bool w4_few(int64_t rows, int64_t nb) {
    return ceil_div(rows, (int64_t)32) * ceil_div(nb, (int64_t)4) <= 256 || nb <= 4;
}
// Whether 8-bit results come by way of fp32 ones in a workspace: the kernel by tiles gives them
// at once, but of few rows its steps of 128 inputs, 0.9 us each, are what it takes.  us by the
// workspace / at once, of 8-bit and fp32 rows: 512 -> 1024 columns, 32 rows 5.3 / 5.7, 6.2 / 8.3,
// 192 rows 6.4 / 5.7, 8.6 / 8.3; 1024 -> 3584, 32 rows 7.4 / 8.0, 9.1 / 12.9, 96 rows (more than
// few) 9.4 / 8.1, 15.1 / 13.1; 2048 -> 2048, 128 rows 11.4 / 12.3, 18.0 / 22.4.
static inline bool w4_by_workspace(int64_t rows, int64_t nb, int64_t kb) {
    return w4_few(rows, nb) && (rows <= 64 || kb > 4);
}

struct QuantRange {
    const void *p;
    int64_t bytes;
};
// Whether an output overlaps an input or another output (null: nothing there).
static inline bool quant_alias(const QuantRange *outs, int n_outs, const QuantRange *ins,
                               int n_ins) {
    for (int i = 0; i < n_outs; ++i) {
        if (!outs[i].p) continue;
        for (int j = 0; j < n_ins; ++j)
            if (ins[j].p && overlaps(outs[i].p, outs[i].bytes, ins[j].p, ins[j].bytes)) return true;
        for (int j = 0; j < i; ++j)
            if (outs[j].p && overlaps(outs[i].p, outs[i].bytes, outs[j].p, outs[j].bytes))
                return true;
    }
    return false;
}

// What the kernels of the product are given.
struct W4Product {
    const void *x;
    const float *x_scales;
    const u32x4 *packed;
    const u32x2 *scales;  // 4 bf16 scales each
    void *y;
    float *y_scales;
    int64_t ld_x;
    int rows, cols;  // of y
    int inner, kb;   // inputs, blocks of inputs
    int nb;          // blocks of outputs
    int q8_groups;   // of a row of x
    // of a launch by tiles: how many, how many of rows, and tiles in 8 of those
    uint32_t tiles;
    int tiles_m;
    FastDiv strip;
};

// The products of x in one type; y_dtype QDC_F32, QDC_BF16 or, gated, QDC_Q8.
int32_t linear_w4_f32(const W4Product &p, int group, bool gated, int32_t y_dtype, hipStream_t s);
int32_t linear_w4_bf16(const W4Product &p, int group, bool gated, int32_t y_dtype, hipStream_t s);
int32_t linear_w4_q8(const W4Product &p, int group, bool gated, int32_t y_dtype, hipStream_t s);

}  // namespace qdc
