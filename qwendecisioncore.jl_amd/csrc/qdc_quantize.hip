// qdc_quantize.hip -- weights into 4 bits and rows into 8, and back.
//
// All of it is one pass over memory, arithmetic hidden behind it.  A wavefront forms a
// block of weights as the product reads it (16 outputs x 128 inputs, 16 bytes a lane):
// the four lanes that hold an output's words share its groups, so a group's maximum is a
// maximum within a lane and two lane swaps.  8-bit rows are formed 4 values a lane, 32
// lanes a group of 128.
#include "qdc_quant.hpp"

namespace qdc {
namespace {

// 8 consecutive values of a row.
__device__ __forceinline__ void load8(const float *p, float (&v)[8]) {
    unpack(load_frag<float, 8>(p), v);
}
__device__ __forceinline__ void load8(const bf16_t *p, float (&v)[8]) { unpack(load_raw(p), v); }

struct Pack {
    void *w;
    u32x4 *packed;
    bf16_t *scales;
    int64_t ld;
    int out, inner, nb, kb;  // out: of gate and of up where gated
    int gated;
};

// The row of w that output n of block b is, -1 for none.
__device__ __forceinline__ int64_t weight_row(const Pack &p, int b, int n) {
    const int j = (p.gated ? b >> 1 : b) * kW4Outputs + n;
    return j < p.out ? (int64_t)j + (p.gated && (b & 1) ? p.out : 0) : -1;
}

// The last 4 bits of w / s to the nearest whole number, ties to even, exactly.
//
// fp32: a product with the inverse may come to the other side of a half than the quotient, but
// what it leaves, w - q s, is exact with FMA (q s has 12 bits, and the rest at most the 24 from
// w's last to s's half), so its side is known: q goes on where more than half of s is left, or
// half of it and q is odd.  1.5 * 2^23 + q has q in its last bits.
__device__ __forceinline__ uint32_t nearest(float w, float s, float inverse, float) {
    w = __builtin_amdgcn_fmed3f(w, -7.0f * s, 7.0f * s);
    const float near = w * inverse + 12582912.0f;
    const uint32_t q = __float_as_uint(near);
    const float rest = __builtin_fmaf(12582912.0f - near, s, w);
    const bool on = size_bits(rest) + (q & 1u) > __float_as_uint(0.5f * s);
    return (on ? q + (rest < 0.0f ? ~0u : 1u) : q) & 15u;
}
// bf16: with 8 bits each, w / s is a half or 2^-9 from it at least, and the product with the
// inverse within 2^-20 of it, so rounded to 2^-16 (the last bit of values from 128 on) it is
// the half where the quotient is; the whole number is then in the last bits of 1.5 * 2^23 more.
__device__ __forceinline__ uint32_t nearest(float w, float, float inverse, bf16_t) {
    const float q = w * inverse + 192.0f - 192.0f;
    return __float_as_uint(__builtin_amdgcn_fmed3f(q, -7.0f, 7.0f) + 12582912.0f) & 15u;
}

template <int G, typename T> __global__ __launch_bounds__(kBlock) void pack_w4(Pack p) {
    const int l = threadIdx.x % kWave, n = l % 16, quarter = l / 16;
    const int unit = blockIdx.x * (kBlock / kWave) + threadIdx.x / kWave;
    if (unit >= p.nb * p.kb) return;
    const int b = unit / p.kb, c = unit % p.kb;
    const int64_t row = weight_row(p, b, n);
    const T *src = reinterpret_cast<const T *>(p.w) + (row < 0 ? 0 : row) * p.ld;
    float v[4][8];
    uint32_t most[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        const int k = c * kW4Inputs + 32 * t + 8 * quarter;
#pragma unroll
        for (int i = 0; i < 8; ++i) v[t][i] = 0.0f;
        if (row >= 0 && k < p.inner) load8(src + k, v[t]);
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) m = max(m, size_bits(v[t][i]));
        // the other three quarters of these 32 inputs
        const auto a = __builtin_amdgcn_permlane16_swap(m, m, false, false);
        m = max(a[0], a[1]);
        const auto h = __builtin_amdgcn_permlane32_swap(m, m, false, false);
        most[t] = max(h[0], h[1]);
    }
    constexpr int T32 = G / 32;
    u32x4 words;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < T32; ++i) m = max(m, most[t / T32 * T32 + i]);
        const bool finite = m < 0x7f800000u;
        const bf16_t held = finite ? from_f32<bf16_t>(__uint_as_float(m) / 7.0f) : (bf16_t)0x7fc0;
        // the smallest scales have no inverse: those groups 2^64 times larger, which is exact
        const float s = to_f32(held), up = s < 0x1p-64f ? 0x1p64f : 1.0f;
        const float larger = s * up, inverse = 1.0f / larger;
        uint32_t word = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float w = v[t][i] * up;
            word |= nearest(w, larger, inverse, T()) << (8 * (i % 4) + 4 * (i / 4));
        }
        words[t] = finite && s > 0.0f ? word : 0u;
        if (t % T32 == 0 && quarter == 0)
            p.scales[((int64_t)unit * (4 / T32) + t / T32) * kW4Outputs + n] = held;
    }
    store_raw(p.packed + (int64_t)unit * kWave + l, words);
}

template <int G, typename T> __global__ __launch_bounds__(kBlock) void unpack_w4(Pack p) {
    const int l = threadIdx.x % kWave, n = l % 16, quarter = l / 16;
    const int unit = blockIdx.x * (kBlock / kWave) + threadIdx.x / kWave;
    if (unit >= p.nb * p.kb) return;
    const int b = unit / p.kb, c = unit % p.kb;
    const int64_t row = weight_row(p, b, n);
    if (row < 0) return;
    const u32x4 words = load_raw(p.packed + (int64_t)unit * kWave + l);
    T *dst = reinterpret_cast<T *>(p.w) + row * p.inner;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        const int k = c * kW4Inputs + 32 * t + 8 * quarter;
        if (k >= p.inner) break;
        const float s =
            to_f32(p.scales[((int64_t)unit * (128 / G) + t / (G / 32)) * kW4Outputs + n]);
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)
            v[i] = (float)((int)(words[t] << (28 - 8 * (i % 4) - 4 * (i / 4))) >> 28) * s;
        store_frag<8>(dst + k, v);
    }
}

struct Rows8 {
    const void *x;
    uint32_t *q;
    float *scales;
    int64_t ld;
    int units, width, groups;
    FastDiv chunks;  // of 256 columns in a row
};

template <typename T> __global__ __launch_bounds__(kBlock) void quantize_q8(Rows8 p) {
    const int l = threadIdx.x % kWave;
    const int unit = blockIdx.x * (kBlock / kWave) + threadIdx.x / kWave;
    if (unit >= p.units) return;
    const int row = (int)fastdiv((uint32_t)unit, p.chunks);
    const int col = 256 * (unit - row * (int)p.chunks.d) + 4 * l;
    const bool in = col < p.width;
    float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (in) unpack(load_frag<T, 4>(reinterpret_cast<const T *>(p.x) + row * p.ld + col), v);
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) m = max(m, size_bits(v[i]));
    const Q8Scale s(group_max<32>(m));
    if (!in) return;
    p.q[((int64_t)row * p.width + col) / 4] = s.word(v);
    if (l % 32 == 0) p.scales[(int64_t)row * p.groups + col / kQ8Group] = s.scale;
}

struct Back8 {
    void *out;
    const u32x2 *q;
    const float *scales;
    int pieces, groups;  // pieces of 8 values
    FastDiv per_row;
};

template <typename T> __global__ __launch_bounds__(kBlock) void dequantize_q8(Back8 p) {
    const int i = blockIdx.x * kBlock + threadIdx.x;
    if (i >= p.pieces) return;
    const int row = (int)fastdiv((uint32_t)i, p.per_row);
    const int at = i - row * (int)p.per_row.d;
    const u32x2 q = p.q[i];
    const float s = p.scales[(int64_t)row * p.groups + at / (kQ8Group / 8)];
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = (float)(int8_t)(q[j / 4] >> (8 * (j % 4))) * s;
    store_frag<8>(reinterpret_cast<T *>(p.out) + 8 * (int64_t)i, v);
}

struct Rms8 {
    float *residual;
    uint32_t *q;
    float *scales;
    const float *x, *add;
    const void *norm;
    const int32_t *mask;
    int rows, width, groups;
    float eps;
};

// A row by WAVES wavefronts, 4 columns a lane, CPL times: held in registers between the
// sum of squares and the 8-bit values.
template <int CPL, int WAVES, typename TW>
__global__ __launch_bounds__(WAVES > 4 ? WAVES * kWave : kBlock) void residual_rms_q8(Rms8 p) {
    constexpr int ROWS = WAVES < 4 ? 4 / WAVES : 1;  // of a workgroup
    __shared__ float part[WAVES > 1 ? WAVES : 1];
    const int l = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const int row = blockIdx.x * ROWS + wave / WAVES;
    if (row >= p.rows) return;  // a workgroup of one row never splits here
    const int at = wave % WAVES;
    const int64_t base = (int64_t)row * p.width;
    f32x4 v[CPL];
    Frag<TW, 4> w[CPL];
#pragma unroll
    for (int c = 0; c < CPL; ++c) {
        const int col = 256 * (c * WAVES + at) + 4 * l;
        v[c] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        w[c] = Frag<TW, 4>{};
        if (col < p.width) {
            v[c] = __builtin_bit_cast(f32x4, load_raw(p.x + base + col));
            if (p.add) v[c] += __builtin_bit_cast(f32x4, load_raw(p.add + base + col));
            w[c] = load_frag<TW, 4>(reinterpret_cast<const TW *>(p.norm) + col);
        }
    }
    float ss = 0.0f;
#pragma unroll
    for (int c = 0; c < CPL; ++c)
#pragma unroll
        for (int j = 0; j < 4; ++j) ss = __builtin_fmaf(v[c][j], v[c][j], ss);
    ss = group_sum<kWave>(ss);
    if constexpr (WAVES > 1) {
        if (l == 0) part[at] = ss;
        __syncthreads();
        ss = part[0];
#pragma unroll
        for (int i = 1; i < WAVES; ++i) ss += part[i];
    }
    const float s = rms_scale(ss, (float)p.width, p.eps);
    const bool keep = !p.mask || p.mask[row] != 0;
#pragma unroll
    for (int c = 0; c < CPL; ++c) {
        const int col = 256 * (c * WAVES + at) + 4 * l;
        float g[4], y[4], r[4];
        unpack(w[c], g);
        uint32_t m = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            r[j] = v[c][j];
            y[j] = keep ? (v[c][j] * s) * (1.0f + g[j]) : 0.0f;
            // behind the row's end 0 * s is NaN where s is
            m = max(m, col < p.width ? size_bits(y[j]) : 0u);
        }
        const Q8Scale q(group_max<32>(m));
        if (col >= p.width) continue;
        if (p.add) store_frag<4>(p.residual + base + col, r);
        p.q[(base + col) / 4] = q.word(y);
        if (l % 32 == 0) p.scales[(int64_t)row * p.groups + col / kQ8Group] = q.scale;
    }
}

}  // namespace
}  // namespace qdc

using namespace qdc;

extern "C" const char *qdc_quant_version(void) { return QDC_HIP_QUANT_VERSION; }

// A wavefront per 256 columns of a row, in workgroups of 4: fewer than 2^32 work-items.
static bool quant_rows(int64_t rows, int64_t width) {
    const int64_t lim = ((int64_t)1 << 26) - 3;
    return rows >= 0 && rows < lim && width > 0 && width < ((int64_t)1 << 24) && width % 16 == 0 &&
           rows * ceil_div(width, (int64_t)256) < lim;
}

extern "C" int32_t qdc_pack_w4(void *packed, void *scales, const void *w, int64_t out,
                               int64_t inner, int64_t ld, int64_t group, int32_t gated,
                               int32_t dtype, hipStream_t stream) {
    if (!valid_dtype(dtype)) return QDC_ERR_DTYPE;
    if (!w4_shape(out, inner, group, gated) || ld < inner || ld % 8 || ld >= ((int64_t)1 << 31))
        return QDC_ERR_SHAPE;
    if (!packed || !scales || !w) return QDC_ERR_NULL;
    if (!aligned16(packed) || !aligned16(scales) || !aligned16(w)) return QDC_ERR_SHAPE;
    const QuantRange outs[] = {{packed, w4_bytes(out, inner, gated)},
                               {scales, w4_scale_bytes(out, inner, group, gated)}};
    const QuantRange ins[] = {{w, ((out - 1) * ld + inner) * elem_size(dtype)}};
    if (quant_alias(outs, 2, ins, 1)) return QDC_ERR_ALIAS;
    Pack p{};
    p.w = const_cast<void *>(w);
    p.packed = reinterpret_cast<u32x4 *>(packed);
    p.scales = reinterpret_cast<bf16_t *>(scales);
    p.ld = ld;
    p.out = (int)(gated ? out / 2 : out);
    p.inner = (int)inner;
    p.nb = (int)w4_rows(out, gated);
    p.kb = (int)w4_cols(inner);
    p.gated = gated != 0;
    const dim3 grid((uint32_t)ceil_div((int64_t)p.nb * p.kb, (int64_t)(kBlock / kWave)));
#define QDC_PACK(G, T) hipLaunchKernelGGL((pack_w4<G, T>), grid, dim3(kBlock), 0, stream, p)
#define QDC_PACK_G(G)                           \
    if (group == G) {                           \
        if (dtype == QDC_F32) QDC_PACK(G, float); \
        else QDC_PACK(G, bf16_t);               \
    }
    QDC_PACK_G(32)
    QDC_PACK_G(64)
    QDC_PACK_G(128)
#undef QDC_PACK
    return launch_status();
}

extern "C" int32_t qdc_unpack_w4(void *w, const void *packed, const void *scales, int64_t out,
                                 int64_t inner, int64_t group, int32_t gated, int32_t dtype,
                                 hipStream_t stream) {
    if (!valid_dtype(dtype)) return QDC_ERR_DTYPE;
    if (!w4_shape(out, inner, group, gated)) return QDC_ERR_SHAPE;
    if (!packed || !scales || !w) return QDC_ERR_NULL;
    if (!aligned16(packed) || !aligned16(scales) || !aligned16(w)) return QDC_ERR_SHAPE;
    const QuantRange outs[] = {{w, out * inner * elem_size(dtype)}};
    const QuantRange ins[] = {{packed, w4_bytes(out, inner, gated)},
                              {scales, w4_scale_bytes(out, inner, group, gated)}};
    if (quant_alias(outs, 1, ins, 2)) return QDC_ERR_ALIAS;
    Pack p{};
    p.w = w;
    p.packed = reinterpret_cast<u32x4 *>(const_cast<void *>(packed));
    p.scales = reinterpret_cast<bf16_t *>(const_cast<void *>(scales));
    p.out = (int)(gated ? out / 2 : out);
    p.inner = (int)inner;
    p.nb = (int)w4_rows(out, gated);
    p.kb = (int)w4_cols(inner);
    p.gated = gated != 0;
    const dim3 grid((uint32_t)ceil_div((int64_t)p.nb * p.kb, (int64_t)(kBlock / kWave)));
#define QDC_PACK(G, T) hipLaunchKernelGGL((unpack_w4<G, T>), grid, dim3(kBlock), 0, stream, p)
    QDC_PACK_G(32)
    QDC_PACK_G(64)
    QDC_PACK_G(128)
#undef QDC_PACK
#undef QDC_PACK_G
    return launch_status();
}

extern "C" int32_t qdc_quantize_q8(void *q, float *scales, const void *x, int64_t rows,
                                   int64_t width, int64_t ld, int32_t dtype, hipStream_t stream) {
    if (!valid_dtype(dtype)) return QDC_ERR_DTYPE;
    if (!quant_rows(rows, width) || ld < width || ld % 8 || ld >= ((int64_t)1 << 31))
        return QDC_ERR_SHAPE;
    if (rows == 0) return QDC_OK;
    if (!q || !scales || !x) return QDC_ERR_NULL;
    if (!aligned16(q) || !aligned16(x) || ((uintptr_t)scales & 3u)) return QDC_ERR_SHAPE;
    const QuantRange outs[] = {{q, rows * width}, {scales, rows * q8_groups(width) * 4}};
    const QuantRange ins[] = {{x, ((rows - 1) * ld + width) * elem_size(dtype)}};
    if (quant_alias(outs, 2, ins, 1)) return QDC_ERR_ALIAS;
    Rows8 p{};
    p.x = x;
    p.q = reinterpret_cast<uint32_t *>(q);
    p.scales = scales;
    p.ld = ld;
    p.width = (int)width;
    p.groups = (int)q8_groups(width);
    p.chunks = make_fastdiv((uint32_t)ceil_div(width, (int64_t)256));
    p.units = (int)(rows * p.chunks.d);
    const dim3 grid((uint32_t)ceil_div((int64_t)p.units, (int64_t)(kBlock / kWave)));
    if (dtype == QDC_F32) hipLaunchKernelGGL((quantize_q8<float>), grid, dim3(kBlock), 0, stream, p);
    else hipLaunchKernelGGL((quantize_q8<bf16_t>), grid, dim3(kBlock), 0, stream, p);
    return launch_status();
}

extern "C" int32_t qdc_dequantize_q8(void *out, const void *q, const float *scales, int64_t rows,
                                     int64_t width, int32_t dtype, hipStream_t stream) {
    if (!valid_dtype(dtype)) return QDC_ERR_DTYPE;
    if (!quant_rows(rows, width)) return QDC_ERR_SHAPE;
    if (rows == 0) return QDC_OK;
    if (!q || !scales || !out) return QDC_ERR_NULL;
    if (!aligned16(q) || !aligned16(out) || ((uintptr_t)scales & 3u)) return QDC_ERR_SHAPE;
    const QuantRange outs[] = {{out, rows * width * elem_size(dtype)}};
    const QuantRange ins[] = {{q, rows * width}, {scales, rows * q8_groups(width) * 4}};
    if (quant_alias(outs, 1, ins, 2)) return QDC_ERR_ALIAS;
    Back8 p{};
    p.out = out;
    p.q = reinterpret_cast<const u32x2 *>(q);
    p.scales = scales;
    p.groups = (int)q8_groups(width);
    p.per_row = make_fastdiv((uint32_t)(width / 8));
    p.pieces = (int)(rows * (width / 8));  // below 2^31: 32 to a chunk of 256 columns
    const dim3 grid((uint32_t)ceil_div((int64_t)p.pieces, (int64_t)kBlock));
    if (dtype == QDC_F32)
        hipLaunchKernelGGL((dequantize_q8<float>), grid, dim3(kBlock), 0, stream, p);
    else hipLaunchKernelGGL((dequantize_q8<bf16_t>), grid, dim3(kBlock), 0, stream, p);
    return launch_status();
}

extern "C" int32_t qdc_residual_rmsnorm_q8(float *residual, void *q, float *scales, const float *x,
                                           const float *add, const void *norm, const int32_t *mask,
                                           int64_t rows, int64_t width, float eps,
                                           int32_t norm_dtype, hipStream_t stream) {
    if (!valid_dtype(norm_dtype)) return QDC_ERR_DTYPE;
    if (!quant_rows(rows, width) || width > 32768) return QDC_ERR_SHAPE;
    if (rows == 0) return QDC_OK;
    if (!q || !scales || !x || !norm || (add && !residual)) return QDC_ERR_NULL;
    if (!add) residual = nullptr;
    if (!aligned16(q) || !aligned16(x) || !aligned16(add) || !aligned16(norm) ||
        !aligned16(residual) || ((uintptr_t)scales & 3u) || ((uintptr_t)mask & 3u))
        return QDC_ERR_SHAPE;
    const int64_t bytes = rows * width * 4;
    const QuantRange outs[] = {{q, rows * width},
                               {scales, rows * q8_groups(width) * 4},
                               {residual, bytes}};
    const QuantRange ins[] = {{norm, width * elem_size(norm_dtype)},
                              {mask, rows * 4},
                              {add, bytes},
                              {x, bytes}};
    // the residual may be x itself
    if (quant_alias(outs, 3, ins, 3) || quant_alias(outs, 2, ins + 3, 1) ||
        (residual && residual != x && overlaps(residual, bytes, x, bytes)))
        return QDC_ERR_ALIAS;
    Rms8 p{};
    p.residual = residual;
    p.q = reinterpret_cast<uint32_t *>(q);
    p.scales = scales;
    p.x = x;
    p.add = add;
    p.norm = norm;
    p.mask = mask;
    p.rows = (int)rows;
    p.width = (int)width;
    p.groups = (int)q8_groups(width);
    p.eps = eps;
#define QDC_RMS8(CPL, WAVES)                                                                     \
    {                                                                                            \
        constexpr int per = WAVES < 4 ? 4 / WAVES : 1;                                           \
        const dim3 grid((uint32_t)ceil_div(rows, (int64_t)per)), block(per * WAVES * kWave);     \
        if (norm_dtype == QDC_F32)                                                               \
            hipLaunchKernelGGL((residual_rms_q8<CPL, WAVES, float>), grid, block, 0, stream, p); \
        else                                                                                     \
            hipLaunchKernelGGL((residual_rms_q8<CPL, WAVES, bf16_t>), grid, block, 0, stream, p); \
        return launch_status();                                                                  \
    }
    if (width <= 256) QDC_RMS8(1, 1)
    if (rows < 256 && width <= 1024) QDC_RMS8(1, 4)
    if (width <= 512) QDC_RMS8(2, 1)
    if (width <= 1024) QDC_RMS8(4, 1)
    if (width <= 2048) QDC_RMS8(2, 4)
    if (width <= 4096) QDC_RMS8(4, 4)
    if (width <= 8192) QDC_RMS8(2, 16)
    QDC_RMS8(8, 16)
#undef QDC_RMS8
}
