// qdc_linear_w4.hpp -- the product of rows with 4-bit weights, for rows of one type.
//
// y[m, n] = sum over groups g of s[n, g] * sum over k in g of q[n, k] x[m, k].  The whole
// numbers enter the matrix instructions as they are (an 8-bit one holds 16 q, a bf16 one
// q / 16 exactly), so the only roundings are those of fp32 sums: a group's sum is scaled and
// added in fp32, and the factor taken out of the result.  fp32 rows enter as three bf16
// terms that hold all 24 bits (8 each, by truncation); 8-bit rows as they are, with whole
// sums, their own scale joining the weight's.
//
// A block of weights is 16 outputs x 128 inputs, 16 bytes a lane in the order of the
// instruction's first operand; x is the second, so that a lane holds one row of the result
// and 4 consecutive outputs.
#pragma once

#include <type_traits>

#include "qdc_quant.hpp"

namespace qdc {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

enum { kF32, kBf16, kQ8 };  // types of x

// A word's 8 whole numbers as bf16, q / 16: the conversion looks at the last 4 bits of a byte
// alone and divides by 16 (from signed bytes 16 q, which take masks, 16384 x 1024 -> 8224 of
// bf16 took 361 us in place of 352, 301 x 2048 -> 6144 of fp32 32.9 in place of 30.0).
constexpr float kBack(bool whole) { return whole ? 0.0625f : 16.0f; }
__device__ __forceinline__ bf16x8 widen(uint32_t word) {
    u32x4 r;
    uint32_t upper = word >> 4;
    asm("" : "+v"(upper));  // a value of its own, whose bytes the conversions select themselves
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint32_t b = i ? upper : word;
        const float v0 = __builtin_amdgcn_cvt_off_f32_i4((int)(b & 0xffu));
        const float v1 = __builtin_amdgcn_cvt_off_f32_i4((int)(b >> 8 & 0xffu));
        const float v2 = __builtin_amdgcn_cvt_off_f32_i4((int)(b >> 16 & 0xffu));
        const float v3 = __builtin_amdgcn_cvt_off_f32_i4((int)(b >> 24));
        // exact in bf16: the upper halves of the fp32 values
        r[2 * i] = __builtin_amdgcn_perm(__float_as_uint(v1), __float_as_uint(v0), 0x07060302u);
        r[2 * i + 1] = __builtin_amdgcn_perm(__float_as_uint(v3), __float_as_uint(v2), 0x07060302u);
    }
    return __builtin_bit_cast(bf16x8, r);
}

// The three bf16 terms of fp32 values, each the upper half of what is left: hi + mid + lo
// is v.  An infinity or NaN is its first term.
__device__ __forceinline__ void terms(const float (&v)[8], u32x4 (&r)[3]) {
    uint32_t h[8], m[8], l[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        h[i] = __float_as_uint(__builtin_canonicalizef(v[i]));  // a NaN with its upper half set
        const bool finite = !__builtin_amdgcn_classf(v[i], 0x207);
        const float rest = finite ? v[i] - __uint_as_float(h[i] & 0xffff0000u) : 0.0f;
        m[i] = __float_as_uint(rest);
        l[i] = __float_as_uint(rest - __uint_as_float(m[i] & 0xffff0000u));
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        r[0][i] = __builtin_amdgcn_perm(h[2 * i + 1], h[2 * i], 0x07060302u);
        r[1][i] = __builtin_amdgcn_perm(m[2 * i + 1], m[2 * i], 0x07060302u);
        r[2][i] = __builtin_amdgcn_perm(l[2 * i + 1], l[2 * i], 0x07060302u);
    }
}

// 4 scales as fp32.
__device__ __forceinline__ f32x4 scales4(u32x2 s) {
    return f32x4{__uint_as_float(s[0] << 16), __uint_as_float(s[0] & 0xffff0000u),
                 __uint_as_float(s[1] << 16), __uint_as_float(s[1] & 0xffff0000u)};
}

// Whole sums as fp32 by a subtraction: they start at 1.5 * 2^23, whose last bit as a float is
// 1, and stay within the 2^22 to either side (128 products of 128 * 127 at most).  With
// conversions in its place 16384 x 1024 -> 8224 took 5% longer.
constexpr int kWhole = 0x4b400000;
// The same in 2^-21: the bits of a float with an exponent lower by that.  1.5 * 2^23 times a
// weight's scale, which the tiles take off as one product, is then within the range of fp32
// for every scale that a finite weight has (up to 2^127 / 3).
constexpr int kSmall = kWhole - (21 << 23);
template <int START> __device__ __forceinline__ float whole(int sum) {
    return __int_as_float(sum) - __int_as_float(START);
}

// The operand of x for 32 inputs of a block: raw words as they are loaded or staged.
template <int X> struct Piece {
    static constexpr int kTerms = X == kF32 ? 3 : 1;
    u32x4 t[kTerms];  // 8 values in bf16; kQ8: 8 bytes in the first two words
};

// total += the block's products.  piece(t): x for the inputs 32 t + 8 (lane / 16) + 0..7.
template <int X, int G, typename F>
__device__ __forceinline__ void block_product(f32x4 &total, u32x4 words, const u32x2 *scales,
                                              float x_scale, F piece) {
    if constexpr (X == kQ8) {
#pragma unroll
        for (int g = 0; g < 128 / G; ++g) {
            i32x4 sum = {kWhole, kWhole, kWhole, kWhole};
            if constexpr (G == 32) {
                const uint32_t w = words[g];
                const u32x2 a = {(w << 4) & 0xf0f0f0f0u, w & 0xf0f0f0f0u};
                const u32x4 x = piece(g).t[0];
                sum = __builtin_amdgcn_mfma_i32_16x16x32_i8(
                    __builtin_bit_cast(long, a), __builtin_bit_cast(long, u32x2{x[0], x[1]}), sum,
                    0, 0, 0);
            } else {
#pragma unroll
                for (int u = g * G / 64; u < (g + 1) * G / 64; ++u) {
                    const uint32_t w0 = words[2 * u], w1 = words[2 * u + 1];
                    const u32x4 a = {(w0 << 4) & 0xf0f0f0f0u, w0 & 0xf0f0f0f0u,
                                     (w1 << 4) & 0xf0f0f0f0u, w1 & 0xf0f0f0f0u};
                    const u32x4 x0 = piece(2 * u).t[0], x1 = piece(2 * u + 1).t[0];
                    sum = __builtin_amdgcn_mfma_i32_16x16x64_i8(
                        __builtin_bit_cast(i32x4, a),
                        __builtin_bit_cast(i32x4, u32x4{x0[0], x0[1], x1[0], x1[1]}), sum, 0, 0, 0);
                }
            }
            const f32x4 s = scales4(scales[g]);
#pragma unroll
            for (int r = 0; r < 4; ++r)
                total[r] = __builtin_fmaf(whole<kWhole>(sum[r]), s[r] * x_scale, total[r]);
        }
    } else {
#pragma unroll
        for (int g = 0; g < 128 / G; ++g) {
            f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int t = g * G / 32; t < (g + 1) * G / 32; ++t) {
                const bf16x8 w = widen(words[t]);
                const Piece<X> x = piece(t);
#pragma unroll
                for (int n = Piece<X>::kTerms - 1; n >= 0; --n)  // the smallest first
                    sum = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                        w, __builtin_bit_cast(bf16x8, x.t[n]), sum, 0, 0, 0);
            }
            const f32x4 s = scales4(scales[g]);
#pragma unroll
            for (int r = 0; r < 4; ++r) total[r] = __builtin_fmaf(sum[r], s[r], total[r]);
        }
    }
}

// 8 values of x from memory, zeros where there are none.
template <int X> __device__ __forceinline__ Piece<X> load_piece(const void *row, int k, bool in) {
    Piece<X> r{};
    if (!in) return r;
    if constexpr (X == kF32) {
        float v[8];
        unpack(load_frag<float, 8>(reinterpret_cast<const float *>(row) + k), v);
        terms(v, r.t);
    } else if constexpr (X == kBf16) {
        r.t[0] = load_raw(reinterpret_cast<const bf16_t *>(row) + k);
    } else {
        const u32x2 h = *reinterpret_cast<const u32x2 *>(reinterpret_cast<const char *>(row) + k);
        r.t[0] = u32x4{h[0], h[1], 0u, 0u};
    }
    return r;
}
template <int X> constexpr int kXBytes = X == kF32 ? 4 : X == kBf16 ? 2 : 1;

// The first `left` of N outputs of T, held in words, from `at` on.  An ordinary store: the cache
// joins what the wavefront's next ones write of a line; and one for all N whatever the
// alignment, as rows of an odd number of outputs start anywhere (16235 x 64 ->
// 1477, fp32 results, by elements 58 us, so 24).
template <typename T, int N>
__device__ __forceinline__ void put_piece(T *at, int left, const uint32_t (&v)[N * sizeof(T) / 4]) {
    constexpr int W = N * (int)sizeof(T) / 4;
    typedef uint32_t Words __attribute__((ext_vector_type(W), aligned(sizeof(T))));
    if (left >= N) {
        Words w;
#pragma unroll
        for (int i = 0; i < W; ++i) w[i] = v[i];
        *reinterpret_cast<Words *>(at) = w;
    } else if (left > 0) {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (i < left) at[i] = sizeof(T) == 4 ? (T)v[i] : (T)(v[i / 2] >> (16 * (i % 2)));
    }
}
// N pieces of 4 outputs of a row, 16 apart, n the first output.
template <typename T, int N>
__device__ __forceinline__ void put(void *y, int cols, int row, int n, const float (&v)[N][4]) {
    typedef typename std::conditional<sizeof(T) == 4, uint32_t, uint16_t>::type Bits;
    Bits *at = reinterpret_cast<Bits *>(y) + (int64_t)row * cols + n;
#pragma unroll
    for (int j = 0; j < N; ++j) {
        if constexpr (sizeof(T) == 4) {
            const uint32_t w[4] = {__float_as_uint(v[j][0]), __float_as_uint(v[j][1]),
                                   __float_as_uint(v[j][2]), __float_as_uint(v[j][3])};
            put_piece<Bits, 4>(at + 16 * j, cols - n - 16 * j, w);
        } else {
            const uint32_t w[2] = {pack_bf16x2(v[j][0], v[j][1]), pack_bf16x2(v[j][2], v[j][3])};
            put_piece<Bits, 4>(at + 16 * j, cols - n - 16 * j, w);
        }
    }
}

// The same in bf16 for a wavefront's 2 or 4 pieces from output n on: the lanes of a row first
// trade pieces, so that each has 8 or 16 outputs side by side and a line is written by two
// instructions in place of four (8-bit rows, 16384 x 1024 -> 8224, 265 -> 257 us).
template <int N>
__device__ __forceinline__ void put_wide(void *y, int cols, int row, bool in, int n, int quarter,
                                         const float (&v)[N][4]) {
    static_assert(N == 2 || N == 4, "pieces");
    uint32_t t[N][2];
#pragma unroll
    for (int j = 0; j < N; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h) t[j][h] = pack_bf16x2(v[j][2 * h], v[j][2 * h + 1]);
    // lane quarter q = 2 a + b: piece [2 a] (of 4) of quarters b and 2 + b, then piece [q] or
    // [b] of quarters in order
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        if constexpr (N == 4)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const auto r = __builtin_amdgcn_permlane32_swap(t[j][h], t[j + 2][h], false, false);
                t[j][h] = r[0];
                t[j + 2][h] = r[1];
            }
#pragma unroll
        for (int j = 0; j < N; j += 2) {
            const auto r = __builtin_amdgcn_permlane16_swap(t[j][h], t[j + 1][h], false, false);
            t[j][h] = r[0];
            t[j + 1][h] = r[1];
        }
    }
    n += N == 4 ? 16 * quarter : 16 * (quarter % 2) + 8 * (quarter / 2);
    bf16_t *at = reinterpret_cast<bf16_t *>(y) + (int64_t)row * cols + n;
#pragma unroll
    for (int j = 0; j < N; j += 2)
        if (in) {
            const uint32_t w[4] = {t[j][0], t[j][1], t[j + 1][0], t[j + 1][1]};
            put_piece<bf16_t, 8>(at + 4 * j, cols - n - 4 * j, w);
        }
}

// ---------------------------------------------------------------- few rows ---
// A workgroup per NB blocks of outputs (pairs of gate and up where gated) and 16 * MT rows,
// whose wavefronts take the blocks of inputs in turn and add up at the end: bound by the
// weights' way from memory and, for a row or two, by one trip there, so every load of a
// wavefront's block leaves at once and x comes straight from the caches.
//
// What it is given, in 64 bytes: a launch with 128 takes the host 0.3 us longer.
struct W4Rows {
    const void *x;
    const float *x_scales;
    const u32x4 *packed;
    const u32x2 *scales;
    void *y;
    uint32_t ld_x;
    int rows, cols, inner, nb;
    int32_t y_dtype;
};
template <int X, int G, int MT, int NB, bool GATED, int WAVES>
__global__ __launch_bounds__(WAVES *kWave) void w4_rows(W4Rows p) {
    const int kb = (p.inner + kW4Inputs - 1) / kW4Inputs;  // and the scales of an 8-bit row
    __shared__ f32x4 parts[WAVES][NB][MT][kWave];
    const int l = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const int quarter = l / 16, b0 = blockIdx.x * NB, m0 = blockIdx.y * 16 * MT;
    f32x4 total[NB][MT];
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int i = 0; i < MT; ++i) total[b][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    for (int c = wave; c < kb; c += WAVES) {
        u32x4 words[NB];
        u32x2 s[NB][128 / G];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const int64_t unit = (int64_t)min(b0 + b, p.nb - 1) * kb + c;
            words[b] = load_stream(p.packed + unit * kWave + l);
#pragma unroll
            for (int g = 0; g < 128 / G; ++g)
                s[b][g] = p.scales[(unit * (128 / G) + g) * 4 + quarter];
        }
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            const int row = m0 + 16 * i + l % 16;
            const bool in = row < p.rows;
            const char *src = reinterpret_cast<const char *>(p.x) +
                              (int64_t)(in ? row : 0) * p.ld_x * kXBytes<X>;
            Piece<X> x[4];
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const int k = c * kW4Inputs + 32 * t + 8 * quarter;
                x[t] = load_piece<X>(src, k, in && k < p.inner);
            }
            float xs = 0.0f;
            if constexpr (X == kQ8)
                if (in) xs = p.x_scales[(int64_t)row * kb + c];
#pragma unroll
            for (int b = 0; b < NB; ++b)
                block_product<X, G>(total[b][i], words[b], s[b], xs,
                                    [&](int t) -> const Piece<X> & { return x[t]; });
        }
    }
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int i = 0; i < MT; ++i) parts[wave][b][i][l] = total[b][i];
    __syncthreads();
    if (wave >= MT) return;
    const int row = m0 + 16 * wave + l % 16;
    if (row >= p.rows) return;
    f32x4 sum[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        sum[b] = parts[0][b][wave][l];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) sum[b] += parts[w][b][wave][l];
    }
    constexpr int PER = GATED ? 2 : 1;
    float v[NB / PER][4];
#pragma unroll
    for (int b = 0; b < NB / PER; ++b)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            v[b][r] = sum[PER * b][r] * kBack(X == kQ8);
            if constexpr (GATED) v[b][r] = silu(v[b][r]) * (sum[2 * b + 1][r] * kBack(X == kQ8));
        }
    const int n = b0 / PER * kW4Outputs + 4 * quarter;
    if (p.y_dtype == QDC_F32) put<float>(p.y, p.cols, row, n, v);
    else put<bf16_t>(p.y, p.cols, row, n, v);
}

// --------------------------------------------------------------- many rows ---
// A workgroup of NW wavefronts takes tiles of NW * NJ blocks of outputs by 16 * MT rows, a
// wavefront NJ blocks of them.  x and the scales go through LDS, a step of 128 inputs while
// the step before is multiplied; the weights, each for one wavefront and in operand order
// already, go to registers.  OUT8: the tile's 16 blocks are gate and up of the 128 columns
// that share a scale of an 8-bit row, whose maximum the wavefronts find together.
template <int X, int G, int MT, int NJ, int NW> struct Staged {
    static constexpr int kRows = 16 * MT, kBlocks = NJ * NW, kThreads = NW * kWave;
    static constexpr int kStep = kThreads / 16 < kRows ? kThreads / 16 : kRows;
    static constexpr int kPass = kRows / kStep;              // pieces of x a thread
    static constexpr int kTerms = Piece<X>::kTerms;
    static constexpr int kLd = X == kQ8 ? 144 : X == kBf16 ? 272 : 256;  // bytes of a row
    static constexpr int kX = kRows * kLd * kTerms;          // x, then the weights' scales
    static constexpr int kScales = kBlocks * (128 / G) * 64;     // (a block's groups, 16 fp32 each),
    static constexpr int kBytes = kX + kScales + 4 * kRows;  // then those of 8-bit rows
    // The most bytes from a row of x to the next: offsets from a tile's first row are 32 bits.
    static constexpr int64_t kFarthest = ((int64_t)1 << 32) / kRows;

    // Where 16 bytes of a row are.  The 16 lanes whose addresses LDS takes at once (0-3, 12-15
    // and 20-27 of a read, and their like) are 16 rows in two quarters: the order of fp32 terms,
    // another one in each row, puts them in all of its banks.  Rows 16 bytes longer than they
    // need to be take 4 of 8 cycles of a read for conflicts, which three terms wait for and
    // one does not.  us by order / longer rows: 301 rows 2048 -> 6144 fp32 29.2 / 31.0; 16384
    // rows 1024 -> 8224 fp32 708 / 723, bf16 312 / 309, 8-bit 262 / 255.
    __device__ static __forceinline__ uint32_t at(int row, int piece) {
        return (uint32_t)(row * kLd + 16 * (X == kF32 ? piece ^ row % 16 : piece));
    }
    // 4 pieces a time further on
    __device__ static __forceinline__ uint32_t along(uint32_t at, uint32_t times) {
        return X == kF32 ? at ^ 64u * times : at + 64u * times;
    }
};

// The tiles of a workgroup.  Workgroups go to the 8 dies in turn, each with a cache of its
// own: a die takes a range of tiles, 8 tiles of rows by all outputs, then the next 8, so
// that it reads its rows once and the weights an eighth as often as it has tiles of rows.
struct Tiles {
    uint32_t first, count, step, at;  // of the die; step: its workgroups

    __device__ explicit Tiles(const W4Product &p) {
        const uint32_t die = blockIdx.x % 8, all = p.tiles;
        first = die * (all / 8) + min(die, all % 8);
        count = all / 8 + (die < all % 8);
        step = gridDim.x / 8 + (die < gridDim.x % 8);
        at = blockIdx.x / 8;  // below count, as the launch has at most a workgroup per tile
    }
    __device__ void place(const W4Product &p, uint32_t i, int &n, int &m) const {
        const uint32_t strip = fastdiv(first + i, p.strip), in = first + i - strip * p.strip.d;
        const uint32_t tall = min(8u, (uint32_t)p.tiles_m - 8 * strip);
        n = (int)(in / tall);
        m = (int)(8 * strip + in % tall);
    }
};

template <int N> __device__ __forceinline__ int round_up(int v) { return (v + N - 1) / N * N; }

template <int X, int G, int MT, int NJ, int NW, bool GATED, bool OUT8>
__global__ __launch_bounds__(NW *kWave, 2) void w4_tiles(W4Product p, int32_t y_dtype) {
    typedef Staged<X, G, MT, NJ, NW> S;
    constexpr int NG = 128 / G, PJ = NJ / 2;  // groups of a step, pairs of blocks
    static_assert(NJ % 2 == 0 && (!OUT8 || S::kBlocks == 16), "");
    __shared__ __align__(16) char tile[2][S::kBytes];
    const int tid = threadIdx.x, l = tid % kWave;
    // known to be one of a wavefront, so that its addresses are scalar
    const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int quarter = l / 16;

    // this thread's pieces of 8 values: the same columns of kPass rows.  Offsets are 32 bits from
    // the tile's first row; rows behind the last one are the last one, and not stored.
    // (Where there are more threads than pieces, and than 1/16 blocks below, they come again.)
    const int k8 = tid % 16, x_row = tid / 16 % S::kStep;
    const uint32_t row_bytes = (uint32_t)p.ld_x * kXBytes<X>;
    uint32_t x_at[S::kPass];
#pragma unroll
    for (int i = 0; i < S::kPass; ++i)
        x_at[i] = (uint32_t)(x_row + S::kStep * i) * row_bytes;
    // and 1/16 of a block's scales (2, 4 or 8 bytes), and a row's
    const uint32_t block_bytes = (uint32_t)p.kb * (32 * NG), q8_bytes = 4 * (uint32_t)p.q8_groups;
    const int st = tid % (16 * S::kBlocks);
    const uint32_t scale_at = (uint32_t)(st / 16) * block_bytes;
    const uint32_t xs_at = (uint32_t)(tid % S::kRows) * q8_bytes;
    typedef typename std::conditional<
        NG == 1, uint16_t, typename std::conditional<NG == 2, uint32_t, u32x2>::type>::type Scales;
    // The raw values of a step on their way, or of two where the registers have room: alone
    // on its unit a workgroup would wait for memory at every step.
    constexpr int RAW = X == kF32 ? 2 : 1;
    constexpr int SETS = NJ * MT <= 4 || (NJ * MT <= 8 && !(X == kQ8 && G == 32)) ? 2 : 1;
    typedef typename std::conditional<X == kQ8, u32x2, u32x4>::type Raw;
    Raw raw[SETS][S::kPass][RAW];
    Scales raw_scales[SETS];
    float raw_xs[SETS];
    u32x4 words[SETS][NJ];
    const uint32_t word_at = 16 * l;
    auto load_w = [&](auto set, int n, int m, int c) {
        c = min(c, p.kb - 1);
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            // behind the last block: loaded, not stored
            const int64_t unit = (int64_t)min(S::kBlocks * n + NJ * wave + j, p.nb - 1) * p.kb + c;
            words[set][j] =
                load_raw(reinterpret_cast<const char *>(p.packed + unit * kWave) + word_at);
        }
        const char *base = reinterpret_cast<const char *>(p.scales) +
                           ((int64_t)S::kBlocks * n * p.kb + c) * (32 * NG);
        const uint32_t most =
            (uint32_t)min(p.nb - 1 - S::kBlocks * n, S::kBlocks - 1) * block_bytes;
        raw_scales[set] = *reinterpret_cast<const Scales *>(
            base + (min(scale_at, most) + (uint32_t)(st % 16 * sizeof(Scales))));
        if constexpr (X == kQ8) {
            const int m0 = m * S::kRows;
            const char *from =
                reinterpret_cast<const char *>(p.x_scales + (int64_t)m0 * p.q8_groups + c);
            raw_xs[set] = *reinterpret_cast<const float *>(
                from + min(xs_at, (uint32_t)min(p.rows - 1 - m0, S::kRows - 1) * q8_bytes));
        }
    };
    auto load_x = [&](auto set, int m, int c) {
        const int m0 = m * S::kRows, k = c * kW4Inputs + 8 * k8;
        const char *base = reinterpret_cast<const char *>(p.x) + (int64_t)m0 * row_bytes;
        const uint32_t most = (uint32_t)min(p.rows - 1 - m0, S::kRows - 1) * row_bytes;
        const uint32_t col = k < p.inner ? (uint32_t)k * kXBytes<X> : 0u;
#pragma unroll
        for (int i = 0; i < S::kPass; ++i)
#pragma unroll
            for (int h = 0; h < RAW; ++h)
                raw[set][i][h] =
                    *reinterpret_cast<const Raw *>(base + (min(x_at[i], most) + col + 16 * h));
    };
    auto stage = [&](auto set, int buf, int c) {
        Raw(&mine)[S::kPass][RAW] = raw[set];
        // zeros behind the last input, where the weights are 0 but a float might be infinite
        const bool ok = (X == kQ8 && SETS == 1) || c * kW4Inputs + 8 * k8 < p.inner;
        float *s = reinterpret_cast<float *>(tile[buf] + S::kX) + st * NG;
        if constexpr (NG == 1) *s = to_f32(raw_scales[set]);
        else if constexpr (NG == 2)
            *reinterpret_cast<f32x2 *>(s) = f32x2{__uint_as_float(raw_scales[set] << 16),
                                                  __uint_as_float(raw_scales[set] & 0xffff0000u)};
        else *reinterpret_cast<f32x4 *>(s) = scales4(raw_scales[set]);
        if constexpr (X == kQ8)
            *reinterpret_cast<float *>(tile[buf] + S::kX + S::kScales + 4 * (tid % S::kRows)) =
                raw_xs[set];
#pragma unroll
        for (int i = 0; i < S::kPass; ++i) {
            // (rows a multiple of 16 apart have one order)
            char *dst = tile[buf] + S::kStep * i * S::kLd;
#pragma unroll
            for (int h = 0; h < RAW; ++h)
#pragma unroll
                for (int e = 0; e < (X == kQ8 ? 2 : 4); ++e)
                    mine[i][h][e] = ok ? mine[i][h][e] : 0u;
            if constexpr (X == kQ8) {
                // the two pieces that an instruction's lane takes lie side by side
                *reinterpret_cast<u32x2 *>(dst + S::at(x_row, 4 * (k8 / 8) + k8 % 4) +
                                           8 * (k8 / 4 % 2)) = mine[i][0];
            } else if constexpr (X == kBf16) {
                *reinterpret_cast<u32x4 *>(dst + S::at(x_row, k8)) = mine[i][0];
            } else {
                float v[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = __uint_as_float(mine[i][e / 4][e % 4]);
                u32x4 t[3];
                terms(v, t);
#pragma unroll
                for (int n = 0; n < 3; ++n)
                    *reinterpret_cast<u32x4 *>(dst + n * S::kRows * S::kLd + S::at(x_row, k8)) = t[n];
            }
        }
    };
    // the scales of 4 outputs of the wavefront's block j in group g of a step
    auto scales = [&](int buf, int j, int g) {
        return *reinterpret_cast<const f32x4 *>(tile[buf] + S::kX +
                                                ((NJ * wave + j) * NG + g) * 64 + 16 * quarter);
    };

    f32x4 total[NJ][MT];
    // A step's products, in units of two blocks by 16 rows whose sums are scaled and added
    // while the next unit's are multiplied: the scheduler, left to itself, starts them all
    // and runs out of registers.
    auto multiply_whole = [&](auto set, int buf, auto &&next) {
        const uint32_t mine = S::at(l % 16, quarter);
        u32x4 x[2][2];
        auto read = [&](int i) {
#pragma unroll
            for (int u = 0; u < 2; ++u)
                x[i % 2][u] = *reinterpret_cast<const u32x4 *>(tile[buf] + 16 * i * S::kLd +
                                                               S::along(mine, u));
        };
        read(0);
        u32x4 a[NJ][2];
        f32x4 s[NJ][NG], bias[NJ];
        float own[MT];
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const uint32_t w0 = words[set][j][2 * u], w1 = words[set][j][2 * u + 1];
                a[j][u] = u32x4{(w0 << 4) & 0xf0f0f0f0u, w0 & 0xf0f0f0f0u, (w1 << 4) & 0xf0f0f0f0u,
                                w1 & 0xf0f0f0f0u};
            }
#pragma unroll
            for (int g = 0; g < NG; ++g) s[j][g] = scales(buf, j, g);
        }
#pragma unroll
        for (int i = 0; i < MT; ++i)
            own[i] = *reinterpret_cast<const float *>(tile[buf] + S::kX + S::kScales +
                                                      4 * (16 * i + l % 16));
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) bias[j][r] = s[j][0][r] * -__int_as_float(kSmall);
        next();
        __builtin_amdgcn_sched_barrier(0);
        i32x4 sum[2][2];
        f32x4 block[2];
#pragma unroll
        for (int n = 0; n <= MT * PJ * NG; ++n) {
            if (n < MT * PJ * NG) {
                const int i = n / (PJ * NG), j0 = n / NG % PJ * 2, g = n % NG;
                if (n % (PJ * NG) == 0 && i + 1 < MT) read(i + 1);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    i32x4 &to = sum[n % 2][j];
                    to = i32x4{kSmall, kSmall, kSmall, kSmall};
                    if constexpr (G == 32) {
                        const u32x4 w = a[j0 + j][g / 2], v = x[i % 2][g / 2];
                        const int h = g % 2 * 2;
                        to = __builtin_amdgcn_mfma_i32_16x16x32_i8(
                            __builtin_bit_cast(long, u32x2{w[h], w[h + 1]}),
                            __builtin_bit_cast(long, u32x2{v[h], v[h + 1]}), to, 0, 0, 0);
                    } else {
#pragma unroll
                        for (int u = g * (G / 64); u < (g + 1) * (G / 64); ++u)
                            to = __builtin_amdgcn_mfma_i32_16x16x64_i8(
                                __builtin_bit_cast(i32x4, a[j0 + j][u]),
                                __builtin_bit_cast(i32x4, x[i % 2][u]), to, 0, 0, 0);
                    }
                }
            }
            __builtin_amdgcn_sched_barrier(0);  // their results are a unit away
            if (n > 0) {
                const int m = n - 1, i = m / (PJ * NG), j0 = m / NG % PJ * 2, g = m % NG;
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float w = s[j0 + j][g][r];
                        const int v = sum[m % 2][j][r];
                        // the first group's subtraction is part of its product: 1.5 * 2^2 of a
                        // scale's 8 bits is exact
                        block[j][r] =
                            g == 0 ? __builtin_fmaf(__int_as_float(v), w, bias[j0 + j][r])
                                   : __builtin_fmaf(whole<kSmall>(v), w, block[j][r]);
                        if (g == NG - 1)
                            total[j0 + j][i][r] =
                                __builtin_fmaf(block[j][r], own[i], total[j0 + j][i][r]);
                    }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    auto multiply_float = [&](auto set, int buf, auto &&next) {
        const uint32_t mine = S::at(l % 16, quarter);
        constexpr int KEEP = G == 128 ? PJ * MT : 2;  // sums alive: all rows' over two halves
        constexpr int UG = G == 32 ? 2 : 1;      // groups in a half
        f32x4 sum[KEEP][2];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            bf16x8 a[NJ][2];
            f32x4 s[NJ][UG];
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
#pragma unroll
                for (int t = 0; t < 2; ++t) a[j][t] = widen(words[set][j][2 * half + t]);
#pragma unroll
                for (int g = 0; g < UG; ++g)
                    s[j][g] = scales(buf, j, G == 128 ? 0 : half * UG + g);
            }
            if (half == 1) next();
            __builtin_amdgcn_sched_barrier(0);
            u32x4 x[2][2][S::kTerms];
            auto read = [&](int i) {
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int n = 0; n < S::kTerms; ++n)
                        x[i % 2][t][n] = *reinterpret_cast<const u32x4 *>(
                            tile[buf] + n * S::kRows * S::kLd + 16 * i * S::kLd +
                            S::along(mine, 2 * half + t));
            };
            read(0);
#pragma unroll
            for (int n = 0; n <= MT * PJ * UG; ++n) {
                if (n < MT * PJ * UG) {
                    const int i = n / (PJ * UG), j0 = n / UG % PJ * 2, g = n % UG;
                    if (n % (PJ * UG) == 0 && i + 1 < MT) read(i + 1);
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        f32x4 &to = sum[n % KEEP][j];
                        if (G != 128 || half == 0) to = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                        for (int t = UG == 2 ? g : 0; t < (UG == 2 ? g + 1 : 2); ++t)
#pragma unroll
                            for (int k = S::kTerms - 1; k >= 0; --k)  // the smallest first
                                to = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                                    a[j0 + j][t], __builtin_bit_cast(bf16x8, x[i % 2][t][k]), to,
                                    0, 0, 0);
                    }
                }
                __builtin_amdgcn_sched_barrier(0);  // their results are a unit away
                if (n > 0 && (G != 128 || half == 1)) {
                    const int m = n - 1, i = m / (PJ * UG), j0 = m / UG % PJ * 2, g = m % UG;
#pragma unroll
                    for (int j = 0; j < 2; ++j)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            total[j0 + j][i][r] = __builtin_fmaf(
                                sum[m % KEEP][j][r], s[j0 + j][g][r], total[j0 + j][i][r]);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    };
    constexpr int NB = GATED ? 2 : 1;
    constexpr float back = X == kQ8 ? kBack(true) * 0x1p21f : kBack(false);
    __shared__ uint32_t sizes[OUT8 ? NW : 1][OUT8 ? S::kRows : 1];
    auto finish = [&](int n, int m) {
        const int n0 = (S::kBlocks * n + NJ * wave) / NB * kW4Outputs + 4 * quarter;
        float act[MT][NJ / NB][4];
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            const int at = 16 * i + l % 16, row = m * S::kRows + at;
            uint32_t most = 0;
#pragma unroll
            for (int j = 0; j < NJ / NB; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    float v = total[NB * j][i][r] * back;
                    if constexpr (GATED) v = silu(v) * (total[2 * j + 1][i][r] * back);
                    act[i][j][r] = v;
                    if (OUT8 && n0 + 16 * j < p.cols) most = max(most, size_bits(v));
                }
            if constexpr (!OUT8) {
                bool narrow = true;
                if constexpr (NJ / NB > 1)
                    if (y_dtype == QDC_BF16) {  // uniform
                        put_wide(p.y, p.cols, row, row < p.rows, n0 - 4 * quarter, quarter,
                                 act[i]);
                        narrow = false;
                    }
                if (narrow && row < p.rows) {
                    if (y_dtype == QDC_F32) put<float>(p.y, p.cols, row, n0, act[i]);
                    else put<bf16_t>(p.y, p.cols, row, n0, act[i]);
                }
            }
            if constexpr (OUT8) {  // over the quarters, then the wavefronts
                const auto a = __builtin_amdgcn_permlane16_swap(most, most, false, false);
                most = max(a[0], a[1]);
                const auto b = __builtin_amdgcn_permlane32_swap(most, most, false, false);
                most = max(b[0], b[1]);
                if (quarter == 0) sizes[wave][at] = most;
            }
        }
        if constexpr (OUT8) {
            __syncthreads();  // before the next tile's sizes there is another, if only a step's
            const int groups = (p.cols + kQ8Group - 1) / kQ8Group;
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                const int at = 16 * i + l % 16, row = m * S::kRows + at;
                if (row >= p.rows) continue;
                uint32_t most = sizes[0][at];
#pragma unroll
                for (int w = 1; w < NW; ++w) most = max(most, sizes[w][at]);
                const Q8Scale s(most);
#pragma unroll
                for (int j = 0; j < NJ / 2; ++j) {
                    if (n0 + 16 * j >= p.cols) continue;
                    *reinterpret_cast<uint32_t *>(reinterpret_cast<char *>(p.y) +
                                                  (int64_t)row * p.cols + n0 + 16 * j) =
                        s.word(act[i][j]);
                }
                if (wave == 0 && quarter == 0)
                    p.y_scales[(int64_t)row * groups + n] = s.scale;
            }
        }
    };

    Tiles mine(p);
    int n, m, buf = 0;
    mine.place(p, mine.at, n, m);
    const std::integral_constant<int, 0> first;
    const std::integral_constant<int, SETS - 1> second;
    load_x(first, m, 0);
    load_w(first, n, m, 0);
    if constexpr (SETS == 2) {
        load_x(second, m, 1);
        load_w(second, n, m, 1);
    }
    stage(first, 0, 0);
    __syncthreads();
    const int steps = round_up<SETS>(p.kb);
    for (;;) {
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int i = 0; i < MT; ++i) total[j][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        // The next tile's first steps are loaded with this one's last, so that memory is not
        // waited for between tiles.  (Behind the last tile: its own again.)
        const uint32_t after = mine.at + mine.step;
        const bool more = after < mine.count;
        int n1, m1;
        mine.place(p, more ? after : mine.at, n1, m1);
        // One block of code: after a branch, the last step's sums would be scaled behind it,
        // all of them held until then.
        for (int c = 0; c < steps; c += SETS) {
            const bool within = c + SETS < steps;
            const int n2 = within ? n : n1, m2 = within ? m : m1, c2 = within ? c + SETS : 0;
            auto step = [&](auto set, auto other, int at, int staged) {
                auto next = [&] {
                    load_w(set, n2, m2, c2 + set);
                    load_x(set, m2, c2 + set);
                };
                if constexpr (X == kQ8) multiply_whole(set, at, next);
                else multiply_float(set, at, next);
                stage(other, at ^ 1, staged);  // read a step ago, a barrier back
                __syncthreads();
            };
            if constexpr (SETS == 2) {
                // an odd number of steps has one more, of rows of zeros
                step(first, second, 0, c + 1);
                step(second, first, 1, c2);
            } else {
                step(first, first, buf, c2);
                buf ^= 1;
            }
        }
        finish(n, m);
        if (!more) return;
        mine.at = after;
        n = n1;
        m = m1;
    }
}

// ---------------------------------------------------------------- dispatch ---
template <int X, int G, int MT, int NB, bool GATED, int WAVES>
int32_t launch_rows(const W4Product &p, int32_t y_dtype, hipStream_t s) {
    const dim3 grid((uint32_t)ceil_div((int64_t)p.nb, (int64_t)NB),
                    (uint32_t)ceil_div((int64_t)p.rows, (int64_t)16 * MT));
    const W4Rows q{p.x,      p.x_scales, p.packed, p.scales, p.y,
                   (uint32_t)p.ld_x, p.rows,     p.cols,   p.inner,  p.nb, y_dtype};
    hipLaunchKernelGGL((w4_rows<X, G, MT, NB, GATED, WAVES>), grid, dim3(WAVES * kWave), 0, s, q);
    return launch_status();
}
template <int X, int G, int MT, int NJ, int NW, bool GATED, bool OUT8>
int32_t launch_tiles(const W4Product &p, int32_t y_dtype, hipStream_t s) {
    // (who launches a taller tile looks at the distance)
    static_assert(MT == 8 || Staged<X, G, MT, NJ, NW>::kFarthest >= kW4RowBytes, "row offsets");
    W4Product q = p;
    const int64_t tiles_n = ceil_div((int64_t)p.nb, (int64_t)NJ * NW);
    q.tiles_m = (int)ceil_div((int64_t)p.rows, (int64_t)16 * MT);
    q.strip = make_fastdiv((uint32_t)(8 * tiles_n));
    const int64_t tiles = tiles_n * q.tiles_m;
    if (tiles >= (int64_t)1 << 30) return QDC_ERR_SHAPE;
    q.tiles = (uint32_t)tiles;
    const uint32_t most = 2048 / NW;  // two wavefronts a SIMD
    const uint32_t grid = tiles < most ? (uint32_t)tiles : most;
    hipLaunchKernelGGL((w4_tiles<X, G, MT, NJ, NW, GATED, OUT8>), dim3(grid), dim3(NW * kWave), 0,
                       s, q, y_dtype);
    return launch_status();
}

// The kernel with the smallest tile of which the chip's 256 units take one each at most; where
// none is large enough the one that is fastest when they take many.  us for 1024 -> 5120,
// groups of 64 (in brackets the workgroups, where they are more than 256):
//   rows x outputs of a tile   16 x 16  16 x 32  32 x 32  32 x 64  32 x 128  32 x 256  64 x 256
//   bf16   16 rows            4.7 (320)    4.4      4.5       -        -         -         -
//          32                 6.0 (640) 5.5 (320)   5.2      6.4       -         -         -
//          96                     -     8.1 (960) 7.4 (480)  6.6       -         -         -
//         128                     -        -     9.4 (640) 11.3 (320) 8.9      11.1        -
//         256                     -        -        -     16.1 (640) 11.8 (320) 11.9     14.9
//         512                     -        -        -        -     16.6 (640) 20 (320)   15.9
//   fp32  301                     -        -        -        -     19.2 (400)  15.4      23.4
// and by tiles of 64 x 256 in 4 wavefronts, two workgroups a unit / 128 x 256 in 8 (fp32: 32 / 64
// rows) 4096 rows: 8-bit 45 / 56, bf16 56 / 62, fp32 127 / 110; 16384: 185 / 189, 233 / 224, 466 /
// 421; 2048 -> 6144 of 1024 rows: 34 / 36, 45 / 39, 71 / 81.
template <int X, int G, bool GATED, bool OUT8>
int32_t launch_many(const W4Product &p, int32_t y_dtype, hipStream_t s) {
    auto tiles = [&](int rows, int blocks) {
        return ceil_div((int64_t)p.rows, (int64_t)rows) * ceil_div((int64_t)p.nb, (int64_t)blocks);
    };
    // 128 outputs or fewer take no tile of 256
    if constexpr (!OUT8)
        if (p.nb <= 8) return launch_tiles<X, G, 2, 2, 4, GATED, false>(p, y_dtype, s);
    if constexpr (X == kF32 || OUT8) {
        if (tiles(16, 16) <= 256) return launch_tiles<X, G, 1, 2, 8, GATED, OUT8>(p, y_dtype, s);
    } else {
        // of 8-bit rows two of these to a unit are faster than one twice as large: us 128 rows
        // 2048 -> 6144 11.5 / 12.2 / 14.7 of 16, 32 rows x 128, 32 x 256; 256 rows 17.7 / 14.7 /
        // 15.3
        constexpr int most = X == kQ8 ? 512 : 256;
        if constexpr (X == kQ8)
            if (tiles(16, 8) <= most) return launch_tiles<X, G, 1, 2, 4, GATED, false>(p, y_dtype, s);
        if (tiles(32, 8) <= most) return launch_tiles<X, G, 2, 2, 4, GATED, false>(p, y_dtype, s);
    }
    if (tiles(32, 16) <= 256) return launch_tiles<X, G, 2, 2, 8, GATED, OUT8>(p, y_dtype, s);
    // groups of 32 of 8-bit rows: more of them would not fit the registers
    if (tiles(64, 16) <= 256 || (X == kF32 && tiles(64, 16) >= 768) || (X == kQ8 && G == 32))
        return launch_tiles<X, G, 4, 2, 8, GATED, OUT8>(p, y_dtype, s);
    if constexpr (X == kF32)  // three terms a row in LDS
        return launch_tiles<X, G, 2, 4, 4, GATED, OUT8>(p, y_dtype, s);
    // 128 rows of the greatest distance are more than a tile's offsets hold
    if constexpr (X == kBf16)
        if (tiles(128, 16) >= 768 && p.ld_x * kXBytes<X> <= Staged<X, G, 8, 2, 8>::kFarthest)
            return launch_tiles<X, G, 8, 2, 8, GATED, OUT8>(p, y_dtype, s);
    if constexpr (X == kBf16 || (X == kQ8 && G != 32))
        return launch_tiles<X, G, 4, 4, 4, GATED, OUT8>(p, y_dtype, s);
    return QDC_ERR_SHAPE;  // not reached
}

template <int X, int G, bool GATED>
int32_t launch(const W4Product &p, int32_t y_dtype, hipStream_t s) {
    if constexpr (GATED)
        if (y_dtype == QDC_Q8) return launch_many<X, G, true, true>(p, y_dtype, s);
    auto fits = [&](int rows, int blocks) {
        return ceil_div((int64_t)p.rows, (int64_t)rows) * ceil_div((int64_t)p.nb, (int64_t)blocks) <=
               256;
    };
    if constexpr (!GATED)
        // (of a row or four the rows cost nothing to read twice: 1024 -> 7168, one row of bf16,
        // 448 workgroups 3.3 us, 224 of two blocks 3.8)
        if (fits(16, 1) || p.nb == 1 || (X != kF32 && p.rows <= 4 && p.nb <= 512)) {
            // a wavefront for each 128 inputs, up to 16: 3584 -> 1024, one row of bf16, 4.1
            // us, of fp32 8.7, with 8 wavefronts 4.3 and 10.4; 256 -> 768 with 4 2.3, 8 2.4
            if (p.kb <= 4) return launch_rows<X, G, 1, 1, false, 4>(p, y_dtype, s);
            if (p.kb < 16) return launch_rows<X, G, 1, 1, false, 8>(p, y_dtype, s);
            return launch_rows<X, G, 1, 1, false, 16>(p, y_dtype, s);
        }
    if (fits(16, 2)) {
        if constexpr (X == kF32)  // 3584 -> 4096 of 8 rows 10.3 us, with 8 11.7; bf16 7.0, 7.1
            if (p.kb >= 16) return launch_rows<X, G, 1, 2, GATED, 16>(p, y_dtype, s);
        return launch_rows<X, G, 1, 2, GATED, 8>(p, y_dtype, s);
    }
    // Groups of 32 of 8-bit rows are nearer to bf16 than to larger ones: twice the sums to scale.
    constexpr bool few_sums = X == kQ8 && G != 32;
    // (outputs of a tile or less: x is read once however many the rows are.  Of 17 to 32 rows two
    // sets of 16 share a weight's widening: 24 rows 1024 -> 7168 bf16 4.9 us, by 16 x 64 5.4)
    if (p.nb <= 2 || (X != kF32 && !few_sums && p.rows <= 32 && fits(32, 2)))
        return launch_rows<X, G, 2, 2, GATED, 8>(p, y_dtype, s);
    // 64 rows 3584 -> 4096 fp32 16.7 us, bf16 10.3, 8-bit 9.7; by 32 x 32 20.5, 10.8, 11.3
    if (fits(16, 4)) return launch_rows<X, G, 1, 4, GATED, 8>(p, y_dtype, s);
    if (fits(32, 4)) {
        // 32 x 64 with the inputs over 8 wavefronts, or 16 x 128 with the outputs over 4: us for
        // 96 rows 512 -> 5120 of bf16 5.5 / 5.1, for 48 rows 2048 -> 6144 9.3 / 11.6, of fp32
        // 16.2 / 17.3, of 8 bits 9.4 / 9.0 (groups of 32: 11.3 / 11.4; 3584 -> 4096 of 96 rows
        // 16.5 / 18.0).  fp32 rows in groups of 32 would not fit the registers of the first:
        // 25.8 / 17.5.
        constexpr bool by_outputs = few_sums || (X == kF32 && G == 32);
        if (p.nb > 4 && (by_outputs || p.kb <= (X == kQ8 ? 16 : 4)))
            return launch_tiles<X, G, 1, 2, 4, GATED, false>(p, y_dtype, s);
        if constexpr (!by_outputs) return launch_rows<X, G, 2, 4, GATED, 8>(p, y_dtype, s);
    }
    return launch_many<X, G, GATED, false>(p, y_dtype, s);
}

template <int X>
int32_t linear_w4(const W4Product &p, int group, bool gated, int32_t y_dtype, hipStream_t s) {
    if (group == 32) return gated ? launch<X, 32, true>(p, y_dtype, s) : launch<X, 32, false>(p, y_dtype, s);
    if (group == 64) return gated ? launch<X, 64, true>(p, y_dtype, s) : launch<X, 64, false>(p, y_dtype, s);
    return gated ? launch<X, 128, true>(p, y_dtype, s) : launch<X, 128, false>(p, y_dtype, s);
}

}  // namespace
}  // namespace qdc
