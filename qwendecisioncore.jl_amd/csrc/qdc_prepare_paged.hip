// qdc_prepare_paged.hip -- per-head zero-centred RMSNorm and half-split partial RoPE
// of q and k heads, each token at its own position, with the K and V rows stored into
// the pages of a cache:
//     s = 1/sqrt(mean(x^2) + eps),  y = x s (1 + w),
//     (y_i, y_{i+half}) <- (y_i c - y_{i+half} s', y_{i+half} c + y_i s')
//
// A group of lanes, a 16-byte chunk of a row each, owns RPG query heads of a token or
// one K and V head: one position, rotation and place for all of them, every row's loads
// before the first is used, and a row's sum one lane-group reduction.  A lane with a
// rotary chunk reads its partner chunk, half a rotary block away, from the same row a
// second time: it is in the cache line the group is fetching anyway, and the other
// lanes read one line there together.
//
// Bound by memory: 16384 tokens of 8 + 2 heads of 256 (bf16, 105 MB read, 105 written)
// 36.3 us = 5.8 TB/s, of 6.5 for a copy: what is between is the chain position -> page ->
// place in front of the K and V stores and the stores' scatter over the pages.  One token
// 2.7 us, a launch and three dependent loads.
#include "qdc_cache.hpp"

namespace qdc {
namespace {

// Small workgroups let stores begin while other rows load (us, 16384 tokens of 8 + 2 heads of
// 256 in bf16, 64 / 128 / 256 / 512 threads: 40.9 / 36.3 / 37.3 / 42.8; other sizes within
// 4% between 64 and 256).
constexpr int kThreads = 128;

struct PreparePaged {
    void *q_out, *k_out, *k_pages, *v_pages;
    const void *q, *k, *v, *q_norm, *k_norm;
    const float *cos, *sin;
    const int32_t *index, *positions, *table;
    int32_t *error_flag;
    int64_t q_tok, q_head, k_tok, k_head, v_tok, v_head, width;
    int64_t total;           // tokens * units of a token: heads / RPG + kv_heads
    FastDiv per_token;       // units of a token
    int heads, kv, half, rows, pages, shift;
    int64_t table_len, reach;  // positions below both are stored
    float eps;
};

// What a lane needs of the rotation: its own chunk's first element e0, its partner's.
template <typename T> struct Turn {
    static constexpr int V = Elem<T>::kVec;
    bool rotary, first;  // in the rotary block, in its first half
    int e0, ep;
    float c[V], s[V];

    __device__ __forceinline__ void place(int lane, int half) {
        e0 = lane * V;
        rotary = e0 < 2 * half;
        first = e0 < half;
        ep = first ? e0 + half : e0 - half;
    }
    __device__ __forceinline__ void load(const PreparePaged &a, int pos) {
        const int64_t at = (int64_t)pos * a.half + (first ? e0 : ep);
#pragma unroll
        for (int q = 0; q < V / 4; ++q) {
            const u32x4 cr = load_raw(a.cos + at + 4 * q), sr = load_raw(a.sin + at + 4 * q);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                c[4 * q + e] = __uint_as_float(cr[e]);
                s[4 * q + e] = __uint_as_float(sr[e]);
            }
        }
    }
};

// A row's chunk, normalised and, with `turned`, rotated; `raw` and `other` hold its own
// and its partner's chunk, w and wp their weights.  WHOLE: the halves of the rotary
// block are whole chunks.
template <typename T, int HD, bool WHOLE>
__device__ __forceinline__ void norm_rope(const PreparePaged &a, const Turn<T> &t, bool turned,
                                          int pos, const T *src, const T *norm, u32x4 raw,
                                          u32x4 other, const float (&w)[Elem<T>::kVec],
                                          const float (&wp)[Elem<T>::kVec],
                                          float (&x)[Elem<T>::kVec]) {
    constexpr int V = Elem<T>::kVec, LPR = HD / V;
    float ss = 0.0f;
    unpack(raw, x);
#pragma unroll
    for (int j = 0; j < V; ++j) ss += x[j] * x[j];
    ss = group_sum<LPR>(ss);
    const float s = rms_scale(ss, (float)HD, a.eps);
#pragma unroll
    for (int j = 0; j < V; ++j) x[j] = (x[j] * s) * (1.0f + w[j]);
    if (!turned) return;
    if constexpr (WHOLE) {
        float p[V];
        unpack(other, p);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float z = (p[j] * s) * (1.0f + wp[j]);
            x[j] = t.first ? x[j] * t.c[j] - z * t.s[j] : x[j] * t.c[j] + z * t.s[j];
        }
    } else {
        const float *cs = a.cos + (int64_t)pos * a.half, *sn = a.sin + (int64_t)pos * a.half;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int e = t.e0 + j;
            if (e >= 2 * a.half) continue;
            const bool first = e < a.half;
            const int ep = first ? e + a.half : e - a.half, ei = first ? e : ep;
            const float z = (to_f32(src[ep]) * s) * (1.0f + to_f32(norm[ep]));
            x[j] = first ? x[j] * cs[ei] - z * sn[ei] : x[j] * cs[ei] + z * sn[ei];
        }
    }
}

template <typename T, int HD, int RPG, bool WHOLE>
__global__ __launch_bounds__(kThreads) void prepare_paged(PreparePaged a) {
    constexpr int V = Elem<T>::kVec, LPR = HD / V, GPB = kThreads / LPR;
    const int lane = threadIdx.x % LPR;
    const int64_t unit = (int64_t)blockIdx.x * GPB + threadIdx.x / LPR;
    if (unit >= a.total) return;  // uniform per lane group
    const uint32_t t = fastdiv((uint32_t)unit, a.per_token);
    const int r = (int)((uint32_t)unit - t * a.per_token.d), q_units = a.heads / RPG;
    const int pos = a.positions[t], row = a.index[t];
    const bool is_q = r < q_units;
    const int h = is_q ? r * RPG : r - q_units;  // the first query head, or the KV head
    const T *norm = (const T *)(is_q ? a.q_norm : a.k_norm);
    const T *src = is_q ? (const T *)a.q + (int64_t)t * a.q_tok + (int64_t)h * a.q_head
                        : (const T *)a.k + (int64_t)t * a.k_tok + (int64_t)h * a.k_head;
    Turn<T> turn;
    turn.place(lane, a.half);
    const bool paired = WHOLE && turn.rotary;
    float w[V], wp[V];
    load_chunk(norm + turn.e0, w);
    load_chunk(norm + (paired ? turn.ep : 0), wp);
    u32x4 raw[RPG], other[RPG], value = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int i = 0; i < RPG; ++i) {
        if (i && !is_q) continue;  // uniform per lane group
        const T *x = src + i * a.q_head;
        raw[i] = load_stream(x + turn.e0);
        other[i] = load_raw(x + (paired ? turn.ep : 0));  // unused: one line for all lanes
    }
    if (!is_q)
        value = load_stream((const T *)a.v + (int64_t)t * a.v_tok + (int64_t)h * a.v_head + turn.e0);
    const bool token = pos >= 0 && row >= 0;
    bool live = token && pos < a.reach && pos < a.table_len && row < a.rows;
    if (live && paired) turn.load(a, pos);
    int64_t place = 0;  // element offset of this K and V row's chunk in its page tensor
    if (live) {
        const int32_t page = a.table[(int64_t)row * a.width + (pos >> a.shift)];
        live = (uint32_t)page < (uint32_t)a.pages;
        place = (((int64_t)page * a.kv + h) << a.shift) + (pos & ((1 << a.shift) - 1));
        place = place * HD + turn.e0;
    }
    if (token && !live && lane == 0 && r == 0) raise_flag(a.error_flag);
    const bool turned = live && turn.rotary;
    float x[V];
    if (is_q) {
        T *dst = (T *)a.q_out + ((int64_t)t * a.heads + h) * HD + turn.e0;
#pragma unroll
        for (int i = 0; i < RPG; ++i) {
            norm_rope<T, HD, WHOLE>(a, turn, turned, pos, src + i * a.q_head, norm, raw[i], other[i], w, wp,
                             x);
            store_chunk(dst + i * HD, x);
        }
        return;
    }
    norm_rope<T, HD, WHOLE>(a, turn, turned, pos, src, norm, raw[0], other[0], w, wp, x);
    if (a.k_out) store_chunk((T *)a.k_out + ((int64_t)t * a.kv + h) * HD + turn.e0, x);
    if (live) {
        // plain stores: the attention that follows reads the pages (as a stream 2% slower)
        *reinterpret_cast<u32x4 *>((T *)a.k_pages + place) = pack(x);
        *reinterpret_cast<u32x4 *>((T *)a.v_pages + place) = value;
    }
}

}  // namespace
}  // namespace qdc

using namespace qdc;

extern "C" const char *qdc_cache_version(void) { return QDC_HIP_CACHE_VERSION; }

extern "C" int32_t qdc_prepare_paged(
    void *q_out, void *k_out, void *k_pages, void *v_pages, const void *q, const void *k,
    const void *v, const void *q_norm, const void *k_norm, const float *cos_table,
    const float *sin_table, const int32_t *index, const int32_t *positions, const int32_t *table,
    int64_t tokens, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t rotary_dim,
    int64_t table_len, int64_t rows, int64_t width, int64_t pages, int64_t page_size,
    int64_t q_tok, int64_t q_head, int64_t k_tok, int64_t k_head, int64_t v_tok, int64_t v_head,
    float eps, int32_t dtype, int32_t *error_flag, hipStream_t stream) {
    if (!valid_dtype(dtype)) return QDC_ERR_DTYPE;
    const int shift = page_shift(page_size);
    if (tokens < 0 || heads <= 0 || kv_heads <= 0 || rows <= 0 || width <= 0 || pages <= 0 ||
        table_len < 0 || rotary_dim < 0 || rotary_dim % 2 || rotary_dim > head_dim || shift < 0 ||
        (head_dim != 64 && head_dim != 128 && head_dim != 256))
        return QDC_ERR_SHAPE;
    const int64_t lim = (int64_t)1 << 31, small = (int64_t)1 << 20;
    if (heads >= small || kv_heads >= small || tokens >= lim || rows >= lim || pages >= lim ||
        width >= lim / 256 || tokens * (heads + 2 * kv_heads) >= ((int64_t)1 << 26))
        return QDC_ERR_SHAPE;
    // Q, K and V rows are read as [tokens, heads] grids of whole 16-byte chunks
    const int64_t es = elem_size(dtype), per = 16 / es;
    if (q_head < head_dim || k_head < head_dim || v_head < head_dim || q_tok < 0 || k_tok < 0 ||
        v_tok < 0 || (q_tok | q_head | k_tok | k_head | v_tok | v_head) % per)
        return QDC_ERR_SHAPE;
    if (tokens == 0) return QDC_OK;
    if (!q_out || !k_pages || !v_pages || !q || !k || !v || !q_norm || !k_norm || !index ||
        !positions || !table || (rotary_dim > 0 && (!cos_table || !sin_table)))
        return QDC_ERR_NULL;
    if (!aligned16(q_out) || !aligned16(k_out) || !aligned16(k_pages) || !aligned16(v_pages) ||
        !aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(q_norm) ||
        !aligned16(k_norm) ||
        (rotary_dim > 0 && (!aligned16(cos_table) || !aligned16(sin_table))))
        return QDC_ERR_SHAPE;
    const int64_t store = pages * kv_heads * page_size * head_dim * es, norm = head_dim * es;
    const int64_t rope = rotary_dim > 0 ? table_len * (rotary_dim / 2) * 4 : 0;
    const Range outs[5] = {{q_out, tokens * heads * head_dim * es},
                           {k_out, k_out ? tokens * kv_heads * head_dim * es : 0},
                           {k_pages, store},
                           {v_pages, store},
                           {error_flag, error_flag ? 4 : 0}};
    const Range ins[10] = {{q, grid_span(tokens, heads, q_tok, q_head, head_dim, es)},
                           {k, grid_span(tokens, kv_heads, k_tok, k_head, head_dim, es)},
                           {v, grid_span(tokens, kv_heads, v_tok, v_head, head_dim, es)},
                           {q_norm, norm}, {k_norm, norm}, {cos_table, rope}, {sin_table, rope},
                           {index, tokens * 4}, {positions, tokens * 4},
                           {table, rows * width * 4}};
    if (any_alias(outs, 5, ins, 10)) return QDC_ERR_ALIAS;
    PreparePaged a{};
    a.q_out = q_out;
    a.k_out = k_out;
    a.k_pages = k_pages;
    a.v_pages = v_pages;
    a.q = q;
    a.k = k;
    a.v = v;
    a.q_norm = q_norm;
    a.k_norm = k_norm;
    a.cos = cos_table;
    a.sin = sin_table;
    a.index = index;
    a.positions = positions;
    a.table = table;
    a.error_flag = error_flag;
    a.q_tok = q_tok;
    a.q_head = q_head;
    a.k_tok = k_tok;
    a.k_head = k_head;
    a.v_tok = v_tok;
    a.v_head = v_head;
    a.width = width;
    a.half = (int)(rotary_dim / 2);
    // Query heads of a lane group: two, four where bf16 rows of 32 MB and more stream by
    // (us, 1 / 2 / 4: 8 x 2048 tokens of 8 + 2 heads of 256 44.5 / 40.5 / 38.5, 64 tokens 3.4
    // / 3.3 / 3.9; fp32 9600 tokens 47.5 / 46.1 / 47.3).
    const bool whole = a.half % (16 / es) == 0;
    const int most = dtype == QDC_BF16 && tokens * heads * head_dim * es >= (32 << 20) ? 4 : 2;
    int rpg = 1;
    while (whole && rpg < most && heads % (2 * rpg) == 0) rpg *= 2;
    a.total = tokens * (heads / rpg + kv_heads);
    a.per_token = make_fastdiv((uint32_t)(heads / rpg + kv_heads));
    a.heads = (int)heads;
    a.kv = (int)kv_heads;
    a.rows = (int)rows;
    a.pages = (int)pages;
    a.shift = shift;
    a.table_len = rotary_dim > 0 ? table_len : lim;
    a.reach = width * page_size;
    a.eps = eps;
#define QDC_PREPARE_ROWS(T, HD, RPG, WHOLE)                                                    \
    if (rpg == RPG && whole == WHOLE) {                                                        \
        constexpr int64_t gpb = kThreads / (HD / Elem<T>::kVec);                                 \
        hipLaunchKernelGGL((prepare_paged<T, HD, RPG, WHOLE>),                                 \
                           dim3((uint32_t)ceil_div(a.total, gpb)), dim3(kThreads), 0, stream, a);\
        return launch_status();                                                                \
    }
#define QDC_PREPARE(T, HD)                                                                     \
    if (head_dim == HD) {                                                                      \
        QDC_PREPARE_ROWS(T, HD, 4, true)                                                       \
        QDC_PREPARE_ROWS(T, HD, 2, true)                                                       \
        QDC_PREPARE_ROWS(T, HD, 1, true)                                                       \
        QDC_PREPARE_ROWS(T, HD, 1, false)                                                      \
    }
    if (dtype == QDC_BF16) {
        QDC_PREPARE(bf16_t, 64)
        QDC_PREPARE(bf16_t, 128)
        QDC_PREPARE(bf16_t, 256)
    }
    QDC_PREPARE(float, 64)
    QDC_PREPARE(float, 128)
    QDC_PREPARE(float, 256)
#undef QDC_PREPARE
#undef QDC_PREPARE_ROWS
    return QDC_ERR_SHAPE;
}
