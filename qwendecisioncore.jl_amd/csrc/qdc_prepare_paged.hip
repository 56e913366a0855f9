// qdc_prepare_paged.hip -- per-head zero-centred RMSNorm and half-split partial RoPE
// of q and k heads, each token at its own position, with the K and V rows stored into
// the pages of a cache:
//     s = 1/sqrt(mean(x^2) + eps),  y = x s (1 + w),
//     (y_i, y_{i+half}) <- (y_i c - y_{i+half} s', y_{i+half} c + y_i s')
//
// A group of lanes owns a row (token, head): one 16-byte chunk a lane, so a row's sum
// is one lane-group reduction and every access of the group covers the whole row.  A
// lane with a rotary chunk reads its partner chunk, half a rotary block away, from the
// same row a second time: it is in the cache line the group is fetching anyway.
#include "qdc_cache.hpp"

namespace qdc {
namespace {

struct PreparePaged {
    void *q_out, *k_out, *k_pages, *v_pages;
    const void *q, *k, *v, *q_norm, *k_norm;
    const float *cos, *sin;
    const int32_t *index, *positions, *table;
    int32_t *error_flag;
    int64_t q_tok, q_head, k_tok, k_head, v_tok, v_head, width;
    int64_t total;           // tokens * (heads + 2 kv_heads)
    FastDiv per_token;       // heads + 2 kv_heads
    int heads, kv, half, rows, pages, shift;
    int64_t table_len, reach;  // positions below both are stored
    float eps;
};

template <typename T, int HD>
__global__ __launch_bounds__(kBlock) void prepare_paged(PreparePaged a) {
    constexpr int V = Elem<T>::kVec, LPR = HD / V, GPB = kBlock / LPR;
    const int lane = threadIdx.x % LPR;
    const int64_t unit = (int64_t)blockIdx.x * GPB + threadIdx.x / LPR;
    if (unit >= a.total) return;  // uniform per lane group
    const uint32_t t = fastdiv((uint32_t)unit, a.per_token);
    const int r = (int)((uint32_t)unit - t * a.per_token.d);
    const int pos = a.positions[t], row = a.index[t];
    const bool is_q = r < a.heads, is_v = r >= a.heads + a.kv;
    const int g = is_q ? r : is_v ? r - a.heads - a.kv : r - a.heads;
    const T *src = is_q   ? (const T *)a.q + (int64_t)t * a.q_tok + (int64_t)g * a.q_head
                   : is_v ? (const T *)a.v + (int64_t)t * a.v_tok + (int64_t)g * a.v_head
                          : (const T *)a.k + (int64_t)t * a.k_tok + (int64_t)g * a.k_head;
    const u32x4 raw = load_stream(src + lane * V);
    const bool token = pos >= 0 && row >= 0;
    bool live = token && pos < a.reach && pos < a.table_len && row < a.rows;
    int64_t place = 0;  // element offset of this row in its page tensor
    if (live) {
        const int32_t page = a.table[(int64_t)row * a.width + (pos >> a.shift)];
        live = (uint32_t)page < (uint32_t)a.pages;
        place = (((int64_t)page * a.kv + g) << a.shift) + (pos & ((1 << a.shift) - 1));
        place = place * HD + lane * V;
    }
    if (token && !live && lane == 0 && r == 0) raise_flag(a.error_flag);
    if (is_v) {
        if (live) *reinterpret_cast<u32x4 *>((T *)a.v_pages + place) = raw;
        return;
    }
    const T *norm = (const T *)(is_q ? a.q_norm : a.k_norm);
    float x[V], w[V], ss = 0.0f;
    unpack(raw, x);
    load_chunk(norm + lane * V, w);
#pragma unroll
    for (int j = 0; j < V; ++j) ss += x[j] * x[j];
    ss = group_sum<LPR>(ss);
    const float s = rms_scale(ss, (float)HD, a.eps);
    const int e0 = lane * V, half = a.half;
    if (live && e0 < 2 * half) {
        const float *cs = a.cos + (int64_t)pos * half, *sn = a.sin + (int64_t)pos * half;
        if (half % V == 0) {  // the whole chunk in one half of the rotary block
            const bool first = e0 < half;
            const int ep = first ? e0 + half : e0 - half, ei = first ? e0 : ep;
            float p[V], wp[V], c[V], d[V];
            load_chunk(src + ep, p);
            load_chunk(norm + ep, wp);
#pragma unroll
            for (int q = 0; q < V / 4; ++q) {
                float c4[4], d4[4];
                load_chunk(cs + ei + 4 * q, c4);
                load_chunk(sn + ei + 4 * q, d4);
#pragma unroll
                for (int e = 0; e < 4; ++e) c[4 * q + e] = c4[e], d[4 * q + e] = d4[e];
            }
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float y = (x[j] * s) * (1.0f + w[j]), z = (p[j] * s) * (1.0f + wp[j]);
                x[j] = first ? y * c[j] - z * d[j] : y * c[j] + z * d[j];
            }
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const int e = e0 + j;
                const float y = (x[j] * s) * (1.0f + w[j]);
                if (e < 2 * half) {
                    const bool first = e < half;
                    const int ep = first ? e + half : e - half, ei = first ? e : ep;
                    const float z = (to_f32(src[ep]) * s) * (1.0f + to_f32(norm[ep]));
                    x[j] = first ? y * cs[ei] - z * sn[ei] : y * cs[ei] + z * sn[ei];
                } else {
                    x[j] = y;
                }
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) x[j] = (x[j] * s) * (1.0f + w[j]);
    }
    if (is_q) {
        store_chunk((T *)a.q_out + ((int64_t)t * a.heads + g) * HD + lane * V, x);
        return;
    }
    if (a.k_out) store_chunk((T *)a.k_out + ((int64_t)t * a.kv + g) * HD + lane * V, x);
    if (live) *reinterpret_cast<u32x4 *>((T *)a.k_pages + place) = pack(x);
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
    a.total = tokens * (heads + 2 * kv_heads);
    a.per_token = make_fastdiv((uint32_t)(heads + 2 * kv_heads));
    a.heads = (int)heads;
    a.kv = (int)kv_heads;
    a.half = (int)(rotary_dim / 2);
    a.rows = (int)rows;
    a.pages = (int)pages;
    a.shift = shift;
    a.table_len = rotary_dim > 0 ? table_len : lim;
    a.reach = width * page_size;
    a.eps = eps;
#define QDC_PREPARE(T, HD)                                                                     \
    if (head_dim == HD) {                                                                      \
        constexpr int64_t gpb = kBlock / (HD / Elem<T>::kVec);                                 \
        hipLaunchKernelGGL((prepare_paged<T, HD>), dim3((uint32_t)ceil_div(a.total, gpb)),     \
                           dim3(kBlock), 0, stream, a);                                        \
        return launch_status();                                                                \
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
    return QDC_ERR_SHAPE;
}
