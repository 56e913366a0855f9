// qdc_paged_attention.hip -- attention of one token's queries over the pages of its
// cache row, with the output gate:
//     out_h = sigmoid(gate_h) * sum_j softmax_j(scale q_h . k_j) v_j,  j <= position.
//
// Every key and value is read once for the (up to 16) query heads that share it, so
// the reads of the pages are all that it has to cost.  The work is cut by what is
// there, not by what could be: the keys of all entries, head after head, in tiles (32
// keys bf16, 16 fp32), are dealt to the workgroups in even parts whatever the lengths
// are.  Each workgroup finds its tiles from the positions by itself; a piece that is not
// all of a head's keys leaves its maximum, sum and unnormalised output in the workspace,
// and a second launch joins the pieces of a head in order.
//
// Scores are formed transposed, S^T = K Q^T on the matrix cores: a lane then holds
// the scores of one head for some keys, the operand layout of O^T = V^T P^T, and the
// running maximum, sum and rescaling are in-lane but for two lane swaps a tile.  Which
// keys and which values sit in a matrix operand's slots is free as long as both
// operands agree, so K, V and the pages' rows go from memory to operands in 16-byte
// pieces with no stop in LDS: V's 8 keys x 8 values of a lane are paired into operands
// with one byte permute each.  For bf16 pages the weights enter the product as two bf16
// terms: rounded to one they would add as much error as the output's own rounding, and
// the matrix cores have time for both.
//
// It is bound by the reads of K and V: 2 rows of 100003 keys of 4 heads of 256 (bf16, 819
// MB, each byte fetched once) 123 us = 6.7 TB/s with its join of 4.6 us behind it, of 7.0
// that a plain streaming read reaches; 2 rows of 100000 of 2 heads of 256 in fp32 (819 MB)
// 128 + 5.2; 96 rows of 0 .. 16384 keys (333 MB) 56 us = 6.0 TB/s.  Where little is read the
// chain positions -> pages -> K -> scores -> join counts: 8 rows of 2048 keys (34 MB) 10.5 +
// 4.0 us, one row of 411 keys (0.4 MB) 5.0 + 3.3, or 6.9 in one launch where the table is so
// narrow that every row must be short.
#include <cfloat>
#include <type_traits>

#include "qdc_cache.hpp"

namespace qdc {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr int kWaves = kBlock / kWave;
constexpr int kHeads = 16;          // query heads of a unit: a matrix operand's columns
constexpr uint32_t kMinTiles = 4;  // fewer a workgroup leave wavefronts without a tile
constexpr int kMaxLogWgs = 9;

// Wavefronts of a workgroup that has a unit to itself, as many as the registers let in,
// and the tiles that it may have.
constexpr int short_waves(int head_dim) { return head_dim == 64 ? 16 : head_dim == 128 ? 8 : 4; }
constexpr int kShortTiles = 2;  // a wavefront's

struct PagedAttention {
    void *out;
    const void *q, *k, *v, *gate;
    const int32_t *table, *index, *positions;
    int32_t *error_flag;
    float *pieces, *stats;  // [2 workgroups][heads of a unit][head_dim], [..][2]
    int64_t q_tok, q_head, gate_tok, gate_head, out_tok, width;
    int n, heads, kv, group, unit_heads, head_groups, rows, pages, shift, log_wgs, join_heads;
    int out_dtype;
    float scale_log2;       // scale * log2(e)
};

template <typename T> constexpr int tile_keys() { return sizeof(T) == 2 ? 32 : 16; }

// Keys of an entry: 0 for one that is no token.
__device__ __forceinline__ int entry_keys(const PagedAttention &a, int row, int pos, bool &bad) {
    bad = row >= a.rows && pos >= 0;
    if (row < 0 || pos < 0 || bad) return 0;
    const int64_t reach = a.width << a.shift;
    bad = pos >= reach;
    return bad ? (int)reach : pos + 1;
}

// What beginning a unit costs, as bytes of pages read in that time: the chain to its page
// numbers and the join of its wavefronts, which for heads of 256 no second workgroup of
// the compute unit fills.  (96 rows of 0 .. 16384 keys of 256, us: 32 KB 78, 64 KB 64,
// 128 KB 56, 256 KB 57; 200 rows of 1 .. 4000 of 64: 17.9, 17.1, 20.0, 24.6.)
constexpr int begin_bytes(int head_dim) { return head_dim > 128 ? 131072 : 65536; }

// How the call's work, entry by entry and unit by unit (KV head and group of its query
// heads), is dealt to the workgroups.  Of up to 64 entries a unit is cut into parts of up
// to `share` tiles, a workgroup each, where that takes no more than the workgroups and no
// more rounds of a tile a wavefront than an even split would.  Anything else is a line
// that is cut evenly: a unit is kBegin tiles' worth for beginning it and then its tiles.
// (us, shares / line: 8 rows of 2048 keys of 256 11.2 / 12.1, 32 of 1000 16.2 /
// 17.1.)
// A wavefront sees 64 entries at a time: lane l holds entry first + l.
// With FIRST it also holds each entry's first page.
template <typename T, int HD, bool FIRST> struct Line {
    static constexpr int TILE = tile_keys<T>();
    static constexpr uint32_t kBegin = begin_bytes(HD) / (TILE * HD * 2 * (int)sizeof(T));
    const PagedAttention &a;
    const uint32_t units;
    int first, row, keys;
    int32_t page;
    uint32_t span, end;    // places of a unit of this entry; the entry's end within the chunk
    uint32_t before, all;  // places of earlier chunks; of this one
    uint32_t share;        // 0: a line

    static __device__ __forceinline__ uint32_t tiles_of(int keys) {
        return ((uint32_t)keys + TILE - 1) / TILE;  // (keys may be 2^31 - 16)
    }
    __device__ __forceinline__ void add_up() {
        const uint32_t tiles = tiles_of(keys);
        span = share ? (tiles + share - 1) / share : keys ? tiles + kBegin : 0u;
        end = (uint32_t)wave_scan((int)(span * units));
        all = __builtin_amdgcn_readlane(end, kWave - 1);
    }
    __device__ __forceinline__ void load(int at) {
        first = at;
        const int i = at + (int)(threadIdx.x % kWave);
        bool bad;
        row = i < a.n ? a.index[i] : -1;
        keys = entry_keys(a, row, i < a.n ? a.positions[i] : -1, bad);
        if constexpr (FIRST) page = keys ? a.table[(int64_t)row * a.width] : -1;
    }
    // all places of the call; leaves the first chunk in place
    __device__ __forceinline__ uint32_t total() {
        before = 0;
        if (a.n <= kWave) {
            load(0);
            const uint32_t tiles = __builtin_amdgcn_readlane(
                wave_scan((int)(tiles_of(keys) * units)), kWave - 1);
            const uint32_t wgs = 1u << a.log_wgs;
            share = max((tiles + wgs - 1) >> a.log_wgs, kMinTiles);
            for (const uint32_t most = (share + kWaves - 1) / kWaves * kWaves; share <= most;
                 ++share) {
                add_up();
                if (all <= wgs) return all;
            }
        }
        share = 0;
        uint32_t sum = 0;
        for (int at = (a.n - 1) / kWave * kWave; at >= 0; at -= kWave) {
            load(at);
            add_up();
            sum += all;
        }
        return sum;
    }
    __device__ __forceinline__ void next() {
        before += all;
        load(first + kWave);
        add_up();
    }
};

// Workgroups that work, as a power of two: fewer where there are few tiles.
__device__ __forceinline__ int log_workers(int log_wgs, uint32_t line) {
    while (log_wgs > 0 && (line >> log_wgs) < kMinTiles) --log_wgs;
    return log_wgs;
}

__device__ __forceinline__ float swap_max(float v) {  // over lanes l, l^16, l^32, l^48
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// What is left of a weight after its leading bf16 term, cut off and not rounded: never
// negative, and for a weight above 0 never 0, so that a value of infinity stays one
// (2^-126 is below half a step of any sum that shows).  The two terms together are
// within 2^-16 of the weight.
__device__ __forceinline__ float rest(float p) {
    return p > 0.0f ? fmaxf(p - __uint_as_float(__float_as_uint(p) & 0xffff0000u), 0x1p-126f)
                    : p;
}

// The gate of N consecutive outputs of head h of entry i, values dim .., loaded ahead of
// the work that it multiplies.
template <typename T, int N>
__device__ __forceinline__ void load_gate(const PagedAttention &a, int i, int h, int dim,
                                          T (&g)[N]) {
    if (!a.gate) return;
    const T *p = (const T *)a.gate + (int64_t)i * a.gate_tok + (int64_t)h * a.gate_head + dim;
#pragma unroll
    for (int j = 0; j < N; ++j) g[j] = p[j];
}

template <typename T, int HD, int N>
__device__ __forceinline__ void store_out(const PagedAttention &a, int i, int h, int dim,
                                          float (&o)[N], bool gated, const T (&g)[N]) {
    if (gated)
#pragma unroll
        for (int j = 0; j < N; ++j) o[j] *= sigmoid(to_f32(g[j]));
    const int64_t at = (int64_t)i * a.out_tok + (int64_t)h * HD + dim;
    if constexpr (N == 4) {
        if (a.out_dtype == QDC_BF16) store_frag((bf16_t *)a.out + at, o);
        else if (a.out_dtype == QDC_F32) store_frag((float *)a.out + at, o);
        else store_frag((split_t *)a.out + at, o);
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            if (a.out_dtype == QDC_BF16) put_elem((bf16_t *)a.out, at + j, o[j]);
            else if (a.out_dtype == QDC_F32) put_elem((float *)a.out, at + j, o[j]);
            else put_elem((split_t *)a.out, at + j, o[j]);
        }
    }
}

// Of an entry without keys: 0 whatever the gate holds.
template <typename T, int HD, int N>
__device__ __forceinline__ void store_zero(const PagedAttention &a, int i, int h, int dim) {
    float zero[N] = {};
    const T gate[N] = {};
    store_out<T, HD, N>(a, i, h, dim, zero, false, gate);
}

// Pages stream by: read as such they come at up to 6.7 TB/s, with plain loads at 5.6.  Rows
// that share pages, such as continuations of one prompt, find them in a cache again: plain
// loads keep them there.  (us, as a stream / plain: 40 prompts of 2000 tokens 34.6 / 37.8;
// 8 with 5 rows each 33.7 / 32.4, 16 of 4000 with 4 rows 71.9 / 53.0, 4 of 8000 with 16
// rows 107 / 80.)
template <bool SHARED, typename P> __device__ __forceinline__ P load_page(const char *p) {
    const P *q = reinterpret_cast<const P *>(p);
    return SHARED ? *q : __builtin_nontemporal_load(q);
}

// Moves within each row of 16 lanes (by 4, 8) and each quad (its lane I to all four).
template <int N> __device__ __forceinline__ float row_rotate(float v) {
    return __int_as_float(
        __builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x120 + N, 0xf, 0xf, true));
}
template <int I> __device__ __forceinline__ float quad_lane(float v) {
    return __int_as_float(
        __builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x55 * I, 0xf, 0xf, true));
}

// One wavefront's operands and sums over its tiles of one head group.
//   K: lane (lr, lg) holds values DS s + V lg .. of key 16 sub + lr.
//   V: values 16 VD c + VD lr .. of keys 16 sub + 4 lg + r.
//   S^T, P: head lr, keys 16 sub + 4 lg + r.   O^T[c][j]: head lr, values
//   16 VD c + VD (4 lg + r) + j.
// FEW, for fp32 and up to 4 heads: sixteen 4 x 4 products with one key's or value's step
// each in place of one of 16 x 16, of which 4 columns would be in use: a quarter of the
// matrix cores' time, which short rows wait for (us, 16 x 16 / 4 x 4: a row of 500 keys of
// 64 9.1 / 7.7, 8 rows of 256 of 128 11.7 / 10.5, 819 MB of 256 134 / 127).  Quad g = lane / 4 %
// 4 and j = lane % 4:
//   K as above, each lg a part of the sum.  S^T, P: head j, keys 4 g + r, the same for all
//   lg.  V: values 16 VD c + VD (4 lg + j) .. of keys 4 g + r.   O[c][e]: head r, values 16
//   VD c + VD (4 lg + j) + e over the keys of quad g.
template <typename T, int HD> struct Lanes {
    static constexpr bool BF = sizeof(T) == 2;
    static constexpr int V = Elem<T>::kVec, SUBS = BF ? 2 : 1, DS = 4 * V, STEPS = HD / DS;
    static constexpr int VD = BF && HD > 64 ? 8 : 4, VC = HD / (16 * VD);
    static constexpr int VW = VD * (int)sizeof(T) / 4;  // registers of a V piece
    typedef uint32_t piece __attribute__((ext_vector_type(VW)));
    u32x4 k[SUBS][STEPS];
    piece v[SUBS][4][VC];
    f32x4 o[VC][VD];
    float base, sum;

    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int c = 0; c < VC; ++c)
#pragma unroll
            for (int j = 0; j < VD; ++j) o[c][j] = f32x4{0.f, 0.f, 0.f, 0.f};
        base = -FLT_MAX;  // finite: a masked score is -inf
        sum = 0.0f;
    }
};

// What the wavefronts of a workgroup share: the queries, and their sums in the end.
template <typename T, int HD, int WAVES> struct Scratch {
    u32x4 q[Lanes<T, HD>::STEPS][kWave];
    float out[WAVES][4][HD + 4], top[WAVES][kHeads], sum[WAVES][kHeads];
};

// Tiles j0 .. j1 - 1 of a unit (KV head and group of its query heads) of an entry, by
// WAVES wavefronts: its outputs, when `whole`, or a piece in slot `slot`.
template <typename T, int HD, int WAVES, bool FEW, bool SHARED>
__device__ __forceinline__ void attend(const PagedAttention &a, int entry, int row, int keys,
                                       int unit, int j0, int j1, bool whole, int64_t slot,
                                       Scratch<T, HD, WAVES> &scratch) {
    typedef Lanes<T, HD> L;
    constexpr int TILE = tile_keys<T>(), KT = kWave / L::SUBS;
    constexpr int VEC = HD / kWave;  // outputs of a thread per pass of 4 heads
    auto &sq = scratch.q;
    auto &so = scratch.out;
    auto &sm = scratch.top;
    auto &sl = scratch.sum;
    const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), l = threadIdx.x % kWave;
    const int lr = l % 16, lg = l / 16;
    const int mask = (1 << a.shift) - 1;
    const uint32_t off_k = (uint32_t)(lr * HD + L::V * lg) * (uint32_t)sizeof(T);
    const int vk = FEW ? lr / 4 : lg, vp = FEW ? l % 4 + 4 * lg : lr;  // V's keys, its piece
    const uint32_t off_v = (uint32_t)(4 * vk * HD + L::VD * vp) * (uint32_t)sizeof(T);
    L x;
    const int kvh = a.head_groups == 1 ? unit : unit / a.head_groups;
    const int hg = unit - kvh * a.head_groups;
    const int head0 = kvh * a.group + hg * kHeads;
    const int gu = min(kHeads, a.group - hg * kHeads);
    const int32_t *pages = a.table + (int64_t)row * a.width;

    const int dim = VEC * l;
    T gate[VEC] = {};
    if (whole && wv < min(gu, 4)) load_gate(a, entry, head0 + wv, dim, gate);
    // this wavefront's tiles: one of every WAVES
    const int jw = j0 + wv, cnt = j1 > jw ? (j1 - jw + WAVES - 1) / WAVES : 0;
    int32_t ids = -1;  // lane l: the page of tile k0 + l / SUBS, sub l % SUBS
    auto fetch_ids = [&](int k0) {
        const int k = k0 + l / L::SUBS;
        const int key = (jw + WAVES * k) * TILE + 16 * (l % L::SUBS);
        if (k < cnt) ids = pages[min(key, keys - 1) >> a.shift];
    };
    fetch_ids(0);
    int limit[L::SUBS];  // keys of the tile's halves that count
    // bytes to the half's first key: its 16 lie in one page, those past the end too
    int64_t from[L::SUBS];
    auto locate = [&](int k) {  // where tile k lies
        if (k && k % KT == 0) fetch_ids(k);
#pragma unroll
        for (int s = 0; s < L::SUBS; ++s) {
            const int key0 = (jw + WAVES * k) * TILE + 16 * s;
            const int id = __builtin_amdgcn_readlane(ids, k % KT * L::SUBS + s);
            const bool ok = (uint32_t)id < (uint32_t)a.pages;
            from[s] = ((((int64_t)(ok ? id : 0) * a.kv + kvh) << a.shift) + (key0 & mask)) *
                      (HD * (int)sizeof(T));
            const int left = min(max(keys - key0, 0), 16);
            limit[s] = ok ? left : 0;
            if (!ok && left && l == 0) raise_flag(a.error_flag);
        }
    };
    auto load_k = [&] {
#pragma unroll
        for (int s = 0; s < L::SUBS; ++s)
#pragma unroll
            for (int i = 0; i < L::STEPS; ++i)
                x.k[s][i] = load_page<SHARED, u32x4>((const char *)a.k + from[s] + off_k +
                                             L::DS * (int)sizeof(T) * i);
    };
    auto load_v = [&] {
#pragma unroll
        for (int s = 0; s < L::SUBS; ++s)
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int c = 0; c < L::VC; ++c)
                    x.v[s][r][c] = load_page<SHARED, typename L::piece>(
                        (const char *)a.v + from[s] + off_v +
                        (r * HD + 16 * L::VD * c) * (int)sizeof(T));
    };
    if (cnt) {
        locate(0);
        load_k();
        load_v();
    }
    // q as the other operand of the scores, heads past the group's repeat its last
    for (int i = threadIdx.x; i < L::STEPS * kWave; i += WAVES * kWave) {
        const int s = i / kWave, ln = i % kWave;
        sq[s][ln] = load_raw((const T *)a.q + (int64_t)entry * a.q_tok +
                             (int64_t)(head0 + min(ln % (FEW ? 4 : 16), gu - 1)) * a.q_head + L::DS * s +
                             L::V * (ln / 16));
    }
    __syncthreads();
    x.clear();
    // tile k; with another after it the loads of that one follow the last use of the
    // registers they fill (in a branch of their own they would be waited for there)
    auto step = [&](int k, auto more) {
        f32x4 sc[L::SUBS];
        if constexpr (FEW) {
            f32x4 part[4];  // chains beside each other
#pragma unroll
            for (int e = 0; e < 4; ++e) part[e] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < L::STEPS; ++i) {
                const u32x4 qf = sq[i][l];
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    part[e] = __builtin_amdgcn_mfma_f32_4x4x1f32(
                        __uint_as_float(x.k[0][i][e]), __uint_as_float(qf[e]), part[e], 0, 0, 0);
            }
            sc[0] = (part[0] + part[1]) + (part[2] + part[3]);
#pragma unroll
            for (int r = 0; r < 4; ++r) sc[0][r] = swap_sum32(swap_sum16(sc[0][r]));
        } else {
#pragma unroll
            for (int s = 0; s < L::SUBS; ++s) sc[s] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < L::STEPS; ++i) {
                const u32x4 qf = sq[i][l];
#pragma unroll
                for (int s = 0; s < L::SUBS; ++s) {
                    if constexpr (L::BF) {
                        sc[s] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                            __builtin_bit_cast(bf16x8, x.k[s][i]), __builtin_bit_cast(bf16x8, qf),
                            sc[s], 0, 0, 0);
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            sc[s] = __builtin_amdgcn_mfma_f32_16x16x4f32(
                                __uint_as_float(x.k[s][i][e]), __uint_as_float(qf[e]), sc[s], 0,
                                0, 0);
                    }
                }
            }
        }
        int now[L::SUBS];
        bool cut = false;
#pragma unroll
        for (int s = 0; s < L::SUBS; ++s) now[s] = limit[s], cut = cut || limit[s] < 16;
        if constexpr (decltype(more)::value) {
            __builtin_amdgcn_sched_barrier(0);
            locate(k + 1);
            load_k();
            __builtin_amdgcn_sched_barrier(0);
        }
        if (cut) {
#pragma unroll
            for (int s = 0; s < L::SUBS; ++s)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    if (4 * vk + r < now[s]) continue;
                    sc[s][r] = -__builtin_inff();
#pragma unroll
                    for (int c = 0; c < L::VC; ++c)  // 0 times what lies there may be NaN
                        x.v[s][r][c] = typename L::piece(0u);
                }
        }
        float top = sc[0][0];
#pragma unroll
        for (int s = 0; s < L::SUBS; ++s)
#pragma unroll
            for (int r = 0; r < 4; ++r) top = fmaxf(top, sc[s][r]);
        if constexpr (FEW) {
            top = fmaxf(top, row_rotate<8>(top));
            top = fmaxf(top, row_rotate<4>(top));
        } else {
            top = swap_max(top);
        }
        top = fmaxf(top * a.scale_log2, x.base);
        if (__any(top > x.base)) {
            const float f = __builtin_amdgcn_exp2f(x.base - top);
            const f32x4 fs = FEW ? f32x4{quad_lane<0>(f), quad_lane<1>(f), quad_lane<2>(f),
                                         quad_lane<3>(f)}
                                 : f32x4{f, f, f, f};
            x.sum *= f;
#pragma unroll
            for (int c = 0; c < L::VC; ++c)
#pragma unroll
                for (int j = 0; j < L::VD; ++j) x.o[c][j] *= fs;
            x.base = top;
        }
        float p[L::SUBS][4];
#pragma unroll
        for (int s = 0; s < L::SUBS; ++s)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                p[s][r] = __builtin_amdgcn_exp2f(
                    __builtin_fmaf(sc[s][r], a.scale_log2, -x.base));
                x.sum += p[s][r];
            }
        if constexpr (L::BF) {
            u32x4 hi, lo;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float p0 = p[i / 2][2 * (i % 2)], p1 = p[i / 2][2 * (i % 2) + 1];
                hi[i] = __builtin_amdgcn_perm(__float_as_uint(p1), __float_as_uint(p0),
                                              0x07060302u);
                lo[i] = pack_bf16x2(rest(p0), rest(p1));
            }
#pragma unroll
            for (int c = 0; c < L::VC; ++c)
#pragma unroll
                for (int j = 0; j < L::VD; ++j) {
                    u32x4 vf;
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        vf[i] = __builtin_amdgcn_perm(
                            x.v[i / 2][2 * (i % 2) + 1][c][j / 2],
                            x.v[i / 2][2 * (i % 2)][c][j / 2],
                            j % 2 ? 0x07060302u : 0x05040100u);
                    const bf16x8 vb = __builtin_bit_cast(bf16x8, vf);
                    x.o[c][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                        vb, __builtin_bit_cast(bf16x8, hi), x.o[c][j], 0, 0, 0);
                    x.o[c][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                        vb, __builtin_bit_cast(bf16x8, lo), x.o[c][j], 0, 0, 0);
                }
        } else {
#pragma unroll
            for (int c = 0; c < L::VC; ++c)
#pragma unroll
                for (int j = 0; j < L::VD; ++j)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float vf = __uint_as_float(x.v[0][r][c][j]);
                        if constexpr (FEW)
                            x.o[c][j] = __builtin_amdgcn_mfma_f32_4x4x1f32(p[0][r], vf, x.o[c][j],
                                                                           0, 0, 0);
                        else
                            x.o[c][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(vf, p[0][r],
                                                                             x.o[c][j], 0, 0, 0);
                    }
        }
        if constexpr (decltype(more)::value) {
            __builtin_amdgcn_sched_barrier(0);
            load_v();
        }
    };
    for (int k = 0; k + 1 < cnt; ++k) step(k, std::true_type{});
    if (cnt) step(cnt - 1, std::false_type{});
    // the wavefronts' sums together, four heads at a time
    if constexpr (FEW) {
        x.sum += row_rotate<8>(x.sum);
        x.sum += row_rotate<4>(x.sum);
    } else {
        x.sum = swap_sum32(swap_sum16(x.sum));
    }
    if (l < (FEW ? 4 : kHeads)) {
        sm[wv][l] = x.base;
        sl[wv][l] = x.sum;
    }
    for (int h0 = 0; h0 < gu; h0 += 4) {
        const int hh = lr - h0;
        if (h0 && whole && wv < min(gu - h0, 4)) load_gate(a, entry, head0 + h0 + wv, dim, gate);
        if constexpr (FEW) {  // the quads' sums, quad g's lanes for head g
#pragma unroll
            for (int c = 0; c < L::VC; ++c) {
                f32x4 mine;
#pragma unroll
                for (int j = 0; j < L::VD; ++j) {
                    f32x4 o = x.o[c][j];
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        o[r] += row_rotate<8>(o[r]);
                        o[r] += row_rotate<4>(o[r]);
                    }
                    mine[j] = vk < 2 ? (vk ? o[1] : o[0]) : (vk == 2 ? o[2] : o[3]);
                }
                *reinterpret_cast<f32x4 *>(&so[wv][vk][16 * L::VD * c + L::VD * vp]) = mine;
            }
        } else if (hh >= 0 && hh < 4) {
#pragma unroll
            for (int c = 0; c < L::VC; ++c)
#pragma unroll
                for (int j = 0; j < L::VD; ++j)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        so[wv][hh][16 * L::VD * c + L::VD * (4 * lg + r) + j] = x.o[c][j][r];
        }
        __syncthreads();
        const int h = h0 + wv;
        if (h < gu && wv < 4) {
            float top = sm[0][h], acc[VEC] = {}, total = 0.0f;
#pragma unroll
            for (int w = 1; w < WAVES; ++w) top = fmaxf(top, sm[w][h]);
#pragma unroll
            for (int w = 0; w < WAVES; ++w) {
                const float f = __builtin_amdgcn_exp2f(sm[w][h] - top);
                total = __builtin_fmaf(f, sl[w][h], total);
#pragma unroll
                for (int e = 0; e < VEC; ++e)
                    acc[e] = __builtin_fmaf(f, so[w][h - h0][dim + e], acc[e]);
            }
            if (whole) {
                const float inv = total == 0.0f ? 0.0f : 1.0f / total;  // 0: no key seen
#pragma unroll
                for (int e = 0; e < VEC; ++e) acc[e] *= inv;
                store_out<T, HD, VEC>(a, entry, head0 + h, dim, acc, a.gate, gate);
            } else {
                float *dst = a.pieces + (slot * a.unit_heads + h) * HD + dim;
#pragma unroll
                for (int e = 0; e < VEC; ++e) dst[e] = acc[e];
                if (l == 0) {
                    float *st = a.stats + (slot * a.unit_heads + h) * 2;
                    st[0] = top;
                    st[1] = total;
                }
            }
        }
        __syncthreads();
    }
}

template <typename T, int HD, bool FEW>
__global__ __launch_bounds__(kBlock, HD > 128 ? 1 : 2) void paged_attention(PagedAttention a) {
    __shared__ __align__(16) Scratch<T, HD, kWaves> scratch;
    Line<T, HD, true> line{a, (uint32_t)(a.kv * a.head_groups)};
    const uint32_t all = line.total();
    uint32_t t = blockIdx.x, t_end = t + (t < all);  // with shares a place is a workgroup's
    if (!line.share) {
        const int lw = log_workers(a.log_wgs, all);
        if (blockIdx.x >> lw) return;
        t = (uint32_t)(((uint64_t)all * blockIdx.x) >> lw);
        t_end = (uint32_t)(((uint64_t)all * (blockIdx.x + 1)) >> lw);
    }
    while (t < t_end) {
        while (line.before + line.all <= t && line.first + kWave < a.n) line.next();
        // the entry and unit that hold place t, and the tiles of it up to t_end
        const uint64_t past = __ballot(line.before + line.end > t);
        if (!past) return;  // the positions changed since they were added up
        const int el = __builtin_ctzll(past);
        const int keys = __builtin_amdgcn_readlane(line.keys, el);
        const int row = __builtin_amdgcn_readlane(line.row, el);
        const uint32_t tiles = line.tiles_of(keys);
        const uint32_t span = __builtin_amdgcn_readlane(line.span, el);
        const uint32_t rel = t - (line.before + __builtin_amdgcn_readlane(line.end, el) -
                                  span * line.units);
        const uint32_t unit = rel / span, p0 = rel - unit * span, p1 = min(span, p0 + (t_end - t));
        uint32_t j0, j1;
        t += p1 - p0;
        if (line.share) {  // part p0 of span
            const uint32_t each = tiles / span, more = tiles - each * span;
            j0 = p0 * each + min(p0, more);
            j1 = j0 + each + (p0 < more);
        } else {
            if (p1 <= line.kBegin) continue;
            j0 = p0 > line.kBegin ? p0 - line.kBegin : 0;
            j1 = p1 - line.kBegin;
        }
        // another entry of the 64 begins with the same page
        const int32_t page = __builtin_amdgcn_readlane(line.page, el);
        const uint64_t same = __ballot(line.page == page);
        const int entry = line.first + el;
        const bool whole = j0 == 0 && j1 == tiles;
        const int64_t slot = 2 * (int64_t)blockIdx.x + (j0 == 0);
        if (same & (same - 1))
            attend<T, HD, kWaves, FEW, true>(a, entry, row, keys, (int)unit, (int)j0, (int)j1,
                                             whole, slot, scratch);
        else
            attend<T, HD, kWaves, FEW, false>(a, entry, row, keys, (int)unit, (int)j0, (int)j1,
                                              whole, slot, scratch);
    }
}

// The same where every row is short: a workgroup for a unit, whole, and no join.
template <typename T, int HD, bool FEW>
__global__ __launch_bounds__(short_waves(HD) * kWave) void paged_attention_short(PagedAttention a) {
    constexpr int TILE = tile_keys<T>(), WAVES = short_waves(HD), VEC = HD / kWave;
    __shared__ __align__(16) Scratch<T, HD, WAVES> scratch;
    const int units = a.kv * a.head_groups;
    const int entry = blockIdx.x / units, unit = blockIdx.x - entry * units;
    const int row = a.index[entry];
    bool bad;
    const int keys = entry_keys(a, row, a.positions[entry], bad);
    if (bad && unit == 0 && threadIdx.x == 0) raise_flag(a.error_flag);
    if (keys) {
        attend<T, HD, WAVES, FEW, false>(a, entry, row, keys, unit, 0, (keys + TILE - 1) / TILE,
                                         true, 0, scratch);
        return;
    }
    const int kvh = unit / a.head_groups, hg = unit - kvh * a.head_groups;
    for (int h = threadIdx.x / kWave; h < min(kHeads, a.group - hg * kHeads); h += WAVES)
        store_zero<T, HD, VEC>(a, entry, kvh * a.group + hg * kHeads + h,
                               VEC * (threadIdx.x % kWave));
}

// A workgroup per entry and head, or join_heads of its heads: the pieces of their keys, in
// order; zeros for an entry without keys; nothing where one workgroup had them all.  (us, 256 / 512 threads: 128
// pieces a head 6.7 / 5.5, 32 5.0 / 4.9, few pieces of 200 x 8 heads 6.2 / 9.2.)
constexpr int64_t kManyPieces = 64;
// Entries times heads from which on a workgroup takes all heads of its entry, so that the
// line is added up once for them.  (us of the whole call, a head each / all: 128 x 8 23.6 /
// 30.1, 512 x 8 67.1 / 62.5, 1024 x 8 147 / 123.)
constexpr int64_t kJoinWgs = 2048;
template <typename T, int HD, int THREADS>
__global__ __launch_bounds__(THREADS) void paged_attention_join(PagedAttention a) {
    constexpr int LPP = HD / 4, PARTS = THREADS / LPP;  // lanes of a piece's row, rows at a time
    __shared__ float top_of[PARTS], sum_of[PARTS];
    __shared__ __align__(16) float so[PARTS][HD];
    const int l = threadIdx.x % kWave, wv = threadIdx.x / kWave;
    const int per_entry = a.heads / a.join_heads, entry = blockIdx.x / per_entry;
    const int h0 = (blockIdx.x - entry * per_entry) * a.join_heads, h1 = h0 + a.join_heads;
    const int dim = HD / kWave * l;
    T gate[HD / kWave] = {};
    if (wv == 0) load_gate(a, entry, h0, dim, gate);
    Line<T, HD, false> line{a, (uint32_t)(a.kv * a.head_groups)};
    const uint32_t all = line.total();
    while (line.first + kWave <= entry) line.next();
    const int keys = __builtin_amdgcn_readlane(line.keys, entry - line.first);
    const uint32_t tiles = line.tiles_of(keys);
    if (h0 == 0 && threadIdx.x == 0) {
        bool bad;
        entry_keys(a, a.index[entry], a.positions[entry], bad);
        if (bad) raise_flag(a.error_flag);
    }
    if (tiles == 0) {
        if (wv == 0)
            for (int h = h0; h < h1; ++h) store_zero<T, HD, HD / kWave>(a, entry, h, dim);
        return;
    }
    const uint32_t span = __builtin_amdgcn_readlane(line.span, entry - line.first);
    const uint32_t start = line.before + __builtin_amdgcn_readlane(line.end, entry - line.first) -
                           span * line.units;
    for (int h = h0; h < h1; ++h) {
        const int kvh = h / a.group, in_group = h - kvh * a.group;
        const int hg = in_group / kHeads, hu = in_group - hg * kHeads;
        const uint32_t at = start + (uint32_t)(kvh * a.head_groups + hg) * span;
        uint32_t w0, w1;  // the workgroups that hold its first and its last tile
        if (line.share) {
            w0 = at;
            w1 = at + span - 1;
        } else {  // that of place t is the last with all * w / 2^lw <= t
            const int lw = log_workers(a.log_wgs, all);
            const uint32_t first = at + line.kBegin;
            w0 = (uint32_t)((((uint64_t)(first + 1) << lw) - 1) / all);
            w1 = (uint32_t)((((uint64_t)(first + tiles) << lw) - 1) / all);
        }
        if (w0 == w1) continue;
        if (h != h0) {
            __syncthreads();  // the scratch is free
            if (wv == 0) load_gate(a, entry, h, dim, gate);
        }
        const int parts = (int)(w1 - w0) + 1;
        auto slot = [&](int p) {
            return ((2 * (int64_t)(w0 + p) + (p == 0)) * a.unit_heads + hu);
        };
        // Each group of LPP lanes runs over every PARTS-th piece, its maximum and sum beside
        // the rows, so that nothing waits for a first pass over the maxima.
        const int part = threadIdx.x / LPP, d4 = 4 * (threadIdx.x % LPP);
        float top = -FLT_MAX, sum = 0.0f;
        f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
        for (int p = part; p < parts; p += PARTS) {
            const f32x4 o = *reinterpret_cast<const f32x4 *>(a.pieces + slot(p) * HD + d4);
            const f32x2 s = *reinterpret_cast<const f32x2 *>(a.stats + 2 * slot(p));
            const float m = fmaxf(top, s[0]);
            const float f = __builtin_amdgcn_exp2f(top - m), g = __builtin_amdgcn_exp2f(s[0] - m);
            top = m;
            sum = __builtin_fmaf(g, s[1], f * sum);
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[e] = __builtin_fmaf(g, o[e], f * acc[e]);
        }
        *reinterpret_cast<f32x4 *>(&so[part][d4]) = acc;
        if (d4 == 0) {
            top_of[part] = top;
            sum_of[part] = sum;
        }
        __syncthreads();
        if (wv) continue;
#pragma unroll
        for (int p = 0; p < PARTS; ++p) top = fmaxf(top, top_of[p]);
        float total = 0.0f, o[HD / kWave] = {};
#pragma unroll
        for (int p = 0; p < PARTS; ++p) {
            const float f = __builtin_amdgcn_exp2f(top_of[p] - top);
            total = __builtin_fmaf(f, sum_of[p], total);
#pragma unroll
            for (int e = 0; e < HD / kWave; ++e) o[e] = __builtin_fmaf(f, so[p][dim + e], o[e]);
        }
        const float inv = total == 0.0f ? 0.0f : 1.0f / total;  // 0: no key seen
#pragma unroll
        for (int e = 0; e < HD / kWave; ++e) o[e] *= inv;
        store_out<T, HD, HD / kWave>(a, entry, h, dim, o, a.gate, gate);
    }
}

// The longest line that a call of these sizes can have, 0 when it is too long or the
// sizes are not taken.
int64_t longest_line(int64_t n, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t width,
                     int64_t page_size, int32_t dtype) {
    if (!valid_dtype(dtype) || n <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads ||
        (head_dim != 64 && head_dim != 128 && head_dim != 256) || width <= 0 ||
        page_shift(page_size) < 0)
        return 0;
    const int64_t lim = (int64_t)1 << 31;
    // the join has a workgroup per head of an entry
    if (heads >= ((int64_t)1 << 20) || n >= ((int64_t)1 << 24) / heads || width >= lim / page_size)
        return 0;
    const int64_t units = kv_heads * ceil_div(heads / kv_heads, (int64_t)kHeads);
    const int64_t tile = dtype == QDC_BF16 ? tile_keys<bf16_t>() : tile_keys<float>();
    const int64_t span = ceil_div(width * page_size, tile) +
                         begin_bytes((int)head_dim) / (tile * head_dim * 2 * elem_size(dtype));
    return span >= lim / units / n ? 0 : span * units * n;
}

// Whether rows of `width` pages are short: at most kShortTiles tiles a wavefront.  The host
// knows the table's width and not the rows: short rows of a wider table are dealt out and
// joined (us a call, a row of 411 keys of 2 fp32 heads of 64: 7.1 in a table of 416 places,
// 8.5 in one of 32768; 8 rows of 2048 of 256, dealt out in both, 12.9 and 13.1).  (The grid
// of a workgroup for each unit stays below 2^32 work-items.)
bool short_rows(int64_t n, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t width,
                int64_t page_size, int32_t dtype) {
    const int64_t tile = dtype == QDC_BF16 ? tile_keys<bf16_t>() : tile_keys<float>();
    const int64_t units = kv_heads * ceil_div(heads / kv_heads, (int64_t)kHeads);
    return width * page_size <= tile * kShortTiles * short_waves((int)head_dim) &&
           n * units < ((int64_t)1 << 22);
}

// Workgroups for a line: one a compute unit for heads of 256, whose operands take half
// the registers of a SIMD for a wavefront, two for smaller ones (us, 256 / 512: bf16 2 x
// 100003 keys of 256 123 / 128, 8 x 2048 12 / 13; of 64, 410 MB 73 / 66; fp32 of 256, 819
// MB 128 / 135, of 64 136 / 124).
int log_workgroups(int64_t line, int64_t head_dim) {
    const int most = head_dim > 128 ? 8 : kMaxLogWgs;
    int lw = 0;
    while (lw < most && ((int64_t)kMinTiles << lw) < line) ++lw;
    return lw;
}

int64_t unit_heads(int64_t heads, int64_t kv_heads) {
    const int64_t g = heads / kv_heads;
    return g < kHeads ? g : kHeads;
}

// Entries of a slice.  Every workgroup adds up its call's line, so a call's time would grow
// with the square of its entries: from twice this many on it is launched slice by slice,
// evenly, of so many entries and more.  (ms, whole / in slices of 1024 / 2048 / 4096, bf16 rows
// of up to 40 keys: 4096 x 4 heads of 64 .172 / .147 / .147 / .170, 131072 65.5 / 5.07 / 4.98 /
// 5.61, 131072 x 8 heads of 256 68.4 / 9.00 / 8.55 / 9.32; up to 600 keys, 3000 x 8 heads of
// 256 .353 / .388 / .373 / .356.)
constexpr int64_t kSlice = 2048;

int32_t launch(PagedAttention a, int64_t head_dim, int32_t dtype, bool brief, bool few,
               void *workspace, hipStream_t stream) {
    const int64_t n = a.n, units = (int64_t)a.kv * a.head_groups;
    const dim3 grid(brief ? (uint32_t)(n * units) : 1u << a.log_wgs);
    a.join_heads = n * a.heads >= kJoinWgs ? a.heads : 1;
    const dim3 join((uint32_t)(n * a.heads / a.join_heads)), block(kBlock);
    const bool many = kManyPieces * n * units <= grid.x;
    a.pieces = reinterpret_cast<float *>(workspace);
    a.stats = a.pieces + (int64_t)2 * grid.x * a.unit_heads * head_dim;
#define QDC_PAGED(T, HD, FEW)                                                                  \
    if (head_dim == HD && few == FEW) {                                                        \
        if (brief) {                                                                           \
            hipLaunchKernelGGL((paged_attention_short<T, HD, FEW>), grid,                      \
                               dim3(short_waves(HD) * kWave), 0, stream, a);                   \
            return launch_status();                                                            \
        }                                                                                      \
        hipLaunchKernelGGL((paged_attention<T, HD, FEW>), grid, block, 0, stream, a);          \
        const int32_t status = launch_status();                                                \
        if (status != QDC_OK) return status;                                                   \
        if (many)                                                                              \
            hipLaunchKernelGGL((paged_attention_join<T, HD, 2 * kBlock>), join,                \
                               dim3(2 * kBlock), 0, stream, a);                                \
        else                                                                                   \
            hipLaunchKernelGGL((paged_attention_join<T, HD, kBlock>), join, block, 0, stream,  \
                               a);                                                             \
        return launch_status();                                                                \
    }
    if (dtype == QDC_BF16) {
        QDC_PAGED(bf16_t, 64, false)
        QDC_PAGED(bf16_t, 128, false)
        QDC_PAGED(bf16_t, 256, false)
    }
    QDC_PAGED(float, 64, true)
    QDC_PAGED(float, 64, false)
    QDC_PAGED(float, 128, true)
    QDC_PAGED(float, 128, false)
    QDC_PAGED(float, 256, true)
    QDC_PAGED(float, 256, false)
#undef QDC_PAGED
    return QDC_ERR_SHAPE;
}

}  // namespace
}  // namespace qdc

using namespace qdc;

extern "C" int64_t qdc_paged_attention_workspace(int64_t n, int64_t heads, int64_t kv_heads,
                                                 int64_t head_dim, int64_t width,
                                                 int64_t page_size, int32_t dtype) {
    const int64_t line = longest_line(n, heads, kv_heads, head_dim, width, page_size, dtype);
    if (line == 0) return -1;
    if (short_rows(n, heads, kv_heads, head_dim, width, page_size, dtype)) return 0;
    // two pieces a workgroup, each with its maximum and sum
    return ((int64_t)2 << log_workgroups(line, head_dim)) * unit_heads(heads, kv_heads) * (head_dim + 2) * 4;
}

extern "C" int32_t qdc_paged_attention(
    void *out, int32_t out_dtype, const void *q, const void *k_pages, const void *v_pages,
    const void *gate, const int32_t *table, const int32_t *index, const int32_t *positions,
    int64_t n, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t rows, int64_t width,
    int64_t pages, int64_t page_size, int64_t q_tok, int64_t q_head, int64_t gate_tok,
    int64_t gate_head, int64_t out_tok, float scale, int32_t dtype, void *workspace,
    int64_t workspace_bytes, int32_t *error_flag, hipStream_t stream) {
    if (!valid_dtype(dtype) || (!valid_dtype(out_dtype) && out_dtype != QDC_BF16X2))
        return QDC_ERR_DTYPE;
    if (n < 0 || rows <= 0 || pages <= 0) return QDC_ERR_SHAPE;
    const int64_t line =
        longest_line(n ? n : 1, heads, kv_heads, head_dim, width, page_size, dtype);
    const int64_t lim = (int64_t)1 << 31;
    if (line == 0 || rows >= lim || pages >= lim) return QDC_ERR_SHAPE;
    const int64_t es = elem_size(dtype), per = 16 / es, oes = elem_size(out_dtype);
    if (q_head < head_dim || q_tok < 0 || (q_tok | q_head) % per || out_tok < heads * head_dim ||
        out_tok % (16 / oes))
        return QDC_ERR_SHAPE;
    if (gate && (gate_head < head_dim || gate_tok < 0 || (gate_tok | gate_head) % per))
        return QDC_ERR_SHAPE;
    if (!(scale > 0.0f) || !(scale * 1.4426950408889634f < __builtin_inff())) return QDC_ERR_RANGE;
    if (n == 0) return QDC_OK;
    const int64_t need = qdc_paged_attention_workspace(n, heads, kv_heads, head_dim, width,
                                                       page_size, dtype);
    if (!out || !q || !k_pages || !v_pages || !table || !index || !positions ||
        (need && !workspace))
        return QDC_ERR_NULL;
    if (!aligned16(out) || !aligned16(q) || !aligned16(k_pages) || !aligned16(v_pages) ||
        !aligned16(gate) || !aligned16(workspace))
        return QDC_ERR_SHAPE;
    if (workspace_bytes < need) return QDC_ERR_SHAPE;
    const int64_t store = pages * kv_heads * page_size * head_dim * es;
    const Range outs[3] = {{out, ((n - 1) * out_tok + heads * head_dim) * oes},
                           {workspace, need},
                           {error_flag, error_flag ? 4 : 0}};
    const Range ins[7] = {
        {q, grid_span(n, heads, q_tok, q_head, head_dim, es)},
        {gate, gate ? grid_span(n, heads, gate_tok, gate_head, head_dim, es) : 0},
        {k_pages, store}, {v_pages, store}, {table, rows * width * 4},
        {index, n * 4}, {positions, n * 4}};
    if (any_alias(outs, 3, ins, 7)) return QDC_ERR_ALIAS;
    PagedAttention a{};
    a.k = k_pages;
    a.v = v_pages;
    a.table = table;
    a.error_flag = error_flag;
    a.q_tok = q_tok;
    a.q_head = q_head;
    a.gate_tok = gate_tok;
    a.gate_head = gate_head;
    a.out_tok = out_tok;
    a.width = width;
    a.heads = (int)heads;
    a.kv = (int)kv_heads;
    a.group = (int)(heads / kv_heads);
    a.unit_heads = (int)unit_heads(heads, kv_heads);
    a.head_groups = (int)ceil_div(heads / kv_heads, (int64_t)kHeads);
    a.rows = (int)rows;
    a.pages = (int)pages;
    a.shift = page_shift(page_size);
    a.out_dtype = out_dtype;
    a.scale_log2 = scale * 1.4426950408889634f;
    const bool brief = need == 0, few = dtype == QDC_F32 && a.group <= 4;
    const int64_t slices = brief || n < 2 * kSlice ? 1 : n / kSlice;
    for (int64_t i = 0; i < slices; ++i) {
        const int64_t i0 = n * i / slices, m = n * (i + 1) / slices - i0;
        a.out = (char *)out + i0 * out_tok * oes;
        a.q = (const char *)q + i0 * q_tok * es;
        a.gate = gate ? (const char *)gate + i0 * gate_tok * es : nullptr;
        a.index = index + i0;
        a.positions = positions + i0;
        a.n = (int)m;
        a.log_wgs = log_workgroups(
            longest_line(m, heads, kv_heads, head_dim, width, page_size, dtype), head_dim);
        const int32_t status = launch(a, head_dim, dtype, brief, few, workspace, stream);
        if (status != QDC_OK) return status;
    }
    return QDC_OK;
}
