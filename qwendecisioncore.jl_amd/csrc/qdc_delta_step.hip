// qdc_delta_step.hip -- one token of a linear attention layer for many cache rows:
//     x = silu(causal conv of the qkv block),  q, k L2-normalised (q also / sqrt(kd)),
//     f = exp(decay),  u = beta (v - f S k),  S <- f S + u k^T,  o = S q,
//     out = o / rms(o) * w * silu(z)
// for the state S [value_dim, key_dim] of each row and value head, as the recurrence
// of qdc_delta_scan.hip between the prologue and the gated norm
// (cpu_delta_recurrent_step!, src/backbone_cpu.jl:681-705).
//
// A workgroup owns one row's state of one head: it is read once into registers, kept
// there through both products and written once, which is nearly all of the traffic
// (2 x 64 KB a head of 128 x 128).  Its loads leave first, and the convolution, norms
// and gates of the token, done again by each head that shares a key head, run while
// they are on the way.  The convolution's window is a ring of `taps` slots by position:
// the new token goes to the slot that is read no more, so no head reads what another
// writes.
//
// Bound by memory: 151 rows of 32 heads of 128 x 128 (317 MB read and written) 109 us = 5.9
// TB/s, of 6.5 for a copy; 64 rows of 16 heads of 128 x 128 (134 MB in all, which the
// last-level cache holds) 23.8 us; one row 5.1 us, two chains of loads and three barriers.
#include <cmath>

#include "qdc_cache.hpp"

namespace qdc {
namespace {

constexpr int kMaxTaps = 8, kMaxValue = 256;

struct DeltaStep {
    void *out;
    const void *proj, *norm;
    void *ring;
    float *state;
    const float *conv, *a_decay, *dt_bias;
    const int32_t *index, *positions;
    int32_t *error_flag;
    int64_t ld, channels;
    int rows, taps, key_heads, heads, groups, value_dim;
    float eps, sqrt_kd;
    int out_dtype;
};

__device__ __forceinline__ float softplus_f(float x) {
    return fmaxf(x, 0.0f) + log1pf(expf(-fabsf(x)));
}

// A state that is larger than what the last-level cache keeps until the next call is
// read and written as a stream.
template <bool STREAM> __device__ __forceinline__ f32x4 load_state(const float *p) {
    const f32x4 *q = reinterpret_cast<const f32x4 *>(p);
    return STREAM ? __builtin_nontemporal_load(q) : *q;
}
template <bool STREAM> __device__ __forceinline__ void store_state(float *p, f32x4 v) {
    f32x4 *q = reinterpret_cast<f32x4 *>(p);
    if (STREAM) __builtin_nontemporal_store(v, q);
    else *q = v;
}

// Threads: twice as many stream a large state 5% faster (us, 317 MB 115 / 109, 134 MB
// 51 / 49), a small one is done sooner without (8 MB 6.5 / 6.9, 67 MB 23.7 / 24.8).
constexpr int step_threads(bool stream) { return stream ? 1024 : 512; }
constexpr int row_lanes(int key_dim) { return key_dim / 4 < 16 ? key_dim / 4 : 16; }

// L lanes a state row, N 16-byte pieces a lane; a pass of the workgroup takes
// kStep / L rows, PASSES passes all of them.  TAPS: the convolution's taps, 0 for any.
template <typename T, int KD, int PASSES, int TAPS, bool STREAM>
__global__ __launch_bounds__(step_threads(STREAM)) void delta_step(DeltaStep a) {
    constexpr int kStep = step_threads(STREAM), L = row_lanes(KD), N = KD / (4 * L);
    constexpr int ROWS = kStep / L;
    static_assert(2 * KD + kMaxValue <= kStep, "a thread a channel");
    __shared__ __align__(16) float qkv[2 * KD + kMaxValue], so[kMaxValue];
    __shared__ float part[kStep / kWave], gates[2];
    const int entry = blockIdx.x, h = blockIdx.y, tid = threadIdx.x, vd = a.value_dim;
    const int row = a.index[entry], pos = a.positions[entry];
    const bool token = row >= 0 && pos >= 0;
    // an address within the cache, whatever the entry holds; what comes from there is
    // used only once the entry has been checked
    const int64_t safe = min(max(row, 0), a.rows - 1);
    const uint32_t p0 = (uint32_t)max(pos, 0);

    // everything a thread reads, the small things first: the token's channels of this
    // head (q | k | v), their window, the gates, and then the state
    const int g = h / a.groups, taps = TAPS ? TAPS : a.taps;
    const int64_t kw = (int64_t)a.key_heads * KD, vw = (int64_t)a.heads * vd, cq = a.channels;
    const T *proj = (const T *)a.proj + entry * a.ld;
    T *ring = (T *)a.ring + safe * taps * cq;
    const bool channel = tid < 2 * KD + vd;
    const int64_t c = tid < KD       ? (int64_t)g * KD + tid
                      : tid < 2 * KD ? kw + (int64_t)g * KD + (tid - KD)
                                     : 2 * kw + (int64_t)h * vd + (tid - 2 * KD);
    constexpr int W = TAPS ? TAPS : kMaxTaps;
    T window[W], z = T(), norm = T();
    float conv[W];
    if (channel) {
        window[0] = proj[c];
#pragma unroll
        for (int lag = 0; lag < W; ++lag) {  // tap taps - 1 - lag
            if (!TAPS && lag >= taps) continue;
            // (without a sign: the sum may pass 2^31)
            if (lag) window[lag] = ring[(p0 + (uint32_t)(taps - lag)) % (uint32_t)taps * cq + c];
            conv[lag] = a.conv[c * taps + (taps - 1 - lag)];
        }
    }
    if (tid < vd) {
        z = proj[cq + (int64_t)h * vd + tid];
        norm = ((const T *)a.norm)[tid];
    }
    const float b_raw = to_f32(proj[cq + vw + a.heads + h]), a_raw = to_f32(proj[cq + vw + h]);
    const float bias = a.dt_bias[h], decay = a.a_decay[h];
    const int lane = tid % L, r0 = tid / L;
    float *state = a.state + (safe * a.heads + h) * vd * KD;
    f32x4 S[PASSES][N];
#pragma unroll
    for (int p = 0; p < PASSES; ++p) {
        const int v = min(r0 + p * ROWS, vd - 1);
#pragma unroll
        for (int n = 0; n < N; ++n)
            S[p][n] = load_state<STREAM>(state + (int64_t)v * KD + 4 * (lane + L * n));
    }

    // a row that an earlier token of the call has: not done twice
    bool bad = token && row >= a.rows;
    if (token)
        for (int j = tid; j < entry; j += kStep)
            bad = bad || (a.index[j] == row && a.positions[j] >= 0);
    const int64_t at = ((int64_t)entry * a.heads + h) * vd;
    auto put = [&](int v, float o) {
        if (a.out_dtype == QDC_BF16) put_elem((bf16_t *)a.out, at + v, o);
        else if (a.out_dtype == QDC_F32) put_elem((float *)a.out, at + v, o);
        else put_elem((split_t *)a.out, at + v, o);
    };
    if (channel) {
        float acc = 0.0f;
#pragma unroll
        for (int lag = W - 1; lag >= 0; --lag)  // the oldest first; before position 0 nothing
            if ((TAPS || lag < taps) && lag <= pos) acc = acc + to_f32(window[lag]) * conv[lag];
        qkv[tid] = silu(acc);
    }
    if (tid == kStep - 1) {
        gates[0] = sigmoid(b_raw);
        gates[1] = expf(decay * softplus_f(a_raw + bias));
    }
    const bool live = !__syncthreads_or(bad) && token;  // uniform
    if (!live) {
        if (tid < vd) put(tid, 0.0f);
        if (token && tid == 0) raise_flag(a.error_flag);
        return;
    }
    if (channel && (tid >= 2 * KD || h % a.groups == 0))  // one head keeps the key head's part
        ring[(int64_t)(pos % taps) * cq + c] = window[0];
    // the squares of q and k, each lane group alike
    float k[N][4], q[N][4], qq = 0.0f, kk = 0.0f;
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            q[n][e] = qkv[4 * (lane + L * n) + e];
            k[n][e] = qkv[KD + 4 * (lane + L * n) + e];
            qq += q[n][e] * q[n][e];
            kk += k[n][e] * k[n][e];
        }
    const float qs = 1.0f / (__builtin_sqrtf(group_sum<L>(qq) + 1e-6f) * a.sqrt_kd);
    const float ks = 1.0f / __builtin_sqrtf(group_sum<L>(kk) + 1e-6f);
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            q[n][e] *= qs;
            k[n][e] *= ks;
        }
    const float beta = gates[0], f = gates[1];
#pragma unroll
    for (int p = 0; p < PASSES; ++p) {
        const int v = r0 + p * ROWS;
        if (v >= vd) continue;  // uniform per lane group
        float sk = 0.0f, sq = 0.0f;
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                S[p][n][e] = pos ? S[p][n][e] * f : 0.0f;  // position 0: from an empty state
                sk = __builtin_fmaf(S[p][n][e], k[n][e], sk);
            }
        const float u = beta * (qkv[2 * KD + v] - group_sum<L>(sk));
#pragma unroll
        for (int n = 0; n < N; ++n) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                S[p][n][e] = __builtin_fmaf(u, k[n][e], S[p][n][e]);
                sq = __builtin_fmaf(S[p][n][e], q[n][e], sq);
            }
            store_state<STREAM>(state + (int64_t)v * KD + 4 * (lane + L * n), S[p][n]);
        }
        sq = group_sum<L>(sq);
        if (lane == 0) so[v] = sq;
    }
    __syncthreads();
    const float o = tid < vd ? so[tid] : 0.0f;
    const float wave = group_sum<kWave>(o * o);
    if (tid % kWave == 0) part[tid / kWave] = wave;
    __syncthreads();
    if (tid >= vd) return;
    float ss = 0.0f;
#pragma unroll
    for (int w = 0; w < kMaxValue / kWave; ++w) ss += part[w];
    const float s = rms_scale(ss, (float)vd, a.eps);
    put(tid, ((o * s) * to_f32(norm)) * silu(to_f32(z)));
}

template <typename T, int KD> int32_t launch(const DeltaStep &a, int64_t n, hipStream_t stream) {
    const dim3 grid((uint32_t)n, (uint32_t)a.heads);
    // Bytes of state from which on it is a stream: half of the last-level cache of 256 MB,
    // which is right for calls repeated on one state (us, replayed, cached / streamed: 67 MB
    // 23.7 / 28.2, 134 MB 55.9 / 51.1, 317 MB 130.7 / 114.8).  What passes between two calls
    // is not known here: with 1 GB of other layers' states in between 67 MB would be ahead as
    // a stream too (33.0 / 28.9).
    const bool stream_state =
        a.taps == 4 && n * a.heads * a.value_dim * KD * 4 >= ((int64_t)128 << 20);
    const dim3 block(step_threads(stream_state));
    const int64_t passes = ceil_div((int64_t)a.value_dim, (int64_t)(block.x / row_lanes(KD)));
#define QDC_STEP_LAUNCH(P, TAPS, STREAM)                                                 \
    hipLaunchKernelGGL((delta_step<T, KD, P, TAPS, STREAM>), grid, block, 0, stream, a);
#define QDC_STEP(P)                                                                      \
    if (passes <= P) {                                                                   \
        if (stream_state) {                                                              \
            QDC_STEP_LAUNCH(P, 4, true)                                                  \
        } else if (a.taps == 4) {                                                        \
            QDC_STEP_LAUNCH(P, 4, false)                                                 \
        } else {                                                                         \
            QDC_STEP_LAUNCH(P, 0, false)                                                 \
        }                                                                                \
        return launch_status();                                                          \
    }
    QDC_STEP(1)
    QDC_STEP(2)
    QDC_STEP(4)
    QDC_STEP(8)
#undef QDC_STEP
#undef QDC_STEP_LAUNCH
    return QDC_ERR_SHAPE;
}

}  // namespace
}  // namespace qdc

using namespace qdc;

extern "C" int32_t qdc_delta_step(void *out, int32_t out_dtype, const void *proj,
                                  int32_t proj_dtype, int64_t ld, const float *conv, int64_t taps,
                                  const float *a_decay, const float *dt_bias, const void *norm,
                                  void *ring, float *state, const int32_t *index,
                                  const int32_t *positions, int64_t n, int64_t rows,
                                  int64_t key_heads, int64_t key_dim, int64_t value_heads,
                                  int64_t value_dim, float eps, int32_t *error_flag,
                                  hipStream_t stream) {
    if (!valid_dtype(proj_dtype) ||
        (out_dtype != proj_dtype && !(out_dtype == QDC_BF16X2 && proj_dtype == QDC_BF16)))
        return QDC_ERR_DTYPE;
    const int64_t lim = (int64_t)1 << 31;
    if (n < 0 || rows <= 0 || rows >= lim || key_heads <= 0 || value_heads <= 0 ||
        key_heads >= 65536 || value_heads >= 65536 || value_heads % key_heads ||
        (key_dim != 32 && key_dim != 64 && key_dim != 128) || value_dim <= 0 || value_dim % 16 ||
        value_dim > kMaxValue || taps <= 0 || taps > kMaxTaps)
        return QDC_ERR_SHAPE;
    const int64_t vw = value_heads * value_dim, channels = 2 * key_heads * key_dim + vw;
    const int64_t es = elem_size(proj_dtype);
    // a workgroup of up to 1024 per entry and head in a grid of fewer than 2^32 work-items
    if (ld < channels + vw + 2 * value_heads || n >= lim || ld >= lim ||
        n * value_heads >= ((int64_t)1 << 22))
        return QDC_ERR_SHAPE;
    if (n == 0) return QDC_OK;
    if (!out || !proj || !conv || !a_decay || !dt_bias || !norm || !ring || !state || !index ||
        !positions)
        return QDC_ERR_NULL;
    if (!aligned16(state)) return QDC_ERR_SHAPE;
    const Range outs[4] = {{out, n * vw * elem_size(out_dtype)},
                           {ring, rows * taps * channels * es},
                           {state, rows * vw * key_dim * 4},
                           {error_flag, error_flag ? 4 : 0}};
    const Range ins[7] = {{proj, ((n - 1) * ld + channels + vw + 2 * value_heads) * es},
                          {conv, channels * taps * 4}, {a_decay, value_heads * 4},
                          {dt_bias, value_heads * 4}, {norm, value_dim * es}, {index, n * 4},
                          {positions, n * 4}};
    if (any_alias(outs, 4, ins, 7)) return QDC_ERR_ALIAS;
    DeltaStep a{};
    a.out = out;
    a.proj = proj;
    a.norm = norm;
    a.ring = ring;
    a.state = state;
    a.conv = conv;
    a.a_decay = a_decay;
    a.dt_bias = dt_bias;
    a.index = index;
    a.positions = positions;
    a.error_flag = error_flag;
    a.ld = ld;
    a.channels = channels;
    a.rows = (int)rows;
    a.taps = (int)taps;
    a.key_heads = (int)key_heads;
    a.heads = (int)value_heads;
    a.groups = (int)(value_heads / key_heads);
    a.value_dim = (int)value_dim;
    a.eps = eps;
    a.sqrt_kd = __builtin_sqrtf((float)key_dim);
    a.out_dtype = out_dtype;
    if (proj_dtype == QDC_BF16) {
        if (key_dim == 128) return launch<bf16_t, 128>(a, n, stream);
        if (key_dim == 64) return launch<bf16_t, 64>(a, n, stream);
        return launch<bf16_t, 32>(a, n, stream);
    }
    if (key_dim == 128) return launch<float, 128>(a, n, stream);
    if (key_dim == 64) return launch<float, 64>(a, n, stream);
    return launch<float, 32>(a, n, stream);
}
