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
#include <cmath>

#include "qdc_cache.hpp"

namespace qdc {
namespace {

constexpr int kStep = 512;  // threads
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

// L lanes a state row, N 16-byte pieces a lane; a pass of the workgroup takes
// kStep / L rows, PASSES passes all of them.
template <typename T, int KD, int PASSES>
__global__ __launch_bounds__(kStep) void delta_step(DeltaStep a) {
    constexpr int L = KD / 4 < 16 ? KD / 4 : 16, N = KD / (4 * L), ROWS = kStep / L;
    __shared__ __align__(16) float qkv[2 * KD + kMaxValue], so[kMaxValue];
    __shared__ float part[kStep / kWave], gates[2];
    const int entry = blockIdx.x, h = blockIdx.y, tid = threadIdx.x, vd = a.value_dim;
    const int row = a.index[entry], pos = a.positions[entry];
    const bool token = row >= 0 && pos >= 0;
    // a row that an earlier token of the call has: not done twice
    bool bad = token && row >= a.rows;
    if (token)
        for (int j = tid; j < entry; j += kStep)
            bad = bad || (a.index[j] == row && a.positions[j] >= 0);
    const bool live = token && !__syncthreads_or(bad);
    const int64_t at = ((int64_t)entry * a.heads + h) * vd;
    auto put = [&](int v, float o) {
        if (a.out_dtype == QDC_BF16) put_elem((bf16_t *)a.out, at + v, o);
        else if (a.out_dtype == QDC_F32) put_elem((float *)a.out, at + v, o);
        else put_elem((split_t *)a.out, at + v, o);
    };
    if (!live) {  // uniform
        for (int v = tid; v < vd; v += kStep) put(v, 0.0f);
        if (token && tid == 0) raise_flag(a.error_flag);
        return;
    }
    const int lane = tid % L, r0 = tid / L;
    float *state = a.state + ((int64_t)row * a.heads + h) * vd * KD;
    f32x4 S[PASSES][N];
#pragma unroll
    for (int p = 0; p < PASSES; ++p)
#pragma unroll
        for (int n = 0; n < N; ++n) {
            S[p][n] = f32x4{0.f, 0.f, 0.f, 0.f};
            if (pos > 0 && r0 + p * ROWS < vd)
                S[p][n] = *reinterpret_cast<const f32x4 *>(state + (int64_t)(r0 + p * ROWS) * KD +
                                                           4 * (lane + L * n));
        }
    // the token's channels of this head: q | k | v
    const int g = h / a.groups;
    const int64_t kw = (int64_t)a.key_heads * KD, cq = a.channels;
    const T *proj = (const T *)a.proj + entry * a.ld;
    T *ring = (T *)a.ring + (int64_t)row * a.taps * cq;
    const bool owner = h % a.groups == 0;  // of the key head's part of the ring
    for (int i = tid; i < 2 * KD + vd; i += kStep) {
        const int64_t c = i < KD       ? (int64_t)g * KD + i
                          : i < 2 * KD ? kw + (int64_t)g * KD + (i - KD)
                                       : 2 * kw + (int64_t)h * vd + (i - 2 * KD);
        const T now = proj[c];
        float acc = 0.0f;
        for (int j = 0; j < a.taps; ++j) {
            const int lag = a.taps - 1 - j;
            if (lag > pos) continue;  // before the row's start
            const T x = lag ? ring[(int64_t)((pos - lag) % a.taps) * cq + c] : now;
            acc = acc + to_f32(x) * a.conv[c * a.taps + j];
        }
        if (owner || i >= 2 * KD) ring[(int64_t)(pos % a.taps) * cq + c] = now;
        qkv[i] = silu(acc);
    }
    if (tid == 0) {
        const int64_t vw = (int64_t)a.heads * vd;
        gates[0] = sigmoid(to_f32(proj[cq + vw + a.heads + h]));
        gates[1] = expf(a.a_decay[h] * softplus_f(to_f32(proj[cq + vw + h]) + a.dt_bias[h]));
    }
    __syncthreads();
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
                S[p][n][e] *= f;
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
            *reinterpret_cast<f32x4 *>(state + (int64_t)v * KD + 4 * (lane + L * n)) = S[p][n];
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
    const float z = to_f32(proj[cq + (int64_t)h * vd + tid]);
    put(tid, ((o * s) * to_f32(((const T *)a.norm)[tid])) * silu(z));
}

template <typename T, int KD> int32_t launch(const DeltaStep &a, int64_t n, hipStream_t stream) {
    const dim3 grid((uint32_t)n, (uint32_t)a.heads), block(kStep);
    constexpr int L = KD / 4 < 16 ? KD / 4 : 16;
    switch (ceil_div((int64_t)a.value_dim, (int64_t)(kStep / L))) {
#define QDC_STEP(P)                                                                   \
    case P:                                                                           \
        hipLaunchKernelGGL((delta_step<T, KD, P>), grid, block, 0, stream, a);        \
        return launch_status();
        QDC_STEP(1)
        QDC_STEP(2)
        QDC_STEP(3)
        QDC_STEP(4)
        QDC_STEP(5)
        QDC_STEP(6)
        QDC_STEP(7)
        QDC_STEP(8)
#undef QDC_STEP
        default: break;
    }
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
    // a workgroup of 512 per entry and head in a grid of fewer than 2^32 work-items
    if (ld < channels + vw + 2 * value_heads || n >= lim || ld >= lim ||
        n * value_heads >= ((int64_t)1 << 23))
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
