// head_norm.hip — queries and keys on their way to an attention outside the 3x3 patch: each
// head's RMS norm with gains and its rotation by position in one pass over q and k
// (slime_ca_qk_norm_rotate), and the gradient of both (slime_ca_qk_norm_rotate_backward).
//
//   n = x w / sqrt(mean x^2 + eps);  (y_u, y_v) = (n_u cos t - n_v sin t, n_u sin t + n_v cos t)
//   t = position * frequency per pair (u, v) of channels
//   backward: g = the gradient of y turned back, a = g w, xh = x / sqrt(mean x^2 + eps):
//   gx = (a - xh mean(a xh)) / sqrt(mean x^2 + eps);  gw = sum over rows and heads of g xh
//
// Both move every element once and are bound by that. A thread owns four pairs of one row
// and walks the heads, so a row's angles are computed once for all of them: per element
// they would cost more instructions than the norm. 16 x 16,384 rows of 2 x 512 bf16: 203 us (5.3
// TB/s; a copy of 1 GiB reaches 4.96); the gradient of 16 x 4096 of them 80 us (5.0 TB/s).
#include "common.hpp"
#include "kernels.hpp"

namespace slime {
namespace {

constexpr int kThreads = 256;
// Heads whose loads are in flight together. Gradients of 16 x 4096 rows of 2 x 512 bf16: 83 us
// with one, 82 with two, 84 with three, 95 with four, whose registers leave three waves a SIMD.
constexpr int kBatch = 2;

// Sine and cosine of pos * freq (radians). The phase is a 64-bit fraction of a turn, and so
// exact modulo whole turns at any position: freq / 2 pi keeps its 53 bits, the phase 32.
// The quarter turn nearest to it leaves |x| <= pi / 4 for the Taylor series, whose next terms are 2e-9 and
// 2e-10.
__device__ __forceinline__ void turn_of(int pos, double freq, float& s, float& c) {
    double f = freq * 0.15915494309189533577;  // 1 / 2 pi
    f -= floor(f);
    // 2^64 f of f < 1 in two exact halves; f that rounds to 1 is no turn at all.
    const double hi = floor(f * 4294967296.0);
    const double lo = floor((f * 4294967296.0 - hi) * 4294967296.0);
    const unsigned long long step = hi >= 4294967296.0 ? 0ull
                                                       : ((unsigned long long)(unsigned)hi << 32) | (unsigned)lo;
    const unsigned phase = (unsigned)((step * (unsigned long long)(long long)pos) >> 32);
    const unsigned quarter = (phase + 0x20000000u) >> 30;
    const float x = (float)(int)(phase - (quarter << 30)) * (6.28318530717958647692f / 4294967296.0f);
    const float z = x * x;
    float sn = __builtin_fmaf(z, 1.0f / 362880.0f, -1.0f / 5040.0f);
    sn = __builtin_fmaf(z, sn, 1.0f / 120.0f);
    sn = __builtin_fmaf(z, sn, -1.0f / 6.0f);
    sn = __builtin_fmaf(z * x, sn, x);
    float cs = __builtin_fmaf(z, -1.0f / 3628800.0f, 1.0f / 40320.0f);
    cs = __builtin_fmaf(z, cs, -1.0f / 720.0f);
    cs = __builtin_fmaf(z, cs, 1.0f / 24.0f);
    cs = __builtin_fmaf(z, cs, -0.5f);
    cs = __builtin_fmaf(z, cs, 1.0f);
    const float a = quarter & 1 ? cs : sn, b = quarter & 1 ? sn : cs;
    s = quarter & 2 ? -a : a;
    c = (quarter + 1) & 2 ? -b : b;
}

// Sum over the kL lanes of one row.
template <int kL>
__device__ __forceinline__ float lanes_sum(float v) {
    if constexpr (kL == 16) return row16_sum(v);
    else return group_sum_n<kL>(v);
}

// A thread's eight channels of one head: c0 .. c0 + 3 and c1 .. c1 + 3, any element's address.
template <typename T>
__device__ __forceinline__ void load8(const T* p, int c0, int c1, float (&x)[8]) {
    if constexpr (sizeof(T) == 2) {
        uint2 a, b;
        __builtin_memcpy(&a, p + c0, 8);
        __builtin_memcpy(&b, p + c1, 8);
        const unsigned w[4] = {a.x, a.y, b.x, b.y};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            x[2 * e] = bf16lo(w[e]);
            x[2 * e + 1] = bf16hi(w[e]);
        }
    } else {
        __builtin_memcpy(x, p + c0, 16);
        __builtin_memcpy(x + 4, p + c1, 16);
    }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, int c0, int c1, const float (&x)[8]) {
    if constexpr (sizeof(T) == 2) {
        const uint2 a = make_uint2(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]));
        const uint2 b = make_uint2(pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7]));
        __builtin_memcpy(p + c0, &a, 8);
        __builtin_memcpy(p + c1, &b, 8);
    } else {
        __builtin_memcpy(p + c0, x, 16);
        __builtin_memcpy(p + c1, x + 4, 16);
    }
}

// The thread's place: lane j of the kL that share a row, its channels, and which of its
// eight values are pair e.
template <int kL, bool kAdjacent>
struct Place {
    static constexpr int kD = 8 * kL;
    int j, c0, c1;
    __device__ __forceinline__ Place() {
        j = threadIdx.x % kL;
        c0 = kAdjacent ? 8 * j : 4 * j;
        c1 = kAdjacent ? 8 * j + 4 : kD / 2 + 4 * j;
    }
    static constexpr int u(int e) { return kAdjacent ? 2 * e : e; }
    static constexpr int v(int e) { return kAdjacent ? 2 * e + 1 : 4 + e; }
    __device__ __forceinline__ void angles(const NormArgs& a, int b, int n, float (&s)[4], float (&c)[4]) const {
        const int* pos = a.positions + b * a.pos_batch + n * a.pos_row;
        const int per = kD / 2 / a.axes;
#pragma unroll
        for (int e = 0; e < 4; ++e) turn_of(pos[(4 * j + e) / per], a.freqs[4 * j + e], s[e], c[e]);
    }
    __device__ __forceinline__ void gains(const float* w, float (&x)[8]) const {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            x[e] = w[c0 + e];
            x[4 + e] = w[c1 + e];
        }
    }
};

// Head e of the q heads followed by the k heads, at row (b, n).
template <typename T>
__device__ __forceinline__ T* head_at(const HeadsArg& q, const HeadsArg& k, int Hq, int e, int b, int n) {
    const HeadsArg& t = e < Hq ? q : k;
    return static_cast<T*>(t.data) + b * t.batch + n * t.row + (e < Hq ? e : e - Hq) * t.head;
}

template <typename T, int kL, bool kAdjacent>
__global__ __launch_bounds__(kThreads) void norm_rotate_kernel(const NormArgs a, const int heads) {
    using P = Place<kL, kAdjacent>;
    const P p;
    const unsigned rows = (unsigned)a.B * a.N;  // below 2^31
    const unsigned row = blockIdx.x * (kThreads / kL) + threadIdx.x / kL;
    if (row >= rows) return;  // whole groups of kL lanes
    const int b = row / (unsigned)a.N, n = row % (unsigned)a.N;
    const int e0 = blockIdx.y * heads, e1 = min(e0 + heads, a.Hq + a.Hkv);
    float s[4], c[4], wq[8], wk[8];
    p.angles(a, b, n, s, c);
    p.gains(a.wq, wq);
    p.gains(a.wk, wk);
    for (int e = e0; e < e1; e += kBatch) {
        float x[kBatch][8];
#pragma unroll
        for (int i = 0; i < kBatch; ++i)
            if (e + i < e1) load8(head_at<const T>(a.q, a.k, a.Hq, e + i, b, n), p.c0, p.c1, x[i]);
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            if (e + i >= e1) break;
            float ss = 0.f;
#pragma unroll
            for (int k = 0; k < 8; ++k) ss = __builtin_fmaf(x[i][k], x[i][k], ss);
            const float r = rsqrtf(lanes_sum<kL>(ss) * (1.0f / P::kD) + a.eps);
            const bool is_q = e + i < a.Hq;
            float y[8];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float nu = x[i][P::u(k)] * r * (is_q ? wq[P::u(k)] : wk[P::u(k)]);
                const float nv = x[i][P::v(k)] * r * (is_q ? wq[P::v(k)] : wk[P::v(k)]);
                y[P::u(k)] = nu * c[k] - nv * s[k];
                y[P::v(k)] = nu * s[k] + nv * c[k];
            }
            store8(head_at<T>(a.oq, a.ok, a.Hq, e + i, b, n), p.c0, p.c1, y);
        }
    }
}

// Blocks walk the rows; each leaves its sums of the gains' gradients in part, and
// gains_join_kernel adds those in block order.
template <typename T, int kL, bool kAdjacent>
__global__ __launch_bounds__(kThreads) void norm_rotate_backward_kernel(const NormArgs a, const int heads) {
    using P = Place<kL, kAdjacent>;
    constexpr int kGroups = kThreads / kL;
    constexpr int kCols = 2 * P::kD, kSegs = kThreads / kCols;  // both gains' channels; threads a channel
    __shared__ float sums[kGroups][kCols];
    __shared__ float segs[kSegs][kCols];
    const P p;
    const int group = threadIdx.x / kL;
    const unsigned rows = (unsigned)a.B * a.N;  // below 2^31
    const int e0 = blockIdx.y * heads, e1 = min(e0 + heads, a.Hq + a.Hkv);
    float wq[8], wk[8], gwq[8], gwk[8];
    p.gains(a.wq, wq);
    p.gains(a.wk, wk);
#pragma unroll
    for (int k = 0; k < 8; ++k) gwq[k] = gwk[k] = 0.f;
    for (unsigned row = blockIdx.x * kGroups + group; row < rows; row += gridDim.x * kGroups) {
        const int b = row / (unsigned)a.N, n = row % (unsigned)a.N;
        float s[4], c[4];
        p.angles(a, b, n, s, c);
        for (int e = e0; e < e1; e += kBatch) {
            float x[kBatch][8], gy[kBatch][8];
#pragma unroll
            for (int i = 0; i < kBatch; ++i)
                if (e + i < e1) {
                    load8(head_at<const T>(a.q, a.k, a.Hq, e + i, b, n), p.c0, p.c1, x[i]);
                    load8(head_at<const T>(a.gq, a.gk, a.Hq, e + i, b, n), p.c0, p.c1, gy[i]);
                }
#pragma unroll
            for (int i = 0; i < kBatch; ++i) {
                if (e + i >= e1) break;
                const bool is_q = e + i < a.Hq;
                float ss = 0.f;
#pragma unroll
                for (int k = 0; k < 8; ++k) ss = __builtin_fmaf(x[i][k], x[i][k], ss);
                const float r = rsqrtf(lanes_sum<kL>(ss) * (1.0f / P::kD) + a.eps);
                float g[8], dot = 0.f;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    g[P::u(k)] = gy[i][P::u(k)] * c[k] + gy[i][P::v(k)] * s[k];
                    g[P::v(k)] = gy[i][P::v(k)] * c[k] - gy[i][P::u(k)] * s[k];
                }
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const float xh = x[i][k] * r, gx = g[k] * xh;
                    gwq[k] += is_q ? gx : 0.f;
                    gwk[k] += is_q ? 0.f : gx;
                    g[k] *= is_q ? wq[k] : wk[k];
                    dot = __builtin_fmaf(g[k], xh, dot);
                    x[i][k] = xh;
                }
                dot = lanes_sum<kL>(dot) * (1.0f / P::kD);
#pragma unroll
                for (int k = 0; k < 8; ++k) g[k] = r * (g[k] - x[i][k] * dot);
                store8(head_at<T>(a.oq, a.ok, a.Hq, e + i, b, n), p.c0, p.c1, g);
            }
        }
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const int d = (k < 4 ? p.c0 : p.c1) + k % 4;
        sums[group][d] = gwq[k];
        sums[group][P::kD + d] = gwk[k];
    }
    __syncthreads();
    const int col = threadIdx.x % kCols, seg = threadIdx.x / kCols;
    float v = 0.f;
#pragma unroll
    for (int i = 0; i < kGroups / kSegs; ++i) v += sums[seg * (kGroups / kSegs) + i][col];
    segs[seg][col] = v;
    __syncthreads();
    if (threadIdx.x < kCols) {
        v = 0.f;
#pragma unroll
        for (int i = 0; i < kSegs; ++i) v += segs[i][threadIdx.x];
        const long long block = (long long)blockIdx.y * gridDim.x + blockIdx.x;
        a.part[block * kCols + threadIdx.x] = v;
    }
}

// The gains' gradients: the blocks' sums, a block here for kJoin channels of both, in fp64.
constexpr int kJoin = 4;
__global__ __launch_bounds__(kThreads) void gains_join_kernel(const NormArgs a, const int blocks) {
    __shared__ double sums[kThreads / kWave][kJoin];
    const int col = threadIdx.x % kJoin, row = threadIdx.x / kJoin, c = blockIdx.x * kJoin + col;
    double v = 0.0;
    constexpr int kRows = kThreads / kJoin, kAhead = 16;  // loads in flight together
    for (int i0 = row; i0 < blocks; i0 += kRows * kAhead) {
        float x[kAhead];
#pragma unroll
        for (int e = 0; e < kAhead; ++e) x[e] = a.part[(long long)min(i0 + e * kRows, blocks - 1) * 2 * a.D + c];
#pragma unroll
        for (int e = 0; e < kAhead; ++e) v += i0 + e * kRows < blocks ? (double)x[e] : 0.0;
    }
#pragma unroll
    for (int step = kJoin; step < kWave; step *= 2) v += __shfl_xor(v, step);
    if (threadIdx.x % kWave < kJoin) sums[threadIdx.x / kWave][col] = v;
    __syncthreads();
    if (threadIdx.x < kJoin) {
        v = (sums[0][col] + sums[1][col]) + (sums[2][col] + sums[3][col]);
        (c < a.D ? a.gwq : a.gwk)[c % a.D] = (float)v;
    }
}

// Heads a thread walks: all of them, fewer where that leaves under two blocks a CU.
int heads_per_thread(const NormArgs& a, long long blocks) {
    const int all = a.Hq + a.Hkv;
    int heads = all;
    while (heads > 1 && blocks * ((all + heads - 1) / heads) < 512) heads = (heads + 1) / 2;
    return heads;
}

constexpr int kMostBlocks = 768;  // of the backward, over the rows: three a CU (512 to 1536: within 4%)

struct Grid {
    unsigned x, y;
    int heads;
};
Grid backward_grid(const NormArgs& a) {
    const long long rows = (long long)a.B * a.N, per = kThreads / (a.D / 8);
    const long long need = (rows + per - 1) / per;
    const long long x = need < kMostBlocks ? need : kMostBlocks;
    const int heads = heads_per_thread(a, x);
    return {(unsigned)x, (unsigned)((a.Hq + a.Hkv + heads - 1) / heads), heads};
}

template <typename T, int kL, bool kAdjacent>
hipError_t forward(const NormArgs& a, hipStream_t s) {
    const long long x = norm_blocks(a);
    const int heads = heads_per_thread(a, x);
    hipLaunchKernelGGL((norm_rotate_kernel<T, kL, kAdjacent>), dim3((unsigned)x, (a.Hq + a.Hkv + heads - 1) / heads),
                       dim3(kThreads), 0, s, a, heads);
    return hipGetLastError();
}
template <typename T, int kL, bool kAdjacent>
hipError_t backward(const NormArgs& a, hipStream_t s) {
    const Grid g = backward_grid(a);
    if (g.x > 0)
        hipLaunchKernelGGL((norm_rotate_backward_kernel<T, kL, kAdjacent>), dim3(g.x, g.y), dim3(kThreads), 0, s, a,
                           g.heads);
    hipLaunchKernelGGL(gains_join_kernel, dim3(2 * a.D / kJoin), dim3(kThreads), 0, s, a, (int)(g.x * g.y));
    return hipGetLastError();
}

template <typename T, int kL>
hipError_t run(const NormArgs& a, bool back, hipStream_t s) {
    if (back) return a.adjacent ? backward<T, kL, true>(a, s) : backward<T, kL, false>(a, s);
    return a.adjacent ? forward<T, kL, true>(a, s) : forward<T, kL, false>(a, s);
}
template <typename T>
hipError_t run_t(const NormArgs& a, bool back, hipStream_t s) {
    switch (a.D) {
        case 8: return run<T, 1>(a, back, s);
        case 16: return run<T, 2>(a, back, s);
        case 32: return run<T, 4>(a, back, s);
        case 64: return run<T, 8>(a, back, s);
        default: return run<T, 16>(a, back, s);
    }
}

}  // namespace

long long norm_blocks(const NormArgs& a) {
    const long long rows = (long long)a.B * a.N, per = kThreads / (a.D / 8);
    return (rows + per - 1) / per;
}
int norm_backward_blocks(const NormArgs& a) {
    const Grid g = backward_grid(a);
    return (int)(g.x * g.y);
}
hipError_t launch_norm_rotate(int dtype, const NormArgs& a, hipStream_t s) {
    return dtype == 1 ? run_t<bf16_t>(a, false, s) : run_t<float>(a, false, s);
}
hipError_t launch_norm_rotate_backward(int dtype, const NormArgs& a, hipStream_t s) {
    return dtype == 1 ? run_t<bf16_t>(a, true, s) : run_t<float>(a, true, s);
}

}  // namespace slime
