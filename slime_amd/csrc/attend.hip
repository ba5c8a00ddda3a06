// attend.hip — attention of cells to cells outside their 3x3 patch (slime_ca_attend): the
// softmax over all seen keys in one pass, with the running maximum and sum of each row.
//
//   s = scale q . k;  out = sum_j exp(s_j - m) v_j / l;  lse = m + log l
//   m = max_j s_j and l = sum_j exp(s_j - m), corrected by exp(m_old - m_new) per key tile.
//
// A wave holds 32 rows, or two sets of them, as columns of S^T = K Q^T and O^T = V^T P^T
// (attend.hpp): every lane has one row's statistics, and P stays in its registers.
//
// What bounds it. Many rows: matrix cores and arithmetic share the card's power. 16,384^2 x 8 x 64
// in bf16 takes 578 to 593 us from card to card (927 to 951 TFLOP/s; a library product of 8192^3
// reaches 1215); the same products and tiles without exponentials, LDS reads and loads take 440. Two sets of rows a wave halve the
// LDS reads (one set 695 us, two 587 of one build). Three blocks of keys in flight (scores,
// weights and product at once) spilled: 656. Deferring the maximum, or two tiles under way
// instead of one, changed nothing. Few rows: the keys' bytes; 16 histories of 8,192 to 16,384,
// 2 heads of 64, 28 us (101 MB, 3.6 TB/s), of which the join of the splits is 4.
#include "attend.hpp"

namespace slime {
namespace {

using namespace at;

constexpr float kLn2 = 0.6931471805599453f;

// The maximum that a row subtracts follows its scores with this slack (in powers of two), so
// that rows whose maximum creeps upward do not rescale their sums at every tile: weights up
// to 2^8 lose nothing in fp32 sums, nor in bf16, whose exponent is fp32's.
constexpr float kSlack = 8.0f;

// One set of 32 rows: its statistics, and its scores' way to weights.
struct Row {
    float m = -INFINITY, l = 0.f;  // the maximum in powers of two, this half's part of the sum
    int lo, hi;

    // Scores of keys that the row does not see; k0: the first key of s.
    __device__ __forceinline__ void mask(f32x16& s, int k0, int half) const {
        const int from = lo - k0 - 4 * half;
        const unsigned n = (unsigned)max(hi - lo + 1, 0);
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = (unsigned)(acc_row(i, 0) - from) < n ? s[i] : -INFINITY;
    }
    // The largest of these scores.
    template <typename... S>
    __device__ __forceinline__ static float top(const f32x16& s, const S&... more) {
        float mx = s[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) mx = fmaxf(mx, s[i]);
        if constexpr (sizeof...(more) > 0) mx = fmaxf(mx, top(more...));
        return mx;
    }
    // Brings the maximum up to both halves' largest score -> what the sums so far are scaled by.
    __device__ __forceinline__ float raise(float mx) {
        const float old = m;
        m = fmaxf(m, both_max(mx));
        const float fix = exp2_fast(old - base());
        l *= fix;
        return fix;
    }
    // A row that has seen no key keeps m = -inf and subtracts 0: exp2(-inf) = 0.
    __device__ __forceinline__ float base() const { return m == -INFINITY ? 0.f : m; }
    __device__ __forceinline__ void weights(f32x16& s, float c) {
        const float sub = base();
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            s[i] = exp2_fast(__builtin_fmaf(s[i], c, -sub));
            sum[i & 3] = i < 4 ? s[i] : sum[i & 3] + s[i];
        }
        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
    }
};

// log2 of the sum of exp2: of the maximum and the sum (a NaN sum stays).
__device__ __forceinline__ float log2_sum(float m, float l) { return l > 0.f || l != l ? m + __log2f(l) : -INFINITY; }
__device__ __forceinline__ float inverse(float l) { return l == 0.f ? 0.f : 1.f / l; }

// Row r of key head hk: its query, head, and place among the rows of lse and of the parts.
struct Place {
    int i, h;
    long long at;
    __device__ __forceinline__ Place(const AttendArgs& a, int b, int hk, int r)
        : i(r / a.group), h(hk * a.group + r % a.group), at(((long long)b * a.Hq + h) * a.Nq + i) {}
    // Four channels from d of the output, or of this split's part of it.
    template <typename T>
    __device__ __forceinline__ void put(const AttendArgs& a, int b, int split, int d, float x, float y, float z,
                                        float w) const {
        const long long rows = (long long)a.B * a.Hq * a.Nq;
        if (a.splits == 1)
            store4(static_cast<T*>(a.out.data) + b * a.out.batch + i * a.out.row + h * a.out.head + d, x, y, z, w);
        else
            store4(a.part + (split * rows + at) * a.D + d, x, y, z, w);
    }
    __device__ __forceinline__ void put_lse(const AttendArgs& a, int split, float m, float l) const {
        const long long rows = (long long)a.B * a.Hq * a.Nq;
        if (a.splits == 1)
            a.lse[at] = log2_sum(m, l) * kLn2;
        else
            a.part[a.splits * rows * a.D + split * rows + at] = log2_sum(m, l);
    }
};

// ---- many rows: four waves of 32 RB rows over shared tiles of 64 keys ----------------------
template <typename T, int DP, int RB, bool kAlive>
__global__ __launch_bounds__(kThreads, DP <= (Elem<T>::kPlanes == 3 ? 64 : 128) ? 2 : 1) void attend_rows_kernel(
    const AttendArgs a, const int row_tiles, const Deal deal) {
    constexpr int kKeys = 64, kRows = 128 * RB;
    using Kv = KeyTile<T, DP, kKeys, kAlive>;
    using G = global_t<T>;
    constexpr int kBufs = key_bufs<T, DP>();
    __shared__ __attribute__((aligned(16))) unsigned char lds_k[kBufs][Kv::kBytes];
    __shared__ __attribute__((aligned(16))) unsigned char lds_v[kBufs][Kv::kBytes];
    const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int head, item;
    if (!deal.at(blockIdx.x, head, item)) return;
    const int split = item % a.splits;
    const int rt = row_tiles - 1 - item / a.splits;  // the longest causal tiles first
    const int hk = head % a.Hkv, b = head / a.Hkv;

    const int R = a.Nq * a.group;
    const Sight sight(a, b);
    const int wg_row = rt * kRows, row0 = wg_row + 32 * RB * wave;
    const Span all(sight, wg_row, wg_row + kRows - 1, R, a.group), mine(sight, row0, row0 + 32 * RB - 1, R, a.group);
    const int tiles = all.hi >= all.lo ? (all.hi - all.lo + kKeys) / kKeys : 0;
    const int per = (tiles + a.splits - 1) / a.splits;
    const int t0 = min(split * per, tiles), t1 = min(t0 + per, tiles);

    const uint8_t* alive = kAlive ? a.alive + b * a.alive_batch : nullptr;
    const Rows krows(static_cast<const G*>(a.k.data) + b * a.k.batch + hk * a.k.head, a.k.row);
    const Rows vrows(static_cast<const G*>(a.v.data) + b * a.v.batch + hk * a.v.head, a.v.row);
    Kv sk, sv;
    auto issue = [&](int t, int buf) {
        const int k0 = all.lo + t * kKeys, n = all.hi + 1 - k0;
        sk.issue(lds_k[buf], krows, alive, k0, n, a.D, tid);
        sv.issue(lds_v[buf], vrows, alive, k0, n, a.D, tid);
    };
    auto finish = [&](int buf) {
        wait_vm0();
        sk.finish(lds_k[buf], tid);
        sv.finish(lds_v[buf], tid);
    };

    Op<T> q[RB][kRowSteps<T, DP>];
    Row row[RB];
#pragma unroll
    for (int n = 0; n < RB; ++n) {
        const int r = row0 + 32 * n + (lane & 31);
        const Place p(a, b, hk, min(r, R - 1));
        row[n].lo = sight.lo(p.i);
        row[n].hi = sight.hi(p.i);
        load_frags<T, DP>(static_cast<const G*>(a.q.data) + b * a.q.batch + p.i * a.q.row + p.h * a.q.head, true, a.D,
                          half, q[n]);
    }
    f32x16 o[RB][DP / 32];
#pragma unroll
    for (int n = 0; n < RB; ++n)
#pragma unroll
        for (int d = 0; d < DP / 32; ++d) o[n][d] = zeros16();
    const float c = a.scale * kLog2e;

#pragma unroll
    for (int i = 0; i < kBufs; ++i) {
        Kv::St::clear_pad(lds_k[i], a.D, tid);
        Kv::St::clear_pad(lds_v[i], a.D, tid);
    }
    if (t0 < t1) issue(t0, 0);
    settle(q);
    if (t0 < t1) {
        finish(0);
        __syncthreads();
    }
    for (int t = t0; t < t1; ++t) {
        const bool more = t + 1 < t1;
        const int k0 = all.lo + t * kKeys, buf = kBufs == 2 ? (t - t0) & 1 : 0, other = kBufs == 2 ? 1 - buf : 0;
        if (more) issue(t + 1, other);
        if (k0 <= mine.hi && k0 + kKeys > mine.lo) {
            f32x16 s[2][RB];
#pragma unroll
            for (int u = 0; u < 2; ++u) scores<T, DP, kKeys, kAlive>(s[u], lds_k[buf], 32 * u, q, lane);
            if (k0 < mine.all_lo || k0 + kKeys - 1 > mine.all_hi) {
#pragma unroll
                for (int n = 0; n < RB; ++n) {
                    row[n].mask(s[0][n], k0, half);
                    row[n].mask(s[1][n], k0 + 32, half);
                }
            }
            float mx[RB];
            bool over = false;
#pragma unroll
            for (int n = 0; n < RB; ++n) {
                mx[n] = Row::top(s[0][n], s[1][n]) * c;
                over = over || mx[n] > row[n].m + kSlack;
            }
            if (__any(over)) {
#pragma unroll
                for (int n = 0; n < RB; ++n) {
                    const float fix = row[n].raise(mx[n]);
#pragma unroll
                    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
                        for (int i = 0; i < 16; ++i) o[n][d][i] *= fix;
                }
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                Probs<T> p[RB];
#pragma unroll
                for (int n = 0; n < RB; ++n) {
                    row[n].weights(s[u][n], c);
                    p[n] = Probs<T>(s[u][n]);
                }
                mma_cols<T, DP, kKeys>(o, lds_v[buf], 32 * u, p, lane);
            }
        }
        if (kBufs == 1) __syncthreads();
        if (more) finish(other);
        __syncthreads();
    }
#pragma unroll
    for (int n = 0; n < RB; ++n) {
        const int r = row0 + 32 * n + (lane & 31);
        const float l = both_sum(row[n].l), inv = inverse(l);
        if (r >= R) continue;
        const Place at(a, b, hk, r);
#pragma unroll
        for (int d = 0; d < DP / 32; ++d)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int ch = 32 * d + 8 * g + 4 * half;
                if (ch < a.D)
                    at.put<G>(a, b, split, ch, o[n][d][4 * g] * inv, o[n][d][4 * g + 1] * inv, o[n][d][4 * g + 2] * inv,
                              o[n][d][4 * g + 3] * inv);
            }
        if (half == 0) at.put_lse(a, split, row[n].m, l);
    }
}

// ---- few rows: four waves share 32 rows and take 32 keys each of a tile of 128 -------------
// They wait for memory, so bf16 weights keep 16 bits here: the output's error is its own rounding,
// 1.4 times that in attend_rows_kernel, whose time more products would add to.
template <typename T>
using KeysProbs = typename std::conditional<sizeof(T) == 2, ProbsInTwo, Probs<T>>::type;

template <typename T, int DP, bool kAlive>
__global__ __launch_bounds__(kThreads) void attend_keys_kernel(const AttendArgs a, const int row_tiles,
                                                               const Deal deal) {
    constexpr int kKeys = 128, kRows = 32;
    using Kv = KeyTile<T, DP, kKeys, kAlive>;
    constexpr int kBufs = 4 * Kv::kBytes <= 160 * 1024 ? 2 : 1, kLds = kBufs * 2 * Kv::kBytes;
    static_assert(kLds >= kWaves * 32 * (DP + 2) * 4, "the waves' results are joined in the tiles' place");
    __shared__ __attribute__((aligned(16))) unsigned char lds[kLds];
    unsigned char(*lds_k)[Kv::kBytes] = reinterpret_cast<unsigned char(*)[Kv::kBytes]>(lds);
    unsigned char(*lds_v)[Kv::kBytes] = lds_k + kBufs;
    const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int head, item;
    if (!deal.at(blockIdx.x, head, item)) return;
    const int split = item % a.splits, rt = row_tiles - 1 - item / a.splits;
    const int hk = head % a.Hkv, b = head / a.Hkv;

    const int R = a.Nq * a.group, row0 = rt * kRows, r = row0 + (lane & 31);
    const Sight sight(a, b);
    const Span all(sight, row0, row0 + kRows - 1, R, a.group);
    const int tiles = all.hi >= all.lo ? (all.hi - all.lo + kKeys) / kKeys : 0;
    const int per = (tiles + a.splits - 1) / a.splits;
    const int t0 = min(split * per, tiles), t1 = min(t0 + per, tiles);
    const uint8_t* alive = kAlive ? a.alive + b * a.alive_batch : nullptr;
    const Rows krows(static_cast<const T*>(a.k.data) + b * a.k.batch + hk * a.k.head, a.k.row);
    const Rows vrows(static_cast<const T*>(a.v.data) + b * a.v.batch + hk * a.v.head, a.v.row);
    Kv sk, sv;
    auto issue = [&](int t, int buf) {
        const int k0 = all.lo + t * kKeys, n = all.hi + 1 - k0;
        sk.issue(lds_k[buf], krows, alive, k0, n, a.D, tid);
        sv.issue(lds_v[buf], vrows, alive, k0, n, a.D, tid);
    };
    auto finish = [&](int buf) {
        wait_vm0();
        sk.finish(lds_k[buf], tid);
        sv.finish(lds_v[buf], tid);
    };
    // A split without tiles goes straight to the waves' results, which lie in the tiles' place: it
    // writes nothing there before, so that no barrier is needed between.
    if (t0 < t1) {
#pragma unroll
        for (int i = 0; i < kBufs; ++i) {
            Kv::St::clear_pad(lds_k[i], a.D, tid);
            Kv::St::clear_pad(lds_v[i], a.D, tid);
        }
        issue(t0, 0);
    }

    Op<T> q[1][kRowSteps<T, DP>];
    Row row;
    {
        const Place p(a, b, hk, min(r, R - 1));
        row.lo = sight.lo(p.i);
        row.hi = sight.hi(p.i);
        load_frags<T, DP>(static_cast<const T*>(a.q.data) + b * a.q.batch + p.i * a.q.row + p.h * a.q.head, true, a.D,
                          half, q[0]);
    }
    f32x16 o[1][DP / 32];
#pragma unroll
    for (int d = 0; d < DP / 32; ++d) o[0][d] = zeros16();
    const float c = a.scale * kLog2e;

    settle(q);
    if (t0 < t1) {
        finish(0);
        __syncthreads();
    }
    for (int t = t0; t < t1; ++t) {
        const bool more = t + 1 < t1;
        const int k0 = all.lo + t * kKeys + 32 * wave, buf = kBufs == 2 ? (t - t0) & 1 : 0;
        if (kBufs == 2 && more) issue(t + 1, 1 - buf);
        const unsigned char *kt = lds_k[buf], *vt = lds_v[buf];
        if (k0 <= all.hi) {
            f32x16 s[1];
            scores<T, DP, kKeys, kAlive>(s, kt, 32 * wave, q, lane);
            if (k0 < all.all_lo || k0 + 31 > all.all_hi) row.mask(s[0], k0, half);
            const float mx = Row::top(s[0]) * c;
            if (__any(mx > row.m + kSlack)) {
                const float fix = row.raise(mx);
#pragma unroll
                for (int d = 0; d < DP / 32; ++d)
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[0][d][i] *= fix;
            }
            row.weights(s[0], c);
            const KeysProbs<T> p[1] = {KeysProbs<T>(s[0])};
            mma_cols<T, DP, kKeys>(o, vt, 32 * wave, p, lane);
        }
        if (kBufs == 1) {
            __syncthreads();
            if (more) issue(t + 1, 0);
        }
        if (more) finish(kBufs == 2 ? 1 - buf : 0);
        __syncthreads();
    }
    // The waves' parts of the rows: each scaled to the joint maximum, added in wave order.
    const float l = both_sum(row.l);
    float* stat = reinterpret_cast<float*>(lds);  // [wave][2][32]
    float* acc = stat + kWaves * 64;              // [wave][32][DP]
    if (half == 0) {
        stat[wave * 64 + lane] = row.m;
        stat[wave * 64 + 32 + lane] = l;
    }
    __syncthreads();
    float mm = stat[lane & 31];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) mm = fmaxf(mm, stat[w * 64 + (lane & 31)]);
    const float base = mm == -INFINITY ? 0.f : mm;
    float ll = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w)
        ll += stat[w * 64 + 32 + (lane & 31)] * exp2_fast(stat[w * 64 + (lane & 31)] - base);
    const float mine = inverse(ll) * exp2_fast(row.m - base);
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const float4 v = make_float4(o[0][d][4 * g] * mine, o[0][d][4 * g + 1] * mine, o[0][d][4 * g + 2] * mine,
                                         o[0][d][4 * g + 3] * mine);
            *reinterpret_cast<float4*>(acc + (wave * 32 + (lane & 31)) * DP + 32 * d + 8 * g + 4 * half) = v;
        }
    if (wave == 0 && half == 0 && r < R) Place(a, b, hk, r).put_lse(a, split, mm, ll);
    __syncthreads();
    for (int e = tid; e < 32 * DP / 4; e += kThreads) {
        const int n = e / (DP / 4), ch = e % (DP / 4) * 4;
        if (row0 + n >= R || ch >= a.D) continue;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float4 x = *reinterpret_cast<const float4*>(acc + (w * 32 + n) * DP + ch);
            v.x += x.x;
            v.y += x.y;
            v.z += x.z;
            v.w += x.w;
        }
        Place(a, b, hk, row0 + n).put<T>(a, b, split, ch, v.x, v.y, v.z, v.w);
    }
}

// out = sum_s 2^(lse_s - lse) out_s over the splits of the keys, in split order.
template <typename T>
__global__ __launch_bounds__(kThreads) void attend_join_kernel(const AttendArgs a) {
    const int per = a.D / 4;
    const long long e = (long long)blockIdx.x * kThreads + threadIdx.x;
    const long long rows = (long long)a.B * a.Hq * a.Nq, row = e / per;
    if (row >= rows) return;
    const int ch = (int)(e % per) * 4;
    const float* ls = a.part + a.splits * rows * a.D + row;
    const float* xs = a.part + row * a.D + ch;
    float m = -INFINITY, l = 0.f;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    // Eight splits' loads in flight together, their sums brought to the maximum so far.
    for (int s0 = 0; s0 < a.splits; s0 += 8) {
        float e[8];
        float4 x[8];
#pragma unroll
        for (int n = 0; n < 8; ++n) {
            const int s = min(s0 + n, a.splits - 1);
            e[n] = ls[s * rows];
            x[n] = *reinterpret_cast<const float4*>(xs + s * rows * a.D);
        }
        const float old = m;
#pragma unroll
        for (int n = 0; n < 8; ++n) m = fmaxf(m, s0 + n < a.splits ? e[n] : -INFINITY);
        const float base = m == -INFINITY ? 0.f : m, fix = exp2_fast(old - base);
        l *= fix;
        v.x *= fix;
        v.y *= fix;
        v.z *= fix;
        v.w *= fix;
#pragma unroll
        for (int n = 0; n < 8; ++n) {
            const float w = s0 + n < a.splits ? exp2_fast(e[n] - base) : 0.f;
            l += w;
            v.x += w * x[n].x;
            v.y += w * x[n].y;
            v.z += w * x[n].z;
            v.w += w * x[n].w;
        }
    }
    const float inv = inverse(l);
    const int i = (int)(row % a.Nq);
    const long long bh = row / a.Nq;
    const int b = (int)(bh / a.Hq), h = (int)(bh % a.Hq);
    store4(static_cast<T*>(a.out.data) + b * a.out.batch + i * a.out.row + h * a.out.head + ch, v.x * inv, v.y * inv,
           v.z * inv, v.w * inv);
    if (ch == 0) a.lse[row] = log2_sum(m, l) * kLn2;
}

template <typename T>
void join(const AttendArgs& a, hipStream_t s) {
    const long long n = (long long)a.B * a.Hq * a.Nq * (a.D / 4);
    hipLaunchKernelGGL(attend_join_kernel<T>, dim3((unsigned)((n + kThreads - 1) / kThreads)), dim3(kThreads), 0, s, a);
}

// T: how many rows meet the keys; K: how few do.
template <typename T, typename K, int DP, bool kAlive>
hipError_t run(const AttendArgs& a, const AttendPlan& p, hipStream_t s) {
    const int tiles = (a.Nq * a.group + p.rows - 1) / p.rows;
    const Deal deal{a.B * a.Hkv, tiles * a.splits};
    const dim3 grid(deal.blocks()), block(kThreads);
    if (p.rows == 32)
        hipLaunchKernelGGL((attend_keys_kernel<K, DP, kAlive>), grid, block, 0, s, a, tiles, deal);
    else if (p.rows == 128)
        hipLaunchKernelGGL((attend_rows_kernel<T, DP, 1, kAlive>), grid, block, 0, s, a, tiles, deal);
    else if constexpr (two_sets(sizeof(K), DP))
        hipLaunchKernelGGL((attend_rows_kernel<T, DP, 2, kAlive>), grid, block, 0, s, a, tiles, deal);
    else
        return hipErrorInvalidValue;  // no such plan
    if (a.splits > 1) join<K>(a, s);
    return hipGetLastError();
}
template <typename T, typename K, int DP>
hipError_t run(const AttendArgs& a, const AttendPlan& p, hipStream_t s) {
    return a.alive ? run<T, K, DP, true>(a, p, s) : run<T, K, DP, false>(a, p, s);
}

template <typename T, typename K>
hipError_t run_t(const AttendArgs& a, const AttendPlan& p, hipStream_t s) {
    return a.D <= 32 ? run<T, K, 32>(a, p, s) : a.D <= 64 ? run<T, K, 64>(a, p, s) : run<T, K, 128>(a, p, s);
}

}  // namespace

AttendPlan attend_plan(int dtype, const AttendArgs& a, int n_cu) {
    AttendPlan p;
    const long long rows = (long long)a.Nq * a.group, heads = (long long)a.B * a.Hkv;
    p.row_splits = 1;
    p.rows = rows <= 32 ? 32 : 128;
    if (two_sets(dtype == 1 ? 2 : 4, a.D) && heads * ((rows + 255) / 256) >= 2LL * n_cu) p.rows = 256;
    // The number of splits, each of two tiles of keys at least, that takes the least time, in products of
    // a tile by 128 rows: a workgroup starts and ends in the time of two. Walks of one length go in
    // rounds of two workgroups a CU (one of fp32 heads of 128, which fill the registers), of which half of
    // one takes 0.8 of its time, or 0.6 where few rows wait for memory; few rows of wide heads (bf16 of
    // 128, fp32 of 64), of which LDS holds one workgroup a CU, have the same fit: a round is two in turn there;
    // walks of many lengths, longest first, end in a quarter of the longest. The parts take 0.15 a
    // thousand rows (fp32 products three times as long beside them) and their join two. Against one
    // workgroup on a CU, or two in fp32 above 32 channels and for few rows, us: 4096 causal x 8 x 64 in
    // bf16 66 -> 42 and in fp32 139 -> 114, 3 x 1337 windowed, 8 over 4 heads of 64, 23 -> 12, 2 x 600 x 8 x
    // 128 26 -> 19; over 82 calls of 51 to 16,384 rows 13 % less time, 3 % above the best splits of each. 52
    // times one row of 8 over 2 heads of 128 on 933 keys 26 -> 21; over 24 calls of few rows, all from
    // memory, 8 % less, 0.3 % above the best.
    const int keys = p.rows == 32 ? 128 : 64, planes = dtype == 1 ? 1 : 3;
    const long long shift = a.align_start ? 0 : (long long)a.Nk - a.Nq;
    auto seen = [&](long long i) {  // keys at most, by the queries up to i
        const long long n = i + shift + 1;
        return a.causal ? (n < 0 ? 0 : n < a.Nk ? n : (long long)a.Nk) : (long long)a.Nk;
    };
    const long long wide = a.window * (a.causal ? 1LL : 2LL) + (p.rows < rows ? p.rows : rows) / a.group;
    const bool cut = a.window > 0 && wide < a.Nk;
    const double sets = p.rows == 256 ? 2.0 : 1.0, longest = sets * ((cut ? wide : seen(a.Nq - 1)) + keys - 1) / keys;
    const double mean = cut ? longest : 0.5 * (longest + sets * (seen(0) + keys - 1) / keys);
    const double wgs = (double)heads * ((rows + p.rows - 1) / p.rows), slots = (p.rows > 32 && planes == 3 && a.D > 64 ? 1.0 : 2.0) * n_cu;
    constexpr int kSplits[] = {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64, 96, 128, 192, 256};
    const double half = p.rows == 32 ? 0.6 : 0.8;
    double least = INFINITY;
    p.splits = 1;
    for (const int s : kSplits) {
        if (s > 1 && 2LL * s > (a.Nk + keys - 1) / keys) break;
        const double l = 2.0 + longest / s, rounds = wgs * s / slots, whole = floor(rounds), rest = rounds - whole;
        double t = l * (whole + (rest > 0.5 ? 1.0 : rest > 0.0 ? half : 0.0));
        if (mean < longest) t = fmax(l * (rounds > 0.5 ? 1.0 : half), rounds * (2.0 + mean / s) + 0.25 * l);
        if (s > 1) t += 2.0 + 0.15e-3 * s * heads * rows / planes;
        if (t < least) {
            least = t;
            p.splits = s;
        }
    }
    return p;
}

double attend_workgroups(const AttendArgs& a, const AttendPlan& p) {
    const double rows = (double)a.Nq * a.group, heads = (double)a.B * a.Hkv;
    const double walks = heads * ceil(rows / p.rows) * p.splits + 8;  // whole eights of them (Deal)
    return p.splits > 1 ? fmax(walks, ceil(heads * rows * (a.D / 4) / kThreads)) : walks;
}

hipError_t launch_attend(int dtype, const AttendArgs& a, const AttendPlan& p, hipStream_t s) {
    return dtype == 1 ? run_t<bf16_t, bf16_t>(a, p, s) : run_t<split_t, float>(a, p, s);
}

}  // namespace slime
