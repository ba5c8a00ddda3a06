// attend_backward.hip — the gradient of slime_ca_attend, from q, k, v, out, the gradient of out
// and each row's log-sum-exp; the probabilities are computed again, never stored.
//
//   P = exp(s - lse), delta = sum_c gout_c out_c, dP = gout v^T, dS = scale P (dP - delta)
//   gq = dS k,  gk = dS^T q,  gv = P^T gout
//
// Without atomics, so the sums have one order: rows' workgroups walk the keys (scores, dP and gq:
// three products), keys' workgroups the rows (scores, dP, gv and gk: four). Seven products in the
// place of the five that one walk with atomics would take. delta is summed first; then both kinds
// of workgroups run in one launch, so that a small call's fill the device together and a large
// call's last ones leave no gap.
//
// What bounds it: 4 x 4096^2 x 8 x 64 in bf16 takes 480 to 507 us from card to card, 1015 to 1070
// TFLOP/s of the products that it makes (a library product of 8192^3 reaches 1215), 680 to 715 of
// the five that it cannot do without. 6144 causal, 8 over 2 heads of 128, takes 364 to 374: 3 + 5
// products, and 20 for the parts' sums.
//
// P and dS are rounded to bf16 before the products that sum them, the type of those products' other
// operands: gradients are off by 1.4 of their own rounding. In fp32 they are three parts.
#include "attend.hpp"

namespace slime {
namespace {

using namespace at;

// delta: a row's 16-byte chunks go to as many neighbouring lanes (1 to 32).
template <typename G>
__global__ __launch_bounds__(kThreads) void attend_delta_kernel(const AttendArgs a, const int lanes) {
    const long long e = (long long)blockIdx.x * kThreads + threadIdx.x, rows = (long long)a.B * a.Hq * a.Nq;
    const long long at = min(e / lanes, rows - 1);  // whole groups of lanes
    const int i = (int)(at % a.Nq), c = (int)(e % lanes) * (16 / (int)sizeof(G));
    const long long bh = at / a.Nq;
    const int b = (int)(bh / a.Hq), h = (int)(bh % a.Hq);
    const uint4 u = load16(static_cast<const G*>(a.out.data) + b * a.out.batch + i * a.out.row + h * a.out.head + c);
    const uint4 v = load16(static_cast<const G*>(a.gout.data) + b * a.gout.batch + i * a.gout.row + h * a.gout.head + c);
    const unsigned x[4] = {u.x, u.y, u.z, u.w}, y[4] = {v.x, v.y, v.z, v.w};
    float sum = 0.f;
#pragma unroll
    for (int n = 0; n < 4; ++n) {
        if constexpr (sizeof(G) == 2) {
            sum = __builtin_fmaf(bf16lo(x[n]), bf16lo(y[n]), sum);
            sum = __builtin_fmaf(bf16hi(x[n]), bf16hi(y[n]), sum);
        } else
            sum = __builtin_fmaf(__builtin_bit_cast(float, x[n]), __builtin_bit_cast(float, y[n]), sum);
    }
    for (int step = lanes / 2; step > 0; step /= 2) sum += __shfl_xor(sum, step);
    if (e % lanes == 0 && e / lanes < rows) a.delta[at] = sum;
}

// log2 of a row's sum; a row that saw no key (lse = -inf) gives every key 2^-inf = 0.
__device__ __forceinline__ float lse_base2(float lse) { return lse == -INFINITY ? INFINITY : lse * kLog2e; }

// A value as the sum of three bf16 (8 bits each, all 24 of it), in the first channels of eight:
// with -1 on the other side, a product of matrices subtracts it from each element of a row.
__device__ __forceinline__ uint4 three_parts(float x) {
    const float a = __builtin_bit_cast(float, __builtin_bit_cast(unsigned, x) & 0xffff0000u), r = x - a;
    const float b = __builtin_bit_cast(float, __builtin_bit_cast(unsigned, r) & 0xffff0000u), c = r - b;
    return make_uint4((__builtin_bit_cast(unsigned, a) >> 16) | __builtin_bit_cast(unsigned, b),
                      __builtin_bit_cast(unsigned, c) >> 16, 0, 0);
}
// What a row that saw no key subtracts from its scores: 2^126, so that every weight is 0.
constexpr float kNoKeys = 8.507059173023462e37f;

// ---- queries' gradient ---------------------------------------------------------------------
// As the forward: a wave holds RB sets of 32 rows as columns, keys come in shared tiles of 64.
template <typename T, int DP, bool kAlive>
struct QShape {
    using Kv = KeyTile<T, DP, 64, kAlive>;
    static constexpr int kBufs = key_bufs<T, DP>(), kLds = kBufs * 2 * Kv::kBytes;
};

template <typename T, int DP, int RB, bool kAlive>
__device__ __forceinline__ void grad_q(const AttendArgs& a, int row_tiles, int head, int item, unsigned char* lds) {
    using Kv = typename QShape<T, DP, kAlive>::Kv;
    using G = global_t<T>;
    constexpr int kKeys = 64, kRows = 128 * RB, kBufs = QShape<T, DP, kAlive>::kBufs;
    unsigned char(*lds_k)[Kv::kBytes] = reinterpret_cast<unsigned char(*)[Kv::kBytes]>(lds);
    unsigned char(*lds_v)[Kv::kBytes] = lds_k + kBufs;
    const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int split = item % a.splits, rt = row_tiles - 1 - item / a.splits;
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
    // The first tile is under way while the rows are read.
#pragma unroll
    for (int i = 0; i < kBufs; ++i) {
        Kv::St::clear_pad(lds_k[i], a.D, tid);
        Kv::St::clear_pad(lds_v[i], a.D, tid);
    }
    if (t0 < t1) issue(t0, 0);
    Op<T> q[RB][kRowSteps<T, DP>], g[RB][kRowSteps<T, DP>];
    float delta[RB], lse2[RB];
    int lo[RB], hi[RB];
#pragma unroll
    for (int n = 0; n < RB; ++n) {
        const int row = row0 + 32 * n + (lane & 31), r = min(row, R - 1), i = r / a.group, h = hk * a.group + r % a.group;
        const long long at = ((long long)b * a.Hq + h) * a.Nq + i;
        lo[n] = sight.lo(i);
        hi[n] = sight.hi(i);
        lse2[n] = a.lse[at];
        load_frags<T, DP>(static_cast<const G*>(a.q.data) + b * a.q.batch + i * a.q.row + h * a.q.head, true, a.D,
                          half, q[n]);
        load_frags<T, DP>(static_cast<const G*>(a.gout.data) + b * a.gout.batch + i * a.gout.row + h * a.gout.head,
                          true, a.D, half, g[n]);
        delta[n] = a.delta[at];
    }
    f32x16 acc[RB][DP / 32];
#pragma unroll
    for (int n = 0; n < RB; ++n)
#pragma unroll
        for (int d = 0; d < DP / 32; ++d) acc[n][d] = zeros16();
    const float c = a.scale * kLog2e;

    settle(q);
    settle(g);
#pragma unroll
    for (int n = 0; n < RB; ++n) {
        asm volatile("" : "+v"(lse2[n]), "+v"(delta[n]));
        lse2[n] = lse_base2(lse2[n]);
    }
    if (t0 < t1) {
        finish(0);
        __syncthreads();
    }
    for (int t = t0; t < t1; ++t) {
        const bool more = t + 1 < t1;
        const int k0 = all.lo + t * kKeys, buf = kBufs == 2 ? (t - t0) & 1 : 0, other = kBufs == 2 ? 1 - buf : 0;
        if (more) issue(t + 1, other);
        const unsigned char *kt = lds_k[buf], *vt = lds_v[buf];
        if (k0 <= mine.hi && k0 + kKeys > mine.lo) {
            const bool part = k0 < mine.all_lo || k0 + kKeys - 1 > mine.all_hi;
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                f32x16 s[RB], gp[RB];
                scores<T, DP, kKeys, kAlive>(s, kt, 32 * u, q, lane);
#pragma unroll
                for (int n = 0; n < RB; ++n) gp[n] = zeros16();
                mma_rows<T, DP, kKeys>(gp, vt, 32 * u, g, lane);
                Probs<T> p[RB];
#pragma unroll
                for (int n = 0; n < RB; ++n) {
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        s[n][i] = exp2_fast(__builtin_fmaf(s[n][i], c, -lse2[n])) * (gp[n][i] - delta[n]);
                    if (part) {
                        const int from = lo[n] - k0 - 4 * half;
                        const unsigned seen = (unsigned)max(hi[n] - lo[n] + 1, 0);
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                            s[n][i] = (unsigned)(32 * u + acc_row(i, 0) - from) < seen ? s[n][i] : 0.f;
                    }
                    p[n] = Probs<T>(s[n]);
                }
                mma_cols<T, DP, kKeys>(acc, kt, 32 * u, p, lane);
            }
        }
        if (kBufs == 1) __syncthreads();
        if (more) finish(other);
        __syncthreads();
    }
    const long long rows_all = (long long)a.B * a.Hq * a.Nq;
#pragma unroll
    for (int n = 0; n < RB; ++n) {
        const int r = row0 + 32 * n + (lane & 31);
        if (r >= R) continue;
        const int i = r / a.group, h = hk * a.group + r % a.group;
        const long long at = ((long long)b * a.Hq + h) * a.Nq + i;
#pragma unroll
        for (int d = 0; d < DP / 32; ++d)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int ch = 32 * d + 8 * e + 4 * half;
                if (ch >= a.D) continue;
                const float x = acc[n][d][4 * e] * a.scale, y = acc[n][d][4 * e + 1] * a.scale,
                            z = acc[n][d][4 * e + 2] * a.scale, w = acc[n][d][4 * e + 3] * a.scale;
                if (a.splits == 1)
                    store4(static_cast<G*>(a.gq.data) + b * a.gq.batch + i * a.gq.row + h * a.gq.head + ch, x, y, z, w);
                else
                    store4(a.part + (split * rows_all + at) * a.D + ch, x, y, z, w);
            }
    }
}

// ---- keys' and values' gradients ----------------------------------------------------------------
// A wave holds KB sets of 32 keys as columns; queries come in shared tiles of 64 of one head,
// with each row's log-sum-exp and delta beside them. Every workgroup walks them from the last
// query to the first, all heads that share the keys at each tile, and the splits take turns: so
// the workgroups of an XCD, wherever a causal mask lets theirs begin, read the same rows at about
// the same time, out of its L2.
//
// Reads from LDS and the products take about as long: for one product of 32 x 32 x 16 the reads
// take 9 cycles of the CU, or 14 along columns, and its four matrix cores finish one every 8. So a
// row's log-sum-exp and delta are three more channels of its two products: two products more, in
// the place of eight reads of 16 bytes and a fourth of the arithmetic on the scores (6144 causal,
// 8 over 2 heads of 128: 444 | 420 us; 4 x 4096^2 x 8 x 64: 498 | 488).
//
// A workgroup takes both gradients of its keys (four products a tile), or where those exceed a
// wave's 256 registers one the keys' gradient (three products) and its neighbour the values'
// (two): one product more (heads of 128: 435 us in one role, which moves its accumulators in and
// out, 398 in two; heads of 64: 507 in one, 609 in two with 64 keys a wave, 770 with 32). Not all
// fit even so: of heads of 128 in bf16 a lane has 8 registers in scratch memory, 22 with living
// cells, of heads of 64 with living cells 6; in fp32 2 for heads of 64 and 16 to 33 of 512 for 128.
// KB is 1 in every call.
enum Part { kBoth, kValues, kKeysOnly };

template <typename T, int DP, int KB>
struct KvShape {
    static constexpr int kKeys = 128 * KB, kRows = 64;
    static constexpr int kTileB = Tile<T, DP, kRows>::kBytes;
    // Each row's log-sum-exp and delta take 16 bytes.
    static constexpr int kInfoB = 16, kBufB = 2 * kTileB + 2 * kRows * kInfoB;
    static constexpr int kBufs = key_bufs<T, DP>();
};

template <typename T, int DP, int KB, Part kPart>
__device__ __forceinline__ void grad_kv(const AttendArgs& a, int head, int item, unsigned char* lds) {
    using Sh = KvShape<T, DP, KB>;
    using G = global_t<T>;
    constexpr int kKeys = Sh::kKeys, kRows = Sh::kRows, kTileB = Sh::kTileB, kBufB = Sh::kBufB;
    constexpr int kInfoB = Sh::kInfoB, kBufs = Sh::kBufs;
    constexpr bool kK = kPart != kValues, kV = kPart != kKeysOnly;
    const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int split = item % a.row_splits, kt = item / a.row_splits;  // the first keys have the most causal rows
    const int hk = head % a.Hkv, b = head / a.Hkv;

    const Sight sight(a, b);
    const int j0 = kt * kKeys, j1 = min(j0 + kKeys, sight.len);
    // The queries that see a key of j0 .. j1 - 1.
    const int i0 = sight.first_query(j0), i1 = min(sight.last_query(j1 - 1), a.Nq - 1);
    const int per_head = j1 > j0 && i1 >= i0 ? (i1 - i0 + kRows) / kRows : 0;
    const int tiles = a.group * per_head, steps = split < tiles ? (tiles - split - 1) / a.row_splits + 1 : 0;

    const int key0 = j0 + 32 * KB * wave;
    Op<T> k[KB][kRowSteps<T, DP>], v[KB][kRowSteps<T, DP>];
    bool ok[KB];
    f32x16 gk[KB][DP / 32], gv[KB][DP / 32];
#pragma unroll
    for (int n = 0; n < KB; ++n) {
        const int key = min(key0 + 32 * n + (lane & 31), a.Nk - 1);
        ok[n] = key0 + 32 * n + (lane & 31) < sight.len;
        if (ok[n] && a.alive) ok[n] = a.alive[b * a.alive_batch + key] != 0;
        load_frags<T, DP>(static_cast<const G*>(a.k.data) + b * a.k.batch + key * a.k.row + hk * a.k.head, ok[n], a.D,
                          half, k[n]);
        if constexpr (kK)
            load_frags<T, DP>(static_cast<const G*>(a.v.data) + b * a.v.batch + key * a.v.row + hk * a.v.head, ok[n],
                              a.D, half, v[n]);
#pragma unroll
        for (int d = 0; d < DP / 32; ++d) gk[n][d] = gv[n][d] = zeros16();
    }
    const float c = a.scale * kLog2e;

    Stage<T, DP, kRows> sq, sg;
    float row_lse = 0.f, row_delta = 0.f;
    // The next tile to load: its head in the group, its last query; and from one to the next.
    int gh = split % a.group, end = i1 - kRows * (split / a.group);
    const int by_head = a.row_splits % a.group, by_row = kRows * (a.row_splits / a.group);
    auto issue = [&](int buf) {
        const int h = hk * a.group + gh, base = max(i0, end - kRows + 1), n = end + 1 - base;
        const Rows q(static_cast<const G*>(a.q.data) + b * a.q.batch + h * a.q.head, a.q.row);
        const Rows g(static_cast<const G*>(a.gout.data) + b * a.gout.batch + h * a.gout.head, a.gout.row);
        sq.issue(lds + buf * kBufB, q, base, n, a.D, tid);
        sg.issue(lds + buf * kBufB + kTileB, g, base, n, a.D, tid);
        // Rows past the last are as rows that saw no key.
        row_lse = -INFINITY;
        row_delta = 0.f;
        if (tid < kRows && tid < n) {
            const long long at = ((long long)b * a.Hq + h) * a.Nq + base + tid;
            row_lse = a.lse[at];
            row_delta = a.delta[at];
        }
        gh += by_head;
        end -= by_row;
        if (gh >= a.group) {
            gh -= a.group;
            end -= kRows;
        }
    };
    auto finish = [&](int buf) {
        wait_vm0();
        // Used here and not before: the compiler would wait for them, and with them for the tile's
        // loads, as soon as they are issued.
        asm volatile("" : "+v"(row_lse), "+v"(row_delta));
        sq.finish(lds + buf * kBufB, tid);
        sg.finish(lds + buf * kBufB + kTileB, tid);
        if (tid < kRows) {
            unsigned char* info = lds + buf * kBufB + 2 * kTileB + tid * kInfoB;
            *reinterpret_cast<uint4*>(info) = three_parts(row_lse == -INFINITY ? kNoKeys : row_lse / a.scale);
            *reinterpret_cast<uint4*>(info + kRows * kInfoB) = three_parts(row_delta);
        }
    };
    // The other operand of those channels: three times -1 in the lower half's.
    const uint4 minus = half ? make_uint4(0, 0, 0, 0) : make_uint4(0xBF80BF80u, 0xBF80u, 0, 0);

    int last = end;
#pragma unroll
    for (int i = 0; i < kBufs; ++i) {
        sq.clear_pad(lds + i * kBufB, a.D, tid);
        sg.clear_pad(lds + i * kBufB + kTileB, a.D, tid);
    }
    if (steps > 0) issue(0);
    settle(k);
    if constexpr (kK) settle(v);
    if (steps > 0) {
        finish(0);
        __syncthreads();
    }
    for (int t = 0; t < steps; ++t) {
        const int next = end, buf = kBufs == 2 ? t & 1 : 0, other = kBufs == 2 ? 1 - buf : 0;
        const bool more = t + 1 < steps;
        if (more) issue(other);
        const unsigned char* qt = lds + buf * kBufB;
        const unsigned char* gt_ = qt + kTileB;
        const unsigned char* info = qt + 2 * kTileB;
        // The wave's keys against the tile's queries: all seen, some, or none.
        const int base = max(i0, last - kRows + 1), key1 = key0 + 32 * KB - 1;
        const bool none = key0 > sight.hi(last) || key1 < sight.lo(base);
        const bool part = key0 < sight.lo(last) || key1 > sight.hi(base) || last - base + 1 < kRows;
        if (!none) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                f32x16 s[KB], ds[KB];
#pragma unroll
                for (int n = 0; n < KB; ++n) s[n] = ds[n] = zeros16();
                const unsigned char* at = info + (32 * u + (lane & 31)) * kInfoB;
                auto products = [&] {
                    mma_rows<T, DP, kRows>(s, qt, 32 * u, k, lane);
                    if constexpr (kK) mma_rows<T, DP, kRows>(ds, gt_, 32 * u, v, lane);
                };
                // In fp32 last: what they subtract rounds the sum once then.
                if constexpr (Elem<T>::kPlanes == 3) products();
                const uint4 ls = *reinterpret_cast<const uint4*>(at);
#pragma unroll
                for (int n = 0; n < KB; ++n) s[n] = mma16(ls, minus, s[n]);
                if constexpr (kK) {
                    const uint4 dl = *reinterpret_cast<const uint4*>(at + kRows * kInfoB);
#pragma unroll
                    for (int n = 0; n < KB; ++n) ds[n] = mma16(dl, minus, ds[n]);
                }
                if constexpr (Elem<T>::kPlanes == 1) products();
#pragma unroll
                for (int n = 0; n < KB; ++n)
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        s[n][i] = exp2_fast(s[n][i] * c);
                        if constexpr (kK) ds[n][i] *= s[n][i];
                    }
                if (part) {
#pragma unroll
                    for (int n = 0; n < KB; ++n) {
                        const int key = key0 + 32 * n + (lane & 31);
                        const int q0 = sight.first_query(key), from = q0 - base - 4 * half;
                        const unsigned seen = (unsigned)max(min(sight.last_query(key), last) - q0 + 1, 0);
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            const bool see = (unsigned)(32 * u + acc_row(i, 0) - from) < seen;
                            s[n][i] = see ? s[n][i] : 0.f;
                            ds[n][i] = see ? ds[n][i] : 0.f;
                        }
                    }
                }
                if constexpr (kV) {
                    Probs<T> p[KB];
#pragma unroll
                    for (int n = 0; n < KB; ++n) p[n] = Probs<T>(s[n]);
                    mma_cols<T, DP, kRows>(gv, gt_, 32 * u, p, lane);
                }
                if constexpr (kK) {
                    Probs<T> p[KB];
#pragma unroll
                    for (int n = 0; n < KB; ++n) p[n] = Probs<T>(ds[n]);
                    mma_cols<T, DP, kRows>(gk, qt, 32 * u, p, lane);
                }
            }
        }
        last = next;
        if (kBufs == 1) __syncthreads();
        if (more) finish(other);
        __syncthreads();
    }
    const long long n_kv = (long long)a.B * a.Nk * a.Hkv * a.D;
#pragma unroll
    for (int n = 0; n < KB; ++n) {
        const int key = key0 + 32 * n + (lane & 31);
        if (key >= a.Nk) continue;
        // Keys that no query may see (past the length, dead) have no gradient, whatever their
        // columns summed.
        auto put = [&](const HeadsArg& out, float* part, const f32x16(&acc)[DP / 32], float scale) {
            float* row = part + split * n_kv + (((long long)b * a.Nk + key) * a.Hkv + hk) * a.D;
            G* at = static_cast<G*>(out.data) + b * out.batch + key * out.row + hk * out.head;
#pragma unroll
            for (int d = 0; d < DP / 32; ++d)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int ch = 32 * d + 8 * i + 4 * half;
                    if (ch >= a.D) continue;
                    float x[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[e] = ok[n] ? acc[d][4 * i + e] * scale : 0.f;
                    if (a.row_splits == 1) store4(at + ch, x[0], x[1], x[2], x[3]);
                    else store4(row + ch, x[0], x[1], x[2], x[3]);
                }
        };
        if constexpr (kK) put(a.gk, a.part_kv, gk[n], a.scale);
        if constexpr (kV) put(a.gv, a.part_kv + a.row_splits * n_kv, gv[n], 1.f);
    }
}

// How the workgroups share the keys' and the values' gradients: by keys alone, but by roles too
// where both gradients' accumulators and the keys' and values' operands exceed 256 registers by far.
template <typename T, int DP>
constexpr int kRoles = DP * Elem<T>::kPlanes >= 128 ? 2 : 1;

template <typename T, int DP>
__device__ __forceinline__ void grad_kv_item(const AttendArgs& a, int head, int item, unsigned char* lds) {
    if constexpr (kRoles<T, DP> == 1)
        grad_kv<T, DP, 1, kBoth>(a, head, item, lds);
    else if (item % 2)
        grad_kv<T, DP, 1, kValues>(a, head, item / 2, lds);
    else
        grad_kv<T, DP, 1, kKeysOnly>(a, head, item / 2, lds);
}

// Both kinds of workgroups: the keys' come first, since theirs is the longer walk.
template <typename T, int DP, int RB, bool kAlive>
__global__ __launch_bounds__(kThreads, 2) void attend_grad_kernel(const AttendArgs a, const int row_tiles, const Deal q,
                                                                  const Deal kv, const int kv_blocks) {
    using Sh = KvShape<T, DP, 1>;
    constexpr int kKv = Sh::kBufs * Sh::kBufB, kQ = QShape<T, DP, kAlive>::kLds;
    __shared__ __attribute__((aligned(16))) unsigned char lds[kKv > kQ ? kKv : kQ];
    int head, item;
    if ((int)blockIdx.x < kv_blocks) {
        if (kv.at(blockIdx.x, head, item)) grad_kv_item<T, DP>(a, head, item, lds);
    } else if (q.at(blockIdx.x - kv_blocks, head, item))
        grad_q<T, DP, RB, kAlive>(a, row_tiles, head, item, lds);
}

// One launch for each where the operands of either need more than 256 registers.
template <typename T, int DP, bool kAlive>
__global__ __launch_bounds__(kThreads) void attend_grad_q_kernel(const AttendArgs a, const int row_tiles, const Deal q) {
    __shared__ __attribute__((aligned(16))) unsigned char lds[QShape<T, DP, kAlive>::kLds];
    int head, item;
    if (q.at(blockIdx.x, head, item)) grad_q<T, DP, 1, kAlive>(a, row_tiles, head, item, lds);
}
template <typename T, int DP>
__global__ __launch_bounds__(kThreads, DP == 64 ? 2 : 1) void attend_grad_kv_kernel(const AttendArgs a, const Deal kv) {
    using Sh = KvShape<T, DP, 1>;
    __shared__ __attribute__((aligned(16))) unsigned char lds[Sh::kBufs * Sh::kBufB];
    int head, item;
    if (kv.at(blockIdx.x, head, item)) grad_kv_item<T, DP>(a, head, item, lds);
}

// One gradient that workgroups summed in parts: rows [B][H][N] (head_first) or [B][N][H] of D.
struct Parts {
    const float* part;  // `parts` of them
    HeadsArg out;
    int parts, N, H;
    bool head_first;
    unsigned blocks;  // of this gradient's rows; 0: there are no parts
};

// Up to three gradients, one after another: out = the sum of their parts, in order.
template <typename G>
__global__ __launch_bounds__(kThreads) void sum_parts_kernel(const Parts gq, const Parts gk, const Parts gv, int B,
                                                             int D) {
    const unsigned k0 = gq.blocks, v0 = k0 + gk.blocks, id = blockIdx.x;
    const Parts& p = id < k0 ? gq : id < v0 ? gk : gv;
    const unsigned block = id < k0 ? id : id < v0 ? id - k0 : id - v0;
    const int per = D / 4;
    const long long e = (long long)block * kThreads + threadIdx.x;
    const long long rows = (long long)B * p.N * p.H, row = e / per;
    if (row >= rows) return;
    const int ch = (int)(e % per) * 4;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
    for (int s = 0; s < p.parts; ++s) {
        const float4 x = *reinterpret_cast<const float4*>(p.part + (s * rows + row) * D + ch);
        v.x += x.x;
        v.y += x.y;
        v.z += x.z;
        v.w += x.w;
    }
    const int lo = p.head_first ? p.N : p.H, in = (int)(row % lo);
    const long long up = row / lo;
    const int mid = (int)(up % (p.head_first ? p.H : p.N)), b = (int)(up / (p.head_first ? p.H : p.N));
    const int n = p.head_first ? in : mid, h = p.head_first ? mid : in;
    store4(static_cast<G*>(p.out.data) + b * p.out.batch + n * p.out.row + h * p.out.head + ch, v.x, v.y, v.z, v.w);
}

template <typename T, int DP, bool kAlive>
hipError_t run(const AttendArgs& a, const AttendPlan& p, hipStream_t s) {
    const int row_tiles = (a.Nq * a.group + p.rows - 1) / p.rows, key_tiles = (a.Nk + 127) / 128;
    const Deal q{a.B * a.Hkv, row_tiles * a.splits}, kv{a.B * a.Hkv, key_tiles * a.row_splits * kRoles<T, DP>};
    const int nq = q.blocks(), nkv = kv.blocks();
    const dim3 block(kThreads);
    if (a.Nq > 0) {
        const int lanes = a.D * (int)sizeof(global_t<T>) / 16;
        const long long n = (long long)a.B * a.Hq * a.Nq * lanes;
        hipLaunchKernelGGL(attend_delta_kernel<global_t<T>>, dim3((unsigned)((n + kThreads - 1) / kThreads)), block, 0, s,
                           a, lanes);
    }
    if constexpr (Elem<T>::kPlanes == 3 && DP >= 64) {
        if (nq > 0) hipLaunchKernelGGL((attend_grad_q_kernel<T, DP, kAlive>), dim3(nq), block, 0, s, a, row_tiles, q);
        if (nkv > 0) hipLaunchKernelGGL((attend_grad_kv_kernel<T, DP>), dim3(nkv), block, 0, s, a, kv);
    } else if (p.rows == 128) {
        if (nq + nkv > 0)
            hipLaunchKernelGGL((attend_grad_kernel<T, DP, 1, kAlive>), dim3(nq + nkv), block, 0, s, a, row_tiles, q, kv,
                               nkv);
    } else if constexpr (two_sets(sizeof(global_t<T>), DP)) {
        if (nq + nkv > 0)
            hipLaunchKernelGGL((attend_grad_kernel<T, DP, 2, kAlive>), dim3(nq + nkv), block, 0, s, a, row_tiles, q, kv,
                               nkv);
    } else
        return hipErrorInvalidValue;  // no such plan
    return hipGetLastError();
}
template <typename T>
hipError_t run_t(const AttendArgs& a, const AttendPlan& p, hipStream_t s) {
    if (a.alive)
        return a.D <= 32 ? run<T, 32, true>(a, p, s) : a.D <= 64 ? run<T, 64, true>(a, p, s) : run<T, 128, true>(a, p, s);
    return a.D <= 32 ? run<T, 32, false>(a, p, s) : a.D <= 64 ? run<T, 64, false>(a, p, s) : run<T, 128, false>(a, p, s);
}

constexpr int kSplits[] = {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64, 96, 128, 192, 256};
constexpr int kMostSplits = sizeof(kSplits) / sizeof(kSplits[0]);

// The workgroups of one kind (queries' or keys'), for each number of splits that leaves a walk two
// tiles: the time that they take together and that of the longest, in products of a tile of 128 rows by
// 64, where a workgroup starts and ends in the time of four; and the rows of fp32 parts, in thousands.
struct Walks {
    double all[kMostSplits], longest[kMostSplits], parts[kMostSplits];
    int n;
    // `products` a tile of the `side` that it walks, of which it sees at most `span`; `rows` of `sums`
    // gradients; `slots` workgroups are resident at once.
    Walks(double workgroups, double slots, double products, long long side, long long span, bool causal, double rows,
          int sums) {
        constexpr double kStart = 4.0;
        const bool cut = span < side;
        const double tiles = (double)(((cut ? span : side) + 63) / 64), mean = causal && !cut ? tiles / 2 : tiles;
        for (n = 0; n < kMostSplits && (n == 0 || 2LL * kSplits[n] <= (side + 63) / 64); ++n) {
            const int s = kSplits[n];
            all[n] = workgroups * (s * kStart + products * mean) / slots;
            longest[n] = kStart + products * tiles / s;
            parts[n] = s > 1 ? 1e-3 * rows * sums * s : 0.0;
        }
    }
};

int padded(int D) { return D <= 32 ? 32 : D <= 64 ? 64 : 128; }
int roles_of(int dtype, int D) { return padded(D) * (dtype == 1 ? 1 : 3) >= 128 ? 2 : 1; }  // kRoles

}  // namespace

AttendPlan attend_grad_plan(int dtype, const AttendArgs& a, int n_cu) {
    AttendPlan p;
    const long long rows = (long long)a.Nq * a.group, heads = (long long)a.B * a.Hkv;
    p.rows = two_sets(dtype == 1 ? 2 : 4, a.D) && heads * ((rows + 255) / 256) >= 2LL * n_cu ? 256 : 128;
    // Of the splits that leave each walk two tiles, those with the fewest parts among the ones whose
    // time above is within a fiftieth of the least. Against splits of each kind by itself, to one or two
    // workgroups a CU, us: in bf16 2 x 2048 x 8 x 128 191 -> 179, 1000, 8 over 2 heads of 128, 72 -> 44,
    // 4096 causal, 8 over 2 heads of 64, 132 -> 94; in fp32 2 x 600 x 8 x 64 84 -> 75. Over 82 calls of
    // 51 to 6144 rows and heads of 32 to 128: 12 % less time, 3 % above the best splits of each call.
    const int planes = dtype == 1 ? 1 : 3, dp = padded(a.D), roles = roles_of(dtype, a.D);
    const bool cut = a.window > 0, one_launch = planes == 1 || dp == 32;
    const double slots_q = (one_launch ? 2.0 : 1.0) * n_cu, slots_kv = (one_launch || dp == 64 ? 2.0 : 1.0) * n_cu;
    const long long seen = a.window * (a.causal ? 1LL : 2LL);
    const Walks q((double)heads * ((rows + p.rows - 1) / p.rows), slots_q, 3.0 * (p.rows / 128), a.Nk,
                  cut ? seen + p.rows / a.group : a.Nk, a.causal, (double)heads * rows, 1);
    const Walks kv((double)heads * ((a.Nk + 127) / 128) * roles, slots_kv, roles == 2 ? 2.5 : 4.0, rows,
                   cut ? (seen + 128) * a.group : rows, a.causal, (double)heads * a.Nk, 2);
    // The time of a call, in the same products. In one launch the queries' workgroups come last: a quarter
    // of their longest is a gap at the end, or else 0.15 of the keys' longest; a launch of its own ends in
    // a quarter of its longest. Parts are then written, read and summed: a tenth of a product a thousand
    // rows (a product in fp32 takes three times as long beside them), and four for the launch.
    auto time_of = [&](int i, int j) {
        const double lq = q.longest[i], lkv = kv.longest[j], parts = q.parts[i] + kv.parts[j];
        const double t = one_launch ? fmax(fmax(lq, lkv), q.all[i] + kv.all[j] + fmax(0.25 * lq, 0.15 * lkv))
                                    : fmax(lq, q.all[i] + 0.25 * lq) + fmax(lkv, kv.all[j] + 0.25 * lkv);
        return t + 0.1 * parts / planes + (parts > 0 ? 4.0 : 0.0);
    };
    double least = INFINITY, fewest = INFINITY;
    for (int i = 0; i < q.n; ++i)
        for (int j = 0; j < kv.n; ++j) least = fmin(least, time_of(i, j));
    p.splits = p.row_splits = 1;
    for (int i = 0; i < q.n; ++i)
        for (int j = 0; j < kv.n; ++j)
            if (q.parts[i] + kv.parts[j] < fewest && time_of(i, j) <= 1.02 * least) {
                fewest = q.parts[i] + kv.parts[j];
                p.splits = kSplits[i];
                p.row_splits = kSplits[j];
            }
    return p;
}

double attend_grad_workgroups(int dtype, const AttendArgs& a, const AttendPlan& p) {
    const double heads = (double)a.B * a.Hkv, rows = (double)a.Nq * a.group;
    const double delta = ceil(heads * rows * (a.D * (dtype == 1 ? 2 : 4) / 16) / kThreads);
    const double walks = heads * (ceil(rows / p.rows) * p.splits + ceil(a.Nk / 128.0) * p.row_splits * roles_of(dtype, a.D)) + 16;
    const double sums = heads * ((p.splits > 1 ? rows : 0.0) + (p.row_splits > 1 ? 2.0 * a.Nk : 0.0)) * (a.D / 4) / kThreads + 3;
    return fmax(delta, fmax(walks, sums));
}

template <typename G>
static hipError_t sum_t(const AttendArgs& a, hipStream_t s) {
    auto blocks = [&](long long rows) { return (unsigned)((rows * (a.D / 4) + kThreads - 1) / kThreads); };
    const long long q = (long long)a.B * a.Hq * a.Nq, k = (long long)a.B * a.Hkv * a.Nk;
    const Parts gq{a.part, a.gq, a.splits, a.Nq, a.Hq, true, a.splits > 1 ? blocks(q) : 0};
    const Parts gk{a.part_kv, a.gk, a.row_splits, a.Nk, a.Hkv, false, a.row_splits > 1 ? blocks(k) : 0};
    Parts gv = gk;
    gv.part += a.row_splits * k * a.D;
    gv.out = a.gv;
    const unsigned n = gq.blocks + gk.blocks + gv.blocks;
    if (n > 0) hipLaunchKernelGGL(sum_parts_kernel<G>, dim3(n), dim3(kThreads), 0, s, gq, gk, gv, a.B, a.D);
    return hipGetLastError();
}
hipError_t launch_attend_grad(int dtype, const AttendArgs& a, const AttendPlan& p, hipStream_t s) {
    const hipError_t e = dtype == 1 ? run_t<bf16_t>(a, p, s) : run_t<split_t>(a, p, s);
    if (e != hipSuccess) return e;
    return dtype == 1 ? sum_t<bf16_t>(a, s) : sum_t<float>(a, s);
}

}  // namespace slime
