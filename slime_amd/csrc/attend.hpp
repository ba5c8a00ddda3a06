// attend.hpp — what the attention kernels share: the tile of rows in LDS and the matrix
// products on it, which keys a query sees, and the walk over the work.
//
// Every product is v_mfma_f32_32x32x16_bf16, or v_mfma_f32_32x32x2_f32 where few rows meet many
// keys in fp32. Of its result a lane holds column n = lane % 32 and, in register i, row
// acc_row(i, lane / 32); as an operand it holds 16 bytes of one row or column. The k index of a
// product may be permuted if both operands agree, so the result of one product is the next
// one's operand as it lies in the registers: scores become probabilities and enter the next
// product without passing through LDS.
//
// "Rows" are queries of one key head: the group = Hq / Hkv query heads that share it are
// packed, row r is query r / group of head r % group, so a key tile is staged once for the
// whole group, and the group's gradients of keys and values are summed by the products.
#pragma once

#include <type_traits>

#include "attend_walk.hpp"
#include "common.hpp"
#include "kernels.hpp"

namespace slime {
namespace at {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr float kLog2e = 1.4426950408889634f;

// ---- 16 bytes of a row, at any element's address ------------------------------------------
// (gfx950 takes global accesses of any alignment; the compiler emits one wide access.)
template <typename T>
__device__ __forceinline__ uint4 load16(const T* p) {
    uint4 v;
    __builtin_memcpy(&v, p, 16);
    return v;
}
template <typename T>
__device__ __forceinline__ void store4(T* p, float a, float b, float c, float d) {
    if constexpr (sizeof(T) == 2) {
        const uint2 v = make_uint2(pack_bf16x2(a, b), pack_bf16x2(c, d));
        __builtin_memcpy(p, &v, 8);
    } else {
        const float4 v = make_float4(a, b, c, d);
        __builtin_memcpy(p, &v, 16);
    }
}

// This lane's value and the other half of the wave's (lane ^ 32), as (lane % 32's, the other's).
__device__ __forceinline__ float2 both(float x) {
    const unsigned v = __builtin_bit_cast(unsigned, x);
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    const unsigned a = r[0], b = r[1];
    return make_float2(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b));
}
__device__ __forceinline__ float both_max(float x) {
    const float2 v = both(x);
    return fmaxf(v.x, v.y);
}
__device__ __forceinline__ float both_sum(float x) {
    const float2 v = both(x);
    return v.x + v.y;
}

// Row of result register i in half h of the wave.
__device__ __forceinline__ constexpr int acc_row(int i, int h) { return 8 * (i / 4) + 4 * h + i % 4; }

// ---- how elements enter the products -----------------------------------------------------------
// bf16 as they are. fp32 either as they are (float), or (split_t) each as the sum of three bf16
// parts, hi + mid + lo, each the rest rounded to nearest: 3 x 8 bits hold all 24. A product of
// two is then six bf16 products, hi hi, hi mid, mid hi, mid mid, hi lo, lo hi; what is left out
// is below 2^-24 of it. Six of 32 cycles a 16 channels take 0.4 of the time of the eight fp32
// products of 64 cycles in their place. (A value that rounds to no finite bf16, above 3.39e38,
// gives NaN.)
struct split_t;
template <typename T>
struct Elem {
    using G = T;  // in global memory
    static constexpr int kBytes = sizeof(T), kPlanes = 1;
};
template <>
struct Elem<split_t> {
    using G = float;
    static constexpr int kBytes = 2, kPlanes = 3;
};
template <typename T>
using global_t = typename Elem<T>::G;
template <typename T>
constexpr bool kBf16Products = Elem<T>::kBytes == 2;

// One lane's operand: 16 bytes of a row or column, of each part.
template <typename T>
struct Op {
    uint4 p[Elem<T>::kPlanes];
};

// Eight values' parts: the bf16 pairs hi[4], mid[4], lo[4].
__device__ __forceinline__ Op<split_t> split8(const float (&x)[8]) {
    unsigned w[3][4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        float a = x[2 * e], b = x[2 * e + 1];
#pragma unroll
        for (int p = 0; p < 3; ++p) {
            w[p][e] = pack_bf16x2(a, b);
            a -= bf16lo(w[p][e]);
            b -= bf16hi(w[p][e]);
        }
    }
    Op<split_t> o;
#pragma unroll
    for (int p = 0; p < 3; ++p) o.p[p] = make_uint4(w[p][0], w[p][1], w[p][2], w[p][3]);
    return o;
}
__device__ __forceinline__ Op<split_t> split8(uint4 lo, uint4 hi) {
    const f32x4 a = __builtin_bit_cast(f32x4, lo), b = __builtin_bit_cast(f32x4, hi);
    const float x[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    return split8(x);
}

// ---- a tile of R rows x DP channels in LDS -------------------------------------------------
// Rows of DP elements (head dims below DP are padded with zeros), their chunks swizzled;
// split_t: three such tiles one after another.
template <typename T, int DP, int R>
struct Tile : Swizzle<DP * Elem<T>::kBytes> {
    static constexpr int kRowB = DP * Elem<T>::kBytes;
    using Swizzle<kRowB>::kChunks;
    using Swizzle<kRowB>::at;
    static constexpr int kSteps = kChunks / 2;  // products of 16 bytes a lane along a row
    static constexpr int kPlaneB = R * kRowB, kBytes = Elem<T>::kPlanes * kPlaneB;

    // Operand of a product along the channels: 16 bytes of row r0 + lane % 32.
    __device__ static __forceinline__ Op<T> row_frag(const unsigned char* t, int r0, int step, int lane) {
        Op<T> f;
#pragma unroll
        for (int p = 0; p < Elem<T>::kPlanes; ++p)
            f.p[p] = *reinterpret_cast<const uint4*>(t + p * kPlaneB + at(r0 + (lane & 31), 2 * step + (lane >> 5)));
        return f;
    }
};
// Operands along a row's channels.
template <typename T, int DP>
constexpr int kRowSteps = Tile<T, DP, 32>::kSteps;

typedef short v4i16 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4i16 lds_v4i16;

// ds_read_b64_tr_b16: in each 16-lane group, lane i receives element i % 4 of the 8 bytes
// that lanes i / 4, 4 + i / 4, 8 + i / 4 and 12 + i / 4 address (in that order).
__device__ __forceinline__ uint2 read_tr16(const unsigned char* p) {
    const v4i16 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (lds_v4i16*)(const __attribute__((address_space(3))) unsigned char*)(p));
    return __builtin_bit_cast(uint2, v);
}

__device__ __forceinline__ f32x16 mma16(uint4 a, uint4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_v, a), __builtin_bit_cast(bf16x8_v, b), c,
                                                   0, 0, 0);
}
__device__ __forceinline__ f32x16 mma(const Op<bf16_t>& a, const Op<bf16_t>& b, f32x16 c) {
    return mma16(a.p[0], b.p[0], c);
}
__device__ __forceinline__ f32x16 mma(const Op<split_t>& a, const Op<split_t>& b, f32x16 c) {
    c = mma16(a.p[0], b.p[2], c);
    c = mma16(a.p[2], b.p[0], c);
    c = mma16(a.p[1], b.p[1], c);
    c = mma16(a.p[0], b.p[1], c);
    c = mma16(a.p[1], b.p[0], c);
    return mma16(a.p[0], b.p[0], c);
}
__device__ __forceinline__ f32x16 mma(const Op<float>& a, const Op<float>& b, f32x16 c) {
    const f32x4 x = __builtin_bit_cast(f32x4, a.p[0]), y = __builtin_bit_cast(f32x4, b.p[0]);
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(x[e], y[e], c, 0, 0, 0);
    return c;
}

__device__ __forceinline__ f32x16 zeros16() {
    f32x16 c;
#pragma unroll
    for (int i = 0; i < 16; ++i) c[i] = 0.f;
    return c;
}

// The 32 x 32 blocks of a product of tile rows r0 .. r0 + 31 (rows of the results) with N
// sets of 32 rows held as operands b (their columns), along the channels, onto c.
template <typename T, int DP, int R, int N>
__device__ __forceinline__ void mma_rows(f32x16 (&c)[N], const unsigned char* t, int r0,
                                         const Op<T> (&b)[N][kRowSteps<T, DP>], int lane) {
#pragma unroll
    for (int s = 0; s < kRowSteps<T, DP>; ++s) {
        const Op<T> f = Tile<T, DP, R>::row_frag(t, r0, s, lane);
#pragma unroll
        for (int n = 0; n < N; ++n) c[n] = mma(f, b[n][s], c[n]);
    }
}

// A 32 x 32 result as the operand of the next product along its rows: bf16 pairs (rounded to
// nearest, at most 2^-8 of each probability: the type its product's other operand has), their
// parts, or fp32.
template <typename T>
struct Probs {
    Op<T> v[2];
    __device__ __forceinline__ Probs() {}
    __device__ __forceinline__ explicit Probs(const f32x16& p) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const float x[8] = {p[8 * t],     p[8 * t + 1], p[8 * t + 2], p[8 * t + 3],
                                p[8 * t + 4], p[8 * t + 5], p[8 * t + 6], p[8 * t + 7]};
            if constexpr (Elem<T>::kPlanes == 3)
                v[t] = split8(x);
            else
                v[t].p[0] = make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]),
                                       pack_bf16x2(x[6], x[7]));
        }
    }
};
template <>
struct Probs<float> {
    f32x16 v;
    __device__ __forceinline__ Probs() {}
    __device__ __forceinline__ explicit Probs(const f32x16& p) : v(p) {}
};
// bf16 pairs with what their rounding left, rounded too: at most 2^-16 of each probability, for a
// second product and five instructions a pair.
struct ProbsInTwo {
    Probs<bf16_t> hi, lo;
    __device__ __forceinline__ explicit ProbsInTwo(const f32x16& p) : hi(p) {
        f32x16 rest;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const uint4& h = hi.v[t].p[0];
            const unsigned w[4] = {h.x, h.y, h.z, h.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                rest[8 * t + 2 * e] = p[8 * t + 2 * e] - bf16lo(w[e]);
                rest[8 * t + 2 * e + 1] = p[8 * t + 2 * e + 1] - bf16hi(w[e]);
            }
        }
        lo = Probs<bf16_t>(rest);
    }
};
template <typename T>
__device__ __forceinline__ f32x16 mma_probs(const Op<T>& a, const Probs<T>& p, int s, f32x16 c) {
    return mma(a, p.v[s], c);
}
__device__ __forceinline__ f32x16 mma_probs(const Op<bf16_t>& a, const ProbsInTwo& p, int s, f32x16 c) {
    return mma(a, p.hi.v[s], mma(a, p.lo.v[s], c));
}

// acc[n][d][.] += sum over tile rows r0 .. r0 + 31 of tile[row][d] p[n][row][.], in blocks of 32
// channels d. The tile is read along its columns: transposing reads (bf16), or one element
// of 32 consecutive channels (fp32).
template <typename T, int DP, int R, typename P, int N>
__device__ __forceinline__ void mma_cols(f32x16 (&acc)[N][DP / 32], const unsigned char* t, int r0,
                                         const P (&p)[N], int lane) {
    using Tl = Tile<T, DP, R>;
    const int half = lane >> 5;
    if constexpr (kBf16Products<T>) {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            // k = 0..3 of the lane's eight: rows r0 + 16 s + 4 half + 0..3; k = 4..7: 8 rows on
            const int ra = r0 + 16 * s + 4 * half + ((lane & 15) >> 2), rb = ra + 8;
            const int col = ((lane >> 4) & 1) * 16 + (lane & 3) * 4;
#pragma unroll
            for (int b = 0; b < DP / 32; ++b) {
                const int c = (32 * b + col) >> 3, off = (col & 4) << 1;
                Op<T> f;
#pragma unroll
                for (int q = 0; q < Elem<T>::kPlanes; ++q) {
                    const uint2 x = read_tr16(t + q * Tl::kPlaneB + Tl::at(ra, c) + off);
                    const uint2 y = read_tr16(t + q * Tl::kPlaneB + Tl::at(rb, c) + off);
                    f.p[q] = make_uint4(x.x, x.y, y.x, y.y);
                }
#pragma unroll
                for (int n = 0; n < N; ++n) acc[n][b] = mma_probs(f, p[n], s, acc[n][b]);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int r = r0 + acc_row(i, half);
#pragma unroll
            for (int b = 0; b < DP / 32; ++b) {
                const int d = 32 * b + (lane & 31);
                const float x = *reinterpret_cast<const float*>(t + Tl::at(r, d >> 2) + ((d & 3) << 2));
#pragma unroll
                for (int n = 0; n < N; ++n)
                    acc[n][b] = __builtin_amdgcn_mfma_f32_32x32x2f32(x, p[n].v[i], acc[n][b], 0, 0, 0);
            }
        }
    }
}

// ---- staging a tile from global memory ---------------------------------------------------------
// Rows of one head: row i at base + i * row_b bytes.
struct Rows {
    const unsigned char* base;
    long long row_b;
    bool direct;  // rows of 16-byte chunks, at most 2^24 bytes apart
    template <typename T>
    __device__ __forceinline__ Rows(const T* p, long long row)
        : base(reinterpret_cast<const unsigned char*>(p)), row_b(row * (long long)sizeof(T)) {
        direct = (((unsigned long long)base | (unsigned long long)row_b) & 15) == 0 &&
                 (unsigned long long)row_b < 1u << 24;
    }
};

// An address that every lane of the wave has alike, in scalar registers that vector instructions
// may have written just before.
__device__ __forceinline__ const unsigned char* uniform(const unsigned char* p) {
    const unsigned long long v = reinterpret_cast<unsigned long long>(p);
    const unsigned lo = __builtin_amdgcn_readfirstlane((unsigned)v), hi = __builtin_amdgcn_readfirstlane((unsigned)(v >> 32));
    return reinterpret_cast<const unsigned char*>((unsigned long long)hi << 32 | lo);
}

// kRows rows of one head into a tile in LDS. Rows of whole 16-byte chunks go there directly
// (global_load_lds: no registers between, so a tile can be under way while another is
// multiplied): the 64 chunks of an instruction lie one after another in LDS, so each lane
// fetches the chunk whose place it fills. A tile of n < kRows rows repeats its last one, which
// no kernel uses (its scores are masked); channels from D on stay the zeros that clear_pad wrote.
// Other rows pass through registers, and rows from n on become zeros. What is split waits in
// registers between issue and finish.
template <typename T, int DP, int kRows, int kThr = kThreads>
struct Stage : Fill<Tile<T, DP, kRows>::kRowB, kRows, kThr> {
    using Tl = Tile<T, DP, kRows>;
    using G = global_t<T>;
    using F = Fill<Tl::kRowB, kRows, kThr>;
    using F::chunk;
    using F::kN;
    using F::kPass;
    using F::place;
    using F::row;
    static constexpr bool kSplit = Elem<T>::kPlanes == 3;
    static constexpr int kElems = 16 / Elem<T>::kBytes, kGlobalB = kElems * (int)sizeof(G);  // of a chunk
    static_assert(kRows <= 128, "offsets of rows 2^24 bytes apart fit 32 bits");
    uint4 v[kSplit ? kN : 1][2];

    // The n rows from `first` on (n >= 1; n >= kRows: a whole tile). Complete for the workgroup
    // after wait_vm0, finish and a barrier.
    __device__ __forceinline__ void issue(unsigned char* tile, const Rows& s, int first, int n, int D, int tid) {
        const unsigned char* p = s.base + first * s.row_b;
        if (s.direct && n >= kRows && D == DP) {
            const unsigned at = lds_addr(tile) + 16 * __builtin_amdgcn_readfirstlane(tid & ~63);
#pragma unroll
            for (int i = 0; i < kN; ++i) {
                const unsigned char* q = uniform(p + i * kPass * s.row_b);
                const unsigned off = (unsigned)row(0, tid) * (unsigned)s.row_b + (unsigned)(kGlobalB * chunk(i, tid));
                if constexpr (kSplit) {
                    v[i][0] = load16(q + off);
                    v[i][1] = load16(q + off + 16);
                } else
                    dma16_lds_v(q, off, at + 16 * i * kThr);
            }
        } else if (!kSplit && s.direct) {
            const unsigned at = lds_addr(tile) + 16 * __builtin_amdgcn_readfirstlane(tid & ~63);
#pragma unroll
            for (int i = 0; i < kN; ++i) {
                const unsigned off =
                    (unsigned)min(row(i, tid), n - 1) * (unsigned)s.row_b + (unsigned)(kGlobalB * chunk(i, tid));
                if (chunk(i, tid) * kElems < D) dma16_lds_v(uniform(p), off, at + 16 * i * kThr);
            }
        } else {
            uint4 w[kN];
#pragma unroll
            for (int i = 0; i < kN; ++i) {
                const int c = chunk(i, tid);
                const bool in = row(i, tid) < n && c * kElems < D;
                const unsigned char* q = p + row(i, tid) * s.row_b + kGlobalB * c;
                if constexpr (kSplit) {
                    v[i][0] = v[i][1] = make_uint4(0, 0, 0, 0);
                    if (in) {
                        v[i][0] = load16(q);
                        v[i][1] = load16(q + 16);
                    }
                } else {
                    w[i] = make_uint4(0, 0, 0, 0);
                    if (in) w[i] = load16(q);
                }
            }
            if constexpr (!kSplit) {
#pragma unroll
                for (int i = 0; i < kN; ++i) *reinterpret_cast<uint4*>(tile + place(i, tid)) = w[i];
            }
        }
    }
    // Zeros in the channels from D on of a tile that direct loads will fill: once, before the first.
    static __device__ __forceinline__ void clear_pad(unsigned char* tile, int D, int tid) {
        if (kSplit || D == DP) return;
#pragma unroll
        for (int i = 0; i < kN; ++i)
            if (chunk(i, tid) * kElems >= D) *reinterpret_cast<uint4*>(tile + place(i, tid)) = make_uint4(0, 0, 0, 0);
    }
    // Zeros for chunk i, after wait_vm0.
    __device__ __forceinline__ void clear(unsigned char* tile, int i, int tid) {
        if constexpr (kSplit)
            v[i][0] = v[i][1] = make_uint4(0, 0, 0, 0);
        else
            *reinterpret_cast<uint4*>(tile + place(i, tid)) = make_uint4(0, 0, 0, 0);
    }
    __device__ __forceinline__ void finish(unsigned char* tile, int tid) const {
        if constexpr (kSplit) {
#pragma unroll
            for (int i = 0; i < kN; ++i) {
                const Op<split_t> o = split8(v[i][0], v[i][1]);
#pragma unroll
                for (int q = 0; q < 3; ++q)
                    *reinterpret_cast<uint4*>(tile + q * Tl::kPlaneB + place(i, tid)) = o.p[q];
            }
        }
    }
};

// This half's 16-byte chunks of a row of D channels in global memory: all of them on their way
// before any is used.
template <typename T, int DP>
struct RowChunks {
    using G = global_t<T>;
    static constexpr int kSteps = kRowSteps<T, DP>, kElems = 16 / Elem<T>::kBytes;
    static constexpr int kN = (int)sizeof(G) / Elem<T>::kBytes;  // chunks of an operand
    uint4 v[kSteps][kN];
    __device__ __forceinline__ RowChunks(const G* row, int D, int half) {
#pragma unroll
        for (int s = 0; s < kSteps; ++s)
#pragma unroll
            for (int n = 0; n < kN; ++n) {
                const int c = (2 * s + half) * kElems;
                v[s][n] = make_uint4(0, 0, 0, 0);
                if (D == DP || c < D) v[s][n] = load16(row + c + n * (16 / (int)sizeof(G)));
            }
    }
};

// One row as operands, from global memory (zeros from D on, or all where !keep).
template <typename T, int DP>
__device__ __forceinline__ void load_frags(const global_t<T>* row, bool keep, int D, int half,
                                           Op<T> (&f)[kRowSteps<T, DP>]) {
    RowChunks<T, DP> x(row, D, half);
#pragma unroll
    for (int s = 0; s < kRowSteps<T, DP>; ++s) {
#pragma unroll
        for (int n = 0; n < x.kN; ++n)
            if (!keep) x.v[s][n] = make_uint4(0, 0, 0, 0);
        if constexpr (Elem<T>::kPlanes == 3)
            f[s] = split8(x.v[s][0], x.v[s][1]);
        else
            f[s].p[0] = x.v[s][0];
    }
}

// ---- which keys a query sees ---------------------------------------------------------------------
struct Sight : SightOf {
    __device__ __forceinline__ Sight(const AttendArgs& a, int b) {
        len = a.Nk;
        if (a.lengths) len = min(max(__builtin_amdgcn_readfirstlane(a.lengths[b]), 0), a.Nk);
        shift = a.align_start ? 0 : len - a.Nq;
        causal = a.causal;
        window = a.window;
    }
};

// The workgroup's rows and the keys that they see. Both bounds grow with the query, so the
// first row's lower and the last row's upper bound hold for all rows between.
struct Span {
    int lo, hi;          // some row sees a key of lo .. hi
    int all_lo, all_hi;  // every row sees the keys of all_lo .. all_hi
    __device__ __forceinline__ Span(const Sight& s, int row0, int row1, int R, int group) {
        const int first = min(row0, R - 1) / group, last = min(row1, R - 1) / group;
        lo = __builtin_amdgcn_readfirstlane(s.lo(first));
        hi = __builtin_amdgcn_readfirstlane(s.hi(last));
        all_lo = __builtin_amdgcn_readfirstlane(s.lo(last));
        all_hi = __builtin_amdgcn_readfirstlane(s.hi(first));
    }
};

// A tile of kKeys keys, or of their values, on its way to LDS. Of dead cells (kAlive) the rows
// become zeros, and a 0 or -inf per key, that the scores start from, follows the tile.
template <typename T, int DP, int kKeys, bool kAlive>
struct KeyTile {
    using St = Stage<T, DP, kKeys>;
    static constexpr int kTileB = St::Tl::kBytes;
    static constexpr int kBytes = kTileB + (kAlive ? kKeys * 4 : 0);
    St st;
    unsigned live[kAlive ? St::kN : 1], key;
    // The n keys from k0 on (n >= kKeys: a whole tile), on their way to buf.
    __device__ __forceinline__ void issue(unsigned char* buf, const Rows& rows, const uint8_t* alive, int k0, int n,
                                          int D, int tid) {
        if constexpr (kAlive) {
            key = tid < kKeys && tid < n ? alive[k0 + tid] : 0;
#pragma unroll
            for (int i = 0; i < St::kN; ++i) {
                const int r = St::row(i, tid);
                live[i] = r < n ? alive[k0 + r] : 0;
            }
        }
        st.issue(buf, rows, k0, n, D, tid);
    }
    // Of the same buf, once this wave's loads are there (wait_vm0): a barrier away from use.
    __device__ __forceinline__ void finish(unsigned char* buf, int tid) {
        if constexpr (kAlive) {
            // Used here and not before: the compiler would wait for them, and with them for the
            // tile's loads, as soon as they are issued.
            asm volatile("" : "+v"(key));
#pragma unroll
            for (int i = 0; i < St::kN; ++i) asm volatile("" : "+v"(live[i]));
#pragma unroll
            for (int i = 0; i < St::kN; ++i)
                if (!live[i]) st.clear(buf, i, tid);
            if (tid < kKeys) reinterpret_cast<float*>(buf + kTileB)[tid] = key ? 0.f : -INFINITY;
        }
        st.finish(buf, tid);
    }
};

// Scores of N sets of 32 rows over the 32 keys from r0 of a tile of R keys in LDS, started
// (kAlive) from the keys' bias that follows the tile.
template <typename T, int DP, int R, bool kAlive, int N>
__device__ __forceinline__ void scores(f32x16 (&s)[N], const unsigned char* kt, int r0,
                                       const Op<T> (&q)[N][kRowSteps<T, DP>], int lane) {
    if constexpr (kAlive) {
        const float* bias = reinterpret_cast<const float*>(kt + Tile<T, DP, R>::kBytes) + r0 + 4 * (lane >> 5);
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const f32x4 x = *reinterpret_cast<const f32x4*>(bias + 8 * g);
#pragma unroll
            for (int n = 0; n < N; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[n][4 * g + e] = x[e];
        }
    } else {
#pragma unroll
        for (int n = 0; n < N; ++n) s[n] = zeros16();
    }
    mma_rows<T, DP, R>(s, kt, r0, q, lane);
}

// Buffers of 64 keys and their values: two, but one for three parts of 64 channels or more, which
// then wait in registers for the products on the tile before.
template <typename T, int DP>
constexpr int key_bufs() {
    return Elem<T>::kPlanes == 3 && DP >= 64 ? 1 : 2;
}

// Waves of 64 rows, whose accumulators and scores fit 256 registers, where there are workgroups
// enough: every tile that a wave reads from LDS serves twice the rows.
constexpr bool two_sets(size_t bytes, int D) { return bytes == 2 && D <= 64; }

// Waits for operands here, before a loop that loads tiles: else the loop's first use of them
// waits for every load under way, at each of its turns.
template <typename T, int N, int S>
__device__ __forceinline__ void settle(Op<T> (&f)[N][S]) {
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
        for (int s = 0; s < S; ++s)
#pragma unroll
            for (int q = 0; q < Elem<T>::kPlanes; ++q) {
                uint4& x = f[n][s].p[q];
                asm volatile("" : "+v"(x.x), "+v"(x.y), "+v"(x.z), "+v"(x.w));
            }
}

}  // namespace at
}  // namespace slime
