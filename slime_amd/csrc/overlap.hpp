// overlap.hpp — whether two strided tensors share a byte of memory.
//
// Plain C++: binding.cpp refuses outputs that lie in an input, and a host program checks the
// answers against a list of all bytes (tests/overlap_check.cpp).
#pragma once

namespace slime {

// A tensor's bytes: runs of `run` bytes at at + sum of i_d stride_d, 0 <= i_d < size_d.
struct Region {
    static constexpr int kDims = 4;
    long long at, run;
    int dims;
    long long size[kDims], stride[kDims];  // strides >= 0, in bytes
    bool empty() const {
        for (int d = 0; d < dims; ++d)
            if (size[d] == 0) return true;
        return false;
    }
};

// The distance of a run of one from a run of the other is a sum of c_t step_t, each c_t in a range of
// whole numbers; equal steps of both are one. From the largest step on, only those c_t are
// tried that the smaller steps can still bring to a distance that overlaps: one or two each
// where steps nest, as views of one allocation's do. Steps that do not nest may need more
// trials than kTrials, and count as an overlap then.
class Overlap {
    static constexpr int kMost = 2 * Region::kDims, kTrials = 100000;
    long long step[kMost], lo[kMost], hi[kMost];
    long long rest_lo[kMost + 1], rest_hi[kMost + 1];  // of the steps from t on
    int n = 0, trials = 0;
    long long below, above;  // a distance overlaps if below < it < above

    void add(long long s, long long from, long long to) {
        if (s == 0 || from == to) return;
        int t = 0;
        while (t < n && step[t] > s) ++t;
        if (t == n || step[t] != s) {
            for (int i = n++; i > t; --i) {
                step[i] = step[i - 1];
                lo[i] = lo[i - 1];
                hi[i] = hi[i - 1];
            }
            step[t] = s;
            lo[t] = hi[t] = 0;
        }
        lo[t] += from;
        hi[t] += to;
    }
    static long long floor_div(long long a, long long b) { return a >= 0 ? a / b : -((-a + b - 1) / b); }
    bool some(int t, long long x) {
        if (x + rest_hi[t] <= below || x + rest_lo[t] >= above) return false;
        if (t == n) return true;
        // below < x + c step + (what the rest adds) < above
        long long c = floor_div(below - rest_hi[t + 1] - x, step[t]) + 1;
        long long last = -floor_div(-(above - rest_lo[t + 1] - x), step[t]) - 1;
        if (c < lo[t]) c = lo[t];
        if (last > hi[t]) last = hi[t];
        for (; c <= last; ++c) {
            if (++trials > kTrials) return true;
            if (some(t + 1, x + c * step[t])) return true;
        }
        return false;
    }
    // Dimensions that lie run to run are part of the run.
    static Region folded(Region r) {
        for (int d = 0; d < r.dims; ++d)
            if (r.size[d] > 1 && r.stride[d] == r.run) {
                r.run *= r.size[d];
                r.size[d] = 1;
                d = -1;
            }
        return r;
    }

public:
    static bool of(const Region& p, const Region& q) {
        if (p.empty() || q.empty()) return false;
        const Region a = folded(p), b = folded(q);
        Overlap o;
        o.below = -b.run;
        o.above = a.run;
        for (int d = 0; d < a.dims; ++d) o.add(a.stride[d], 1 - a.size[d], 0);
        for (int d = 0; d < b.dims; ++d) o.add(b.stride[d], 0, b.size[d] - 1);
        o.rest_lo[o.n] = o.rest_hi[o.n] = 0;
        for (int t = o.n - 1; t >= 0; --t) {
            o.rest_lo[t] = o.rest_lo[t + 1] + o.lo[t] * o.step[t];
            o.rest_hi[t] = o.rest_hi[t + 1] + o.hi[t] * o.step[t];
        }
        return o.some(0, b.at - a.at);
    }
};

}  // namespace slime
