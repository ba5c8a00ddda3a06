// Host check of slime_amd/csrc/overlap.hpp: random views against a list of all their bytes, and the
// views that callers have, at sizes that no list could hold.
//
// -DPLANT_OVERLAP: a mistake in what is expected, which the check must report.
#include "../slime_amd/csrc/overlap.hpp"

#include <cstdio>
#include <random>
#include <vector>

using namespace slime;

namespace {

int errors = 0;
void expect(bool got, bool want, const char* what, long long n) {
    if (got != want && ++errors < 9) std::printf("%s %lld: %d, expected %d\n", what, n, got, want);
}

void mark(const Region& r, int d, long long at, std::vector<char>& bytes) {
    if (d == r.dims) {
        for (long long i = 0; i < r.run; ++i) bytes[at + i] = 1;
        return;
    }
    for (long long i = 0; i < r.size[d]; ++i) mark(r, d + 1, at + i * r.stride[d], bytes);
}

bool listed(const Region& a, const Region& b) {
    std::vector<char> x(100000, 0), y(100000, 0);
    mark(a, 0, a.at, x);
    mark(b, 0, b.at, y);
    for (size_t i = 0; i < x.size(); ++i)
        if (x[i] && y[i]) return true;
    return false;
}

}  // namespace

int main() {
    std::mt19937 rng(1);
    auto pick = [&](int n) { return (long long)(rng() % n); };
    int both = 0, none = 0;
    for (int i = 0; i < 20000; ++i) {
        Region r[2];
        const long long common[3] = {8 + pick(40), 40 + pick(200), 300 + pick(900)};
        for (Region& x : r) {
            x.at = pick(3000);
            x.run = 1LL << pick(4);
            x.dims = (int)pick(4) + 1;
            for (int d = 0; d < x.dims; ++d) {
                x.size[d] = pick(6) + (pick(20) != 0);
                x.stride[d] = pick(2) ? common[pick(3)] : pick(400);
            }
        }
        bool want = listed(r[0], r[1]);
        (want ? both : none)++;
#ifdef PLANT_OVERLAP
        if (i == 777) want = !want;
#endif
        expect(Overlap::of(r[0], r[1]), want, "case", i);
        expect(Overlap::of(r[1], r[0]), want, "turned case", i);
    }
    if (both < 2000 || none < 2000) std::printf("%d overlap, %d do not\n", both, none), ++errors;

    // Queries, keys and values side by side in one product of 2^21 rows of 24 heads of 64 in bf16.
    const long long rows = 1 << 21, row = 24 * 128;
    auto heads = [&](long long at, long long h) {
        return Region{at, 2, 4, {16, rows / 16, h, 64}, {rows / 16 * row, row, 128, 2}};
    };
    expect(Overlap::of(heads(0, 8), heads(8 * 128, 8)), false, "packed, head", 8);
    expect(Overlap::of(heads(0, 8), heads(7 * 128, 8)), true, "packed, head", 7);
    expect(Overlap::of(heads(0, 8), heads(row - 128, 1)), false, "packed, last head", 0);
    expect(Overlap::of(heads(0, 8), heads(row - 126, 1)), true, "packed, across the row", 0);
    // One row of a cache of 65, another row, and a new tensor behind it.
    auto cache = [&](long long t, long long n) { return Region{t * 1024, 2, 4, {1 << 20, n, 8, 64}, {65 * 1024, 1024, 128, 2}}; };
    expect(Overlap::of(cache(64, 1), cache(0, 64)), false, "cache, row", 64);
    expect(Overlap::of(cache(63, 1), cache(0, 64)), true, "cache, row", 63);
    expect(Overlap::of(cache(0, 65), Region{(65LL << 20) * 1024, 2, 1, {1 << 20}, {2}}), false, "behind", 0);
    expect(Overlap::of(cache(0, 65), Region{(65LL << 20) * 1024 - 2, 2, 1, {1 << 20}, {2}}), true, "behind", -2);
    // Broadcast: one row for all.
    expect(Overlap::of(Region{0, 2, 2, {1 << 20, 64}, {0, 2}}, Region{128, 2, 2, {9, 64}, {128, 2}}), false, "broadcast", 0);
    expect(Overlap::of(Region{0, 2, 2, {1 << 20, 64}, {0, 2}}, Region{126, 2, 2, {9, 64}, {128, 2}}), true, "broadcast", 1);
    if (errors) return std::printf("%d errors\n", errors), 1;
    std::printf("OK\n");
    return 0;
}
