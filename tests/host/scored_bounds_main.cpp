// The intervals of keys and rows that the scored attention kernels walk and mask by (om_attention_scored.hpp,
// om_attention_scored_mm.hpp), against the rule itself in 64 bits, at sizes up to the largest that the entry points accept.
// Prints each broken promise and a last line "checks broken".
#include <algorithm>
#include <cstdio>
#include <random>
#include <vector>

#include "../../onemodel-csharp_amd/csrc/om_attention_scored_mm.hpp"

using namespace osc;

static long checks, broken;
static void expect(bool ok, const char *what, const Rule &u, int a, int b, int pre) {
    checks++;
    if (ok) return;
    if (broken++ < 20)
        std::printf("%s lq=%d lk=%d G=%d causal=%d window=%d pre=%d at %d %d\n", what, u.lq, u.lk, u.G, u.causal, u.window, pre, a, b);
}

// Whether some / every (position, key) of the rectangle is visible. The rule without prefix asks for i - j in an interval.
static void rect(const Rule &u, int64_t i0, int64_t i1, int64_t j0, int64_t j1, int64_t pre, bool &some, bool &all) {
    const int64_t far = (int64_t)1 << 40, lo = u.causal ? 0 : u.window ? -(int64_t)u.window + 1 : -far, hi = u.window ? (int64_t)u.window - 1 : far;
    const int64_t k0 = std::max(j0, pre);  // the keys from here on are under the rule
    some = j0 < pre;
    all = true;
    if (k0 <= j1) {
        const int64_t least = i0 - j1, most = i1 - k0;
        some = some || (least <= hi && most >= lo);
        all = least >= lo && most <= hi;
    }
}

static void check(const Rule &u, int prefix, std::mt19937_64 &rng) {
    const int rows = u.G * u.lq, pre = prefix;
    auto some_of = [&](int n, std::vector<int> extra) {  // block starts: the ends, the extras and a few drawn ones
        std::vector<int> at = {0, n - 1};
        for (int e : extra) at.push_back(e);
        for (int i = 0; i < 12; i++) at.push_back((int)(rng() % (uint64_t)n));
        for (int &x : at) x = std::min(std::max(x, 0), n - 1);
        return at;
    };
    const int near = pre < 0 ? 0 : std::min(pre, u.lk);
    for (int k : some_of(u.lk, {near - 1, near - 17, near, u.off, u.off - u.window, u.lk - u.window}))
        for (int width : {1, 4, 32, 128}) {
            const int j0 = k / width * width, j1 = std::min(j0 + width, u.lk) - 1;
            int r0, r1;
            row_range(u, j0, j1, pre, r0, r1);
            expect(0 <= r0 && r0 <= r1 && r1 <= rows, "row_range leaves the rows", u, j0, j1, pre);
            const RowBand band(u, j0, j1, pre);
            for (int r : some_of(rows, {r0 - 1, r0, r1 - 1, r1, r1 + 31, 132096 % std::max(rows, 1)}))
                for (int step : {1, 32}) {
                    const int f0 = r / step * step, f1 = f0 + step - 1, last = std::min(f1, rows - 1);
                    bool some, all;
                    rect(u, (int64_t)f0 / u.G + u.off, (int64_t)last / u.G + u.off, j0, j1, pre, some, all);
                    expect(!band.all(f0, f1) || all, "RowBand::all", u, f0, j0, pre);
                    expect(band.some(f0, f1) || !some, "RowBand::some", u, f0, j0, pre);
                    if (step == 1) expect((r0 <= f0 && f0 < r1) || !some, "row_range leaves out a row", u, f0, j0, pre);
                    if (step == 1 && width == 1) {
                        const int pos = f0 / u.G + u.off;
                        expect(in_reach(u, pos - j0, j0, pre) == some, "in_reach", u, pos, j0, pre);
                        expect(keys_seen(u, pos, 0, pre).has(j0) == some, "keys_seen", u, pos, j0, pre);
                        expect(rows_seeing(u, j0, 0, pre).has(pos) == some, "rows_seeing", u, pos, j0, pre);
                    }
                }
        }
    for (int r : some_of(rows, {}))
        for (int width : {1, 3, 32, 128}) {
            const int f0 = r / width * width, last = std::min(f0 + width, rows) - 1;
            const int i0 = f0 / u.G + u.off, i1 = last / u.G + u.off;
            int lo, hi;
            key_range(u, i0, i1, pre, lo, hi);
            expect(0 <= lo && hi < u.lk, "key_range leaves the keys", u, i0, i1, pre);
            const Band band(u, i0, i1, pre);
            for (int k : some_of(u.lk, {lo - 1, lo, hi, hi + 1, near - 1, near}))
                for (int step : {1, 32}) {
                    const int j0 = k / step * step, j1 = j0 + step - 1, end = std::min(j1, u.lk - 1);
                    bool some, all;
                    rect(u, i0, i1, j0, end, pre, some, all);
                    expect(!band.all(j0, j1) || (all && j1 < u.lk), "Band::all", u, i0, j0, pre);
                    expect(band.some(j0, j1) || !some, "Band::some", u, i0, j0, pre);
                    if (step == 1) expect((lo <= j0 && j0 <= hi) || !some, "key_range leaves out a key", u, i0, j0, pre);
                }
        }
}

int main() {
    std::mt19937_64 rng(7);
    auto rule = [](int lq, int lk, int G, int causal, int window) {
        Rule u = {};
        u.B = u.Hk = 1;
        u.G = G;
        u.lq = lq;
        u.lk = lk;
        u.d = 1;
        u.off = lk - lq;
        u.causal = causal;
        u.window = window >= std::max(lq, lk) ? 0 : window;  // as make_rule has it
        return u;
    };
    const int most = 1 << 30;
    for (int causal : {0, 1})
        for (int pre : {0, 100, 1 << 24, INT32_MAX, -4}) {
            check(rule(8, 1 << 25, 128, causal, 1024), pre, rng);
            check(rule(200, 1 << 20, 4096, causal, 5), pre, rng);
            check(rule(1, most, 1 << 20, causal, 3), pre, rng);
            check(rule(1 << 20, most, 1 << 10, causal, 70000), pre, rng);
            check(rule(most, most, 1, causal, most - 1), pre, rng);
            check(rule(most, most, 1, causal, INT32_MAX - 5), pre, rng);
            check(rule(most, 1, 1, causal, most - 3), pre, rng);
            check(rule(1, most, most, causal, 1), pre, rng);
        }
    auto drawn = [&](int64_t top) { return (int)std::max<double>(1.0, std::exp2(std::uniform_real_distribution<>(0, std::log2((double)top))(rng))); };
    for (int n = 0; n < 3000; n++) {
        const int G = drawn(n % 2 ? 64 : most), lq = drawn(most / G), lk = drawn(most);
        check(rule(lq, lk, G, (int)(rng() % 2), rng() % 3 ? drawn(INT32_MAX) : 0), rng() % 2 ? 0 : drawn(2 * (int64_t)lk), rng);
    }
    std::printf("%ld %ld\n", checks, broken);
    return 0;
}
