// CPU test of the shares' arithmetic (voltattn_amd/csrc/va_shares.hpp): built with g++ and run by
// tests/test_shares.py; checks random totals and batches, prints "shares: ok".
#include "va_shares.hpp"

#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

#define CHECK(c)                                                          \
    do {                                                                  \
        if (!(c)) {                                                       \
            std::fprintf(stderr, "%s:%d: check failed: %s\n", __FILE__, __LINE__, #c); \
            std::exit(1);                                                 \
        }                                                                 \
    } while (0)

static std::mt19937 rng(7);
static int pick(int lo, int hi) { return lo + (int)(rng() % (uint32_t)(hi - lo + 1)); }

// Every unit is in one share, and the shares go by what they should.
template <int BM> static void starts(int total, int nwg, int shift) {
    const va::Shares<BM> s{total, nwg, shift};
    CHECK(s.start(0) == 0);
    const int n = s.shares();
    CHECK(n >= 1 && n <= nwg);
    for (int w = 0; w < nwg; ++w) {
        const int len = s.start(w + 1) - s.start(w);
        CHECK(len >= 0);
        CHECK(w < n ? len > 0 : len == 0);
        if (s.by_age()) {
            constexpr int AGES = va::Shares<BM>::AGES;
            const int of = nwg / 8 / AGES, age = w % (nwg / 8) / of;
            const double part = va::Shares<BM>::AGE[age + 1] - va::Shares<BM>::AGE[age];
            const double want = (double)total * part / (8.0 * va::Shares<BM>::AGE[AGES] * of);
            CHECK(len > want - 1 && len < want + 1);          // both ends are rounded down
        } else {
            CHECK(len <= s.share());
        }
    }
    CHECK(s.start(n) == total && s.start(nwg) == total && s.start(nwg + 7) == total);
}

// A batch's blocks, cut as the kernels cut them: every tile of every block in one piece, in order, the first unit
// with the first tile; of a cut block one piece begins it and one ends it.
template <int BM> static void batch(int nwg, int shift, int setup, int blocks, int most) {
    struct Block { int first, units, tiles; };
    std::vector<Block> b;
    int total = 0;
    while ((int)b.size() < blocks) {                          // sequences of blocks that begin ever later
        const int n = pick(1, 9), t0 = pick(1, most), step = pick(0, 3);
        const int slope = (step << shift) + (shift ? pick(0, (1 << shift) - 1) : 0), head = (t0 + setup) << shift;
        for (int rb = 0; rb < n; ++rb) {
            const Block x{total, head + rb * slope, std::max(1, t0 + rb * step + pick(0, 1))};
            b.push_back(x);
            total += x.units;
        }
    }
    const va::Shares<BM> s{total, nwg, shift};
    std::vector<int> at(b.size(), 0), begins(b.size(), 0), ends(b.size(), 0), pieces(b.size(), 0);
    for (int w = 0; w < nwg; ++w) {
        int u = s.start(w);
        const int end = s.start(w + 1);
        while (u < end) {
            const int i = (int)(std::upper_bound(b.begin(), b.end(), u, [](int x, const Block& y) { return x < y.first; }) - b.begin()) - 1;
            const int t0 = va::tiles_ahead(u - b[i].first, b[i].units, b[i].tiles, shift), t1 = va::tiles_ahead(end - b[i].first, b[i].units, b[i].tiles, shift);
            u = std::min(end, b[i].first + b[i].units);
            CHECK(t0 >= 0 && t0 <= t1 && t1 <= b[i].tiles && t0 == at[i]);
            if (t0 >= t1) continue;
            at[i] = t1;
            begins[i] += t0 == 0;
            ends[i] += t1 == b[i].tiles;
            ++pieces[i];
        }
    }
    for (size_t i = 0; i < b.size(); ++i) CHECK(at[i] == b[i].tiles && begins[i] == 1 && ends[i] == 1 && pieces[i] >= 1);
}

template <int BM> static void all() {
    const int fixed[] = {1, 2, 7, 8, 24, 48, 100, 512, 767, 768, 1000};
    for (int i = 0; i < 3000; ++i) {
        const int nwg = i % 2 ? fixed[pick(0, 10)] : pick(1, 1024), shift = pick(0, 4);
        starts<BM>(pick(1, 1 << pick(0, 30)), nwg, shift);
        starts<BM>(std::max(1, (nwg << (shift + 4)) + pick(-2, 2)), nwg, shift);      // where shares begin to go by age
        batch<BM>(nwg, shift, pick(0, 2), pick(1, 400), 1 << pick(0, 8));
    }
}

int main() {
    all<16>();
    all<32>();
    all<128>();
    all<256>();
    std::puts("shares: ok");
    return 0;
}
