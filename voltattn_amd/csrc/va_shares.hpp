// va_shares.hpp — how the units of a batch are cut into shares (va_attend.hpp): scalars only, so that
// tests/cpp/test_shares.cpp walks the same code on the host.
#pragma once
#include <cstdint>

#ifdef __HIPCC__
#define VA_SHARES_FN __host__ __device__ __forceinline__
#else
#define VA_SHARES_FN inline
#endif

namespace va {

// Units 0 .. total - 1, 2^shift of them to a tile, in shares for nwg work-groups of BM rows to a block: units
// start(w) .. start(w + 1) - 1 are work-group w's. The work-groups of a CU do not get on equally: its oldest
// waves go first. With equal shares of many rows those of 128-row blocks, three to a CU, ended after 508, 650 and
// 752 us (10 prompts' chunks over up to 16 K positions), those of 256-row blocks, two, after 3272 and 3977 (8 K
// tokens over 32 K positions); shares by age (10 : 8 : 6 and 8 : 6) take these calls from 670 to 650 us and from
// 3900 to 3810. A launch fills the GPU in the order of its blocks, an age after the other, eight XCDs in turn.
template <int BM> struct Shares {
    static constexpr int AGES = BM == 128 ? 3 : BM == 256 ? 2 : 1;
    static constexpr int AGE[4] = {0, AGES == 3 ? 10 : 8, AGES == 3 ? 18 : 14, 24};   // what the work-groups up to an age take
    int total, nwg, shift;
    VA_SHARES_FN bool by_age() const { return AGES > 1 && nwg % (8 * AGES) == 0 && total >> (shift + 4) >= nwg; }
    VA_SHARES_FN int share() const {
        const int x = (total + nwg - 1) / nwg, tile = 1 << shift;
        return x >= 8 * tile ? x : (x + tile - 1) & -tile;   // whole tiles, where they are few
    }
    VA_SHARES_FN int shares() const { return by_age() ? nwg : (total + share() - 1) / share(); }
    VA_SHARES_FN int start(int w) const {
        if (!by_age()) {
            const long long at = (long long)w * share();
            return at < total ? (int)at : total;
        }
        if (w >= nwg) return total;
        const int per = nwg / 8, of = per / AGES, x = w / per, j = w - x * per, age = j / of;
        const int p = (x * AGE[AGES] + AGE[age]) * of + (j - age * of) * (AGE[age + 1] - AGE[age]), all = 8 * AGE[AGES] * of;
        return total / all * p + (int)((uint32_t)(total % all) * (uint32_t)p / (uint32_t)all);
    }
};

// The tiles of a block ahead of its unit x: in proportion, the first tile with the first unit.
VA_SHARES_FN int tiles_ahead(int x, int units, int tiles, int shift) {
    if (x >= units) return tiles;
    if (x <= 0) return 0;
    if (units == tiles << shift) return (x + (1 << shift) - 1) >> shift;   // the same, without the division
    return (int)__builtin_ceil((double)x * tiles / units);
}

} // namespace va
