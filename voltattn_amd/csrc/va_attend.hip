// va_attend.hip — launches of the kernels of va_attend.hpp.
#include "va_attend.hpp"
#include <algorithm>

namespace va {

// Tiles that beginning a block is worth (its queries and first tile have to come, its sums to go): 5 to 11 us
// on a full GPU. Of 0, 2 and 4 a decoding batch (64 sequences, up to 8 K positions, 8 K/V heads) takes 73,
// 62.5 and 63.5 us, a step with four prompts' chunks among 36 tokens 199, 175 and 177, chunks of 10 prompts
// 680, 670 and 667.
constexpr int SETUP = 2;

AttendForm attend_form(int D, int B, int total, int hkv, int group, int cap, int cus) {
    (void)D;
    AttendForm f;
    const double mean = (double)total * group / B;
    f.rows = mean <= 16 ? 16 : mean <= 32 ? 32 : mean <= 2048 ? 128 : 256;
    const long long bn = f.rows >= 128 ? 64 : 128;
    // every sequence's last block may be a part, as may the rows before the first and behind the last one
    const long long blocks = std::min((long long)total * group, (long long)total * group / f.rows + B + 2) * hkv;
    f.tiles = blocks * std::max(1LL, (cap + bn - 1) / bn);
    f.groups = std::max(1LL, std::min(f.tiles, (f.rows == 128 ? 3LL : 2LL) * cus));   // total = 0: no tiles
    f.setup = f.tiles / f.groups >= 8 ? SETUP : 0;
    // the numbering, of which the slope may make twice the tiles, has to end below 2^31
    f.shift = 4;
    while (f.shift > 0 && (f.tiles + f.setup * blocks) << f.shift > 1 << 29) --f.shift;
    return f;
}

size_t attend_ws_floats(const AttendForm& f, int D) { return (size_t)2 * f.groups * f.rows * (D + 2) + f.groups * sizeof(AttendNote) / sizeof(float); }

template <int D, int G>
static hipError_t launch(const AttendArgs& a, hipStream_t stream) {
    const dim3 grid((unsigned)(a.nwg + 7) / 8 * 8), block(256);
    hipError_t e;
#define VA_ATTEND(KERNEL, BM, PW)                                                                       \
    do {                                                                                                    \
        hipLaunchKernelGGL((KERNEL), grid, block, 0, stream, a);                                            \
        e = hipGetLastError();                                                                              \
        if (e == hipSuccess && a.nwg > 1) {                                                                 \
            const dim3 mgrid((unsigned)((size_t)a.nwg * (BM / (32 / PW))));                                 \
            hipLaunchKernelGGL((attend_merge<D, BM, PW>), mgrid, block, 0, stream, a);                  \
            e = hipGetLastError();                                                                          \
        }                                                                                                   \
    } while (0)
    if (a.form == 16) VA_ATTEND((attend_few<D, G, 1>), 16, 4);
    else if (a.form == 32) VA_ATTEND((attend_few<D, G, 2>), 32, 4);
    else if (a.form == 128) VA_ATTEND((attend_wide<D, G, 1>), 128, 1);
    else VA_ATTEND((attend_wide<D, G, 2>), 256, 1);
#undef VA_ATTEND
    return e;
}

hipError_t launch_attend(int D, int G, const AttendArgs& args, hipStream_t stream) {
    AttendArgs a = args;
    a.by_group = FastDiv::of((uint32_t)a.group);
    const long long span = (long long)a.group * (a.form >= 128 ? 64 : 128);
    a.slope = (int)((((long long)a.form << a.shift) + span / 2) / span);
    if (D == 128) return G == 32 ? launch<128, 32>(a, stream) : launch<128, 64>(a, stream);
    return G == 32 ? launch<64, 32>(a, stream) : launch<64, 64>(a, stream);
}

} // namespace va
