// va_attend.hip — launches of the kernels of va_attend.hpp.
#include "va_attend.hpp"
#include <algorithm>

namespace va {

// Tiles that beginning a block is worth (its queries and first tile have to come, its sums to go): 5 to 11 us
// on a full GPU. Of 0, 2 and 4 a decoding batch (64 sequences, up to 8 K positions, 8 K/V heads) takes 73,
// 62.5 and 63.5 us, a step with four prompts' chunks among 36 tokens 199, 175 and 177, chunks of 10 prompts
// 680, 670 and 667.
constexpr int SETUP = 2;

// Rows to a block, by a sequence's mean rows to a K/V head (the lengths are on the device). In us, 4 query heads
// to each of 8 K/V heads of 128 dimensions: one token over 4 K positions with blocks of 16 rows 11.9, of 32 15.1;
// 16 sequences over 4 K with 16 rows to a head 40.3 and 42.3, with 24 52.2 and 43.7; with 32 rows and blocks of 32
// 45.2, of 128 57.4; with 64 rows 83 (16), 61 (128). 2 x 4 K tokens over 8 K positions with blocks of 128 rows
// 869, of 256 836, 8 K tokens over 32 K 3880 and 3615; with 2048 rows both take 306, and blocks of 128 waste less of
// uneven batches. (All of batches whose sequences are alike: the mean says little of one long chunk beside many
// tokens, whose rows then share the tokens' short blocks. 127 tokens and a chunk of 512 take 215 us, 111 and 71
// apart.) One launch for all of a batch: of a step with four chunks among 36 tokens two (16-row blocks
// for the tokens, 128-row blocks for the chunks) took 157 against 158.
AttendForm attend_form(int B, int total, int hkv, int group, int cap, int cus) {
    AttendForm f;
    const double mean = (double)total * group / B;
    f.rows = mean <= 16 ? 16 : mean <= 32 ? 32 : mean <= 2048 ? 128 : 256;
    const long long bn = f.rows >= 128 ? 64 : 128;
    // every sequence's last block may be a part, as may the rows before the first and behind the last one
    const long long blocks = std::min((long long)total * group, (long long)total * group / f.rows + B + 2) * hkv;
    f.tiles = blocks * std::max(1LL, (cap + bn - 1) / bn);
    // what fills the card: 128 rows leave room for three work-groups on a CU, the others for two
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
