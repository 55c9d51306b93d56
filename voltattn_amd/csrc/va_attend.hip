// va_attend.hip — launches of the kernels of va_attend.hpp.
#include "va_attend.hpp"
#include <algorithm>

namespace va {

AttendForm attend_form(int D, int B, int total, int hkv, int group, int cap, int cus) {
    (void)D;
    AttendForm f;
    const double mean = (double)total * group / B;
    f.rows = mean <= 16 ? 16 : mean <= 32 ? 32 : mean <= 2048 ? 128 : 256;
    const long long bn = f.rows >= 128 ? 64 : 128;
    // every sequence's last block may be a part, as may the rows before the first and behind the last one
    const long long blocks = std::min((long long)total * group, (long long)total * group / f.rows + B + 2) * hkv;
    f.tiles = blocks * std::max(1LL, (cap + bn - 1) / bn);
    f.groups = std::min(f.tiles, (f.rows == 128 ? 3LL : 2LL) * cus);
    return f;
}

size_t attend_ws_floats(const AttendForm& f, int D) { return (size_t)2 * f.groups * f.rows * (D + 2); }

template <int D, int G>
static hipError_t launch(const AttendArgs& a, hipStream_t stream) {
    const dim3 grid((unsigned)(a.nwg + 7) / 8 * 8), block(256);
    hipError_t e;
#define VA_ATTEND(KERNEL, BM, BN, PW)                                                                       \
    do {                                                                                                    \
        hipLaunchKernelGGL((KERNEL), grid, block, 0, stream, a);                                            \
        e = hipGetLastError();                                                                              \
        if (e == hipSuccess && a.nwg > 1) {                                                                 \
            const dim3 mgrid((unsigned)((size_t)a.nwg * (BM / (32 / PW))));                                 \
            hipLaunchKernelGGL((attend_merge<D, BM, BN, PW>), mgrid, block, 0, stream, a);                  \
            e = hipGetLastError();                                                                          \
        }                                                                                                   \
    } while (0)
    if (a.form == 16) VA_ATTEND((attend_few<D, G, 1>), 16, 128, 4);
    else if (a.form == 32) VA_ATTEND((attend_few<D, G, 2>), 32, 128, 4);
    else if (a.form == 128) VA_ATTEND((attend_wide<D, G, 1>), 128, 64, 1);
    else VA_ATTEND((attend_wide<D, G, 2>), 256, 64, 1);
#undef VA_ATTEND
    return e;
}

hipError_t launch_attend(int D, int G, const AttendArgs& args, hipStream_t stream) {
    AttendArgs a = args;
    a.by_group = FastDiv::of((uint32_t)a.group);
    if (D == 128) return G == 32 ? launch<128, 32>(a, stream) : launch<128, 64>(a, stream);
    return G == 32 ? launch<64, 32>(a, stream) : launch<64, 64>(a, stream);
}

} // namespace va
