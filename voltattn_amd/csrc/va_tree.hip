// va_tree.hip — launches of the tree kernels (va_tree.hpp).
#include "va_tree.hpp"
#include <algorithm>

namespace va {

// The row block that holds all rows of a K/V head, up to 128 rows, reads K and V once and
// fills the card from about 4 tiles to a CU on. Below, one work-group to a CU takes the
// next narrower block: fewer pieces to join, each with fewer rows, outweigh reading K and V twice.
// One sequence, 64 rows to a K/V head (8 of them, q8), narrower : wider: 4096 positions (2 tiles)
// 16.6 : 22.8 us, 32768 (16 tiles) 47.2 : 39.2 us; 128 rows, 4096 positions 19.9 : 28.6 us;
// 16 sequences of 8192 positions, 128 rows, q4 78.9 : 63.2 us.
TreeForm tree_form(int kind, int D, int B, int hkv, int rows, int cap, int cus) {
    TreeForm f;
    f.qw = rows <= 32 ? 1 : rows <= 64 ? 2 : 4;
    auto count = [&]() {
        const long long bm = 32 * f.qw, bn = f.qw == 1 ? TreeTile<1>::BN : TreeTile<2>::BN;
        return (long long)B * hkv * ((rows + bm - 1) / bm) * std::max(1LL, (cap + bn - 1) / bn);
    };
    f.tiles = count();
    f.groups = (long long)tree_waves(kind, D, f.qw) * cus;
    if (f.qw > 1 && f.tiles <= 4LL * cus) {
        f.qw /= 2;
        f.tiles = count();
        f.groups = cus;
    }
    f.groups = std::min(f.groups, f.tiles);
    return f;
}

template <int KIND, int D, int G>
static hipError_t launch(const TreeArgs& a, hipStream_t stream) {
    const dim3 grid((unsigned)(a.nwg + 7) / 8 * 8), block(256);
    // rows to a merging work-group, and waves to a row's pieces: 32 and 1, or 8 and 4 where the former
    // would leave CUs idle. The whole call, 8 and 4 : 32 and 1, 16 drafts and 32 query heads over 8192
    // positions q8: 512 rows 24.7 : 32.5 us, 2048 46.5 : 48.4, 4096 69.5 : 70.1, 8192 114.3 : 114.1, 16384 203.8 : 201.6
    const bool few = (long long)a.B * a.T * a.hkv * a.group <= 8192;
    const int mr = few ? 8 : 32;
    const dim3 mgrid((unsigned)((size_t)a.B * a.hkv * ((a.T * a.group + mr - 1) / mr)));
    hipError_t e;
#define VA_TREE(QW)                                                                        \
    do {                                                                                   \
        hipLaunchKernelGGL((tree_attend<KIND, D, G, QW>), grid, block, 0, stream, a);      \
        e = hipGetLastError();                                                             \
        if (e == hipSuccess) {                                                             \
            if (few) hipLaunchKernelGGL((tree_merge<D, QW, 4>), mgrid, block, 0, stream, a); \
            else hipLaunchKernelGGL((tree_merge<D, QW, 1>), mgrid, block, 0, stream, a);   \
            e = hipGetLastError();                                                         \
        }                                                                                  \
    } while (0)
    switch (a.qw) {
        case 1: VA_TREE(1); break;
        case 2: VA_TREE(2); break;
        default: VA_TREE(4); break;
    }
#undef VA_TREE
    return e;
}

template <int KIND>
static hipError_t launch_kind(int D, int G, const TreeArgs& a, hipStream_t stream) {
    if (D == 128) return G == 32 ? launch<KIND, 128, 32>(a, stream) : launch<KIND, 128, 64>(a, stream);
    return G == 32 ? launch<KIND, 64, 32>(a, stream) : launch<KIND, 64, 64>(a, stream);
}

hipError_t launch_tree(int kind, int D, int G, const TreeArgs& a, hipStream_t stream) {
    switch (kind) {
        case KF16: return D == 128 ? launch<KF16, 128, 64>(a, stream) : launch<KF16, 64, 64>(a, stream);
        case KQ8: return launch_kind<KQ8>(D, G, a, stream);
        case KQ4: return launch_kind<KQ4>(D, G, a, stream);
        default: return launch_kind<KQ3>(D, G, a, stream);
    }
}

} // namespace va
