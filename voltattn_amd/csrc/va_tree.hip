// va_tree.hip — launches of the tree kernels (va_tree.hpp).
#include "va_tree.hpp"

namespace va {

// Waves side by side over the query rows of a K/V head.
static int tree_qw(int rows) { return rows <= 32 ? 1 : rows <= 64 ? 2 : 4; }

int tree_rows(int rows) { return 32 * tree_qw(rows); }
int tree_tile(int rows) { return tree_qw(rows) == 1 ? TreeTile<1>::BN : TreeTile<2>::BN; }
int tree_groups_per_cu(int D, int rows) { return tree_waves(D, tree_qw(rows)); }

template <int KIND, int D, int G>
static hipError_t launch(const TreeArgs& a, hipStream_t stream) {
    const dim3 grid((unsigned)a.nwg), block(256);
    const bool few = (long long)a.B * a.T * a.hkv * a.group <= 8192;   // 32 to a work-group would leave CUs idle
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
    switch (tree_qw(a.T * a.group)) {
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
