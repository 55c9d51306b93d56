// va_tree.hpp — attention of drafted tokens over a paged cache (va_decode_tree).
//
// Sequence b has ctx positions of context and n drafted tokens (a tree), whose K/V
// rows are the positions ctx .. ctx + n - 1. Draft i attends every position of the
// context and the drafts j whose bit is set in mask[b][i]:
//   o_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp2((q_i.k_j - m_i) * log2(e)/sqrt(D)),
// a row to which nothing is visible is zero. The n * (Hq/Hkv) query rows of a K/V head
// share every K/V row, so both products run on the matrix cores, 32 rows to a wave as
// the columns of va_wide.hpp's tiles.
//
// Work-group: 4 waves, QW of them side by side over the query rows (BM = 32 QW) and
// KW = 4/QW over the K/V rows of a tile of BN. A tile is fetched into registers while
// its predecessor is computed, unpacked into LDS as exact fp16 codes (one unpack for all
// query rows) and its group scales beside it; K's scales are applied to each group's part
// of the dot product in fp32, V's to the weights: p * s is rounded once, to fp16 (RNE),
// an independent error of 2^-12 of each weight, and the output's own rounding to fp16 is
// as large. fp16 holds p * s from 2^-24 to 65504: the lazy maximum lets p grow to 2^SLACK
// and starts it at 2^OFF, so that no scale of a cache made from fp16 values (|v| <= 65504)
// overflows and weights far below the largest one keep their digits.
//
// Work split: the tiles of all (sequence, K/V head, row block), numbered one behind the
// other, are cut into equal shares, one to a work-group. A row block inside one share is
// finished there; the pieces of one that several shares cut go to ws (slot 2w: the
// piece that work-group w begins with, 2w + 1: the one it ends with) and tree_merge
// joins them.
#pragma once
#include "va_kernels.hpp"
#include "va_wide.hpp"

namespace va {

// ------------------------------------------------------------ unpacking --
// A unit is what one lane fetches of a tile at once: UB bytes of a row, UE values.
template <int KIND> struct Unit {
    static constexpr int UB = KIND == KQ3 ? 12 : 16;
    static constexpr int UE = UB * 8 / KindBits<KIND>::num;
    static constexpr int W = UB / 4;
};
template <int W> struct Words { uint32_t w[W]; };

__device__ __forceinline__ f16x2 as_f16x2(uint32_t x) { return __builtin_bit_cast(f16x2, x); }
__device__ __forceinline__ f16x8 join4(f16x2 a, f16x2 b, f16x2 c, f16x2 d) {
    return f16x8{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}
// Four codes, one to a byte of w, as fp16 pairs 1024 + n, less `bias`: exact.
__device__ __forceinline__ void bytes_to_f16(uint32_t w, _Float16 bias, f16x2& a, f16x2& b) {
    const f16x2 z = {bias, bias};
    a = as_f16x2(__builtin_amdgcn_perm(0x64646464u, w, 0x04010400u)) - z;
    b = as_f16x2(__builtin_amdgcn_perm(0x64646464u, w, 0x04030402u)) - z;
}
// A unit's values in order, as exact fp16 codes (f16: the values).
template <int KIND>
__device__ __forceinline__ void unpack_unit(const Words<Unit<KIND>::W>& u, f16x8 (&out)[Unit<KIND>::UE / 8]) {
    if constexpr (KIND == KF16) {
        out[0] = __builtin_bit_cast(f16x8, u32x4{u.w[0], u.w[1], u.w[2], u.w[3]});
    } else if constexpr (KIND == KQ8) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            f16x2 a, b, c, d;
            bytes_to_f16(u.w[2 * i] ^ 0x80808080u, (_Float16)1152.f, a, b);
            bytes_to_f16(u.w[2 * i + 1] ^ 0x80808080u, (_Float16)1152.f, c, d);
            out[i] = join4(a, b, c, d);
        }
    } else if constexpr (KIND == KQ4) {
        const f16x2 lo = {(_Float16)1032.f, (_Float16)1032.f}, hi = {(_Float16)72.f, (_Float16)72.f};
        const f16x2 r16 = {(_Float16)0.0625f, (_Float16)0.0625f};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t w = u.w[i], x = w >> 8;
            // nibbles (0,4), (1,5), (2,6), (3,7): n - 8, the upper ones from 1024 + 16n
            const uint32_t p04 = __builtin_bit_cast(uint32_t, as_f16x2((w & 0x000F000Fu) | 0x64006400u) - lo);
            const uint32_t p15 = __builtin_bit_cast(uint32_t, as_f16x2((w & 0x00F000F0u) | 0x64006400u) * r16 - hi);
            const uint32_t p26 = __builtin_bit_cast(uint32_t, as_f16x2((x & 0x000F000Fu) | 0x64006400u) - lo);
            const uint32_t p37 = __builtin_bit_cast(uint32_t, as_f16x2((x & 0x00F000F0u) | 0x64006400u) * r16 - hi);
            out[i] = __builtin_bit_cast(f16x8, u32x4{__builtin_amdgcn_perm(p15, p04, 0x05040100u), __builtin_amdgcn_perm(p37, p26, 0x05040100u),
                                                     __builtin_amdgcn_perm(p15, p04, 0x07060302u), __builtin_amdgcn_perm(p37, p26, 0x07060302u)});
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {                       // 24 bits, eight codes, at bit 24i
            const int at = 24 * i;
            const uint32_t low = u.w[at / 32], high = at / 32 + 1 < 3 ? u.w[at / 32 + 1] : 0u;
            const uint32_t g = at % 32 ? __builtin_amdgcn_alignbit(high, low, at % 32) : low;
            uint32_t c[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const uint32_t x = (g >> (12 * j)) & 0xFFFu, t = (x | (x << 10)) & 0x003F003Fu;
                c[j] = (t | (t << 5)) & 0x07070707u;        // one code to a byte
            }
            f16x2 a, b, d, e;
            bytes_to_f16(c[0], (_Float16)1028.f, a, b);
            bytes_to_f16(c[1], (_Float16)1028.f, d, e);
            out[i] = join4(a, b, d, e);
        }
    }
}

// p and p * scale stay within fp16: the weights start at 2^OFF and may grow by 2^SLACK
// before the maximum follows. A scale of a cache of fp16 values is at most 65504/127 (q8),
// 65504/7 (q4), 65504/3 (q3).
template <int KIND> struct WeightRange;
template <> struct WeightRange<KF16> { static constexpr float off = 4.f, slack = 8.f; };
template <> struct WeightRange<KQ8>  { static constexpr float off = 3.f, slack = 3.f; };
template <> struct WeightRange<KQ4>  { static constexpr float off = 0.f, slack = 2.f; };
template <> struct WeightRange<KQ3>  { static constexpr float off = 0.f, slack = 1.f; };

// ------------------------------------------------------------- work split --
// A sequence's part in the numbering: nothing for one without drafts or with lengths
// out of range (whose rows tree_merge fills).
struct TreeSeq {
    int ctx, n, len;      // len = ctx + n
    int tiles, blocks;    // K/V tiles, row blocks per K/V head
    bool bad;
};
template <int BM, int BN>
__device__ __forceinline__ TreeSeq tree_seq(const TreeArgs& a, int b) {
    TreeSeq s;
    s.ctx = a.ctx_lens[b];
    s.n = a.sizes ? a.sizes[b] : a.T;
    s.bad = s.ctx < 0 || s.n < 0 || s.n > a.T || s.ctx > a.cap - s.n;
    s.len = s.bad ? 0 : s.ctx + s.n;
    s.tiles = (s.len + BN - 1) / BN;
    s.blocks = s.bad ? 0 : (s.n * a.group + BM - 1) / BM;
    return s;
}
template <int BM, int BN>
__device__ __forceinline__ int tree_units(const TreeArgs& a, int b) {
    if (b >= a.B) return 0;
    const TreeSeq s = tree_seq<BM, BN>(a, b);
    return s.tiles * s.blocks * a.hkv;
}
// Sum over the sequences below `upto` (all: a.B); every wave by itself.
template <int BM, int BN>
__device__ __forceinline__ int tree_units_below(const TreeArgs& a, int upto) {
    int sum = 0;
    for (int b0 = 0; b0 < upto; b0 += 64) {
        const int b = b0 + (int)__lane_id();
        sum += __builtin_amdgcn_readlane(wave_scan(b < upto ? tree_units<BM, BN>(a, b) : 0), 63);
    }
    return sum;
}
__device__ __forceinline__ int tree_share(const TreeArgs& a, int units) {
    return max((units + a.nwg - 1) / a.nwg, a.min_share);
}
// Tile `at` of the numbering: its sequence and the number of that sequence's first tile.
template <int BM, int BN>
__device__ __forceinline__ bool tree_find(const TreeArgs& a, int at, int& seq, int& first) {
    int before = 0;
    for (int b0 = 0; b0 < a.B; b0 += 64) {
        const int b = b0 + (int)__lane_id(), u = tree_units<BM, BN>(a, b), upto = before + wave_scan(u);
        const uint64_t hit = __ballot(upto > at);
        if (hit) {
            const int l = __builtin_ctzll(hit);
            seq = b0 + l;
            first = __builtin_amdgcn_readlane(upto, l) - __builtin_amdgcn_readlane(u, l);
            return true;
        }
        before = __builtin_amdgcn_readlane(upto, 63);
    }
    return false;
}

// --------------------------------------------------------------- kernel --
template <int QW> struct TreeTile {
    static constexpr int BM = 32 * QW, KW = 4 / QW;
    static constexpr int BN = QW == 1 ? 128 : 64;
    static constexpr int KB = BN / 32 / KW;                 // 32-row blocks of a tile per wave
};

template <int KIND, int D, int G, int QW>
__global__ __launch_bounds__(256, KIND == KF16 && QW == 1 ? 1 : 2) void tree_attend(TreeArgs a) {
    using T = TreeTile<QW>;
    constexpr int BM = T::BM, BN = T::BN, KW = T::KW, KB = T::KB;
    constexpr int KS = D / 16, DB = D / 32;
    constexpr int NG = KIND == KF16 ? 1 : D / G;            // scale groups of a row
    constexpr bool SCALED = KIND != KF16;
    constexpr int ROWB = RowBytes<KIND, D>::value;
    constexpr int UPR = D / Unit<KIND>::UE;                 // units per row
    constexpr int UNITS = BN * UPR;                         // of one tensor's tile
    constexpr int UPT = (UNITS + 255) / 256;                // per lane
    constexpr int TILE = BN * 2 * D;
    constexpr int HALVES = BN / 64;                         // a page holds at least 64 rows
    constexpr int RSRCS = 256 / UPR > 64 ? 1 : HALVES;      // halves that a wave fetches from
    constexpr int SCB = SCALED ? NG * BN * 2 : 0;           // bytes of a tile's scales, [group][row]
    constexpr int COMB = KW > 1 ? 4 * 32 * (D + 4) * 4 : 0; // the KW partial sums, over the tiles
    constexpr int LDS = 2 * TILE + 2 * SCB > COMB ? 2 * TILE + 2 * SCB : COMB;
    __shared__ __align__(1024) uint8_t lds[LDS];

    const int tid = (int)threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), half = lane >> 5;
    const int qw = wave % QW, kw = wave / QW;
    lds_u8* kt = (lds_u8*)lds;
    lds_u8* vt = kt + TILE;
    lds_u8* skt = vt + TILE;
    lds_u8* svt = skt + SCB;
    WideAddr<D> ad;
    ad.init(lane);

    const int units = tree_units_below<BM, BN>(a, a.B);
    const int share = tree_share(a, units);
    // consecutive shares on one XCD (work-groups are dealt to the eight in turn): the row
    // blocks of a K/V head lie next to each other and read the same rows
    const int wg = (a.nwg & 7) == 0 ? (int)(blockIdx.x & 7) * (a.nwg >> 3) + (int)(blockIdx.x >> 3) : (int)blockIdx.x;
    int at = wg * share;
    const int end = min(units, at + share);
    while (at < end) {
        int b, first;
        if (!tree_find<BM, BN>(a, at, b, first)) return;
        b = uniform(b);
        const TreeSeq sq = tree_seq<BM, BN>(a, b);
        const int in = at - first, blk = in / sq.tiles;     // (K/V head, row block) of the sequence
        const int hk = uniform(blk / sq.blocks), rb = uniform(blk - hk * sq.blocks);
        const int t0 = uniform(in - blk * sq.tiles), t1 = uniform(min(sq.tiles, t0 + (end - at)));
        const int rows = sq.n * a.group;
        const int row = rb * BM + qw * 32 + (lane & 31);
        const int rc = min(row, rows - 1), node = rc / a.group, hq = hk * a.group + (rc - node * a.group);
        uint64_t mask = a.mask[(size_t)b * a.T + node];
        if (sq.n < 64) mask &= (1ull << sq.n) - 1;
        f16x8 q[KS];
        {
            const uint16_t* qp = a.q + (((size_t)b * a.T + node) * a.hkv * a.group + hq) * D + 8 * half;
#pragma unroll
            for (int s = 0; s < KS; ++s) q[s] = *reinterpret_cast<const f16x8*>(qp + 16 * s);
        }
        const int32_t* table = a.block_table + (size_t)b * a.max_pages;

        Words<Unit<KIND>::W> kr[UPT], vr[UPT];
        uint32_t scr[2] = {0, 0};                           // lane's scales of K (lanes 0..127) or V
        bool bad = false;
        auto fetch = [&](int t) {
            // the rows of each half of the tile, 64 to a page at least: pool row and how many there are
            size_t first_row[HALVES];
            int left[HALVES];
#pragma unroll
            for (int x = 0; x < HALVES; ++x) {
                const int j = t * BN + x * 64;
                left[x] = max(min(64, sq.len - j), 0);
                int page = left[x] > 0 ? table[j >> a.page_shift] : 0;
                if (page < 0 || page >= a.num_pages) {
                    bad = true;
                    left[x] = page = 0;
                }
                first_row[x] = (((size_t)page * a.hkv + hk) << a.page_shift) + (size_t)(j & ((1 << a.page_shift) - 1));
            }
            __amdgpu_buffer_rsrc_t rk[RSRCS], rv[RSRCS];
#pragma unroll
            for (int x = 0; x < RSRCS; ++x) {
                const bool up = RSRCS < HALVES ? wave >= 2 : x == 1;
                const size_t r = uniform64(up ? first_row[HALVES - 1] : first_row[0]);
                const uint32_t bytes = (uint32_t)(uniform(up ? left[HALVES - 1] : left[0]) * ROWB);
                rk[x] = make_rsrc(a.k + r * ROWB, bytes);
                rv[x] = make_rsrc(a.v + r * ROWB, bytes);
            }
#pragma unroll
            for (int i = 0; i < UPT; ++i) {
                const int u = i * 256 + tid, r = u / UPR, x = RSRCS == 1 ? 0 : (i * 256 / UPR) >> 6;
                const uint32_t off = (uint32_t)((r & 63) * ROWB + (u % UPR) * Unit<KIND>::UB);
                if (UNITS % 256 == 0 || u < UNITS) {
                    if constexpr (Unit<KIND>::W == 4) {
                        const u32x4 ka = ld128(rk[x], off, 0), va = ld128(rv[x], off, 0);
                        kr[i] = {{ka.x, ka.y, ka.z, ka.w}};
                        vr[i] = {{va.x, va.y, va.z, va.w}};
                    } else {
                        const u32x3 ka = ld96(rk[x], off, 0), va = ld96(rv[x], off, 0);
                        kr[i] = {{ka.x, ka.y, ka.z}};
                        vr[i] = {{va.x, va.y, va.z}};
                    }
                }
            }
            if constexpr (SCALED) {
                const bool up = HALVES == 2 && (wave & 1);
                const size_t r = up ? first_row[HALVES - 1] : first_row[0];
                const int n = up ? left[HALVES - 1] : left[0];
                scr[0] = scr[1] = 0;
                if ((HALVES == 2 || !(wave & 1)) && lane < n) {
                    const uint16_t* p = (wave < 2 ? a.sk : a.sv) + (r + (size_t)lane) * NG;
                    if constexpr (NG == 1) scr[0] = p[0];
                    else scr[0] = *reinterpret_cast<const uint32_t*>(p);
                    if constexpr (NG == 4) scr[1] = *reinterpret_cast<const uint32_t*>(p + 2);
                }
            }
        };
        auto stage = [&]() {
#pragma unroll
            for (int i = 0; i < UPT; ++i) {
                const int u = i * 256 + tid, r = u / UPR, c = (u % UPR) * (Unit<KIND>::UE / 8);
                if (UNITS % 256 == 0 || u < UNITS) {
                    f16x8 x[Unit<KIND>::UE / 8], y[Unit<KIND>::UE / 8];
                    unpack_unit<KIND>(kr[i], x);
                    unpack_unit<KIND>(vr[i], y);
#pragma unroll
                    for (int e = 0; e < Unit<KIND>::UE / 8; ++e) {
                        const int to = r * 2 * D + (((c + e) ^ swz<D>(r)) << 4);
                        *reinterpret_cast<lds_f16x8*>(kt + to) = x[e];
                        *reinterpret_cast<lds_f16x8*>(vt + to) = y[e];
                    }
                }
            }
            if constexpr (SCALED) {
                const int r = tid & 127;
                if (r < BN) {
                    lds_u8* s = tid < 128 ? skt : svt;
#pragma unroll
                    for (int g = 0; g < NG; ++g)
                        *reinterpret_cast<__attribute__((address_space(3))) uint16_t*>(s + (g * BN + r) * 2) =
                            (uint16_t)(scr[g / 2] >> (16 * (g & 1)));
                }
            }
        };

        f32x16 o[DB] = {};
        float m = -__builtin_inff(), l = 0.f;               // m: raw scores; p = exp2((s - m) qscale + OFF)
        fetch(t0);
        for (int t = t0; t < t1; ++t) {
            __syncthreads();                                // the last tile (or sum) is read
            stage();
            if (t + 1 < t1) fetch(t + 1);
            __syncthreads();
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) {
                const int r32 = (kw * KB + kb) * 32;        // the block's first row in the tile
                const int j = t * BN + r32;
                f32x16 s = {};
                if constexpr (SCALED) {
#pragma unroll
                    for (int g = 0; g < NG; ++g) {
                        f32x16 acc = {};
#pragma unroll
                        for (int i = g * G / 16; i < (g + 1) * G / 16; ++i)
                            acc = mfma_32x32x16(lds_row8(kt + r32 * 2 * D, ad.k[i]), q[i], acc);
#pragma unroll
                        for (int v4 = 0; v4 < 4; ++v4) {
                            const f16x4 sc = *reinterpret_cast<__attribute__((address_space(3))) f16x4*>(skt + (g * BN + r32 + 8 * v4 + 4 * half) * 2);
#pragma unroll
                            for (int e = 0; e < 4; ++e) s[4 * v4 + e] = __builtin_fmaf(acc[4 * v4 + e], (float)sc[e], s[4 * v4 + e]);
                        }
                    }
                } else {
                    s = wide_scores<D>(kt + r32 * 2 * D, ad, q);
                }
                if (j + 32 > sq.ctx) {                      // drafts, or rows behind the sequence
                    const int d = sq.ctx - j;               // below 32: where the drafts begin
                    uint32_t seen = d > 0 ? ((1u << d) - 1u) | (uint32_t)(mask << d) : d > -64 ? (uint32_t)(mask >> -d) : 0u;
                    seen >>= 4 * half;
#pragma unroll
                    for (int v = 0; v < 16; ++v) s[v] = seen & (1u << (8 * (v / 4) + v % 4)) ? s[v] : -__builtin_inff();
                }
                float top = s[0];
#pragma unroll
                for (int v = 1; v < 16; ++v) top = fmaxf(top, s[v]);
                top = halves_max(top);
                if (__any((top - m) * a.qscale > WeightRange<KIND>::slack)) {   // also the first one: m = -inf
                    const float to = fmaxf(m, top);
                    const float f = to == m ? 1.f : fast_exp2((m - to) * a.qscale);
                    m = to;
                    l *= f;
#pragma unroll
                    for (int db = 0; db < DB; ++db) o[db] *= f;
                }
                const float base = m == -__builtin_inff() ? 0.f : m * a.qscale - WeightRange<KIND>::off;
#pragma unroll
                for (int v = 0; v < 16; ++v) {
                    s[v] = fast_exp2(__builtin_fmaf(s[v], a.qscale, -base));
                    l += s[v];
                }
                lds_u8* vb = vt + r32 * 2 * D;
                if constexpr (SCALED) {
#pragma unroll
                    for (int g = 0; g < NG; ++g) {
                        f16x8 p[2];
#pragma unroll
                        for (int v4 = 0; v4 < 4; ++v4) {
                            const f16x4 sc = *reinterpret_cast<__attribute__((address_space(3))) f16x4*>(svt + (g * BN + r32 + 8 * v4 + 4 * half) * 2);
#pragma unroll
                            for (int e = 0; e < 4; ++e) p[v4 / 2][4 * (v4 & 1) + e] = (_Float16)(s[4 * v4 + e] * (float)sc[e]);
                        }
#pragma unroll
                        for (int tt = 0; tt < 2; ++tt)
#pragma unroll
                            for (int db = g * G / 32; db < (g + 1) * G / 32; ++db) {
                                const uint32_t to = (uint32_t)(tt * 16 * 2 * D);
                                o[db] = mfma_32x32x16(lds_tr8(vb, ad.v[db][0] + to, ad.v[db][1] + to), p[tt], o[db]);
                            }
                    }
                } else {
                    f16x8 p[2];
#pragma unroll
                    for (int v = 0; v < 16; ++v) p[v / 8][v % 8] = (_Float16)s[v];
                    wide_values<D>(vb, ad, p, o);
                }
            }
        }
        l = halves_sum(l);
        if (bad) l = __builtin_nanf("");

        const bool whole = t0 == 0 && t1 == sq.tiles;
        const int slot = 2 * wg + (t0 == 0 ? 1 : 0);
        float* part = a.ws + (size_t)slot * BM * (D + 2);   // [BM][D] sums, then [BM][2] (m, l)
        const int r = qw * 32 + (lane & 31);
        uint16_t* out = a.out + (((size_t)b * a.T + node) * a.hkv * a.group + hq) * D;
        auto finish = [&](float mm, float ll, int d, float x0, float x1, float x2, float x3) {
            if (row >= rows) return;
            if (whole) {
                const float inv = ll == 0.f ? 0.f : 1.f / ll;
                const bool none = ll == 0.f;
                f16x4 w = {(_Float16)(none ? 0.f : x0 * inv), (_Float16)(none ? 0.f : x1 * inv),
                           (_Float16)(none ? 0.f : x2 * inv), (_Float16)(none ? 0.f : x3 * inv)};
                *reinterpret_cast<f16x4*>(out + d) = w;
            } else {
                *reinterpret_cast<f32x4*>(part + (size_t)r * D + d) = f32x4{x0, x1, x2, x3};
                if (d == 0) *reinterpret_cast<u32x2*>(part + (size_t)BM * D + 2 * r) =
                    u32x2{__builtin_bit_cast(uint32_t, mm * a.qscale), __builtin_bit_cast(uint32_t, ll)};
            }
        };
        if constexpr (KW == 1) {
#pragma unroll
            for (int db = 0; db < DB; ++db)
#pragma unroll
                for (int g = 0; g < 4; ++g)
                    finish(m, l, 32 * db + 8 * g + 4 * half, o[db][4 * g], o[db][4 * g + 1], o[db][4 * g + 2], o[db][4 * g + 3]);
        } else {
            // the KW waves of these rows: sums side by side in LDS, then each wave joins a part of the columns
            __syncthreads();
            __attribute__((address_space(3))) float* cs = (__attribute__((address_space(3))) float*)lds;
            constexpr int RS = D + 4;                       // row stride: rows four banks apart
            __attribute__((address_space(3))) float* mine = cs + (wave * 32 + (lane & 31)) * RS;
#pragma unroll
            for (int db = 0; db < DB; ++db)
#pragma unroll
                for (int g = 0; g < 4; ++g)
                    *reinterpret_cast<__attribute__((address_space(3))) f32x4*>(mine + 32 * db + 8 * g + 4 * half) =
                        f32x4{o[db][4 * g], o[db][4 * g + 1], o[db][4 * g + 2], o[db][4 * g + 3]};
            if (half == 0) {
                mine[D] = m;
                mine[D + 1] = l;
            }
            __syncthreads();
            float mm = -__builtin_inff();
#pragma unroll
            for (int k = 0; k < KW; ++k) mm = fmaxf(mm, cs[((k * QW + qw) * 32 + (lane & 31)) * RS + D]);
            float ll = 0.f, f[KW];
#pragma unroll
            for (int k = 0; k < KW; ++k) {
                const __attribute__((address_space(3))) float* x = cs + ((k * QW + qw) * 32 + (lane & 31)) * RS;
                f[k] = x[D] == mm ? 1.f : fast_exp2((x[D] - mm) * a.qscale);
                ll = __builtin_fmaf(f[k], x[D + 1], ll);
            }
            // (K/V-row wave kw, half) of 2 KW: columns 4 (kw 2 + half) + 8 KW i
#pragma unroll
            for (int i = 0; i < D / (8 * KW); ++i) {
                const int d = 4 * (kw * 2 + half) + 8 * KW * i;
                f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int k = 0; k < KW; ++k) {
                    const f32x4 x = *reinterpret_cast<__attribute__((address_space(3))) f32x4*>(cs + ((k * QW + qw) * 32 + (lane & 31)) * RS + d);
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[e] = __builtin_fmaf(f[k], x[e], s[e]);
                }
                finish(mm, ll, d, s[0], s[1], s[2], s[3]);
            }
        }
        at += t1 - t0;
    }
}

// Joins the pieces of the row blocks that several shares cut, and fills the rows that no
// work-group has: zeros for drafts behind a sequence's last one and for sequences of
// length 0, NaN for sequences whose lengths are out of range. A wave per output row.
template <int D, int QW>
__global__ __launch_bounds__(256) void tree_merge(TreeArgs a) {
    constexpr int BM = TreeTile<QW>::BM, BN = TreeTile<QW>::BN, E = D / 64;
    const int lane = (int)__lane_id();
    const int hq = a.hkv * a.group;
    const long long n = (long long)a.B * a.T * hq;
    const long long i = (long long)blockIdx.x * 4 + uniform((int)threadIdx.x >> 6);
    if (i >= n) return;
    const int b = (int)(i / (a.T * hq)), in = (int)(i - (long long)b * a.T * hq), node = in / hq, h = in - node * hq;
    uint16_t* out = a.out + (size_t)i * D + lane * E;
    const TreeSeq sq = tree_seq<BM, BN>(a, b);
    float x[E] = {};
    if (sq.bad) {
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = __builtin_nanf("");
    } else if (node < sq.n) {
        const int hk = h / a.group, r = node * a.group + (h - hk * a.group);
        const int share = tree_share(a, tree_units_below<BM, BN>(a, a.B));
        const int t0 = tree_units_below<BM, BN>(a, b) + (hk * sq.blocks + r / BM) * sq.tiles;
        const int w0 = t0 / share, w1 = (t0 + sq.tiles - 1) / share;
        if (w0 == w1) return;                               // finished by its work-group
        float m = -__builtin_inff(), l = 0.f;
        for (int w = w0; w <= w1; ++w) {
            const float* part = a.ws + (size_t)(2 * w + (w == w0 ? 1 : 0)) * BM * (D + 2);
            const float mw = part[(size_t)BM * D + 2 * (r % BM)], lw = part[(size_t)BM * D + 2 * (r % BM) + 1];
            const float to = fmaxf(m, mw);
            const float f = m == to ? 1.f : fast_exp2(m - to), g = mw == to ? 1.f : fast_exp2(mw - to);
            m = to;
            l = __builtin_fmaf(g, lw, l * f);
#pragma unroll
            for (int e = 0; e < E; ++e) x[e] = __builtin_fmaf(g, part[(size_t)(r % BM) * D + lane * E + e], x[e] * f);
        }
        const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = l == 0.f ? 0.f : x[e] * inv;
    }
#pragma unroll
    for (int e = 0; e < E; ++e) out[e] = f2h_rne(x[e]);
}

} // namespace va
