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
// KW = 4/QW over the K/V rows of a tile of BN. The sums are fp32, the weights are rounded
// to fp16 (RNE) for the second product, each off by at most 2^-11 of itself (see WeightRange for
// small ones), independently of each other, which adds to the output about the error of its own
// rounding to fp16. Scales, by the row block:
//   QW <= 2: a tile is fetched into registers while its predecessor is computed, unpacked
//     into LDS as exact fp16 codes and its group scales beside it; K's scales are applied to
//     each group's part of the dot product in fp32, V's to the weights (p * s is what is
//     rounded, relative to the largest scale so far: see WeightRange).
//   QW = 4: 128 rows share one unpacking, so the scales are applied there, which leaves the
//     waves' loop as it is for fp16 rows: K becomes two fp16 terms whose sum is code * scale
//     to 22 bits (twice the products of S, but no scaling of 128 x 64 scores per group), V is
//     rounded to fp16, each value off by at most 2^-11 of itself. Both are halved, in the codes,
//     where it is exact, so that code * scale up to 131008 fits; what is below fp16's normal numbers
//     there is off by 2^-24 at most. fp16 rows go straight to LDS (wide_walk).
// The output's error against 64 bits, in units of its own rounding to fp16 alone (44 x 58 drafts over
// 1985 positions, N(0, 1) rows): fp16 rows 1.38; 128-row blocks q8 1.70, q4 1.63, q3 1.50. There
// weights as two fp16 terms would give 1.42, 1.33 and 1.20, with a third more products:
// 24 x 32 drafts q4 138 -> 158 us; blocks of 64 rows, which round no V, 180 -> 272 us (8192 positions, q8).
// Measured (MI355X, D = 128): 24 x 32 drafts over up to 16384 positions q4 135 us (394 TFLOP/s
// of the two products; unpacking and K's second term bound it, the pieces' 11 us of joining
// next), 4 x 64 drafts over up to 8003 positions f16, 8 query heads to a K/V head, 61.5 us
// (493 TFLOP/s), one sequence's 16 drafts over 4096 positions q8 17.8 us (latency: a launch
// of two kernels, 2 tiles of work to a CU).
//
// Work split: the tiles of all (sequence, K/V head, row block), numbered one behind the
// other, are cut into equal shares, one to a work-group. A row block inside one share is
// finished there; the pieces of one that several shares cut go to ws (slot 2w: the
// piece that work-group w begins with, 2w + 1: the one it ends with) and tree_merge
// joins them.
//
// Tiles with drafts, or rows behind the sequence, are masked: see wide_clean for V's infinite
// and NaN values there.
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
// Four codes, one to a byte of w, as fp16 pairs 1024 + n, less 1024 + bias (HALF: half of that, 512 +
// n/2, less 512 + bias/2): exact.
template <bool HALF> __device__ __forceinline__ void bytes_to_f16(uint32_t w, float bias, f16x2& a, f16x2& b) {
    const _Float16 x = (_Float16)((1024.f + bias) * (HALF ? 0.5f : 1.f));
    const f16x2 z = {x, x};
    constexpr uint32_t HIGH = HALF ? 0x60606060u : 0x64646464u;
    a = as_f16x2(__builtin_amdgcn_perm(HIGH, w, 0x04010400u)) - z;
    b = as_f16x2(__builtin_amdgcn_perm(HIGH, w, 0x04030402u)) - z;
}
// A unit's values in order, as exact fp16 codes, or halves of codes (f16: the values).
template <int KIND, bool HALF>
__device__ __forceinline__ void unpack_unit(const Words<Unit<KIND>::W>& u, f16x8 (&out)[Unit<KIND>::UE / 8]) {
    if constexpr (KIND == KF16) {
        out[0] = __builtin_bit_cast(f16x8, u32x4{u.w[0], u.w[1], u.w[2], u.w[3]});
    } else if constexpr (KIND == KQ8) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            f16x2 a, b, c, d;
            bytes_to_f16<HALF>(u.w[2 * i] ^ 0x80808080u, 128.f, a, b);
            bytes_to_f16<HALF>(u.w[2 * i + 1] ^ 0x80808080u, 128.f, c, d);
            out[i] = join4(a, b, c, d);
        }
    } else if constexpr (KIND == KQ4) {
        constexpr float H = HALF ? 0.5f : 1.f;
        constexpr uint32_t LOW = HALF ? 0x60006000u : 0x64006400u;   // 512 + n/2, or 1024 + n
        const f16x2 lo = f16x2((_Float16)(1032.f * H)), hi = f16x2((_Float16)(72.f * H)), r16 = f16x2((_Float16)(0.0625f * H));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t w = u.w[i], x = w >> 8;
            // nibbles (0,4), (1,5), (2,6), (3,7): n - 8, the upper ones from 1024 + 16n
            const uint32_t p04 = __builtin_bit_cast(uint32_t, as_f16x2((w & 0x000F000Fu) | LOW) - lo);
            const uint32_t p15 = __builtin_bit_cast(uint32_t, as_f16x2((w & 0x00F000F0u) | 0x64006400u) * r16 - hi);
            const uint32_t p26 = __builtin_bit_cast(uint32_t, as_f16x2((x & 0x000F000Fu) | LOW) - lo);
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
            bytes_to_f16<HALF>(c[0], 4.f, a, b);
            bytes_to_f16<HALF>(c[1], 4.f, d, e);
            out[i] = join4(a, b, d, e);
        }
    }
}

template <int AUX> __device__ __forceinline__ u32x4 load128(__amdgpu_buffer_rsrc_t r, uint32_t off) {
    return __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, AUX);
}
template <int AUX> __device__ __forceinline__ u32x3 load96(__amdgpu_buffer_rsrc_t r, uint32_t off) {
    return __builtin_amdgcn_raw_buffer_load_b96(r, off, 0, AUX);
}

// The range of the weights' operand: the largest weight is held as 2^off at least and may grow
// by 2^slack before the maximum follows. SCALED: times V's group scale over a power of two
// 2^ve above every scale so far (see scale_top), so that the operand stays below 2^15 for any
// finite scale, and a product of weight and scale keeps fp16's 11 bits down to 2^-26 of the
// largest weight times the largest scale.
template <bool SCALED> struct WeightRange { static constexpr float off = WIDE_OFF, slack = WIDE_SLACK; };
template <> struct WeightRange<true> { static constexpr float off = 12.f, slack = 3.f; };

__device__ __forceinline__ f16x4 lds_scales(const lds_u8* p, uint32_t at) {
    return *reinterpret_cast<const __attribute__((address_space(3))) f16x4*>(p + at);
}

// ------------------------------------------------------------- work split --
// A sequence's part in the numbering: nothing for one without drafts or with lengths
// out of range (whose rows tree_merge fills).
struct TreeSeq {
    int ctx, n, len;      // len = ctx + n
    int tiles, blocks;    // K/V tiles, row blocks per K/V head
    bool bad;
    int first;            // the sequence's first tile in the numbering
};
// The numbering, by one wave: lane i has sequence b0 + i of the current 64.
template <int BM, int BN> struct TreePlan {
    const TreeArgs& a;
    int b0 = -1, ctx, n, upto = 0;               // upto: tiles up to and with the lane's sequence
    int total = 0;                               // of the batch
    __device__ __forceinline__ void make(TreeSeq& s) const {
        s.bad = s.ctx < 0 || s.n < 0 || s.n > a.T || s.ctx > a.cap - s.n;
        s.len = s.bad ? 0 : s.ctx + s.n;
        s.tiles = s.len / BN + (s.len % BN != 0);           // len + BN may pass 2^31, as (t + 1) * BN below
        s.blocks = s.bad ? 0 : (s.n * a.group + BM - 1) / BM;
    }
    __device__ __forceinline__ void load(int from, int before) {
        const int b = from + (int)__lane_id();
        TreeSeq s{};
        if (b < a.B) {
            s.ctx = a.ctx_lens[b];
            s.n = a.sizes ? a.sizes[b] : a.T;
        }
        make(s);
        b0 = from;
        ctx = s.ctx;
        n = s.n;
        upto = before + wave_scan(b < a.B ? s.tiles * s.blocks * a.hkv : 0);
    }
    __device__ __forceinline__ explicit TreePlan(const TreeArgs& args) : a(args) {
        for (int from = 0; from < a.B; from += 64) {
            load(from, total);
            total = __builtin_amdgcn_readlane(upto, 63);
        }
    }
    // Brings in the 64 that sequence b is among, or that tile `at` is in (b < 0).
    __device__ __forceinline__ void seek(int b, int at) {
        if (a.B <= 64) return;
        int before = 0;
        for (int from = 0; from < a.B; from += 64) {
            load(from, before);
            before = __builtin_amdgcn_readlane(upto, 63);
            if (b >= 0 ? b < from + 64 : at < before) return;
        }
    }
    __device__ __forceinline__ TreeSeq lane(int l) const {
        TreeSeq s;
        s.ctx = __builtin_amdgcn_readlane(ctx, l);
        s.n = __builtin_amdgcn_readlane(n, l);
        make(s);
        s.first = __builtin_amdgcn_readlane(upto, l) - s.tiles * s.blocks * a.hkv;
        return s;
    }
    __device__ __forceinline__ TreeSeq sequence(int b) {
        seek(b, 0);
        return lane(b - b0);
    }
    // The sequence that tile at < total is in.
    __device__ __forceinline__ TreeSeq at(int tile, int& b) {
        seek(-1, tile);
        const int l = __builtin_ctzll(__ballot(upto > tile));
        b = b0 + l;
        return lane(l);
    }
    __device__ __forceinline__ int share() const { return max((total + a.nwg - 1) / a.nwg, 1); }
    __device__ __forceinline__ int shares(int share) const { return (total + share - 1) / share; }
};

// --------------------------------------------------------------- kernel --
// The infinite and NaN ones of values c .. c + 3 of position j's V row, as its tile would hold
// them, 0 for the others.
template <int KIND, int D, int G, bool EXACT2>
__device__ __forceinline__ f32x4 tree_odd(const uint8_t* v, const uint16_t* sv, int page_shift, int num_pages, int hkv, int page, int hk, int j, int c) {
    f32x4 x = {};
    if (page < 0 || page >= num_pages) return x;
    const size_t r = (((size_t)page * hkv + hk) << page_shift) + (size_t)(j & ((1 << page_shift) - 1));
    const uint8_t* row = v + r * RowBytes<KIND, D>::value;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int d = c + e;
        if constexpr (KIND == KF16) {
            x[e] = wide_odd((float)reinterpret_cast<const _Float16*>(row)[d]);
        } else {
            int n;
            if constexpr (KIND == KQ8) n = (int8_t)row[d];
            else if constexpr (KIND == KQ4) n = ((row[d >> 1] >> (4 * (d & 1))) & 15) - 8;
            else {
                const uint8_t* p = row + 3 * (d >> 3);      // eight codes in 24 bits
                n = (int)(((uint32_t)p[0] | (uint32_t)p[1] << 8 | (uint32_t)p[2] << 16) >> (3 * (d & 7)) & 7u) - 4;
            }
            const _Float16 s = __builtin_bit_cast(_Float16, sv[r * (D / G) + d / G]);
            if constexpr (EXACT2) x[e] = wide_odd((float)((_Float16)(0.5f * (float)n) * s));
            else x[e] = wide_odd((float)s) == 0.f ? 0.f : (float)n * (float)s;
        }
    }
    return x;
}

// Work-groups that fit a CU (waves to a SIMD): their registers decide.
constexpr int tree_waves(int kind, int D, int qw) { return qw < 4 ? 2 : D == 128 || kind == KF16 ? 3 : 4; }
template <int QW> struct TreeTile {
    static constexpr int BM = 32 * QW, KW = 4 / QW;
    static constexpr int BN = QW == 1 ? 128 : 64;
    static constexpr int KB = BN / 32 / KW;                 // 32-row blocks of a tile per wave
};

template <int KIND, int D, int G, int QW>
__global__ __launch_bounds__(256, tree_waves(KIND, D, QW)) void tree_attend(TreeArgs a) {
    using T = TreeTile<QW>;
    constexpr int BM = T::BM, BN = T::BN, KW = T::KW, KB = T::KB;
    constexpr int KS = D / 16, DB = D / 32;
    constexpr int NG = KIND == KF16 ? 1 : D / G;            // scale groups of a row
    constexpr bool EXACT2 = KIND != KF16 && QW == 4;        // K as two fp16 terms
    constexpr bool SCALED = KIND != KF16 && !EXACT2;
    constexpr int ROWB = RowBytes<KIND, D>::value;
    constexpr int UPR = D / Unit<KIND>::UE;                 // units per row
    constexpr int UNITS = BN * UPR;                         // of one tensor's tile
    constexpr int UPT = (UNITS + 255) / 256;                // per lane
    constexpr int TILE = BN * 2 * D;
    // A tile is fetched while its predecessor is computed, or, by the widest row blocks, when it is
    // its turn: three work-groups fit a CU without its registers and cover each other's waits
    constexpr bool AHEAD = QW != 4;
    constexpr int AUX = QW == 4 ? 0 : VA_LOAD_AUX;      // the row blocks of a K/V head read the same rows
    using WR = WeightRange<SCALED>;
    constexpr int GP = QW == 1 ? 1 : NG > 2 ? 2 : NG, VP = GP;   // scale groups that are in registers at once
    constexpr int HALVES = BN / 64;                         // a page holds at least 64 rows
    constexpr int RSRCS = 256 / UPR > 64 ? 1 : HALVES;      // halves that a wave fetches from
    constexpr int SCB = SCALED ? NG * BN * 2 : 0;           // bytes of a tile's scales, [group][row]
    constexpr int TILES = (QW == 4 ? 3 : 2) * TILE + 2 * SCB;   // QW = 4: also K's second terms, or K of the next tile
    constexpr int ES = 68;                                  // epilogue: 64 columns of a row, the next four banks on
    constexpr int EPI = 4 * 32 * ES * 4;
    constexpr int LDS = TILES > EPI + 1024 ? TILES : EPI + 1024;
    __shared__ __align__(1024) uint8_t lds[LDS + 16];
    lds_int* odd = (lds_int*)((lds_u8*)lds + LDS);          // infinite or NaN values were left out
    lds_int* scale_top = odd + 1;                           // SCALED: the largest of V's scales so far in each half of a tile

    const int tid = (int)threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
    // the thread's number, made anew: what is computed from it is not held across loops
    auto fresh_tid = [&]() {
        int x = tid;
        asm volatile("" : "+v"(x));
        return x;
    };
    const int qw = wave % QW, kw = wave / QW;
    lds_u8* kt = (lds_u8*)lds;
    lds_u8* vt = kt + TILE;
    lds_u8* skt = vt + TILE;                                // scales, or K's second terms
    lds_u8* svt = skt + SCB;
    const float qs = a.qscale * (EXACT2 ? 2.f : 1.f);       // K and V are halved there
    WideAddr<D> ad0;
    ad0.init(lane, kw * KB * 32);

    if (tid == 0) *odd = 0;
    int wg = 0, at = 0, end = 0;
    do {                                                    // the pieces of the share; each finds its place anew
        const int lane = fresh_tid() & 63, half = lane >> 5;
        TreePlan<BM, BN> plan(a);                           // (holding the plan would cost the loop's registers)
        if (end == 0) {
            // consecutive shares on one XCD (work-groups are dealt to the eight in turn), as many on
            // each: the row blocks of a K/V head lie next to each other and read the same rows
            const int share = plan.share(), per = (plan.shares(share) + 7) >> 3;
            if ((int)(blockIdx.x >> 3) >= per) return;
            wg = (int)(blockIdx.x & 7) * per + (int)(blockIdx.x >> 3);
            at = wg * share;
            end = min(plan.total, at + share);
            if (at >= end) return;
        }
        int b;
        const TreeSeq sq = plan.at(at, b);
        const int in = at - sq.first, blk = in / sq.tiles;  // (K/V head, row block) of the sequence
        const int hk = uniform(blk / sq.blocks), rb = uniform(blk - hk * sq.blocks);
        const int t0 = uniform(in - blk * sq.tiles), t1 = uniform(min(sq.tiles, t0 + (end - at)));
        const uint32_t sat = (uint32_t)((kw * KB * 32 + 4 * half) * 2);   // the lane's scales in a group
        const int rows = sq.n * a.group;
        const int row = rb * BM + qw * 32 + (lane & 31);
        const int rc = min(row, rows - 1), node = rc / a.group, hq = hk * a.group + (rc - node * a.group);
        const uint64_t bits = a.mask[(size_t)b * a.T + node];
        f16x8 q[KS];
        {
            const uint16_t* qp = a.q + (((size_t)b * a.T + node) * a.hkv * a.group + hq) * D + 8 * half;
#pragma unroll
            for (int s = 0; s < KS; ++s) q[s] = *reinterpret_cast<const f16x8*>(qp + 16 * s);
        }
        const int32_t* table = a.block_table + (size_t)b * a.max_pages;

        Words<Unit<KIND>::W> kr[UPT], vr[UPT];
        uint32_t scr[2] = {0, 0};                           // lane's scales of K (lanes 0..127) or V
        uint32_t ksu[UPT], vsu[UPT];                        // EXACT2: of its units
        bool bad = false;
        auto fetch = [&](int t) {
            const int tid = fresh_tid(), lane = tid & 63;
            // the rows of each half of the tile, 64 to a page at least: pool row and how many there are
            size_t first_row[HALVES];
            int left[HALVES];
#pragma unroll
            for (int x = 0; x < HALVES; ++x) {
                const int j = t * BN + x * 64;
                left[x] = max(min(64, sq.len - t * BN - x * 64), 0);
                int page = left[x] > 0 ? table[j >> a.page_shift] : 0;
                if (page < 0 || page >= a.num_pages) {
                    bad = true;
                    left[x] = page = 0;
                }
                first_row[x] = (((size_t)page * a.hkv + hk) << a.page_shift) + (size_t)(j & ((1 << a.page_shift) - 1));
            }
            __amdgpu_buffer_rsrc_t rk[RSRCS], rv[RSRCS], rsk[RSRCS], rsv[RSRCS];
#pragma unroll
            for (int x = 0; x < RSRCS; ++x) {
                const bool up = RSRCS < HALVES ? wave >= 2 : x == 1;
                const size_t r = uniform64(up ? first_row[HALVES - 1] : first_row[0]);
                const uint32_t bytes = (uint32_t)(uniform(up ? left[HALVES - 1] : left[0]) * ROWB);
                rk[x] = make_rsrc(a.k + r * ROWB, bytes);
                rv[x] = make_rsrc(a.v + r * ROWB, bytes);
                if constexpr (EXACT2) {
                    rsk[x] = make_rsrc(a.sk + r * NG, bytes / ROWB * NG * 2);
                    rsv[x] = make_rsrc(a.sv + r * NG, bytes / ROWB * NG * 2);
                }
            }
#pragma unroll
            for (int i = 0; i < UPT; ++i) {
                const int u = i * 256 + tid, r = u / UPR, x = RSRCS == 1 ? 0 : (i * 256 / UPR) >> 6;
                const uint32_t off = (uint32_t)((r & 63) * ROWB + (u % UPR) * Unit<KIND>::UB);
                if (UNITS % 256 == 0 || u < UNITS) {
                    if constexpr (Unit<KIND>::W == 4) {
                        const u32x4 ka = load128<AUX>(rk[x], off), va = load128<AUX>(rv[x], off);
                        kr[i] = {{ka.x, ka.y, ka.z, ka.w}};
                        vr[i] = {{va.x, va.y, va.z, va.w}};
                    } else {
                        const u32x3 ka = load96<AUX>(rk[x], off), va = load96<AUX>(rv[x], off);
                        kr[i] = {{ka.x, ka.y, ka.z}};
                        vr[i] = {{va.x, va.y, va.z}};
                    }
                    if constexpr (EXACT2) {
                        const uint32_t so = (uint32_t)(((r & 63) * NG + (u % UPR) * Unit<KIND>::UE / G) * 2);
                        ksu[i] = ld16(rsk[x], so, 0);
                        vsu[i] = ld16(rsv[x], so, 0);
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
        int ve = -24;                                       // SCALED: V's scales so far are below 2^ve; else unused
        auto hides = [&](int t) { return t * BN > sq.ctx - BN; };   // drafts, or rows behind the sequence
        auto stage = [&](int t) {
            const int tid = fresh_tid();
            const bool clean = hides(t);
            bool any = false;
#pragma unroll
            for (int i = 0; i < UPT; ++i) {
                const int u = i * 256 + tid, r = u / UPR, c = (u % UPR) * (Unit<KIND>::UE / 8);
                if (UNITS % 256 == 0 || u < UNITS) {
                    f16x8 x[Unit<KIND>::UE / 8];
                    unpack_unit<KIND, EXACT2>(kr[i], x);
                    const f16x8 ks = EXACT2 ? f16x8(__builtin_bit_cast(_Float16, (uint16_t)ksu[i])) : f16x8{};
#pragma unroll
                    for (int e = 0; e < Unit<KIND>::UE / 8; ++e) {
                        const int to = r * 2 * D + (((c + e) ^ swz<D>(r)) << 4);
                        if constexpr (EXACT2) {
                            const f16x8 hi = x[e] * ks;
                            *reinterpret_cast<lds_f16x8*>(skt + to) = __builtin_elementwise_fma(x[e], ks, -hi);
                            x[e] = hi;
                        }
                        *reinterpret_cast<lds_f16x8*>(kt + to) = x[e];
                    }
                    if (!AHEAD) __builtin_amdgcn_sched_barrier(0);   // one operand's values in registers at a time
                    unpack_unit<KIND, EXACT2>(vr[i], x);
                    const f16x8 vs = EXACT2 ? f16x8(__builtin_bit_cast(_Float16, (uint16_t)vsu[i])) : f16x8{};
#pragma unroll
                    for (int e = 0; e < Unit<KIND>::UE / 8; ++e) {
                        const int to = r * 2 * D + (((c + e) ^ swz<D>(r)) << 4);
                        if constexpr (EXACT2) x[e] *= vs;
                        if constexpr (!SCALED) {
                            u32x4 y = __builtin_bit_cast(u32x4, x[e]);
                            if (clean) any |= wide_clean(y);
                            x[e] = __builtin_bit_cast(f16x8, y);
                        }
                        *reinterpret_cast<lds_f16x8*>(vt + to) = x[e];
                    }
                    if (!AHEAD) __builtin_amdgcn_sched_barrier(0);
                }
            }
            if constexpr (SCALED) {
                const int r = tid & 127;
                if (r < BN) {
                    lds_u8* s = tid < 128 ? skt : svt;
                    if (tid >= 128) {
                        u32x4 y = {scr[0], scr[1], 0u, 0u};
                        const bool odds = wide_clean(y);
                        if (clean) {                        // odd values of V are those of its scales
                            any = odds;
                            scr[0] = y.x;
                            scr[1] = y.y;
                        }
                        int top = 0;                        // as bits, which order like the values
#pragma unroll
                        for (int g = 0; g < NG; ++g) top = max(top, (int)(y[g / 2] >> (16 * (g & 1)) & 0x7FFFu));
                        // rarely one of 2^ve or more
                        const int limit = ve < -14 ? 1 << (ve + 24) : (ve + 15) << 10;
                        if (t == t0 || __any(top >= limit)) {
                            top = wave_scan_max(top);
                            if ((tid & 63) == 63) scale_top[(tid >> 6) & 1] = top;
                        }
                    }
#pragma unroll
                    for (int g = 0; g < NG; ++g)
                        *reinterpret_cast<__attribute__((address_space(3))) uint16_t*>(s + (g * BN + r) * 2) =
                            (uint16_t)(scr[g / 2] >> (16 * (g & 1)));
                }
            }
            if (any) *odd = 1;
        };

        // keeps the operands' loads ahead of the arithmetic that covers their latency; with few
        // query rows the fetches bound, and the registers are theirs
        auto order = []() {
            if constexpr (QW == 2) __builtin_amdgcn_sched_barrier(0);
        };
        f32x16 o[DB] = {};
        float m = -__builtin_inff(), l = 0.f;               // m: raw scores; p = exp2((s - m) qscale + OFF - ve); QW = 4: as wide_weights'
        if constexpr (AHEAD) fetch(t0);
        const uint64_t mask = sq.n < 64 ? bits & ((1ull << sq.n) - 1) : bits;
        // takes the positions that a row does not see out of a block of scores; d: where the drafts begin,
        // from the block's first position
        auto hide = [&](int d, f32x16& s) {
            if (d >= 32) return;                            // no drafts, nor rows behind the sequence
            uint32_t seen = d > 0 ? ((1u << d) - 1u) | (uint32_t)(mask << d) : d > -64 ? (uint32_t)(mask >> -d) : 0u;
            seen >>= 4 * half;
#pragma unroll
            for (int v = 0; v < 16; ++v) s[v] = seen & (1u << (8 * (v / 4) + v % 4)) ? s[v] : -__builtin_inff();
        };
        auto hide_tile = [&](int t, f32x16 (&s)[KB]) {
#pragma unroll
            for (int b = 0; b < KB; ++b) hide(sq.ctx - t * BN - 32 * b, s[b]);
        };
        if constexpr (KIND == KF16 && QW == 4) {
            size_t at = 0, next = 0;                        // pool row of the tile fetched, and of its successor
            int left = 0, ahead = 0;
            auto tile = [&](const uint8_t* pool, lds_u8* to) {
                WideFetch<D>(wave, fresh_tid() & 63, ROWB)(make_rsrc(pool + uniform64(at) * ROWB, (uint32_t)(uniform(left) * ROWB)), to);
            };
            auto seek = [&](int t) {
                const int j = t * BN;
                ahead = min(64, sq.len - j);
                int page = table[j >> a.page_shift];
                if (page < 0 || page >= a.num_pages) {
                    bad = true;
                    ahead = page = 0;
                }
                next = (((size_t)page * a.hkv + hk) << a.page_shift) + (size_t)(j & ((1 << a.page_shift) - 1));
            };
            seek(t0);
            __syncthreads();                                // the last piece's sums are read
            wide_walk<D, 2>(kt, ad0, q, t0, t1, qs,
                [&](int t, lds_u8* to) {
                    at = next;
                    left = ahead;
                    if (t + 1 < t1) seek(t + 1);
                    tile(a.k, to);
                },
                [&](int, lds_u8* to) { tile(a.v, to); },    // called before its successor's K is fetched
                hides, hide_tile, odd, m, l, o);
        } else if constexpr (QW == 4) {
            for (int t = t0; t < t1; ++t) {
                __syncthreads();                            // the last tile, or sums, are read
                fetch(t);
                stage(t);
                __syncthreads();
                const WideAddr<D> ad = ad0.fresh();
                f32x16 s[KB];
                wide_scores<D, KB, 2, true>(kt, skt, ad, q, s);
                hide_tile(t, s);
                f16x8 p[KB][2];
                wide_weights<D, KB>(s, qs, m, l, o, p);
                wide_values<D, KB>(vt, ad, p, o);
            }
        } else for (int t = t0; t < t1; ++t) {
            __syncthreads();                                // the last tile, or sums, are read
            stage(t);
            if (t + 1 < t1) fetch(t + 1);
            __syncthreads();
            int vtop = 0;                                   // used when the scores are there
            if constexpr (SCALED) vtop = HALVES == 2 ? max(scale_top[0], scale_top[1]) : scale_top[0];
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) {
                const WideAddr<D> ad = ad0.fresh();
                const uint32_t at32 = (uint32_t)(kb * 64 * D);   // the block's rows, in bytes
                f32x16 s = {};
                f16x8 kf[KS];
#pragma unroll
                for (int i = 0; i < KS; ++i) kf[i] = lds_row8(kt, ad.k(i) + at32);
                order();
                if constexpr (SCALED) {
#pragma unroll
                    for (int g0 = 0; g0 < NG; g0 += GP) {
                        f32x16 acc[GP] = {};
#pragma unroll
                        for (int i = 0; i < G / 16; ++i)
#pragma unroll
                            for (int g = 0; g < GP; ++g) acc[g] = mfma_32x32x16(kf[(g0 + g) * G / 16 + i], q[(g0 + g) * G / 16 + i], acc[g]);
                        order();
                        f16x4 sc[GP][4];
#pragma unroll
                        for (int g = 0; g < GP; ++g)
#pragma unroll
                            for (int v4 = 0; v4 < 4; ++v4) sc[g][v4] = lds_scales(skt, sat + (uint32_t)(((g0 + g) * BN + kb * 32 + 8 * v4) * 2));
#pragma unroll
                        for (int g = 0; g < GP; ++g)
#pragma unroll
                            for (int v = 0; v < 16; ++v) s[v] = __builtin_fmaf(acc[g][v], (float)sc[g][v / 4][v % 4], s[v]);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < KS; ++i) s = mfma_32x32x16(kf[i], q[i], s);
                }
                // V's operands are on their way while the weights are made
                order();
                f16x8 vf[2][DB];
#pragma unroll
                for (int tt = 0; tt < 2; ++tt)
#pragma unroll
                    for (int db = 0; db < DB; ++db) {
                        const uint32_t to = at32 + (uint32_t)(tt * 32 * D);
                        vf[tt][db] = lds_tr8(vt, ad.v(db, 0) + to, ad.v(db, 1) + to);
                    }
                f16x4 vsc[NG][4];
                if constexpr (SCALED) {
#pragma unroll
                    for (int g = 0; g < VP; ++g)
#pragma unroll
                        for (int v4 = 0; v4 < 4; ++v4) vsc[g][v4] = lds_scales(svt, sat + (uint32_t)((g * BN + kb * 32 + 8 * v4) * 2));
                }
                order();
                hide(sq.ctx - t * BN - (kw * KB + kb) * 32, s);
                float grown = 1.f;                          // 2^-(what ve grows by)
                if constexpr (SCALED) {
                    static_assert(KB == 1, "one rescale per tile");
                    const int to = (int)(__builtin_bit_cast(uint32_t, h2f((uint32_t)uniform(vtop))) >> 23) - 126;   // below 2^to
                    if (to > ve) {
                        grown = __builtin_bit_cast(float, (uint32_t)(127 + ve - to) << 23);
                        ve = to;
                    }
                }
                float top = s[0];
#pragma unroll
                for (int v = 1; v < 16; ++v) top = fmaxf(top, s[v]);
                top = halves_max(top);
                if (grown < 1.f || __any((top - m) * qs > WR::slack)) {   // also the first one: m = -inf
                    const float to = fmaxf(m, top);
                    const float f = (to == m ? 1.f : fast_exp2((m - to) * qs)) * grown;
                    m = to;
                    l *= f;
#pragma unroll
                    for (int db = 0; db < DB; ++db) o[db] *= f;
                }
                const float base = m == -__builtin_inff() ? 0.f : m * qs - WR::off + (SCALED ? (float)ve : 0.f);
#pragma unroll
                for (int v = 0; v < 16; ++v) {
                    s[v] = fast_exp2(__builtin_fmaf(s[v], qs, -base));
                    l += s[v];
                }
                f16x8 p[2];
                if constexpr (!SCALED) {
#pragma unroll
                    for (int v = 0; v < 16; ++v) p[v / 8][v % 8] = (_Float16)s[v];
                }
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    if constexpr (SCALED) {
                        if (g + VP < NG)
#pragma unroll
                            for (int v4 = 0; v4 < 4; ++v4) vsc[g + VP][v4] = lds_scales(svt, sat + (uint32_t)(((g + VP) * BN + kb * 32 + 8 * v4) * 2));
#pragma unroll
                        for (int v = 0; v < 16; ++v)    // + 0: one instruction, the product rounded to fp16 once
                            p[v / 8][v % 8] = (_Float16)__builtin_fmaf(s[v], (float)vsc[g][v / 4][v % 4], 0.f);
                    }
#pragma unroll
                    for (int tt = 0; tt < 2; ++tt)
#pragma unroll
                        for (int db = g * DB / NG; db < (g + 1) * DB / NG; ++db) o[db] = mfma_32x32x16(vf[tt][db], p[tt], o[db]);
                }
            }
        }
        l = halves_sum(l);
        if (bad) l = __builtin_nanf("");

        // The sums, 64 columns at a time, go through LDS: the KW waves of the same rows are joined
        // there, and a row leaves in one piece (a row per lane leaves 32 bytes at a time: one
        // sequence, 16 drafts over 4096 positions q8, 26.4 us with it).
        const bool whole = t0 == 0 && t1 == sq.tiles;
        const int slot = 2 * wg + (t0 == 0 ? 1 : 0);
        // [BM][D] sums, then [BM][2] (m, l). Of few rows they are written through to memory (sc1): what is
        // dirty in the L2s is written back when the kernel ends, which nothing covers there (one
        // sequence's 64 rows 17.5 us, 18.0 through the L2s). The widest blocks' pieces, begun and ended
        // at different times, go through the L2s (4 x 512 rows f16 62.5 us, 65.0 written through).
        constexpr int PART_AUX = QW == 4 ? 0 : 16;
        const __amdgpu_buffer_rsrc_t part = make_rsrc(a.ws + (size_t)uniform(slot) * BM * (D + 2), BM * (D + 2) * 4);
        __attribute__((address_space(3))) float* es = (__attribute__((address_space(3))) float*)lds;
        __attribute__((address_space(3))) float* ml = es + EPI / 4;     // [wave][32][2]
#pragma unroll
        for (int c0 = 0; c0 < D; c0 += 64) {
            const int tid = fresh_tid(), lane = tid & 63, half = lane >> 5;
            __syncthreads();
#pragma unroll
            for (int db = 0; db < 2; ++db)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const f32x16& x = o[c0 / 32 + db];
                    *reinterpret_cast<__attribute__((address_space(3))) f32x4*>(es + (wave * 32 + (lane & 31)) * ES + 32 * db + 8 * g + 4 * half) =
                        f32x4{x[4 * g], x[4 * g + 1], x[4 * g + 2], x[4 * g + 3]};
                }
            if (c0 == 0 && half == 0) {
                ml[(wave * 32 + lane) * 2] = m;
                ml[(wave * 32 + lane) * 2 + 1] = l;
            }
            __syncthreads();
            const int c = (tid & 15) * 4;
#pragma unroll 1
            for (int r0 = 0; r0 < BM; r0 += 16) {
                const int r = r0 + (tid >> 4), at0 = r & 31, w0 = r >> 5;
                float mm = ml[(w0 * 32 + at0) * 2], ll = ml[(w0 * 32 + at0) * 2 + 1];
                f32x4 x = *reinterpret_cast<__attribute__((address_space(3))) f32x4*>(es + (w0 * 32 + at0) * ES + c);
                if constexpr (KW > 1) {
                    const float m0 = mm;
#pragma unroll
                    for (int k = 1; k < KW; ++k) mm = fmaxf(mm, ml[((k * QW + w0) * 32 + at0) * 2]);
                    const float f0 = m0 == mm ? 1.f : fast_exp2((m0 - mm) * qs);
                    ll *= f0;
                    x *= f0;
#pragma unroll
                    for (int k = 1; k < KW; ++k) {
                        const int w = (k * QW + w0) * 32 + at0;
                        const float mk = ml[w * 2], f = mk == mm ? 1.f : fast_exp2((mk - mm) * qs);
                        const f32x4 y = *reinterpret_cast<__attribute__((address_space(3))) f32x4*>(es + w * ES + c);
                        ll = __builtin_fmaf(f, ml[w * 2 + 1], ll);
#pragma unroll
                        for (int e = 0; e < 4; ++e) x[e] = __builtin_fmaf(f, y[e], x[e]);
                    }
                }
                const int to = rb * BM + r;
                if (to >= rows) continue;
                if (EXACT2) x *= 2.f;
                if (SCALED) {                           // out of the units of 2^ve
                    const float f = __builtin_bit_cast(float, (uint32_t)(127 + ve) << 23);
                    ll *= f;
                    x *= f;
                }
                if (*odd) {                             // what was left out, to the rows that see it
                    const int nd = to / a.group;
                    const uint64_t bits = a.mask[(size_t)b * a.T + nd];
#pragma unroll 1
                    for (int j = max(t0, sq.ctx / BN) * BN; j < (t1 < sq.tiles ? t1 * BN : sq.len); ++j)
                        if (j < sq.ctx || (bits >> (j - sq.ctx) & 1)) 
                            x += tree_odd<KIND, D, G, EXACT2>(a.v, a.sv, a.page_shift, a.num_pages, a.hkv, table[j >> a.page_shift], hk, j, c0 + c);
                }
                if (whole) {
                    const float inv = ll == 0.f ? 0.f : 1.f / ll;
                    f16x4 y;
#pragma unroll
                    for (int e = 0; e < 4; ++e) y[e] = (_Float16)(ll == 0.f ? 0.f : x[e] * inv);
                    const int nd = to / a.group;
                    *reinterpret_cast<f16x4*>(a.out + (((size_t)b * a.T + nd) * a.hkv * a.group + hk * a.group + (to - nd * a.group)) * D + c0 + c) = y;
                } else {
                    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, x), part, (uint32_t)(r * D + c0 + c) * 4, 0, PART_AUX);
                    if (c0 == 0 && c == 0)
                        __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, (f32x2{QW == 4 ? mm : mm * qs, ll})), part, (uint32_t)(BM * D + 2 * r) * 4, 0, PART_AUX);
                }
            }
        }
        at += t1 - t0;
    } while (at < end);
}

// Joins the pieces of the row blocks that several shares cut (bound by reading them: 66 KB for each
// 128 rows; 11 us for the 24 x 32 drafts above), and fills the rows that no
// work-group has: zeros for drafts behind a sequence's last one and for sequences of
// length 0, NaN for sequences whose lengths are out of range. A work-group has 32/PW rows of
// one (sequence, K/V head), eight lanes to a row with D/8 columns each; PW of its waves
// share the pieces of the same rows (few rows, many pieces), joined through LDS.
template <int D, int QW, int PW>
__global__ __launch_bounds__(256) void tree_merge(TreeArgs a) {
    constexpr int BM = TreeTile<QW>::BM, BN = TreeTile<QW>::BN, V = D / 32, MR = 32 / PW;
    constexpr int U = 4;                                    // pieces in flight
    __shared__ float s_part[PW > 1 ? 4 * 8 * D : 1], s_ml[PW > 1 ? 4 * 8 * 2 : 1];
    const int lane = (int)__lane_id(), wave = uniform((int)threadIdx.x >> 6);
    const int all = a.T * a.group, per = (all + MR - 1) / MR;   // rows of a K/V head, work-groups
    const int bh = (int)blockIdx.x / per, b = bh / a.hkv, hk = bh - b * a.hkv;
    const int base = ((int)blockIdx.x - bh * per) * MR;     // MR rows never leave a row block
    const int row = base + (PW > 1 ? 0 : wave * 8) + (lane >> 3), r = row % BM, pw = PW > 1 ? wave : 0;
    TreePlan<BM, BN> plan(a);
    const TreeSeq sq = plan.sequence(b);
    const int rows = sq.bad ? 0 : sq.n * a.group;
    const int share = plan.share(), t0 = sq.first + (hk * sq.blocks + base / BM) * sq.tiles;
    const int w0 = t0 / share, w1 = (t0 + sq.tiles - 1) / share;
    if (base + MR <= rows && w0 == w1) return;              // finished by their work-group
    constexpr size_t STEP = (size_t)BM * (D + 2);
    const float* col = a.ws + (size_t)r * D + (lane & 7) * 4;
    const float* ml = a.ws + (size_t)BM * D + 2 * r;
    float m = -__builtin_inff(), l = 0.f;
    f32x4 x[V] = {};
    if (w0 != w1 && base < rows) {
        for (int p0 = w0 + pw; p0 <= w1; p0 += U * PW) {
            f32x2 s[U];
            f32x4 y[U][V];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int p = min(p0 + u * PW, w1);         // the last one again: not used
                const size_t at = (size_t)(2 * p + (p == w0 ? 1 : 0)) * STEP;
                s[u] = *reinterpret_cast<const f32x2*>(ml + at);
#pragma unroll
                for (int v = 0; v < V; ++v) y[u][v] = *reinterpret_cast<const f32x4*>(col + at + 32 * v);
            }
            float to = m;
#pragma unroll
            for (int u = 0; u < U; ++u) to = fmaxf(to, s[u].x);
            const float f = m == to ? 1.f : fast_exp2(m - to);
            m = to;
            l *= f;
#pragma unroll
            for (int v = 0; v < V; ++v) x[v] *= f;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (p0 + u * PW > w1) continue;
                const float g = s[u].x == to ? 1.f : fast_exp2(s[u].x - to);
                l = __builtin_fmaf(g, s[u].y, l);
#pragma unroll
                for (int v = 0; v < V; ++v)
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[v][e] = __builtin_fmaf(g, y[u][v][e], x[v][e]);
            }
        }
    }
    if constexpr (PW > 1) {
        float* mine = s_part + (wave * 8 + (lane >> 3)) * D + (lane & 7) * 4;
#pragma unroll
        for (int v = 0; v < V; ++v) *reinterpret_cast<f32x4*>(mine + 32 * v) = x[v];
        if ((lane & 7) == 0) {
            s_ml[(wave * 8 + (lane >> 3)) * 2] = m;
            s_ml[(wave * 8 + (lane >> 3)) * 2 + 1] = l;
        }
        __syncthreads();
        if (wave != 0) return;
        float to = m;
#pragma unroll
        for (int w = 1; w < PW; ++w) to = fmaxf(to, s_ml[(w * 8 + (lane >> 3)) * 2]);
        const float f = m == to ? 1.f : fast_exp2(m - to);
        l *= f;
#pragma unroll
        for (int v = 0; v < V; ++v) x[v] *= f;
#pragma unroll
        for (int w = 1; w < PW; ++w) {
            const float mw = s_ml[(w * 8 + (lane >> 3)) * 2], g = mw == to ? 1.f : fast_exp2(mw - to);
            l = __builtin_fmaf(g, s_ml[(w * 8 + (lane >> 3)) * 2 + 1], l);
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const f32x4 y = *reinterpret_cast<const f32x4*>(mine + w * 8 * D + 32 * v);
#pragma unroll
                for (int e = 0; e < 4; ++e) x[v][e] = __builtin_fmaf(g, y[e], x[v][e]);
            }
        }
    }
    if (row >= all || (row < rows && w0 == w1)) return;
    const int node = row / a.group;
    uint16_t* out = a.out + (((size_t)b * a.T + node) * a.hkv * a.group + hk * a.group + (row - node * a.group)) * D + (lane & 7) * 4;
    const float inv = l == 0.f ? 0.f : 1.f / l, none = sq.bad ? __builtin_nanf("") : 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        f16x4 y;
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = (_Float16)(row >= rows ? none : l == 0.f ? 0.f : x[v][e] * inv);
        *reinterpret_cast<f16x4*>(out + 32 * v) = y;
    }
}

} // namespace va
