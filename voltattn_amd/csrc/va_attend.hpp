// va_attend.hpp — attention of the newest tokens over a cache of e4m3 codes with a scale for
// each block of G positions and head (va_attend_paged).
//
// Sequence b has n new tokens (n = 1: a decode step) whose K/V rows are the last of its len
// positions. Row i attends positions 0 .. len - n + i:
//   o_i = sum_j p_ij sv_j v_j / sum_j p_ij,  p_ij = exp2(sk_j (q_i.k_j) log2(e)/sqrt(D) - m_i),
// with codes k, v and scales sk, sv that are one value for a whole tile, so that neither is
// applied to elements: K's goes into the factor of the scores, V's into the conversion of the
// codes to fp16 (v_cvt_scalef32, a power of two, exact) and what is left of it, in [1, 2), into
// the weights. Codes as fp16 are exact; sums, maxima and outputs are fp32. The weights are
// rounded to fp16 (RNE) for the second product, each off by at most 2^-11 of itself.
//
// The n * (Hq/Hkv) rows (token, head of the group) of a K/V head are cut into blocks; a block's
// work is the tiles of positions up to its last row's. Blocks have costs in units (a tile's and
// what it takes to begin one); all blocks' units, numbered one behind the other (sequence, K/V
// head, block), are cut into shares, one to a work-group, and a block's tiles go to the shares as its
// units do. The pieces of blocks that several shares cut go to ws (slot 2w: the piece that
// work-group w begins with, 2w + 1: the one it ends with) and attend_merge joins them.
#pragma once
#include "va_kernels.hpp"
#include "va_shares.hpp"
#include "va_wide.hpp"

namespace va {

typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) i32x2 lds_i32x2;
typedef __attribute__((address_space(3))) u32x4 lds_u32x4;
typedef __attribute__((address_space(3))) float lds_float;

// ------------------------------------------------------------- work split --
// The lane's (thread's) number, made anew: what is computed from it is not held across loops.
__device__ __forceinline__ int fresh(int x) {
    asm volatile("" : "+v"(x));
    return x;
}

// Constants that are not held in registers across loops either.
__device__ __forceinline__ float local_nan() {
    float x;
    asm volatile("v_mov_b32 %0, 0x7fc00000" : "=v"(x));
    return x;
}
__device__ __forceinline__ float local_minus_inf() {
    float x;
    asm volatile("v_mov_b32 %0, 0xff800000" : "=v"(x));
    return x;
}

// A block of BM rows of a sequence and K/V head; uniform. The rows are those between two consecutive
// bounds 0, cu[0], .., cu[B], total (each limited to what lies between its predecessor and total);
// those before the first and behind the last sequence (seq: -1), and of sequences whose lengths are
// out of range, are blocks of one tile that only store their rows.
template <int BM, int BN> struct AttendBlock {
    int seq, begin, n, len;
    int hk, rb;               // K/V head, block of rows
    int first, units, tiles;  // its first unit in the numbering, how many; its tiles
    static __device__ __forceinline__ int blocks(const AttendArgs& a, int n) { return (n * a.group + BM - 1) / BM; }
    static __device__ __forceinline__ bool bad(const AttendArgs& a, int seq, int len) { return seq < 0 || len < 0 || len > a.cap; }
    static __device__ __forceinline__ int tiles_of(const AttendArgs& a, int seq, int n, int len, int rb) {
        if (bad(a, seq, len)) return 1;
        const int i1 = min(n - 1, (int)a.by_group.div((uint32_t)(rb * BM + BM - 1)));
        const int seen = len - n + i1 + 1;       // positions that the block's last row sees
        return seen <= 0 ? 1 : (seen - 1) / BN + 1;
    }
    // The units of block rb are head + rb * slope, which for blocks that begin ever later is near its tiles.
    static __device__ __forceinline__ int head(const AttendArgs& a, int seq, int n, int len) {
        if (bad(a, seq, len)) return 1 << a.shift;
        return (tiles_of(a, seq, n, len, n <= len ? 0 : max(blocks(a, n), 1) - 1) + a.setup) << a.shift;
    }
    static __device__ __forceinline__ int slope(const AttendArgs& a, int seq, int n, int len) { return bad(a, seq, len) || n > len ? 0 : a.slope; }
    __device__ __forceinline__ bool bad(const AttendArgs& a) const { return bad(a, seq, len); }
    __device__ __forceinline__ void size(const AttendArgs& a) {
        units = uniform(head(a, seq, n, len) + rb * slope(a, seq, n, len));
        tiles = uniform(tiles_of(a, seq, n, len, rb));
    }
    // The block behind this one, unless that is another sequence's.
    __device__ __forceinline__ bool next(const AttendArgs& a) {
        if (rb + 1 < blocks(a, n)) ++rb;
        else if (hk + 1 < a.hkv) {
            ++hk;
            rb = 0;
        } else return false;
        first += units;
        size(a);
        return true;
    }
    // The tiles ahead of unit first + x.
    __device__ __forceinline__ int ahead(const AttendArgs& a, int x) const { return tiles_ahead(x, units, tiles, a.shift); }
};

// The numbering, by one wave: lane i has span from + i of the current 64.
template <int BM, int BN> struct AttendPlan {
    using Block = AttendBlock<BM, BN>;
    const AttendArgs& a;
    int from = -1, before = 0, prev = 0;         // before: units ahead of the 64; prev: the bound ahead of the next ones
    int begin = 0, n = 0, len = 0;
    int count = 0, upto = 0;                     // units of the lane's span, and up to and with it
    int total = 0;                               // units of the batch
    __device__ __forceinline__ int spans() const { return a.cu ? a.B + 2 : a.B; }
    __device__ __forceinline__ int seq_of(int i) const { return !a.cu ? (i < a.B ? i : -1) : i >= 1 && i <= a.B ? i - 1 : -1; }
    static __device__ __forceinline__ int ahead(int head, int slope, int rb) { return rb * head + (int)((long long)rb * (rb - 1) / 2) * slope; }   // units of blocks 0 .. rb - 1
    __device__ __forceinline__ void load(int at, int units, int bound) {
        from = at;
        before = units;
        const int i = at + (fresh((int)threadIdx.x) & 63);
        const int seq = seq_of(i);
        len = seq >= 0 ? a.seq_lens[seq] : 0;
        if (a.cu) {
            int e = i <= a.B ? a.cu[i] : a.total;
            e = max(0, min(e, a.total));
            e = max(bound, wave_scan_max(e));    // bounds never fall back
            begin = __builtin_amdgcn_update_dpp(bound, e, 0x138, 0xF, 0xF, false);   // wave shift right by one
            n = i <= a.B + 1 ? e - begin : 0;
            prev = __builtin_amdgcn_readlane(e, 63);
        } else {
            begin = i;
            n = i < a.B;
        }
        count = ahead(Block::head(a, seq, n, len), Block::slope(a, seq, n, len), Block::blocks(a, n)) * a.hkv;
        upto = before + wave_scan(count);
    }
    // all: counts the batch's units (else only to find blocks)
    __device__ __forceinline__ explicit AttendPlan(const AttendArgs& args, bool all = true) : a(args) {
        for (int at = 0; at < (all ? spans() : 1); at += 64) {
            load(at, total, prev);
            total = __builtin_amdgcn_readlane(upto, 63);
        }
    }
    // The block that unit `at` < total is in.
    __device__ __forceinline__ Block find(int at) {
        if (spans() > 64) {                      // on from the last block's, if this one is behind it
            if (at < before) load(0, 0, 0);
            while (at >= __builtin_amdgcn_readlane(upto, 63)) load(from + 64, __builtin_amdgcn_readlane(upto, 63), prev);
        }
        const int l = __builtin_ctzll(__ballot(upto > at));
        Block b;
        b.seq = seq_of(from + l);
        b.begin = __builtin_amdgcn_readlane(begin, l);
        b.n = __builtin_amdgcn_readlane(n, l);
        b.len = __builtin_amdgcn_readlane(len, l);
        const int nb = Block::blocks(a, b.n), of = __builtin_amdgcn_readlane(count, l), per = of / a.hkv;
        const int head = Block::head(a, b.seq, b.n, b.len), slope = Block::slope(a, b.seq, b.n, b.len);
        const int start = __builtin_amdgcn_readlane(upto, l) - of;
        b.hk = uniform((at - start) / per);
        const int in = at - start - b.hk * per;
        b.rb = 0;
        for (int step = nb; step > 1;) {         // the last block whose units begin at `in` or before: among step from rb on
            step = (step + 63) / 64;
            const int rb = b.rb + (fresh((int)threadIdx.x) & 63) * step;
            b.rb += step * (__builtin_popcountll(__ballot(rb < nb && ahead(head, slope, rb) <= in)) - 1);
        }
        b.rb = uniform(b.rb);
        b.first = uniform(start + b.hk * per + ahead(head, slope, b.rb));
        b.size(a);
        return b;
    }
    __device__ __forceinline__ Shares<BM> shares() const { return Shares<BM>{total, a.nwg, a.shift}; }
};

// What attend_merge has to know of work-group w, behind the pieces in ws: whether it begins a block
// that others go on with (its rows, else 0; its first token, K/V head and number), and whether it goes
// on with one (head: 1, and 2 if it ends it).
struct AttendNote {
    int rows, begin, hk, rb;
    int head, unused[3];
};
template <int D, int BM> __device__ __forceinline__ AttendNote* attend_note(const AttendArgs& a, int w) {
    return reinterpret_cast<AttendNote*>(a.ws + (size_t)2 * a.nwg * BM * (D + 2)) + w;
}
template <int D, int BM, int BN> __device__ __forceinline__ void attend_write_note(const AttendArgs& a, int w, const AttendBlock<BM, BN>& b, int t0, int t1) {
    AttendNote* to = attend_note<D, BM>(a, w);
    if (t0 == 0) *reinterpret_cast<i32x4*>(to) = i32x4{min(BM, b.n * a.group - b.rb * BM), b.begin, b.hk, b.rb};
    else to->head = t1 == b.tiles ? 2 : 1;
}
// The share of a work-group; its note is empty at first.
template <int D, int BM, int BN> struct AttendShare {
    int wg, at, end;
    __device__ __forceinline__ AttendShare(const AttendArgs& a, const AttendPlan<BM, BN>& plan) {
        const Shares<BM> shares = plan.shares();
        const int per = (shares.shares() + 7) >> 3, x = (int)blockIdx.x & 7, j = (int)blockIdx.x >> 3;   // neighbours on one XCD
        wg = j < per ? x * per + j : 8 * per + x * ((int)(gridDim.x >> 3) - per) + j - per;
        if (wg < a.nwg && threadIdx.x == 0) {
            i32x4* to = reinterpret_cast<i32x4*>(attend_note<D, BM>(a, wg));
            to[0] = to[1] = i32x4{};
        }
        at = j < per ? uniform(shares.start(wg)) : 0;
        end = j < per ? uniform(shares.start(wg + 1)) : 0;
    }
};

// -------------------------------------------------------------- cache tiles --
// Where the tiles of a sequence's K/V head lie: lane i has tile base + i of STEP positions at
// BASE positions from the tile's start on; scales as two fp16 (of its halves, if G is less than STEP).
template <int STEP, int G> struct Places {
    int base = -1, page = -1;
    uint32_t sk = 0, sv = 0;
    // at: position of tile `first`'s part, `stride` positions from tile to tile; those from `end` on are not looked at
    __device__ __forceinline__ void load(const AttendArgs& a, const int32_t* table, int hk, int tile, int tiles, int stride, int off, int end) {
        base = tile;
        const int t = tile + (fresh((int)threadIdx.x) & 63);
        const long long j64 = (long long)t * stride + off;
        const bool on = t < tiles && j64 < end;
        const int j = on ? (int)j64 : 0;
        page = on ? table[j >> a.page_shift] : -1;
        if (page < 0 || page >= a.num_pages) page = -1;
        sk = sv = 0;
        if (page >= 0) {
            const size_t at = ((((size_t)page * a.hkv + hk) << a.page_shift) + (size_t)(j & ((1 << a.page_shift) - 1))) / G;
            if constexpr (STEP > G) {
                const uint32_t own = end - j <= G ? 0xFFFFu : 0xFFFFFFFFu;   // what lies behind the last position is not the sequence's
                sk = *reinterpret_cast<const uint32_t*>(a.sk + at) & own;
                sv = *reinterpret_cast<const uint32_t*>(a.sv + at) & own;
            } else {
                sk = a.sk[at] * 0x10001u;
                sv = a.sv[at] * 0x10001u;
            }
        }
    }
};

// A tile's part under one pair of scales, all uniform: K's scale times the scores' factor, V's
// scale as 2^(e + more), 0 <= more < 1, and whether the part has no finite values (a page outside
// the pool, a scale that is infinite or NaN): rows that see it are NaN. `more` goes into the
// exponent of the weights, and what it adds to their sum is taken out with less = 2^-more.
struct Scales {
    float qs, more, less;
    int e;                // NONE: V's scale is 0
    bool bad;
    static constexpr int NONE = -1000;
    __device__ __forceinline__ void set(uint32_t sk, uint32_t sv, float qscale, bool there) {
        sk &= 0x7FFFu;
        sv &= 0x7FFFu;
        bad = !there || sk >= 0x7C00u || sv >= 0x7C00u;
        const uint32_t k = bad ? 0u : wide_bits(sk), v = bad ? 0u : wide_bits(sv);
        // a hidden position's score is -infinity, which a factor of 0 would make NaN
        qs = uniformf(qscale * __builtin_bit_cast(float, k ? k : 0x0D800000u));      // 2^-100
        e = v ? (int)(v >> 23) - 127 : NONE;
        more = 0.f;
        less = 1.f;
        if (v & 0x7FFFFFu) {                     // no power of two
            const float x = __builtin_bit_cast(float, (v & 0x7FFFFFu) | 0x3F800000u);
            more = uniformf(__builtin_amdgcn_logf(x));
            less = uniformf(1.f / x);
        }
    }
    // The bits of a finite fp16 number's fp32 value, on the scalar unit.
    static __device__ __forceinline__ uint32_t wide_bits(uint32_t h) {
        if (h >= 0x400u) return (h << 13) + (112u << 23);
        if (h == 0) return 0;
        const int p = 31 - __builtin_clz(h);     // h 2^-24, its highest bit 2^p
        return ((uint32_t)(p + 103) << 23) + ((h << (23 - p)) & 0x7FFFFFu);
    }
};
__device__ __forceinline__ float power(int e) { return __builtin_bit_cast(float, (uint32_t)(127 + e) << 23); }   // -126 <= e <= 127

// The output's sums are in units of 2^unit. A part's codes go to fp16 times 2^(e - unit), exact for
// -15 <= e - unit <= 7 (an e4m3 code is a multiple of 2^-9 below 2^9, an fp16 number one of 2^-24
// below 2^16); another unit is taken where a part needs it.
__device__ __forceinline__ bool unit_fits(const Scales& s, int unit) {
    const int d = s.e - unit;
    return s.e == Scales::NONE || (d >= -15 && d <= 7);
}
__device__ __forceinline__ int unit_for(const Scales& s, int unit) { return unit_fits(s, unit) ? unit : s.e; }
// One for both parts of a tile: where their scales are more than 2^22 apart, the smaller one's excess
// goes to its weights (which keep their 11 bits down to 2^-7 of a row's largest then).
__device__ __forceinline__ int unit_for(Scales (&s)[2], int unit) {
    if (unit_fits(s[0], unit) && unit_fits(s[1], unit)) return unit;
    const int top = max(s[0].e, s[1].e), low = min(s[0].e, s[1].e);   // not both NONE
    const int u = low == Scales::NONE ? top : max(top - 7, min(top, low + 15));
#pragma unroll
    for (int b = 0; b < 2; ++b)
        if (s[b].e != Scales::NONE && s[b].e < u - 15) {
            s[b].more += (float)(s[b].e - u + 15);
            s[b].less *= power(u - 15 - s[b].e);
            s[b].e = u - 15;
        }
    return u;
}
__device__ __forceinline__ float factor_of(const Scales& s, int unit) { return power(s.e == Scales::NONE ? -120 : s.e - unit); }

// Four codes as fp16, times the power of two f.
__device__ __forceinline__ void codes_to_f16(uint32_t w, float f, f16x2& a, f16x2& b) {
    a = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, f, false));
    b = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, f, true));
}
__device__ __forceinline__ f16x8 codes_to_f16x8(uint32_t w0, uint32_t w1, float f) {
    f16x2 a, b, c, d;
    codes_to_f16(w0, f, a, b);
    codes_to_f16(w1, f, c, d);
    return f16x8{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}
// Takes the NaN codes out of w (0 in their place); whether there were any. They are the only values
// that are not finite, and 0 times them is NaN: tiles that some row does not wholly see go into the
// product without them, and the rows that see them become NaN afterwards.
__device__ __forceinline__ bool codes_clean(u32x4& w) {
    uint32_t any = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const uint32_t odd = ((w[e] & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;   // 0x7F carries into bit 7
        w[e] &= ~(odd | (odd - (odd >> 7)));
        any |= odd;
    }
    return any != 0;
}
// Which of the codes c .. c + 3 of position j's V row are NaN, a bit to each.
template <int D>
__device__ __forceinline__ uint32_t attend_odd(const AttendArgs& a, const int32_t* table, int hk, int j, int c) {
    const int page = table[j >> a.page_shift];
    if (page < 0 || page >= a.num_pages) return 0;
    const size_t r = (((size_t)page * a.hkv + hk) << a.page_shift) + (size_t)(j & ((1 << a.page_shift) - 1));
    const uint32_t w = *reinterpret_cast<const uint32_t*>(a.v + r * D + c);
    uint32_t nan = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) nan |= (((w >> (8 * e)) & 0x7Fu) == 0x7Fu ? 1u : 0u) << e;
    return nan;
}

// The lazy maximum, as WIDE_OFF and WIDE_SLACK, with room for the part of V's scale below 2.
constexpr float ATT_OFF = 10.f, ATT_SLACK = 4.f;

// A weight is exp2 of a fused product less the maximum, whose product was rounded: where the maximum is far from 0,
// digits that only one of the two has are whole powers of two (from 2^27 on weights would pass fp16's range, from 2^30
// on the largest may become 0), and `more` is lost in the maximum's last step. A wave with a row whose maximum is far
// therefore makes its scores less the maximum first, of products rounded once. (Scores far from a maximum that is not
// have the weight 0.) No model has such scores; whether there are any is looked at where a maximum grows. (10 prompts'
// chunks 645 us without, 651 with it; 8 K tokens over 32 K positions 3674 and 3689.)
constexpr float ATT_FAR = 4096.f;
__device__ __forceinline__ bool is_far(float m) { return __builtin_fabsf(m) >= ATT_FAR && m != -__builtin_inff(); }
__device__ __forceinline__ float rounded_product(float x, float y) {
#pragma clang fp contract(off)
    return x * y;
}
// The lazy maximum's next value. Its last step may be more than ATT_OFF.
__device__ __forceinline__ float next_max(float m, float top) {
    const float to = fmaxf(m, top - ATT_OFF);
    return top - to > ATT_OFF + ATT_SLACK ? top : to;
}

// ---------------------------------------------------------------- one or few rows --
// Block: 16 NB rows as columns of 16x16x32 products; the four waves take 32 positions each of a tile
// of 128, every wave by itself until the piece ends. K comes from memory in the operand's layout
// (a lane has 16 bytes of a row, dimensions 16h .. and 64 + 16h ..: the k index is a free
// permutation, and q is laid out likewise); V is transposed through the wave's own LDS with
// ds_read_b64_tr_b8 (lane i of 16 addresses half i%2 of row i/2 and receives column i of the eight
// rows; probed on MI355X). A lane's slots of the second product are the positions whose scores it
// holds: 4h + 0..3 and 16 + 4h + 0..3.
//
// Bound by memory: 32 heads over 64 K positions (537 MB) 85 us, 6.3 TB/s of the 7.3 that plain reads reach; 64
// sequences over up to 8 K positions (303 MB) 56 us, where every work-group begins two blocks; one token over
// 4 K positions 7 us, the chain of lengths, table, scales and tile. Three work-groups on a CU (161 registers,
// one V tile ahead) do 64 K positions in 91 us.

template <int D> __device__ __forceinline__ int few_swz(int row) {
    return D == 128 ? ((row >> 1) & 1) | ((row >> 4) & 1) << 1 | ((row >> 2) & 1) << 2 : ((row >> 4) & 1) | ((row >> 2) & 1) << 1;
}

template <int D, int G, int NB>
__global__ __launch_bounds__(256, 2) void attend_few(AttendArgs a) {
    constexpr int BM = 16 * NB, BN = 128, KC = D / 64, DT = D / 16, VL = D / 32;   // 16-byte loads of a lane per 16 rows of K, of V's 32 rows
    constexpr int VB = 32 * D;                               // bytes of a wave's V part
    constexpr int VAHEAD = NB > 1 && D == 128 ? 1 : 2;       // V tiles on their way (K: 2): what the registers hold
    constexpr int ES = D + 4;                                // epilogue: floats of a row, the next four banks on
    constexpr int EPI = 4 * 16 * ES * 4, ML = 4 * 16 * 2 * 4;
    constexpr int LDS = 4 * VB > EPI + ML ? 4 * VB : EPI + ML;
    __shared__ __align__(1024) uint8_t lds[LDS + 16];
    lds_int* odds = (lds_int*)((lds_u8*)lds + LDS);          // of each wave, in the epilogue: whether it has left out NaN codes

    const int tid = (int)threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), h = lane >> 4, c16 = lane & 15;
    lds_u8* vt = (lds_u8*)lds + wave * VB;
    AttendPlan<BM, BN> plan(a);
    const AttendShare<D, BM, BN> share(a, plan);
    const int wg = share.wg, end = share.end;
    int at = share.at;
    AttendBlock<BM, BN> blk;
    blk.tiles = 0;

    auto fresh_lane = [&]() { return fresh(lane); };
    while (at < end) {
        if (blk.tiles == 0 || !blk.next(a)) blk = plan.find(at);
        const int hk = blk.hk, rb = blk.rb, n = blk.n, begin = blk.begin, seq = blk.seq, len = blk.len, tiles = blk.tiles;
        const int t0 = uniform(blk.ahead(a, at - blk.first)), t1 = uniform(blk.ahead(a, end - blk.first));
        const int rows = n * a.group, hq = a.hkv * a.group;
        at = uniform(min(end, blk.first + blk.units));
        if (t0 >= t1) continue;
        if (blk.bad(a)) {
            const float x = seq < 0 ? 0.f : __builtin_nanf("");
            for (int i = fresh(tid); i < BM * (D / 8); i += 256) {
                const int r = rb * BM + i / (D / 8);
                if (r >= rows) break;
                const int tok = (int)a.by_group.div((uint32_t)r);
                *reinterpret_cast<f16x8*>(a.out + ((size_t)(begin + tok) * hq + hk * a.group + (r - tok * a.group)) * D + (i % (D / 8)) * 8) = f16x8((_Float16)x);
            }
            continue;
        }
        const int ctx = len - n;
        const int32_t* table = a.block_table + (size_t)seq * a.max_pages;
        f16x8 q[NB][D / 32];
        int last[NB];                                        // the last position that the lane's row sees
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const int r = min(rb * BM + b * 16 + c16, rows - 1), tok = (int)a.by_group.div((uint32_t)r);
            last[b] = ctx + tok;
            const uint16_t* qp = a.q + ((size_t)(begin + tok) * hq + hk * a.group + (r - tok * a.group)) * D + 16 * h;
#pragma unroll
            for (int s = 0; s < D / 32; ++s) q[b][s] = *reinterpret_cast<const f16x8*>(qp + (s >> 1) * 64 + (s & 1) * 8);
        }
        const int all = ctx + (int)a.by_group.div((uint32_t)min(rb * BM, rows - 1));   // every row sees positions up to this one

        Places<32, G> pl;
        u32x4 kr[2][2 * KC], vr[VAHEAD][VL];
        size_t vat[2];                                       // V of the tiles fetched
        uint32_t vbytes[2];
        Scales sc[2];
        bool on[2] = {false, false};
        auto fetch_v = [&](int b) {
            const __amdgpu_buffer_rsrc_t rv = make_rsrc(a.v + vat[b], vbytes[b]);
#pragma unroll
            for (int i = 0; i < VL; ++i) vr[b % VAHEAD][i] = ld128(rv, (uint32_t)(i * 1024 + fresh_lane() * 16), 0);
        };
        auto fetch_rows = [&](int t, int b) {
            if (t >= pl.base + 64 || pl.base < 0) pl.load(a, table, hk, t, t1, BN, wave * 32, len);
            const int l = t - pl.base, page = __builtin_amdgcn_readlane(pl.page, l), j = t * BN + wave * 32;
            const int left = page < 0 ? 0 : max(0, min(32, len - j));
            on[b] = j < len;
            const size_t row = uniform64((((size_t)(page < 0 ? 0 : page) * a.hkv + hk) << a.page_shift) + (size_t)(j & ((1 << a.page_shift) - 1)));
            const uint32_t bytes = (uint32_t)(uniform(left) * D);
            const __amdgpu_buffer_rsrc_t rk = make_rsrc(a.k + row * D, bytes);
            vat[b] = row * D;
            vbytes[b] = bytes;
            const int lane = fresh_lane(), h = lane >> 4, c16 = lane & 15;
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int c = 0; c < KC; ++c) kr[b][i * KC + c] = ld128(rk, (uint32_t)((16 * i + c16) * D + 64 * c + 16 * h), 0);
            if (VAHEAD == 2) fetch_v(b);
        };
        auto scales_of = [&](int t, int b) {
            const int l = t - pl.base;
            sc[b].set((uint32_t)__builtin_amdgcn_readlane((int)pl.sk, l), (uint32_t)__builtin_amdgcn_readlane((int)pl.sv, l), a.qscale,
                      __builtin_amdgcn_readlane(pl.page, l) >= 0);
        };
        auto fetch = [&](int t, int b) {
            fetch_rows(t, b);
            scales_of(t, b);
        };
        f32x4 o[NB][DT] = {};
        float m[NB], l[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            m[b] = -__builtin_inff();
            l[b] = 0.f;
        }
        int unit = 0, far = 0;                               // far: some row's maximum is
        bool odd = false;                                    // this lane has left out NaN codes
        auto tile = [&](int t, int b) {
            if (!on[b]) return;                              // nothing there, nor behind it: uniform
            const int j0 = t * BN + wave * 32;
            const Scales s = sc[b];
            const int lane = fresh_lane(), h = lane >> 4, c16 = lane & 15;
            // LDS addresses: the lane's V chunks as they arrived (row of load 0; each load is 1024 / D rows
            // on), and its half rows for the transposing reads
            const int vrow = lane * 16 / D, vchunk = lane % (D / 16);
            const int trow = c16 / 2 < 4 ? 4 * h + c16 / 2 : 12 + 4 * h + c16 / 2;
            const int tr0 = trow * D + (c16 & 1) * 8, trx = few_swz<D>(trow);
            f32x4 x[2][NB] = {};
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int c = 0; c < KC; ++c) {
                    const u32x4 w = kr[b][i * KC + c];
                    const f16x8 k0 = codes_to_f16x8(w.x, w.y, 1.f), k1 = codes_to_f16x8(w.z, w.w, 1.f);
#pragma unroll
                    for (int y = 0; y < NB; ++y) {
                        x[i][y] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, q[y][2 * c], x[i][y], 0, 0, 0);
                        x[i][y] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, q[y][2 * c + 1], x[i][y], 0, 0, 0);
                    }
                }
            const bool hides = j0 + 31 > all;
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < VL; ++i) {
                u32x4 w = vr[b % VAHEAD][i];
                if (hides) odd |= codes_clean(w);
                const int row = vrow + i * (1024 / D);
                *reinterpret_cast<lds_u32x4*>(vt + row * D + ((vchunk ^ few_swz<D>(row)) << 4)) = w;
            }
            if (VAHEAD == 1 && t + 1 < t1) fetch_v(b ^ 1);
            if (s.bad) {
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int y = 0; y < NB; ++y) x[i][y] = f32x4{__builtin_nanf(""), __builtin_nanf(""), __builtin_nanf(""), __builtin_nanf("")};
            }
            if (hides) {
#pragma unroll
                for (int y = 0; y < NB; ++y)
#pragma unroll
                    for (int i = 0; i < 2; ++i)
#pragma unroll
                        for (int v = 0; v < 4; ++v) x[i][y][v] = j0 + 16 * i + 4 * h + v > last[y] ? -__builtin_inff() : x[i][y][v];
            }
            float top[NB];
            bool grows = false;
#pragma unroll
            for (int y = 0; y < NB; ++y) {
                top[y] = x[0][y][0];
#pragma unroll
                for (int e = 1; e < 8; ++e) top[y] = fmaxf(top[y], x[e / 4][y][e % 4]);
                top[y] = rounded_product(rows_max(top[y]), s.qs);
                grows |= top[y] - m[y] > ATT_OFF + ATT_SLACK;    // also at the first one: m = -inf
            }
            const int to_unit = unit_for(s, unit);
            if (__any(grows) || to_unit != unit) {
                const float u = power(unit - to_unit);
                unit = to_unit;
                bool away = false;
#pragma unroll
                for (int y = 0; y < NB; ++y) {
                    const float to = next_max(m[y], top[y]), f = to == m[y] ? 1.f : fast_exp2(m[y] - to);
                    m[y] = to;
                    l[y] *= f;
#pragma unroll
                    for (int d = 0; d < DT; ++d) o[y][d] *= f * u;
                    away |= is_far(m[y]);
                }
                far = __any(away);
            }
            if (__builtin_expect(far, 0)) {                  // from here on the scores are less the maximum
#pragma unroll
                for (int y = 0; y < NB; ++y)
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[e / 4][y][e % 4] = rounded_product(x[e / 4][y][e % 4], s.qs) - (m[y] == -__builtin_inff() ? 0.f : m[y]);
            }
            const float qs = uniformf(far ? 1.f : s.qs);
            f16x8 p[NB];
#pragma unroll
            for (int y = 0; y < NB; ++y) {
                const float up = s.more - (far || m[y] == -__builtin_inff() ? 0.f : m[y]);
                float sum = 0.f;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float w = fast_exp2(__builtin_fmaf(x[e / 4][y][e % 4], qs, up));
                    sum += w;
                    p[y][e] = (_Float16)w;
                }
                l[y] = __builtin_fmaf(sum, s.less, l[y]);
            }
            const float f = factor_of(s, unit);
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                const i32x2 w = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i32x2*)(vt + tr0 + ((d ^ trx) << 4)));
                const f16x8 vv = codes_to_f16x8((uint32_t)w.x, (uint32_t)w.y, f);
#pragma unroll
                for (int y = 0; y < NB; ++y) o[y][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vv, p[y], o[y][d], 0, 0, 0);
            }
        };
        fetch_rows(t0, 0);                                   // the first rows do not wait for their scales
        if (VAHEAD == 1) fetch_v(0);
        if (t0 + 1 < t1) fetch_rows(t0 + 1, 1);
        scales_of(t0, 0);
        if (t0 + 1 < t1) scales_of(t0 + 1, 1);
        int t = t0;
        do {
            tile(t, 0);
            if (t + 2 < t1) fetch(t + 2, 0);
            if (t + 1 < t1) tile(t + 1, 1);
            if (t + 3 < t1) fetch(t + 3, 1);
            t += 2;
        } while (t < t1);

        const bool whole = t0 == 0 && t1 == tiles;
        if (!whole && fresh(tid) == 0) attend_write_note<D, BM, BN>(a, wg, blk, t0, t1);
        float* part = a.ws + (size_t)(2 * wg + (t0 == 0 ? 1 : 0)) * BM * (D + 2);   // [BM][D] sums, then [BM][2] (m, l)
        lds_float* es = (lds_float*)lds;
        lds_float* ml = es + EPI / 4;
        const float scale = power(unit);
        odds[wave] = __any(odd) != 0;                        // read between this epilogue's barriers only: nothing to clear
#pragma unroll
        for (int y = 0; y < NB; ++y) {
            const float ly = rows_sum(l[y]);
            __syncthreads();
#pragma unroll
            for (int d = 0; d < DT; ++d) *reinterpret_cast<__attribute__((address_space(3))) f32x4*>(es + (wave * 16 + c16) * ES + 16 * d + 4 * h) = o[y][d] * scale;
            if (h == 0) {
                ml[(wave * 16 + c16) * 2] = m[y];
                ml[(wave * 16 + c16) * 2 + 1] = ly;
            }
            __syncthreads();
            const i32x4 left = *reinterpret_cast<__attribute__((address_space(3))) i32x4*>(odds);
            const bool any = uniform(left.x | left.y | left.z | left.w) != 0;
            for (int i = tid; i < 16 * (D / 4); i += 256) {
                const int r = i / (D / 4), c = i % (D / 4) * 4, to = rb * BM + y * 16 + r;
                if (to >= rows) break;
                float mm = ml[r * 2];
#pragma unroll
                for (int w = 1; w < 4; ++w) mm = fmaxf(mm, ml[(w * 16 + r) * 2]);
                float ll = 0.f;
                f32x4 x = {};
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const float mw = ml[(w * 16 + r) * 2], f = mw == mm ? 1.f : fast_exp2(mw - mm);
                    ll = __builtin_fmaf(f, ml[(w * 16 + r) * 2 + 1], ll);
                    const f32x4 z = *reinterpret_cast<__attribute__((address_space(3))) f32x4*>(es + (w * 16 + r) * ES + c);
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[e] = __builtin_fmaf(f, z[e], x[e]);
                }
                const int tok = (int)a.by_group.div((uint32_t)to);
                if (any) {                                   // NaN codes that were left out, to the rows that see them
                    uint32_t nan = 0;
                    for (int j = max(max(t0 * BN, all + 1 - BN), 0); j <= min(ctx + tok, t1 * BN - 1); ++j) nan |= attend_odd<D>(a, table, hk, j, c);
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[e] = nan >> e & 1 ? __builtin_nanf("") : x[e];
                }
                if (whole) {
                    const float inv = ll == 0.f ? 0.f : 1.f / ll;
                    f16x4 w;
#pragma unroll
                    for (int e = 0; e < 4; ++e) w[e] = (_Float16)(ll == 0.f ? 0.f : x[e] * inv);
                    *reinterpret_cast<f16x4*>(a.out + ((size_t)(begin + tok) * hq + hk * a.group + (to - tok * a.group)) * D + c) = w;
                } else {
                    *reinterpret_cast<f32x4*>(part + (y * 16 + r) * D + c) = x;
                    if (c == 0) *reinterpret_cast<f32x2*>(part + BM * D + 2 * (y * 16 + r)) = f32x2{mm, ll};
                }
            }
        }
        __syncthreads();                                     // the sums are read, odds too
    }
}

// ----------------------------------------------------------------- many rows --
// Block: 128 CB rows, 32 CB to a wave as the columns of 32x32x16 products (S^T = K Q^T, O^T = V^T P^T,
// lane layout as in va_wide.hpp). A tile of 64 positions comes straight to LDS as codes (16 KB of K and
// V) while its predecessor is computed, and every wave turns them into fp16 as it reads its operands.
// K: a lane reads 16 codes of its row, two steps' worth (chunk 2j + half: the k index is a free
// permutation, q is laid out likewise). V: ds_read_b64_tr_b8, the slots of wide_values' positions.
// The 16-byte chunks of a row lie XORed with wide_swz_k / wide_swz_v, so that neither read meets a
// bank twice. CB = 2: every operand, once converted, feeds two products; more than half of the wave's
// query operands wait in LDS (step by step, 16 bytes of each lane), which its registers do not hold
// beside the sums of 64 rows.
//
// A wave's products go before the other waves' weights (s_setprio): they need the issue port for a
// moment each and the matrix cores for long; without it the oldest wave of a SIMD goes first, the
// others fall behind, and the last work-groups of a CU finish alone (8 K tokens over 32 K positions: 4336
// us without, 3998 with it, before shares went by age).
//
// Bound by the matrix cores and what shares the issue port with them: those 8 K tokens (32 heads, 8 K/V
// heads of 128 dimensions) take 3690 to 3780 us, 1020 to 1040 TFLOP/s at the 1.9 GHz that the power allows; a
// large product of the library does 1173 to 1465.
//
// A lane has two score blocks of 32 positions at a time: both halves of a tile against one row (CB =
// 1), or one half against a row of each group (CB = 2).
template <int D> __device__ __forceinline__ int wide_swz_k(int row) { return D == 128 ? (row >> 1) & 7 : (row >> 2) & 3; }
template <int D> __device__ __forceinline__ int wide_swz_v(int row) {
    return D == 128 ? ((row >> 1) & 1) << 1 | ((row >> 3) & 1) << 2 : ((row >> 3) & 1) << 1;
}

// Steps whose query operands of the first group are in registers.
constexpr int wide_steps(int D, int CB) { return CB == 2 && D == 128 ? 5 : D / 16; }

// S^T; at: the tile's K (CB = 2: the half's); q2: this lane's query operands in LDS, the first group's
// that are not in registers, and the second group's.
// The next step's reads are on their way while a step's codes are converted and multiplied.
template <int D, int CB>
__device__ __forceinline__ void wide_keys(const lds_u8* k, uint32_t at, const f16x8 (&q)[wide_steps(D, CB)], const lds_u8* q2, f32x16 (&s)[2]) {
    s[0] = s[1] = f32x16{};
    if constexpr (CB == 1) {
        u32x4 w[2][2];
        auto read = [&](int j) {
#pragma unroll
            for (int b = 0; b < 2; ++b) w[j & 1][b] = *reinterpret_cast<const lds_u32x4*>(k + (at ^ (uint32_t)(j << 5)) + b * 32 * D);
        };
        read(0);
#pragma unroll
        for (int j = 0; j < D / 32; ++j) {
            __builtin_amdgcn_sched_barrier(0);
            if (j + 1 < D / 32) read(j + 1);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int b = 0; b < 2; ++b) s[b] = mfma_32x32x16(codes_to_f16x8(w[j & 1][b][2 * x], w[j & 1][b][2 * x + 1], 1.f), q[2 * j + x], s[b]);
        }
    } else {
        constexpr int KS = D / 16, QR = wide_steps(D, CB);
        u32x4 w[2];
        f16x8 z[2][2];
        auto read_k = [&](int j) { w[j & 1] = *reinterpret_cast<const lds_u32x4*>(k + (at ^ (uint32_t)(j << 5))); };
        auto read_q = [&](int i) {
            z[i & 1][1] = lds_row8(q2, (uint32_t)((KS - QR + i) * 1024));
            if (i >= QR) z[i & 1][0] = lds_row8(q2, (uint32_t)((i - QR) * 1024));
        };
        read_k(0);
        read_q(0);
#pragma unroll
        for (int i = 0; i < KS; ++i) {
            __builtin_amdgcn_sched_barrier(0);
            if (i % 2 == 0 && i / 2 + 1 < KS / 2) read_k(i / 2 + 1);
            if (i + 1 < KS) read_q(i + 1);
            __builtin_amdgcn_sched_barrier(0);
            const f16x8 y = codes_to_f16x8(w[(i >> 1) & 1][2 * (i & 1)], w[(i >> 1) & 1][2 * (i & 1) + 1], 1.f);
            s[0] = mfma_32x32x16(y, i < QR ? q[i < QR ? i : 0] : z[i & 1][0], s[0]);
            s[1] = mfma_32x32x16(y, z[i & 1][1], s[1]);
        }
    }
    __builtin_amdgcn_sched_barrier(0);
}
// O^T += V^T P^T; at: the tile's V (CB = 2: the half's); f: what the blocks' codes are multiplied by.
template <int D, int CB>
__device__ __forceinline__ void wide_sums(lds_u8* v, uint32_t at, const float (&f)[2], const f16x8 (&p)[2][2], f32x16 (&o)[CB][D / 32]) {
    constexpr int DB = D / 32, N = 4 / CB;                   // 16 positions to a step
    i32x2 w[2][DB];
    auto read = [&](int i) {
#pragma unroll
        for (int db = 0; db < DB; ++db)
            w[i & 1][db] = __builtin_amdgcn_ds_read_tr8_b64_v2i32(reinterpret_cast<lds_i32x2*>(v + (at ^ (uint32_t)(db << 5)) + i * 16 * D));
    };
    read(0);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        __builtin_amdgcn_sched_barrier(0);
        if (i + 1 < N) read(i + 1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int db = 0; db < DB; ++db) {
            const f16x8 y = codes_to_f16x8((uint32_t)w[i & 1][db].x, (uint32_t)w[i & 1][db].y, f[CB == 1 ? i >> 1 : 0]);
            o[0][db] = mfma_32x32x16(y, p[CB == 1 ? i >> 1 : 0][i & 1], o[0][db]);
            if constexpr (CB == 2) o[1][db] = mfma_32x32x16(y, p[1][i & 1], o[1][db]);
        }
    }
    __builtin_amdgcn_sched_barrier(0);
}
// The weights of two score blocks: of one row under the scales sc[0] and sc[1] (CB = 1), or of two rows
// under sc[0]. The maxima and the unit of the sums follow where they have to.
template <int D, int CB>
__device__ __forceinline__ void wide_softmax(f32x16 (&s)[2], const Scales* sc, int to_unit, int& unit, int& far, float (&m)[CB], float (&l)[CB],
                                             f32x16 (&o)[CB][D / 32], f16x8 (&p)[2][2]) {
    float top[CB];
#pragma unroll
    for (int c = 0; c < CB; ++c) top[c] = -__builtin_inff();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        float x = s[i][0];
#pragma unroll
        for (int v = 1; v < 16; ++v) x = fmaxf(x, s[i][v]);
        const int c = CB == 1 ? 0 : i;
        top[c] = fmaxf(top[c], rounded_product(x, sc[CB == 1 ? i : 0].qs));
    }
    bool grows = false;
#pragma unroll
    for (int c = 0; c < CB; ++c) {
        top[c] = halves_max(top[c]);
        grows |= top[c] - m[c] > ATT_OFF + ATT_SLACK;        // also at the first one: m = -inf
    }
    if (__any(grows) || to_unit != unit) {
        const float u = power(unit - to_unit);
        unit = to_unit;
        bool away = false;
#pragma unroll
        for (int c = 0; c < CB; ++c) {
            const float to = next_max(m[c], top[c]), f = to == m[c] ? 1.f : fast_exp2(m[c] - to);
            m[c] = to;
            l[c] *= f;
            const float g = f * u;
#pragma unroll
            for (int db = 0; db < D / 32; ++db) o[c][db] *= g;
            away |= is_far(m[c]);
        }
        far = __any(away);
    }
    if (__builtin_expect(far, 0)) {                          // from here on the scores are less the maximum
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int c = CB == 1 ? 0 : i;
#pragma unroll
            for (int v = 0; v < 16; ++v) s[i][v] = rounded_product(s[i][v], sc[CB == 1 ? i : 0].qs) - (m[c] == -__builtin_inff() ? 0.f : m[c]);
        }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int c = CB == 1 ? 0 : i;
        const Scales& x = sc[CB == 1 ? i : 0];
        const float qs = uniformf(far ? 1.f : x.qs), up = x.more - (far || m[c] == -__builtin_inff() ? 0.f : m[c]);
        float sum = 0.f;
#pragma unroll
        for (int v = 0; v < 16; ++v) {
            const float w = fast_exp2(__builtin_fmaf(s[i][v], qs, up));
            sum += w;
            p[i][v / 8][v % 8] = (_Float16)w;
        }
        l[c] = __builtin_fmaf(sum, x.less, l[c]);
    }
}

template <int D, int G, int CB>
__global__ __launch_bounds__(256, CB == 1 ? 3 : 2) void attend_wide(AttendArgs a) {
    constexpr int BM = 128 * CB, BN = 64, KS = D / 16, DB = D / 32, RAW = BN * D, N = RAW / 4096;
    constexpr int QR = wide_steps(D, CB), QB = (CB * KS - QR) * 1024;   // bytes of a wave's query operands in LDS
    __shared__ __align__(1024) uint8_t lds[4 * RAW + 4 * QB];   // K of two tiles, V of two
    lds_u8* kt = (lds_u8*)lds;
    lds_u8* vt = kt + 2 * RAW;

    const int tid = (int)threadIdx.x, wave = uniform(tid >> 6);
    lds_u8* q2 = vt + 2 * RAW + wave * QB;
    auto fresh_lane = [&]() { return fresh(tid) & 63; };
    // addresses of the lane's operands in a tile, and in q2
    auto key_at = [&](int tile) {
        const int x = fresh_lane(), row = x & 31;
        return (uint32_t)(tile + row * D + (((x >> 5) ^ wide_swz_k<D>(row)) << 4));
    };
    auto value_at = [&](int tile) {
        const int x = fresh_lane(), e = (x & 15) >> 1, pos = 4 * (x >> 5) + (e & 3) + 8 * (e >> 2);
        return (uint32_t)(tile + pos * D + ((((x >> 4) & 1) ^ wide_swz_v<D>(pos)) << 4) + (x & 1) * 8);
    };
    int at = 0, end = 0, wg = 0;
    AttendBlock<BM, BN> blk;
    blk.tiles = 0;
    do {
        if (blk.tiles == 0 || !blk.next(a)) {
            AttendPlan<BM, BN> plan(a, end == 0);            // (holding the plan would cost the loop's registers)
            if (end == 0) {
                const AttendShare<D, BM, BN> share(a, plan);
                wg = share.wg;
                at = share.at;
                end = share.end;
                if (at >= end) return;
            }
            blk = plan.find(at);
        }
        const int hk = blk.hk, rb = blk.rb, n = blk.n, begin = blk.begin, seq = blk.seq, len = blk.len, tiles = blk.tiles;
        const int t0 = uniform(blk.ahead(a, at - blk.first)), t1 = uniform(blk.ahead(a, end - blk.first));
        const int rows = n * a.group, hq = a.hkv * a.group;
        at = uniform(min(end, blk.first + blk.units));
        if (t0 >= t1) continue;
        if (blk.bad(a)) {
            const float x = seq < 0 ? 0.f : __builtin_nanf("");
            for (int i = fresh(tid); i < BM * (D / 8); i += 256) {
                const int r = rb * BM + i / (D / 8);
                if (r >= rows) break;
                const int tok = (int)a.by_group.div((uint32_t)r);
                *reinterpret_cast<f16x8*>(a.out + ((size_t)(begin + tok) * hq + hk * a.group + (r - tok * a.group)) * D + (i % (D / 8)) * 8) = f16x8((_Float16)x);
            }
            continue;
        }
        const int ctx = len - n;
        const int32_t* table = a.block_table + (size_t)seq * a.max_pages;
        // the wave's rows; the work-groups of a CU begin with different waves, so that the few rows of
        // short blocks do not all meet on one SIMD
        const int row0 = uniform(rb * BM + ((wave + (int)(blockIdx.x >> 8)) & 3) * CB * 32);
        // the lane's row of the block in the wave's group c
        auto row_of = [&](int c, int& half, int& row, int& rc, int& tok) {
            const int x = fresh_lane();
            half = x >> 5;
            row = row0 + c * 32 + (x & 31);
            rc = min(row, rows - 1);
            tok = (int)a.by_group.div((uint32_t)rc);
        };
        const int all = ctx + (int)a.by_group.div((uint32_t)(rb * BM));                                       // that every row of the block sees
        const int mine = ctx + (int)a.by_group.div((uint32_t)min(row0, rows - 1));                            // .. of the wave
        const int most = row0 < rows ? ctx + (int)a.by_group.div((uint32_t)min(row0 + CB * 32, rows) - 1u) : -1;   // that some row of the wave sees
        f16x8 q[QR];
#pragma unroll
        for (int c = CB - 1; c >= 0; --c) {
            int half, row, rc, tok;
            row_of(c, half, row, rc, tok);
            const uint16_t* qp = a.q + ((size_t)(begin + tok) * hq + hk * a.group + (rc - tok * a.group)) * D + 16 * half;
            lds_u8* to = q2 + fresh_lane() * 16;
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                const f16x8 x = *reinterpret_cast<const f16x8*>(qp + (s >> 1) * 32 + (s & 1) * 8);
                if (c == 0 && s < QR) q[s < QR ? s : 0] = x;
                else *reinterpret_cast<lds_f16x8*>(to + (c == 1 ? KS - QR + s : s - QR) * 1024) = x;
            }
        }
        Places<64, G> pl;
        uint32_t sk = 0, sv = 0;                             // of the tile that is fetched
        bool there = false;
        auto fetch = [&](int t, int to) {
            if (pl.base < 0 || t >= pl.base + 64) pl.load(a, table, hk, t, t1, BN, 0, len);
            const int x = t - pl.base, page = __builtin_amdgcn_readlane(pl.page, x), j = t * BN;
            sk = (uint32_t)__builtin_amdgcn_readlane((int)pl.sk, x);
            sv = (uint32_t)__builtin_amdgcn_readlane((int)pl.sv, x);
            there = page >= 0;
            const uint32_t bytes = (uint32_t)(there ? max(0, min(BN, len - j)) : 0) * D;
            const size_t r = ((((size_t)(there ? page : 0) * a.hkv + hk) << a.page_shift) + (size_t)(j & ((1 << a.page_shift) - 1))) * D;
            const __amdgpu_buffer_rsrc_t k = make_rsrc(a.k + uniform64(r), uniform((int)bytes)), v = make_rsrc(a.v + uniform64(r), uniform((int)bytes));
            // the lane's place in LDS, and the chunk that belongs there; the next KB's is the same with another XOR
            const int lane = fresh_lane(), off = wave * N * 1024, row = (off + lane * 16) / D, c = lane % (D / 16);
            const uint32_t kc = (uint32_t)(row * D + ((c ^ wide_swz_k<D>(row)) << 4)), vc = (uint32_t)(row * D + ((c ^ wide_swz_v<D>(row)) << 4));
#pragma unroll
            for (int i = 0; i < N; ++i) {
                static_assert(D == 128 || N == 1, "1 KB is 8 rows: bit 2 of row >> 1, bit 0 of row >> 3");
                __builtin_amdgcn_raw_ptr_buffer_load_lds(k, kt + to + off + i * 1024, 16, (kc ^ (uint32_t)(i << 6)) + (uint32_t)(i * 1024), 0, 0, 0);
                __builtin_amdgcn_raw_ptr_buffer_load_lds(v, vt + to + off + i * 1024, 16, (vc ^ (uint32_t)(i << 6)) + (uint32_t)(i * 1024), 0, 0, 0);
            }
        };
        f32x16 o[CB][DB] = {};
        float m[CB], l[CB];
#pragma unroll
        for (int c = 0; c < CB; ++c) {
            m[c] = -__builtin_inff();
            l[c] = 0.f;
        }
        int unit = 0, far = 0;                               // far: some row's maximum is
        bool odd = false;                                    // this wave has left out NaN codes
        __syncthreads();                                     // the last piece's tiles are read
        fetch(t0, 0);
        // tile t is there, for every wave; its successor is on its way
        auto arrive = [&](int t, int cur) {
            __builtin_amdgcn_sched_barrier(0);
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __builtin_amdgcn_sched_barrier(0);
            if (t * BN + BN - 1 > all) {                     // positions that some row of the block does not see
                lds_u32x4* p = reinterpret_cast<lds_u32x4*>(vt + cur + wave * (N * 1024)) + fresh_lane();
                bool any = false;
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    u32x4 w = p[i * 64];
                    if (codes_clean(w)) {
                        any = true;
                        p[i * 64] = w;
                    }
                }
                odd |= __any(any) != 0;
            }
            __builtin_amdgcn_sched_barrier(0);
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
            __builtin_amdgcn_sched_barrier(0);
            if (t + 1 < t1) fetch(t + 1, cur ^ RAW);
        };
        const int tw = most < 0 ? t0 : max(t0, min(t1, most / BN + 1));   // tiles that this wave sees a part of
        int t = t0, cur = 0;
        for (; t < tw; ++t, cur ^= RAW) {
            Scales sc[2];
            sc[0].set(sk & 0xFFFFu, sv & 0xFFFFu, a.qscale, there);
            sc[1].set(sk >> 16, sv >> 16, a.qscale, there);
            const int to_unit = unit_for(sc, unit);
            arrive(t, cur);
#pragma unroll
            for (int h = 0; h < CB; ++h) {                   // CB = 2: half by half
                f32x16 s[2];
                __builtin_amdgcn_s_setprio(1);
                wide_keys<D, CB>(kt, key_at(cur) + (uint32_t)(h * 32 * D), q, q2 + (QB ? fresh_lane() * 16 : 0), s);
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    if (sc[CB == 1 ? i : h].bad) s[i] = f32x16(local_nan());
                if (t * BN + BN - 1 > mine) {
                    const float hidden = local_minus_inf();
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        int half, row, rc, tok;
                        row_of(CB == 1 ? 0 : i, half, row, rc, tok);
                        const int lim = ctx + tok - t * BN - 32 * (CB == 1 ? i : h) - 4 * half;   // the last position that the row sees, from the lane's first one
#pragma unroll
                        for (int v = 0; v < 16; ++v) s[i][v] = 8 * (v / 4) + v % 4 > lim ? hidden : s[i][v];
                    }
                }
                f16x8 p[2][2];
                __builtin_amdgcn_s_setprio(0);
                wide_softmax<D, CB>(s, sc + (CB == 1 ? 0 : h), to_unit, unit, far, m, l, o, p);
                __builtin_amdgcn_s_setprio(1);
                const float f[2] = {factor_of(sc[CB == 1 ? 0 : h], unit), factor_of(sc[1], unit)};
                wide_sums<D, CB>(vt, value_at(cur) + (uint32_t)(h * 32 * D), f, p, o);
            }
            __builtin_amdgcn_s_setprio(0);
        }
        for (; t < t1; ++t, cur ^= RAW) arrive(t, cur);
        const bool whole = t0 == 0 && t1 == tiles;
        if (!whole && fresh(tid) == 0) attend_write_note<D, BM, BN>(a, wg, blk, t0, t1);
        __syncthreads();                                     // the last tile is read
        if ((fresh(tid) & 63) == 0) reinterpret_cast<lds_int*>(kt)[wave] = odd;
        __syncthreads();
        bool any = false;                                    // some wave has
#pragma unroll
        for (int w = 0; w < 4; ++w) any |= uniform(reinterpret_cast<lds_int*>(kt)[w]) != 0;
        const float scale = power(unit);
#pragma unroll
        for (int c = 0; c < CB; ++c) {
            const float lc = halves_sum(l[c]);
            int half, row, rc, tok;
            row_of(c, half, row, rc, tok);
#pragma unroll
            for (int db = 0; db < DB; ++db) o[c][db] *= scale;
            if (row >= rows) continue;
            if (any) {                                       // NaN codes that were left out, to the rows that see them
                uint64_t nan = 0;                            // of the lane's values, in order
#pragma unroll 1
                for (int j = max(max(t0 * BN, all + 1 - BN), 0); j <= min(ctx + tok, t1 * BN - 1); ++j)
#pragma unroll 1
                    for (int d = 0; d < D / 8; ++d) nan |= (uint64_t)attend_odd<D>(a, table, hk, j, 8 * d + 4 * half) << (4 * d);
#pragma unroll
                for (int d = 0; d < D / 2; ++d) o[c][d / 16][d % 16] = nan >> d & 1 ? local_nan() : o[c][d / 16][d % 16];
            }
            if (whole) {
                uint16_t* out = a.out + ((size_t)(begin + tok) * hq + hk * a.group + (rc - tok * a.group)) * D + 4 * half;
                const float inv = lc == 0.f ? 0.f : 1.f / lc;
#pragma unroll
                for (int db = 0; db < DB; ++db)
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        f16x4 w;
#pragma unroll
                        for (int i = 0; i < 4; ++i) w[i] = (_Float16)(lc == 0.f ? 0.f : o[c][db][4 * g + i] * inv);
                        *reinterpret_cast<f16x4*>(out + 32 * db + 8 * g) = w;
                    }
            } else {
                float* part = a.ws + (size_t)(2 * wg + (t0 == 0 ? 1 : 0)) * BM * (D + 2);
                const int r = row - rb * BM;
#pragma unroll
                for (int db = 0; db < DB; ++db)
#pragma unroll
                    for (int g = 0; g < 4; ++g)
                        *reinterpret_cast<f32x4*>(part + r * D + 32 * db + 8 * g + 4 * half) =
                            f32x4{o[c][db][4 * g], o[c][db][4 * g + 1], o[c][db][4 * g + 2], o[c][db][4 * g + 3]};
                if (half == 0) *reinterpret_cast<f32x2*>(part + BM * D + 2 * r) = f32x2{m[c], lc};
            }
        }
    } while (at < end);
}

// ------------------------------------------------------------------- merge --
// Joins the pieces of the block that work-group w begins and does not end (if it does): MR rows to a
// work-group, eight lanes to a row with D/8 columns each; PW of the waves share the same rows' pieces.
// 4 to 5 us for few rows (the launch, the notes, the pieces); 22 and 31 us for 128- and 256-row blocks on
// a full card (65 and 130 KB a piece, written and read again).
template <int D, int BM, int PW>
__global__ __launch_bounds__(256) void attend_merge(AttendArgs a) {
    constexpr int MR = 32 / PW, V = D / 32, U = 4;           // U: pieces in flight
    __shared__ float s_part[PW > 1 ? 4 * 8 * D : 1], s_ml[PW > 1 ? 4 * 8 * 2 : 1];
    const int lane = (int)__lane_id(), wave = uniform((int)threadIdx.x >> 6);
    const int w0 = (int)blockIdx.x / (BM / MR), base = (int)(blockIdx.x % (BM / MR)) * MR;
    auto head_of = [&](int p) { return p == w0 ? 1 : p < a.nwg ? attend_note<D, BM>(a, p)->head : 2; };
    const AttendNote note = *attend_note<D, BM>(a, w0);
    int head = head_of(w0 + lane);                           // (with the note, not after it)
    const int rows = uniform(note.rows);
    if (base >= rows) return;
    const int r = base + (PW > 1 ? 0 : wave * 8) + (lane >> 3), pw = PW > 1 ? wave : 0;
    constexpr size_t STEP = (size_t)BM * (D + 2);
    const int rc = min(r, rows - 1);                         // (a row that is there)
    const float* col = a.ws + (size_t)rc * D + (lane & 7) * 4;
    const float* ml = a.ws + (size_t)BM * D + 2 * rc;
    float m = -__builtin_inff(), l = 0.f;
    f32x4 x[V] = {};
    for (int from = w0;; from += 64) {
        // which of the 64 work-groups from there on have a piece; with PW > 1 the waves share them
        if (from != w0) head = head_of(from + lane);
        const uint64_t last = __ballot(head == 2);
        uint64_t there = __ballot(head != 0 && (PW == 1 || lane % PW == pw));
        if (last) there &= (last ^ (last - 1));              // up to the first that ends it
        while (there) {
            f32x2 s[U];
            f32x4 y[U][V];
            bool on[U];
            int k = 0;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                on[u] = there != 0;
                if (on[u]) k = __builtin_ctzll(there);       // else the last one again: not used
                there &= there - 1;
                const size_t at = (size_t)(2 * (from + k) + (from + k == w0 ? 1 : 0)) * STEP;
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
                if (!on[u]) continue;
                const float g = s[u].x == to ? 1.f : fast_exp2(s[u].x - to);
                l = __builtin_fmaf(g, s[u].y, l);
#pragma unroll
                for (int v = 0; v < V; ++v)
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[v][e] = __builtin_fmaf(g, y[u][v][e], x[v][e]);
            }
        }
        if (last) break;
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
    if (r >= rows) return;
    const int row = note.rb * BM + r, tok = (int)a.by_group.div((uint32_t)row);
    uint16_t* out = a.out + ((size_t)(note.begin + tok) * a.hkv * a.group + note.hk * a.group + (row - tok * a.group)) * D + (lane & 7) * 4;
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        f16x4 y;
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = (_Float16)(l == 0.f ? 0.f : x[v][e] * inv);
        *reinterpret_cast<f16x4*>(out + 32 * v) = y;
    }
}

} // namespace va
