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
// work is the tiles of positions up to its last row's. All blocks' tiles, numbered one behind the
// other (sequence, K/V head, block, tile), are cut into equal shares, one to a work-group; the
// pieces of blocks that several shares cut go to ws (slot 2w: the piece that work-group w begins
// with, 2w + 1: the one it ends with) and attend_merge joins them.
#pragma once
#include "va_kernels.hpp"
#include "va_wide.hpp"

namespace va {

typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) i32x2 lds_i32x2;
typedef __attribute__((address_space(3))) u32x4 lds_u32x4;
typedef __attribute__((address_space(3))) float lds_float;

// ------------------------------------------------------------- work split --
// The rows between two consecutive bounds 0, cu[0], .., cu[B], total (each limited to what lies
// between its predecessor and total); those before the first and behind the last sequence, and
// sequences whose lengths are out of range, are blocks of one tile that only store their rows.
struct AttendSpan {
    int seq;              // -1: rows of no sequence
    int begin, n, len;
    int first;            // its first tile in the numbering
    __device__ __forceinline__ bool bad(int cap) const { return len < 0 || len > cap; }
};
struct AttendBlock {
    AttendSpan s;
    int hk, rb;           // K/V head, block of rows
    int first, tiles;     // its first tile in the numbering, how many
};

// The numbering, by one wave: lane i has span from + i of the current 64.
template <int BM, int BN> struct AttendPlan {
    const AttendArgs& a;
    int from = -1, prev = 0;                     // prev: the bound ahead of the next 64
    int begin = 0, n = 0, len = 0;
    int count = 0, upto = 0;                     // tiles of the lane's span, and up to and with it
    int total = 0;                               // tiles of the batch
    __device__ __forceinline__ int spans() const { return a.cu ? a.B + 2 : a.B; }
    __device__ __forceinline__ int seq_of(int i) const { return !a.cu ? (i < a.B ? i : -1) : i >= 1 && i <= a.B ? i - 1 : -1; }
    __device__ __forceinline__ int blocks(int rows) const { return (rows + BM - 1) / BM; }
    __device__ __forceinline__ int tiles(int seq, int n, int len, int rb) const {
        if (seq < 0 || len < 0 || len > a.cap) return 1;
        const int i1 = min(n - 1, (int)a.by_group.div((uint32_t)(rb * BM + BM - 1)));
        const int seen = len - n + i1 + 1;       // positions that the block's last row sees
        return seen <= 0 ? 1 : (seen - 1) / BN + 1;
    }
    __device__ __forceinline__ void load(int at, int before, int bound) {
        from = at;
        const int i = at + (int)__lane_id();
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
        const int seq = seq_of(i);
        len = seq >= 0 ? a.seq_lens[seq] : 0;
        int sum = 0;
        for (int rb = 0, nb = blocks(n * a.group); rb < nb; ++rb) sum += tiles(seq, n, len, rb);
        count = sum * a.hkv;
        upto = before + wave_scan(count);
    }
    __device__ __forceinline__ explicit AttendPlan(const AttendArgs& args) : a(args) {
        for (int at = 0; at < spans(); at += 64) {
            load(at, total, prev);
            total = __builtin_amdgcn_readlane(upto, 63);
        }
    }
    // The block that tile `at` < total is in.
    __device__ __forceinline__ AttendBlock find(int at) {
        if (spans() > 64) {
            int before = 0, bound = 0;
            for (int f = 0; f < spans(); f += 64) {
                load(f, before, bound);
                before = __builtin_amdgcn_readlane(upto, 63);
                bound = prev;
                if (at < before) break;
            }
        }
        const int l = __builtin_ctzll(__ballot(upto > at));
        AttendBlock b;
        b.s.seq = seq_of(from + l);
        b.s.begin = __builtin_amdgcn_readlane(begin, l);
        b.s.n = __builtin_amdgcn_readlane(n, l);
        b.s.len = __builtin_amdgcn_readlane(len, l);
        const int nb = blocks(b.s.n * a.group), of = __builtin_amdgcn_readlane(count, l), per = of / a.hkv;
        b.s.first = __builtin_amdgcn_readlane(upto, l) - of;
        b.hk = (at - b.s.first) / per;
        int in = at - b.s.first - b.hk * per;
        for (int r0 = 0;; r0 += 64) {
            const int rb = r0 + (int)__lane_id();
            const int t = rb < nb ? tiles(b.s.seq, b.s.n, b.s.len, rb) : 0;
            const int up = wave_scan(t), all = __builtin_amdgcn_readlane(up, 63);
            if (in < all) {
                const int k = __builtin_ctzll(__ballot(up > in));
                b.rb = r0 + k;
                b.tiles = __builtin_amdgcn_readlane(t, k);
                b.first = at - in + __builtin_amdgcn_readlane(up, k) - b.tiles;
                return b;
            }
            in -= all;
        }
    }
    __device__ __forceinline__ int share() const { return max((total + a.nwg - 1) / a.nwg, 1); }
    __device__ __forceinline__ int shares(int share) const { return (total + share - 1) / share; }
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
        const int t = tile + (int)__lane_id();
        const long long j64 = (long long)t * stride + off;
        const bool on = t < tiles && j64 < end;
        const int j = on ? (int)j64 : 0;
        page = on ? table[j >> a.page_shift] : -1;
        if (page < 0 || page >= a.num_pages) page = -1;
        sk = sv = 0;
        if (page >= 0) {
            const size_t at = ((((size_t)page * a.hkv + hk) << a.page_shift) + (size_t)(j & ((1 << a.page_shift) - 1))) / G;
            if constexpr (STEP > G) {
                sk = *reinterpret_cast<const uint32_t*>(a.sk + at);
                sv = *reinterpret_cast<const uint32_t*>(a.sv + at);
            } else {
                sk = a.sk[at] * 0x10001u;
                sv = a.sv[at] * 0x10001u;
            }
        }
    }
};

// A tile's part under one pair of scales, all uniform: K's scale times the scores' factor, V's
// scale as 2^e times `more` in [1, 2), and whether the part has no finite values (a page outside
// the pool, a scale that is infinite or NaN): rows that see it are NaN.
struct Scales {
    float qs, more;
    int e;                // NONE: V's scale is 0
    bool bad;
    static constexpr int NONE = -1000;
    __device__ __forceinline__ void set(uint32_t sk, uint32_t sv, float qscale, bool there) {
        sk &= 0x7FFFu;
        sv &= 0x7FFFu;
        bad = !there || sk >= 0x7C00u || sv >= 0x7C00u;
        // a hidden position's score is -infinity, which a factor of 0 would make NaN
        const float k = uniformf(h2f(bad ? 0u : sk)), v = uniformf(h2f(bad ? 0u : sv));
        qs = k > 0.f ? qscale * k : 0x1p-100f;
        const uint32_t b = __builtin_bit_cast(uint32_t, v);
        e = b ? (int)(b >> 23) - 127 : NONE;
        more = b ? __builtin_bit_cast(float, (b & 0x7FFFFFu) | 0x3F800000u) : 1.f;
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
            s[b].more *= power(s[b].e - u + 15);
            s[b].e = u - 15;
        }
    return u;
}
__device__ __forceinline__ float factor_of(const Scales& s, int unit) { return s.e == Scales::NONE ? 0x1p-120f : power(s.e - unit); }

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
// NaN where one of the codes c .. c + 3 of position j's V row is NaN, else 0.
template <int D>
__device__ __forceinline__ f32x4 attend_odd(const AttendArgs& a, const int32_t* table, int hk, int j, int c) {
    f32x4 x = {};
    const int page = table[j >> a.page_shift];
    if (page < 0 || page >= a.num_pages) return x;
    const size_t r = (((size_t)page * a.hkv + hk) << a.page_shift) + (size_t)(j & ((1 << a.page_shift) - 1));
    const uint32_t w = *reinterpret_cast<const uint32_t*>(a.v + r * D + c);
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (((w >> (8 * e)) & 0x7Fu) == 0x7Fu) x[e] = __builtin_nanf("");
    return x;
}

// The lazy maximum, as WIDE_OFF and WIDE_SLACK, with room for the part of V's scale below 2.
constexpr float ATT_OFF = 10.f, ATT_SLACK = 4.f;

// ---------------------------------------------------------------- one or few rows --
// Block: 16 NB rows as columns of 16x16x32 products; the four waves take 32 positions each of a tile
// of 128, every wave by itself until the piece ends. K comes from memory in the operand's layout
// (a lane has 16 bytes of a row, dimensions 16h .. and 64 + 16h ..: the k index is a free
// permutation, and q is laid out likewise); V is transposed through the wave's own LDS with
// ds_read_b64_tr_b8 (lane i of 16 addresses half i%2 of row i/2 and receives column i of the eight
// rows; probed on MI355X). A lane's slots of the second product are the positions whose scores it
// holds: 4h + 0..3 and 16 + 4h + 0..3.
typedef float f32x4v __attribute__((ext_vector_type(4)));

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
    lds_int* odd = (lds_int*)((lds_u8*)lds + LDS);

    const int tid = (int)threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), h = lane >> 4, c16 = lane & 15;
    lds_u8* vt = (lds_u8*)lds + wave * VB;
    if (tid == 0) *odd = 0;
    AttendPlan<BM, BN> plan(a);
    const int share = plan.share(), per = (plan.shares(share) + 7) >> 3;
    if ((int)(blockIdx.x >> 3) >= per) return;
    const int wg = (int)(blockIdx.x & 7) * per + (int)(blockIdx.x >> 3);
    int at = wg * share;
    const int end = min(plan.total, at + share);

    // the thread's number, made anew: what is computed from it is not held across loops
    auto fresh_lane = [&]() {
        int x = lane;
        asm volatile("" : "+v"(x));
        return x;
    };
    while (at < end) {
        const AttendBlock blk = plan.find(at);
        const int hk = uniform(blk.hk), rb = uniform(blk.rb), n = uniform(blk.s.n), begin = uniform(blk.s.begin), seq = uniform(blk.s.seq);
        const int len = uniform(blk.s.len), tiles = uniform(blk.tiles), t0 = uniform(at - blk.first), t1 = uniform(min(tiles, t0 + (end - at)));
        const int rows = n * a.group, hq = a.hkv * a.group;
        at += t1 - t0;
        if (seq < 0 || blk.s.bad(a.cap)) {
            const float x = seq < 0 ? 0.f : __builtin_nanf("");
            for (int i = tid; i < BM * (D / 8); i += 256) {
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
        auto fetch = [&](int t, int b) {
            if (t >= pl.base + 64 || pl.base < 0) pl.load(a, table, hk, t, t1, BN, wave * 32, len);
            const int l = t - pl.base, page = __builtin_amdgcn_readlane(pl.page, l), j = t * BN + wave * 32;
            const int left = page < 0 ? 0 : max(0, min(32, len - j));
            sc[b].set((uint32_t)__builtin_amdgcn_readlane((int)pl.sk, l), (uint32_t)__builtin_amdgcn_readlane((int)pl.sv, l), a.qscale, page >= 0);
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
        f32x4 o[NB][DT] = {};
        float m[NB], l[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            m[b] = -__builtin_inff();
            l[b] = 0.f;
        }
        int unit = 0;
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
            bool any = false;
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < VL; ++i) {
                u32x4 w = vr[b % VAHEAD][i];
                if (hides) any |= codes_clean(w);
                const int row = vrow + i * (1024 / D);
                *reinterpret_cast<lds_u32x4*>(vt + row * D + ((vchunk ^ few_swz<D>(row)) << 4)) = w;
            }
            if (any) *odd = 1;
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
                top[y] = rows_max(top[y]) * s.qs;
                grows |= top[y] - m[y] > ATT_OFF + ATT_SLACK;    // also at the first one: m = -inf
            }
            const int to_unit = unit_for(s, unit);
            if (__any(grows) || to_unit != unit) {
                const float u = power(unit - to_unit);
                unit = to_unit;
#pragma unroll
                for (int y = 0; y < NB; ++y) {
                    const float to = fmaxf(m[y], top[y] - ATT_OFF), f = to == m[y] ? 1.f : fast_exp2(m[y] - to);
                    m[y] = to;
                    l[y] *= f;
#pragma unroll
                    for (int d = 0; d < DT; ++d) o[y][d] *= f * u;
                }
            }
            f16x8 p[NB];
#pragma unroll
            for (int y = 0; y < NB; ++y) {
                const float base = m[y] == -__builtin_inff() ? 0.f : m[y];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float w = fast_exp2(__builtin_fmaf(x[e / 4][y][e % 4], s.qs, -base));
                    l[y] += w;
                    p[y][e] = (_Float16)(w * s.more);
                }
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
        fetch(t0, 0);
        if (VAHEAD == 1) fetch_v(0);
        if (t0 + 1 < t1) fetch(t0 + 1, 1);
        int t = t0;
        do {
            tile(t, 0);
            if (t + 2 < t1) fetch(t + 2, 0);
            if (t + 1 < t1) tile(t + 1, 1);
            if (t + 3 < t1) fetch(t + 3, 1);
            t += 2;
        } while (t < t1);

        const bool whole = t0 == 0 && t1 == tiles;
        float* part = a.ws + (size_t)(2 * wg + (t0 == 0 ? 1 : 0)) * BM * (D + 2);   // [BM][D] sums, then [BM][2] (m, l)
        lds_float* es = (lds_float*)lds;
        lds_float* ml = es + EPI / 4;
        const float scale = power(unit);
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
                if (*odd)                                    // NaN codes that were left out, to the rows that see them
                    for (int j = max(t0 * BN, all + 1 - BN); j <= min(ctx + tok, t1 * BN - 1); ++j)
                        if (j >= 0) x += attend_odd<D>(a, table, hk, j, c);
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
        __syncthreads();                                     // the sums are read, odd too
        if (tid == 0) *odd = 0;
    }
}

// ----------------------------------------------------------------- many rows --
// The weights of two parts of 32 positions; qs, more: of each.
template <int D>
__device__ __forceinline__ void attend_weights(const f32x16 (&s)[2], const Scales (&sc)[2], int to_unit, int& unit, float& m, float& l, f32x16 (&o)[D / 32], f16x8 (&p)[2][2]) {
    float top = -__builtin_inff();
#pragma unroll
    for (int b = 0; b < 2; ++b) {
        float x = s[b][0];
#pragma unroll
        for (int v = 1; v < 16; ++v) x = fmaxf(x, s[b][v]);
        top = fmaxf(top, x * sc[b].qs);
    }
    top = halves_max(top);
    if (__any(top - m > ATT_OFF + ATT_SLACK) || to_unit != unit) {   // also at the first one: m = -inf
        const float to = fmaxf(m, top - ATT_OFF), f = to == m ? 1.f : fast_exp2(m - to);
        m = to;
        l *= f;
        const float g = f * power(unit - to_unit);
        unit = to_unit;
#pragma unroll
        for (int db = 0; db < D / 32; ++db) o[db] *= g;
    }
    const float base = m == -__builtin_inff() ? 0.f : m;
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int v = 0; v < 16; ++v) {
            const float e = fast_exp2(__builtin_fmaf(s[b][v], sc[b].qs, -base));
            l += e;
            p[b][v / 8][v % 8] = (_Float16)(e * sc[b].more);
        }
}

// Block: 128 rows, 32 to a wave as the columns of va_wide.hpp's tiles. A tile of 64 positions comes
// to LDS as codes while its predecessor is computed (16 KB of K and V, each wave a quarter), and every
// wave turns what it fetched into fp16 rows that all four read.
template <int D, int G>
__global__ __launch_bounds__(256, 3) void attend_wide(AttendArgs a) {
    constexpr int BM = 128, BN = 64, KS = D / 16, DB = D / 32, TILE = BN * 2 * D, RAW = BN * D, N = RAW / 4096;
    __shared__ __align__(1024) uint8_t lds[2 * TILE + 2 * RAW + 16];
    lds_u8* kt = (lds_u8*)lds;
    lds_u8* vt = kt + TILE;
    lds_u8* rk = vt + TILE;
    lds_u8* rv = rk + RAW;
    lds_int* odd = (lds_int*)(rv + RAW);

    const int tid = (int)threadIdx.x, wave = uniform(tid >> 6);
    if (tid == 0) *odd = 0;
    WideAddr<D> ad0;
    ad0.init(tid & 63);
    // the lane, made anew: what is computed from it is not held across loops
    auto fresh_lane = [&]() {
        int x = tid & 63;
        asm volatile("" : "+v"(x));
        return x;
    };
    int at = 0, end = 0, wg = 0;
    do {
        AttendBlock blk;
        {
            AttendPlan<BM, BN> plan(a);                      // (holding the plan would cost the loop's registers)
            if (end == 0) {
                const int share = plan.share(), per = (plan.shares(share) + 7) >> 3;
                if ((int)(blockIdx.x >> 3) >= per) return;
                wg = (int)(blockIdx.x & 7) * per + (int)(blockIdx.x >> 3);
                at = wg * share;
                end = min(plan.total, at + share);
                if (at >= end) return;
            }
            blk = plan.find(at);
        }
        const int hk = uniform(blk.hk), rb = uniform(blk.rb), n = uniform(blk.s.n), begin = uniform(blk.s.begin), seq = uniform(blk.s.seq);
        const int len = uniform(blk.s.len), tiles = uniform(blk.tiles), t0 = uniform(at - blk.first), t1 = uniform(min(tiles, t0 + (end - at)));
        const int rows = n * a.group, hq = a.hkv * a.group;
        at += t1 - t0;
        if (seq < 0 || blk.s.bad(a.cap)) {
            const float x = seq < 0 ? 0.f : __builtin_nanf("");
            for (int i = tid; i < BM * (D / 8); i += 256) {
                const int r = rb * BM + i / (D / 8);
                if (r >= rows) break;
                const int tok = (int)a.by_group.div((uint32_t)r);
                *reinterpret_cast<f16x8*>(a.out + ((size_t)(begin + tok) * hq + hk * a.group + (r - tok * a.group)) * D + (i % (D / 8)) * 8) = f16x8((_Float16)x);
            }
            continue;
        }
        const int ctx = len - n;
        const int32_t* table = a.block_table + (size_t)seq * a.max_pages;
        // the lane's row of the block
        auto row_of = [&](int& half, int& row, int& rc, int& tok) {
            const int x = fresh_lane();
            half = x >> 5;
            row = rb * BM + wave * 32 + (x & 31);
            rc = min(row, rows - 1);
            tok = (int)a.by_group.div((uint32_t)rc);
        };
        const int all = ctx + (int)a.by_group.div((uint32_t)(rb * BM));                                       // that every row of the block sees
        const int mine = ctx + (int)a.by_group.div((uint32_t)min(rb * BM + wave * 32, rows - 1));             // .. of the wave
        f16x8 q[KS];
        {
            int half, row, rc, tok;
            row_of(half, row, rc, tok);
            const uint16_t* qp = a.q + ((size_t)(begin + tok) * hq + hk * a.group + (rc - tok * a.group)) * D + 8 * half;
#pragma unroll
            for (int s = 0; s < KS; ++s) q[s] = *reinterpret_cast<const f16x8*>(qp + 16 * s);
        }
        Places<64, G> pl;
        uint32_t sk = 0, sv = 0;                             // of the tile that is fetched
        bool there = false;
        auto fetch = [&](int t) {
            if (pl.base < 0 || t >= pl.base + 64) pl.load(a, table, hk, t, t1, BN, 0, len);
            const int x = t - pl.base, page = __builtin_amdgcn_readlane(pl.page, x), j = t * BN;
            sk = (uint32_t)__builtin_amdgcn_readlane((int)pl.sk, x);
            sv = (uint32_t)__builtin_amdgcn_readlane((int)pl.sv, x);
            there = page >= 0;
            const int left = there ? max(0, min(BN, len - j)) : 0;
            const size_t r = uniform64((((size_t)(there ? page : 0) * a.hkv + hk) << a.page_shift) + (size_t)(j & ((1 << a.page_shift) - 1)));
            const uint32_t bytes = (uint32_t)(uniform(left) * D);
            const __amdgpu_buffer_rsrc_t k = make_rsrc(a.k + r * D, bytes), v = make_rsrc(a.v + r * D, bytes);
            const int lane = fresh_lane();
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const uint32_t off = (uint32_t)((wave * N + i) * 1024);
                __builtin_amdgcn_raw_ptr_buffer_load_lds(k, rk + off, 16, off + (uint32_t)lane * 16u, 0, 0, 0);
                __builtin_amdgcn_raw_ptr_buffer_load_lds(v, rv + off, 16, off + (uint32_t)lane * 16u, 0, 0, 0);
            }
        };
        f32x16 o[DB] = {};
        float m = -__builtin_inff(), l = 0.f;
        int unit = 0;
        fetch(t0);
        for (int t = t0; t < t1; ++t) {
            Scales sc[2];
            sc[0].set(sk & 0xFFFFu, sv & 0xFFFFu, a.qscale, there);
            sc[1].set(sk >> 16, sv >> 16, a.qscale, there || t * BN + 32 >= len);
            const int to_unit = unit_for(sc, unit);
            const bool hides = t * BN + BN - 1 > all;
            // what this wave fetched has arrived; every wave has read the last tile (or the last piece's flag)
            __builtin_amdgcn_sched_barrier(0);
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
            __builtin_amdgcn_sched_barrier(0);
            {
                const float f = wave < 2 ? factor_of(sc[0], to_unit) : factor_of(sc[1], to_unit);
                const int lane = fresh_lane();
                bool any = false;
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const int off = (wave * N + i) * 1024 + lane * 16, r = off / D, c = off % D / 8;
                    const int to0 = r * 2 * D + ((c ^ swz<D>(r)) << 4), to1 = r * 2 * D + (((c + 1) ^ swz<D>(r)) << 4);
                    const u32x4 kw = *reinterpret_cast<lds_u32x4*>(rk + off);
                    u32x4 vw = *reinterpret_cast<lds_u32x4*>(rv + off);
                    *reinterpret_cast<lds_f16x8*>(kt + to0) = codes_to_f16x8(kw.x, kw.y, 1.f);
                    *reinterpret_cast<lds_f16x8*>(kt + to1) = codes_to_f16x8(kw.z, kw.w, 1.f);
                    if (hides) any |= codes_clean(vw);
                    *reinterpret_cast<lds_f16x8*>(vt + to0) = codes_to_f16x8(vw.x, vw.y, f);
                    *reinterpret_cast<lds_f16x8*>(vt + to1) = codes_to_f16x8(vw.z, vw.w, f);
                }
                if (any) *odd = 1;
            }
            __builtin_amdgcn_sched_barrier(0);
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
            __builtin_amdgcn_sched_barrier(0);
            if (t + 1 < t1) fetch(t + 1);
            const WideAddr<D> ad = ad0.fresh();
            f32x16 s[2];
            wide_scores<D, 2, 2, false>(kt, nullptr, ad, q, s);
            if (sc[0].bad || sc[1].bad) {
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int v = 0; v < 16; ++v) s[b][v] = sc[b].bad ? __builtin_nanf("") : s[b][v];
            }
            if (t * BN + BN - 1 > mine) {
                int half, row, rc, tok;
                row_of(half, row, rc, tok);
                const int lim = ctx + tok - t * BN - 4 * half;   // the last position that the row sees, from the lane's first one
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int v = 0; v < 16; ++v) s[b][v] = 32 * b + 8 * (v / 4) + v % 4 > lim ? -__builtin_inff() : s[b][v];
            }
            f16x8 p[2][2];
            attend_weights<D>(s, sc, to_unit, unit, m, l, o, p);
            wide_values<D, 2>(vt, ad, p, o);
        }
        l = halves_sum(l);
        __syncthreads();                                     // the last tile is read, odd is whole
        const bool whole = t0 == 0 && t1 == tiles, any = *odd != 0;
        __syncthreads();
        if (tid == 0) *odd = 0;
        const float scale = power(unit);
#pragma unroll
        for (int db = 0; db < DB; ++db) o[db] *= scale;
        int half, row, rc, tok;
        row_of(half, row, rc, tok);
        const int last = ctx + tok;
        if (row < rows) {
            if (any)                                         // NaN codes that were left out, to the rows that see them
#pragma unroll 1
                for (int j = max(max(t0 * BN, all + 1 - BN), 0); j <= min(last, t1 * BN - 1); ++j)
#pragma unroll
                    for (int d = 0; d < D / 8; ++d) {
                        const f32x4 x = attend_odd<D>(a, table, hk, j, 8 * d + 4 * half);
#pragma unroll
                        for (int i = 0; i < 4; ++i) o[d / 4][4 * (d % 4) + i] += x[i];
                    }
            if (whole) {
                uint16_t* out = a.out + ((size_t)(begin + tok) * hq + hk * a.group + (rc - tok * a.group)) * D + 4 * half;
                const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
                for (int db = 0; db < DB; ++db)
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        f16x4 w;
#pragma unroll
                        for (int i = 0; i < 4; ++i) w[i] = (_Float16)(l == 0.f ? 0.f : o[db][4 * g + i] * inv);
                        *reinterpret_cast<f16x4*>(out + 32 * db + 8 * g) = w;
                    }
            } else {
                float* part = a.ws + (size_t)(2 * wg + (t0 == 0 ? 1 : 0)) * BM * (D + 2);
                const int r = row - rb * BM;
#pragma unroll
                for (int db = 0; db < DB; ++db)
#pragma unroll
                    for (int g = 0; g < 4; ++g)
                        *reinterpret_cast<f32x4*>(part + r * D + 32 * db + 8 * g + 4 * half) = f32x4{o[db][4 * g], o[db][4 * g + 1], o[db][4 * g + 2], o[db][4 * g + 3]};
                if (half == 0) *reinterpret_cast<f32x2*>(part + BM * D + 2 * r) = f32x2{m, l};
            }
        }
    } while (at < end);
}

// ------------------------------------------------------------------- merge --
// Joins the pieces of the block that share w begins and does not end (if it does): MR rows to a
// work-group, eight lanes to a row with D/8 columns each; PW of the waves share the same rows' pieces.
template <int D, int BM, int BN, int PW>
__global__ __launch_bounds__(256) void attend_merge(AttendArgs a) {
    constexpr int MR = 32 / PW, V = D / 32, U = 4;           // U: pieces in flight
    __shared__ float s_part[PW > 1 ? 4 * 8 * D : 1], s_ml[PW > 1 ? 4 * 8 * 2 : 1];
    const int lane = (int)__lane_id(), wave = uniform((int)threadIdx.x >> 6);
    const int w0 = (int)blockIdx.x / (BM / MR), base = (int)(blockIdx.x % (BM / MR)) * MR;
    AttendPlan<BM, BN> plan(a);
    const int share = plan.share(), cut = (w0 + 1) * share;
    if ((long long)(w0 + 1) * share >= plan.total) return;
    const AttendBlock blk = plan.find(cut - 1);
    const int rows = blk.s.n * a.group - blk.rb * BM;        // of the block, BM at most
    if (blk.first < w0 * share || blk.first + blk.tiles <= cut || base >= rows) return;
    const int w1 = (blk.first + blk.tiles - 1) / share;
    const int r = base + (PW > 1 ? 0 : wave * 8) + (lane >> 3), pw = PW > 1 ? wave : 0;
    constexpr size_t STEP = (size_t)BM * (D + 2);
    const float* col = a.ws + (size_t)r * D + (lane & 7) * 4;
    const float* ml = a.ws + (size_t)BM * D + 2 * r;
    float m = -__builtin_inff(), l = 0.f;
    f32x4 x[V] = {};
    if (r < rows) {
        for (int p0 = w0 + pw; p0 <= w1; p0 += U * PW) {
            f32x2 s[U];
            f32x4 y[U][V];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int p = min(p0 + u * PW, w1);          // the last one again: not used
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
    if (r >= rows) return;
    const int row = blk.rb * BM + r, tok = (int)a.by_group.div((uint32_t)row);
    uint16_t* out = a.out + ((size_t)(blk.s.begin + tok) * a.hkv * a.group + blk.hk * a.group + (row - tok * a.group)) * D + (lane & 7) * 4;
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
