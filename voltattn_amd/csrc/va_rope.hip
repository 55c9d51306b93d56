// va_rope.hip — the rows that a projection gives, into a paged cache with the position rotation
// applied on the way (va_append_rope). With t = position * freq[i], a pair (x, y) of dimensions
// (i, i + R/2), or (2i, 2i + 1), of q and k becomes
//   x' = (x cos t - y sin t) scaling,   y' = (x sin t + y cos t) scaling     (i < R/2),
// the dimensions from R on and v stay. k and v go to the cache, q (and k, if asked) to fp16 rows.
//
// The angle is position * freq / 2 pi turns in 64 bits, less its whole turns; v_sin_f32 and
// v_cos_f32 take turns and are off by 2^-22.9 at most there (measured over [-1/2, 1/2]), so that a
// rotated value is off by 2^-21 of its pair's length for any position, and is rounded once. (Polynomials in
// fp32, off by 2^-24, cost 4 us of 32 for 5500 rows and 8 of 91 for 17600.)
//
// A lane has 8 consecutive dimensions of a row and head (16 bytes), D/8 lanes a head. Bound by memory
// where there are many rows: 17600 rows of 32 + 2 x 8 heads of 128 dimensions into blocks of 64, with the
// rotated k, 91 us (4.7 TB/s of what has to be read and written; a large copy takes 5.15). What counts
// beside it are instructions: frequencies in turns once for all rows of a lane, one product and one
// fused addition to a value, no test of a value that the conversion makes itself (105 us before). Few rows:
// 3 to 5 us, the chain of bounds, start, page and rows. Which form a launch takes goes by the mean rows of its
// sequences: 127 tokens and 1000 rows of another sequence take 128 us (block format), 9.6 and 12 apart.
//
// Row formats (f16, q8, q4, q3): rows are independent; a wave has one row and some of its heads, so
// that angles and the page are found once. The block format (e4m3 codes, a power of two for each G
// positions and head): what one call writes of a block is written by one group of lanes, which
// finds the block's largest value first; a block that holds rows already keeps its scale or has
// them scaled anew (the codes times a power of two: exact but for e4m3's subnormal numbers).
#include "va_pack.hpp"
#include "va_kernels.hpp"

#include <algorithm>

namespace va {

constexpr double TURN = 0.15915494309189533577;   // 1 / 2 pi

// Row r's sequence (-1: none), its first row and the row behind its last one; uniform. A bound below
// its predecessor counts as equal to it, and none leaves 0 .. total.
struct RowSeq {
    int seq, begin, end;
};
__device__ __forceinline__ RowSeq row_seq(const RopeArgs& a, int r) {
    if (!a.cu) return RowSeq{r, r, r + 1};
    int bound = 0;
    for (int i0 = 0; i0 <= a.B; i0 += 64) {
        const int i = i0 + (int)__lane_id();
        const int e = i <= a.B ? max(0, min(a.cu[i], a.total)) : a.total;
        const uint64_t hit = __ballot(e > r && i <= a.B);
        const int l = hit ? __builtin_ctzll(hit) : 64;
        const int top = wave_scan_max((int)__lane_id() < l ? e : 0);
        bound = max(bound, __builtin_amdgcn_readlane(top, 63));
        if (hit) {
            const int b = i0 + l - 1;
            return RowSeq{b < 0 ? -1 : b, bound, __builtin_amdgcn_readlane(e, l)};
        }
    }
    return RowSeq{-1, r, a.total};
}

// Pool row of sequence seq's position p and K/V head 0 over page_rows, or -1 where it is not written.
__device__ __forceinline__ long long pool_row(const RopeArgs& a, int seq, long long p, int& in) {
    in = 0;
    if (p < 0 || p > 0x7FFFFFFFLL) return -1;
    const int pi = (int)a.by_page.div((uint32_t)p);
    if (pi >= a.max_pages) return -1;
    const int page = a.block_table[(size_t)seq * a.max_pages + pi];
    if (page < 0 || page >= a.num_pages) return -1;
    in = (int)p - pi * a.page_rows;
    return page;
}

// cos and sin of a lane's dimensions d .. d + 7 at a position, times scaling; neighbours share a
// pair's angle if pairs is set. lead: the lane has the pairs' first dimensions (pairs: both).
struct Turn {
    float c[8], s[8];     // s: with the sign that the pair's other value takes (pairs: as it is)
};
// What a lane's dimensions turn by in a position, in turns.
struct Rates {
    double f[8];
    bool on, lead;
};
__device__ __forceinline__ Rates rates_of(const RopeArgs& a, int d) {
    Rates r;
    const int half = a.rot >> 1;
    r.on = d < a.rot;
    r.lead = a.pairs || d < half;
    const int i0 = !r.on ? 0 : a.pairs ? d >> 1 : d < half ? d : d - half;
    const f32x4 f0 = *reinterpret_cast<const f32x4*>(a.freq + i0);      // i0 is a multiple of 4
    f32x4 f1 = f0;
    if (!a.pairs) f1 = *reinterpret_cast<const f32x4*>(a.freq + i0 + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        r.f[e] = TURN * (double)f0[e];
        r.f[4 + e] = TURN * (double)f1[e];
    }
    return r;
}
__device__ __forceinline__ void set_turn(Turn& t, const RopeArgs& a, const Rates& r, double at) {
    const float sign = a.pairs || !r.lead ? a.scaling : -a.scaling;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        if (e >= 4 && a.pairs) break;
        double x = at * r.f[e];
        x -= __builtin_rint(x);
        const float y = (float)x;
        t.c[e] = __builtin_amdgcn_cosf(y) * a.scaling;
        t.s[e] = __builtin_amdgcn_sinf(y) * sign;
    }
}
// The other halves of a lane's pairs lie at element offset d0 + other() (the lane's own, if pairs is set).
__device__ __forceinline__ int other(const RopeArgs& a, int d) {
    const int half = a.rot >> 1;
    return a.pairs || d >= a.rot ? d : d < half ? d + half : d - half;
}
__device__ __forceinline__ void values8(const u32x4& w, float (&x)[8]) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        x[2 * k] = h2f_lo(w[k]);
        x[2 * k + 1] = h2f_hi(w[k]);
    }
}
__device__ __forceinline__ void turn8(const Turn& t, bool on, bool pairs, const u32x4& own, const u32x4& oth, float (&x)[8]) {
    values8(own, x);
    if (!on) return;
    if (pairs) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float p = x[2 * i], q = x[2 * i + 1];
            x[2 * i] = __builtin_fmaf(p, t.c[i], -q * t.s[i]);
            x[2 * i + 1] = __builtin_fmaf(p, t.s[i], q * t.c[i]);
        }
    } else {
        float y[8];
        values8(oth, y);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = __builtin_fmaf(x[e], t.c[e], y[e] * t.s[e]);
    }
}
__device__ __forceinline__ u32x4 halves8(const float (&x)[8]) {
    u32x4 w;
#pragma unroll
    for (int k = 0; k < 4; ++k) w[k] = (uint32_t)f2h_rne(x[2 * k]) | (uint32_t)f2h_rne(x[2 * k + 1]) << 16;
    return w;
}

// --------------------------------------------------------------- row formats --
// 8 elements of a row of k or v, at element `to` of the pool.
template <int BITS, int G>
__device__ __forceinline__ void store_row8(const float (&x)[8], const u32x4& as_is, bool rotated, bool on, size_t to, uint8_t* pages, uint16_t* scales) {
    if constexpr (BITS == 16) {
        if (on) stream_store(reinterpret_cast<u32x4*>(pages + to * 2), rotated ? halves8(x) : as_is);
    } else {
        float amax = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) amax = fmaxf(amax, __builtin_fabsf(x[e]));
        const uint16_t sb = quant_scale<BITS>(group_max<G / 8>(amax));
        int code[8];
        quant_codes<BITS, 8>(x, h2f(sb), code);
        pack_store<BITS, 8>(code, pages, to, on);
        if (on && to % G == 0) scales[to / G] = sb;
    }
}

// One row's heads, D/8 lanes to a head: q's, and k's and v's too for the row formats (BITS > 0).
template <int BITS, int D, int G, bool MANY>
__device__ __forceinline__ void rope_heads(const RopeArgs& a, int r, int j0, int j1) {
    constexpr int L = D / 8, PER = 64 / L, U = 4;            // lanes of a head, heads of a wave at once; U: of those in flight
    const int lane = (int)__lane_id(), d = lane % L * 8, g = lane / L;
    const RowSeq rs = row_seq(a, r);
    const int heads = a.hq + (BITS ? 2 * a.hkv : 0);
    if (rs.seq < 0) {                                        // a row of no sequence
        for (int j = j0; j < j1; ++j) {
            const int head = j * PER + g;
            if (head < a.hq) *reinterpret_cast<u32x4*>(a.q_out + ((size_t)r * a.hq + head) * D + d) = u32x4{0u, 0u, 0u, 0u};
            else if (BITS && a.k_out && head < a.hq + a.hkv) *reinterpret_cast<u32x4*>(a.k_out + ((size_t)r * a.hkv + head - a.hq) * D + d) = u32x4{0u, 0u, 0u, 0u};
        }
        if (MANY && a.k_out && j0 == 0)                      // no block has it
            for (int hk = g; hk < a.hkv; hk += PER) *reinterpret_cast<u32x4*>(a.k_out + ((size_t)r * a.hkv + hk) * D + d) = u32x4{0u, 0u, 0u, 0u};
        return;
    }
    const long long p = (long long)a.start[rs.seq] + (r - rs.begin);
    int in = 0;
    long long page = -1;
    if (BITS) page = pool_row(a, rs.seq, p, in);
    const int oth = other(a, d);
    const Rates rates = rates_of(a, d);
    Turn t;
    set_turn(t, a, rates, a.places ? (double)a.places[r] : (double)p);
    for (int jb = j0; jb < j1; jb += U) {
        u32x4 w[U], v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int head = (jb + u) * PER + g;
            w[u] = v[u] = u32x4{0u, 0u, 0u, 0u};
            if (jb + u >= j1 || head >= heads) continue;
            const uint16_t* src = head < a.hq ? a.q + (size_t)r * a.q_row + (size_t)head * a.q_head
                                : head < a.hq + a.hkv ? a.k + (size_t)r * a.k_row + (size_t)(head - a.hq) * a.k_head
                                                      : a.v + (size_t)r * a.v_row + (size_t)(head - a.hq - a.hkv) * a.v_head;
            w[u] = *reinterpret_cast<const u32x4*>(src + d);
            if (!a.pairs && rates.on && head < a.hq + a.hkv) v[u] = *reinterpret_cast<const u32x4*>(src + oth);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int head = (jb + u) * PER + g;
            if (jb + u >= j1 || head >= heads) continue;
            float x[8];
            if (head < a.hq) {
                turn8(t, rates.on, a.pairs, w[u], v[u], x);
                *reinterpret_cast<u32x4*>(a.q_out + ((size_t)r * a.hq + head) * D + d) = rates.on ? halves8(x) : w[u];
            } else if constexpr (BITS != 0) {
                const bool is_k = head < a.hq + a.hkv;
                const int hk = head - a.hq - (is_k ? 0 : a.hkv);
                const bool turned = is_k && rates.on;
                if (is_k) turn8(t, rates.on, a.pairs, w[u], v[u], x);
                else values8(w[u], x);
                if (is_k && a.k_out) *reinterpret_cast<u32x4*>(a.k_out + ((size_t)r * a.hkv + hk) * D + d) = turned ? halves8(x) : w[u];
                const size_t to = page < 0 ? (size_t)d : (((size_t)page * a.hkv + hk) * a.page_rows + in) * D + d;
                store_row8<BITS, G>(x, w[u], turned, page >= 0, to, is_k ? a.kp : a.vp, is_k ? a.ks : a.vs);
            }
        }
    }
}

// -------------------------------------------------------------- block format --
// The exponent of the smallest power of two from 2^-24 to 2^15 whose 448-fold is not below top.
__device__ __forceinline__ int block_exponent(float top) {
    const uint32_t b = __builtin_bit_cast(uint32_t, top);
    const int e = (int)(b >> 23) - 135 + ((b & 0x7FFFFFu) > 0x600000u ? 1 : 0);    // 448 = 1.75 * 2^8
    return max(-24, min(e, 15));
}
__device__ __forceinline__ uint16_t power16(int e) { return (uint16_t)(e >= -14 ? (e + 15) << 10 : 1 << (e + 24)); }

// The largest finite |x|.
__device__ __forceinline__ float finite_top(const float (&x)[8], float top) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float y = __builtin_fabsf(x[e]);
        top = fmaxf(top, y < __builtin_inff() ? y : 0.f);
    }
    return top;
}
// Codes of x / s (inv = 1 / s, exact where s is a power of two): RNE, at most 448, NaN for what is not finite.
__device__ __forceinline__ u32x2 codes8(const float (&x)[8], float s, float inv, bool exact) {
    float y[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float z = exact ? x[e] * inv : x[e] / s;
        y[e] = __builtin_fabsf(x[e]) < __builtin_inff() ? __builtin_amdgcn_fmed3f(z, -448.f, 448.f) : __builtin_nanf("");
    }
    u32x2 w;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        int c = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * k], y[4 * k + 1], 0, false);
        w[k] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[4 * k + 2], y[4 * k + 3], c, true);
    }
    return w;
}
__device__ __forceinline__ u32x2 plain8(const float (&x)[8], float inv) {
    u32x2 w;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        int c = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * k] * inv, x[4 * k + 1] * inv, 0, false);
        w[k] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[4 * k + 2] * inv, x[4 * k + 3] * inv, c, true);
    }
    return w;
}
// Held codes under a scale 1/f as large.
__device__ __forceinline__ uint32_t scaled4(uint32_t w, float f) {
    const auto a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    int c = __builtin_amdgcn_cvt_pk_fp8_f32(a[0] * f, a[1] * f, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(b[0] * f, b[1] * f, c, true);
}

// A block's scale: what the new rows need, or the held one (held rows: those before them in the
// block), whichever is larger; a held scale that is not finite stays. scale: as it is stored; s: its
// value; keep: what the held codes are to be multiplied by (1: left as they are).
struct BlockScale {
    uint16_t bits;
    float s, keep;
    bool exact;           // s is a power of two
};
__device__ __forceinline__ BlockScale block_scale(float top, bool held, uint16_t old) {
    BlockScale b;
    const int e = block_exponent(top);
    b.bits = power16(e);
    b.s = h2f(b.bits);
    b.keep = 1.f;
    b.exact = true;
    if (held) {
        old &= 0x7FFFu;
        const float o = h2f(old);
        if (old >= b.bits) {                                 // as numbers too: fp16's bits order like the values
            b.bits = old;
            if (old < 0x7C00u) {
                b.s = o;
                b.exact = (old & 0x3FFu) == 0 || (old < 0x400u && (old & (old - 1)) == 0);
            }
        } else {
            b.keep = o / b.s;
        }
    }
    return b;
}

// Few rows to a sequence: D/8 lanes have what this call writes of a block (whose first new row is r)
// of a K/V head, k or v.
template <int D, int G>
__device__ __forceinline__ void rope_block_few(const RopeArgs& a, int r, int j) {
    constexpr int L = D / 8, PER = 64 / L;
    const int lane = (int)__lane_id(), d = lane % L * 8, slot = j * PER + lane / L;
    const RowSeq rs = row_seq(a, r);
    const bool is_k = slot < a.hkv, on = slot < 2 * a.hkv;
    const int hk = is_k ? slot : slot - a.hkv;
    if (rs.seq < 0) {
        if (on && is_k && a.k_out) *reinterpret_cast<u32x4*>(a.k_out + ((size_t)r * a.hkv + hk) * D + d) = u32x4{0u, 0u, 0u, 0u};
        return;
    }
    const long long p = (long long)a.start[rs.seq] + (r - rs.begin);
    const int at = (int)(p & (G - 1));
    if (r != rs.begin && at != 0) return;                    // not the block's first new row
    const int n = min(rs.end - r, G - at);
    if (!on) return;
    int in;
    const long long page = pool_row(a, rs.seq, p, in);
    const size_t row0 = page < 0 ? 0 : ((size_t)page * a.hkv + hk) * a.page_rows + (in - at);       // the block's first
    uint16_t* scales = is_k ? a.ks : a.vs;
    uint8_t* pool = is_k ? a.kp : a.vp;
    const uint16_t old = page >= 0 && at > 0 ? scales[row0 / G] : (uint16_t)0;
    const int oth = other(a, d);
    const uint16_t* src = is_k ? a.k + (size_t)hk * a.k_head : a.v + (size_t)hk * a.v_head;
    const long long stride = is_k ? a.k_row : a.v_row;
    const Rates rates = rates_of(a, d);
    Turn t;
    float x[8];
    auto row = [&](int i) {
        const uint16_t* s = src + (size_t)(r + i) * stride;
        const u32x4 w = *reinterpret_cast<const u32x4*>(s + d);
        if (!is_k) return values8(w, x);
        u32x4 v = {0u, 0u, 0u, 0u};
        if (!a.pairs) v = *reinterpret_cast<const u32x4*>(s + oth);
        set_turn(t, a, rates, a.places ? (double)a.places[r + i] : (double)(p + i));
        turn8(t, rates.on, a.pairs, w, v, x);
    };
    float top = 0.f;
    for (int i = 0; i < n; ++i) {
        row(i);
        top = finite_top(x, top);
    }
    top = group_max<L>(top);
    const BlockScale b = block_scale(top, at > 0, old);
    const float inv = 1.f / b.s;
    if (page >= 0 && at > 0 && b.keep != 1.f)
        for (int i = 0; i < at; ++i) {
            u32x2* c = reinterpret_cast<u32x2*>(pool + (row0 + i) * D + d);
            u32x2 w = *c;
            w.x = scaled4(w.x, b.keep);
            w.y = scaled4(w.y, b.keep);
            *c = w;
        }
    for (int i = 0; i < n; ++i) {
        if (n > 1) row(i);
        if (is_k && a.k_out) *reinterpret_cast<u32x4*>(a.k_out + ((size_t)(r + i) * a.hkv + hk) * D + d) = halves8(x);
        if (page >= 0) *reinterpret_cast<u32x2*>(pool + (row0 + at + i) * D + d) = codes8(x, b.s, inv, b.exact);
    }
    if (page >= 0 && d == 0) scales[row0 / G] = b.bits;
}

// Many rows: a work-group has the block `item` of them all.
template <int D, int G>
__device__ __forceinline__ void rope_block_many(const RopeArgs& a, int item, int slot, float* s_top) {
    constexpr int L = D / 8, RP = 256 / L, PASS = G / RP > 0 ? G / RP : 1;     // rows at once
    const int lane = (int)__lane_id();
    int seq = -1, begin = 0, n = 0;
    long long p = 0;                                         // of the first new row
    {
        constexpr int SH = G == 32 ? 5 : 6;
        int before = 0, prev = 0;
        for (int i0 = 0; i0 <= a.B && seq < 0; i0 += 64) {
            const int i = i0 + lane;
            const int first = i >= 1 && i <= a.B ? a.start[i - 1] : 0;
            int e = i <= a.B ? a.cu[i] : a.total;
            e = max(0, min(e, a.total));
            e = max(prev, wave_scan_max(e));
            const int f = __builtin_amdgcn_update_dpp(prev, e, 0x138, 0xF, 0xF, false);   // wave shift right by one
            const int c = i >= 1 && i <= a.B ? e - f : 0;
            const long long st = first;
            const int blocks = c > 0 ? (int)(((st + c - 1) >> SH) - (st >> SH)) + 1 : 0;
            const int upto = before + wave_scan(blocks);
            const uint64_t hit = __ballot(upto > item);
            if (hit) {
                const int l = __builtin_ctzll(hit);
                seq = i0 + l - 1;
                const int k = item - (__builtin_amdgcn_readlane(upto, l) - __builtin_amdgcn_readlane(blocks, l));
                const int all = __builtin_amdgcn_readlane(c, l);
                const long long s0 = __builtin_amdgcn_readlane(first, l);
                p = k == 0 ? s0 : ((s0 >> SH) + k) * G;
                begin = __builtin_amdgcn_readlane(f, l) + (int)(p - s0);
                n = min(all - (int)(p - s0), G - (int)(p & (G - 1)));
            }
            before = __builtin_amdgcn_readlane(upto, 63);
            prev = __builtin_amdgcn_readlane(e, 63);
        }
    }
    if (seq < 0) return;                                     // the same for the whole work-group
    const bool is_k = slot < a.hkv;
    const int hk = is_k ? slot : slot - a.hkv, at = (int)(p & (G - 1)), tid = (int)threadIdx.x;
    const int d = tid % L * 8, r0 = tid / L, oth = other(a, d);
    const uint16_t* src = is_k ? a.k + (size_t)begin * a.k_row + (size_t)hk * a.k_head : a.v + (size_t)begin * a.v_row + (size_t)hk * a.v_head;
    const long long stride = is_k ? a.k_row : a.v_row;
    u32x4 w[PASS], v[PASS];
#pragma unroll
    for (int i = 0; i < PASS; ++i) {
        const uint16_t* s = src + (size_t)min(r0 + i * RP, n - 1) * stride;
        w[i] = *reinterpret_cast<const u32x4*>(s + d);
        v[i] = w[i];
        if (is_k && !a.pairs) v[i] = *reinterpret_cast<const u32x4*>(s + oth);
    }
    // (behind the rows' loads: the page and the held scale are two more waits)
    int in;
    const long long page = pool_row(a, seq, p, in);
    const size_t row0 = page < 0 ? 0 : ((size_t)page * a.hkv + hk) * a.page_rows + (in - at);
    uint16_t* scales = is_k ? a.ks : a.vs;
    uint8_t* pool = is_k ? a.kp : a.vp;
    const uint16_t old = page >= 0 && at > 0 ? scales[row0 / G] : (uint16_t)0;
    float x[PASS][8], top = 0.f;                             // (rows past the last are that one again)
    if (is_k) {
        const Rates rates = rates_of(a, d);
        const double first = (double)p;                      // (p may pass 32 bits: rows that are not written are turned all the same)
#pragma unroll
        for (int i = 0; i < PASS; ++i) {
            Turn t;
            const int r = r0 + i * RP, rr = min(r, n - 1);
            set_turn(t, a, rates, a.places ? (double)a.places[begin + rr] : first + (double)rr);
            turn8(t, rates.on, a.pairs, w[i], v[i], x[i]);
            if (a.k_out && r < n) *reinterpret_cast<u32x4*>(a.k_out + ((size_t)(begin + r) * a.hkv + hk) * D + d) = rates.on ? halves8(x[i]) : w[i];
        }
    } else {
#pragma unroll
        for (int i = 0; i < PASS; ++i) values8(w[i], x[i]);
    }
    if (page < 0) return;
    auto all_max = [&](float y) {
        y = wave_max(y);
        if (lane == 0) s_top[tid >> 6] = y;
        __syncthreads();
        return fmaxf(fmaxf(s_top[0], s_top[1]), fmaxf(s_top[2], s_top[3]));
    };
#pragma unroll
    for (int i = 0; i < PASS; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) top = fmaxf(top, __builtin_fabsf(x[i][e]));   // NaN: passed over
    top = all_max(top);
    if (top == __builtin_inff()) {                           // of the finite ones, then
        top = 0.f;
#pragma unroll
        for (int i = 0; i < PASS; ++i) top = finite_top(x[i], top);
        __syncthreads();
        top = all_max(top);
    }
    const BlockScale b = block_scale(top, at > 0, old);
    const float inv = 1.f / b.s;
    if (at > 0 && b.keep != 1.f)
        for (int i = r0; i < at; i += RP) {
            u32x2* c = reinterpret_cast<u32x2*>(pool + (row0 + i) * D + d);
            u32x2 y = *c;
            y.x = scaled4(y.x, b.keep);
            y.y = scaled4(y.y, b.keep);
            *c = y;
        }
    // (where nothing can be above 448 the conversion itself does the rest: infinities become NaN)
    const bool plain = b.exact && top <= 448.f * b.s;
#pragma unroll
    for (int i = 0; i < PASS; ++i)
        if (r0 + i * RP < n) *reinterpret_cast<u32x2*>(pool + (row0 + at + r0 + i * RP) * D + d) = plain ? plain8(x[i], inv) : codes8(x[i], b.s, inv, b.exact);
    if (tid == 0) scales[row0 / G] = b.bits;
}

// ------------------------------------------------------------------- launches --
// What a launch is made of: `blocks` work-groups for the block format's k and v, the others for heads
// of rows, `per` turns of a wave's heads to each wave.
struct RopeForm {
    bool many;
    long long items, blocks;      // block format
    int turns, per;               // turns of all of a row's heads
    long long waves;              // of the heads
};

template <int BITS, int D, int G, bool MANY>
__global__ __launch_bounds__(256) void append_rope(RopeArgs a, int heads, int per) {
    constexpr int PER = 512 / D;                             // heads of a wave at once
    __shared__ float s_top[4];
    const int wave = uniform((int)threadIdx.x >> 6);
    int wg = (int)blockIdx.x;
    if constexpr (BITS == 0) {
        if (wg >= heads) {                                   // the blocks come last (first: 37 instead of 35.5 us, side by side: 38.5)
            wg -= heads;
            if constexpr (MANY) {
                const int slots = 2 * a.hkv, item = wg / slots;
                rope_block_many<D, G>(a, item, wg - item * slots, s_top);
            } else {
                const int turns = (2 * a.hkv + PER - 1) / PER;
                const int w = wg * 4 + wave, r = w / turns;
                if (r < a.total) rope_block_few<D, G>(a, r, w - r * turns);
            }
            return;
        }
    }
    const int turns = (a.hq + (BITS ? 2 * a.hkv : 0) + PER - 1) / PER, parts = (turns + per - 1) / per;
    const int w = wg * 4 + wave, r = w / parts, j0 = (w - r * parts) * per;
    if (r < a.total) rope_heads<BITS, D, G, MANY>(a, r, j0, min(j0 + per, turns));
}

static RopeForm rope_form(int bits, int D, int G, const RopeArgs& a) {
    RopeForm f{};
    const int at_once = 512 / D;
    const int heads = a.hq + (bits ? 2 * a.hkv : 0);
    f.turns = (heads + at_once - 1) / at_once;
    if (bits == 0) {
        f.many = (long long)a.total >= 16LL * a.B;
        f.items = std::min((long long)a.total, (long long)a.total / G + 2LL * a.B);
        f.blocks = f.many ? f.items * 2 * a.hkv : ((long long)a.total * ((2 * a.hkv + at_once - 1) / at_once) + 3) / 4;
    }
    // One turn to a wave until there are waves enough to fill the card. 5500 rows of 32 heads with 5 turns
    // to a wave (8192 waves) take 35.6 us, with all 8 of them 32.6; with one 53.
    const long long all = (long long)a.total * f.turns;
    f.per = (int)std::max(1LL, std::min((long long)f.turns, all / 4096));
    f.waves = heads > 0 ? (long long)a.total * ((f.turns + f.per - 1) / f.per) : 0;
    return f;
}

long long rope_groups(int bits, int D, int G, const RopeArgs& a) {
    const RopeForm f = rope_form(bits, D, G, a);
    return f.blocks + (f.waves + 3) / 4;
}

template <int BITS, int G>
static hipError_t launch_bits(int D, const RopeArgs& a, hipStream_t stream) {
    const RopeForm f = rope_form(BITS, D, G, a);
    const int heads = (int)((f.waves + 3) / 4);
    const dim3 grid((unsigned)(f.blocks + heads)), block(256);
    if (D == 128) {
        if (BITS == 0 && f.many) hipLaunchKernelGGL((append_rope<BITS, 128, G, BITS == 0>), grid, block, 0, stream, a, heads, f.per);
        else hipLaunchKernelGGL((append_rope<BITS, 128, G, false>), grid, block, 0, stream, a, heads, f.per);
    } else {
        if (BITS == 0 && f.many) hipLaunchKernelGGL((append_rope<BITS, 64, G, BITS == 0>), grid, block, 0, stream, a, heads, f.per);
        else hipLaunchKernelGGL((append_rope<BITS, 64, G, false>), grid, block, 0, stream, a, heads, f.per);
    }
    return hipGetLastError();
}

hipError_t launch_rope(int bits, int D, int G, const RopeArgs& args, hipStream_t stream) {
    RopeArgs a = args;
    a.by_page = FastDiv::of((uint32_t)a.page_rows);
    if (bits == 16) return launch_bits<16, 32>(D, a, stream);
    if (G == 32) return bits == 8 ? launch_bits<8, 32>(D, a, stream) : bits == 4 ? launch_bits<4, 32>(D, a, stream) : bits == 3 ? launch_bits<3, 32>(D, a, stream) : launch_bits<0, 32>(D, a, stream);
    return bits == 8 ? launch_bits<8, 64>(D, a, stream) : bits == 4 ? launch_bits<4, 64>(D, a, stream) : bits == 3 ? launch_bits<3, 64>(D, a, stream) : launch_bits<0, 64>(D, a, stream);
}

} // namespace va
