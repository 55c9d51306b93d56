// va_wide.hpp — attention of 32 query rows per wave against tiles of K/V rows
// on the matrix cores (gfx950 MFMA 32x32x16 f16), shared by the prompt kernel
// (va_prefill.hip) and the tree kernel (va_tree.hip).
//
// Both products are computed transposed, so that a query row is a column, which
// one lane of each half-wave holds, and its softmax statistics are plain per-lane
// scalars:
//   S^T = K Q^T    A = 32 K rows, B = the wave's 32 query rows, k = dimensions;
//   O^T = V^T P^T  A = V^T (32 dimensions), B = P^T, k = K/V rows.
// MFMA lane layout (probed on MI355X): lane l, half h = l/32, holds
// A[l%32][8h+e] and B[8h+e][l%32] (e = 0..7) and receives D[8(v/4)+4h+v%4][l%32]
// (v = 0..15). The k index of the second product is a free permutation, so the
// registers of S^T are its B operand as they are: slot (h, e) of step t is K/V
// row 16t + 8(e/4) + 4h + e%4.
//
// K and V tiles lie in LDS as fp16 rows of 2D bytes whose 16-byte chunks are
// permuted by XOR with swz(row): both the K reads (32 rows, one chunk) and the
// transposing V reads (4 rows, four adjacent chunks) then touch every bank once.
// The V reads are ds_read_b64_tr_b16: of the 4x4 blocks that 16 lanes address
// (lane i: row i/4, values 4(i%4)..+3) lane i receives column i, rows 0..3
// (probed on MI355X).
#pragma once
#include "va_device.hpp"

namespace va {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef short    s16x4 __attribute__((ext_vector_type(4)));
typedef float    f32x2 __attribute__((ext_vector_type(2)));
typedef float    f32x16 __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) uint8_t lds_u8;
typedef __attribute__((address_space(3))) int lds_int;
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
typedef __attribute__((address_space(3))) f16x8 lds_f16x8;

__device__ __forceinline__ f32x16 mfma_32x32x16(const f16x8& a, const f16x8& b, const f32x16& c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

// XOR of the 16-byte chunk index of LDS row `row`. D = 128: a row is all 64 banks,
// so the four rows of a transposing read go to its four quarters; D = 64: two rows
// share the banks, so pairs of rows go to its two halves.
template <int D> __device__ __forceinline__ int swz(int row) {
    return D == 128 ? ((row & 3) << 2) | ((row >> 2) & 3) : ((row & 2) << 1) | ((row >> 2) & 3);
}

// The running maximum that weights are relative to follows lazily: the largest weight is held as
// 2^WIDE_OFF at least (fp16 keeps the digits of a weight down to 2^-14, so down to 2^-24 of it)
// and may grow by 2^WIDE_SLACK before sums and output are rescaled, which a wave then rarely does.
// (2^4 with room for 2^8 left the weights 16 below a row's maximum, e^-16, 5 bits; five prompts of up
// to 261 tokens took 12.2 us with it, 12.3 now, the longer ones the same.)
constexpr float WIDE_OFF = 10.f, WIDE_SLACK = 5.f;

// x combined over the two half-waves (lanes l and l^32).
__device__ __forceinline__ float halves_max(float x) {
    unsigned a = __builtin_bit_cast(unsigned, x), b = a;
    permlane32_swap(a, b);
    return fmaxf(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b));
}
__device__ __forceinline__ float halves_sum(float x) {
    unsigned a = __builtin_bit_cast(unsigned, x), b = a;
    permlane32_swap(a, b);
    return __builtin_bit_cast(float, a) + __builtin_bit_cast(float, b);
}

// LDS addresses of a wave's operands in a K tile and a V tile (byte offsets from
// the tile's start). Rows 32 apart differ by 64D bytes in the address only, and the
// chunks of one row by an XOR, so that three registers are enough; fresh() keeps the
// compiler from holding all their XORs across a loop.
template <int D> struct WideAddr {
    uint32_t k0, v0[2];
    // row0: the tile's row that the wave's blocks begin at, a multiple of 32
    __device__ __forceinline__ void init(int lane, int row0 = 0) {
        const int h = lane >> 5, row = lane & 31;
        k0 = (uint32_t)((row0 + row) * 2 * D + ((h ^ swz<D>(row)) << 4));
        const int i = lane & 15;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int key = 8 * r + 4 * h + (i >> 2), chunk = 2 * ((lane >> 4) & 1) + ((i & 3) >> 1);
            v0[r] = (uint32_t)((row0 + key) * 2 * D + ((chunk ^ swz<D>(key)) << 4) + (i & 1) * 8);
        }
    }
    __device__ __forceinline__ WideAddr fresh() const {
        WideAddr a = *this;
        asm volatile("" : "+v"(a.k0), "+v"(a.v0[0]), "+v"(a.v0[1]));
        return a;
    }
    __device__ __forceinline__ uint32_t k(int s) const { return k0 ^ (uint32_t)(s << 5); }          // chunk of step s of this lane's row
    __device__ __forceinline__ uint32_t v(int db, int r) const { return v0[r] ^ (uint32_t)(db << 6); }   // V^T block db, rows 8r + ..
};

__device__ __forceinline__ f16x8 lds_row8(const lds_u8* p, uint32_t at) {
    return *reinterpret_cast<const lds_f16x8*>(p + at);
}
__device__ __forceinline__ f16x8 lds_tr8(lds_u8* p, uint32_t a, uint32_t b) {
    const f16x4 x = __builtin_bit_cast(f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_s16x4*>(p + a)));
    const f16x4 y = __builtin_bit_cast(f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_s16x4*>(p + b)));
    return __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
}

// Order for the scheduler of N matrix products with R LDS reads each, in the scheduling
// region that this call ends: the reads of the next DEEP products are always on their way.
template <int N, int R, int DEEP> __device__ __forceinline__ void feed_mfma() {
    __builtin_amdgcn_sched_group_barrier(0x100, DEEP * R, 0);
#pragma unroll
    for (int i = 0; i < N - DEEP; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, R, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, DEEP, 0);
}

// O^T += V^T P^T over NB 32-row V blocks from `v` on; p: their S^T registers as fp16.
template <int D, int NB>
__device__ __forceinline__ void wide_values(lds_u8* v, const WideAddr<D>& ad, const f16x8 (&p)[NB][2], f32x16 (&o)[D / 32]) {
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int db = 0; db < D / 32; ++db) {
                const uint32_t at = (uint32_t)((b * 32 + t * 16) * 2 * D);
                o[db] = mfma_32x32x16(lds_tr8(v, ad.v(db, 0) + at, ad.v(db, 1) + at), p[b][t], o[db]);
            }
    feed_mfma<NB * D / 16, 2, 4>();
    __builtin_amdgcn_sched_barrier(0);
}

// A row that a query row does not see has the weight 0 there, and 0 times an infinite or NaN value
// is NaN: tiles with such rows go into the product without these values, and who sees them adds
// them to the finished sums. `x` without them; whether there are any.
__device__ __forceinline__ bool wide_clean(u32x4& x) {
    uint32_t any = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const uint32_t odd = ((x[e] & 0x7C007C00u) + 0x04000400u) & 0x80008000u;   // an exponent of ones carries into bit 15
        any |= odd;
        x[e] &= ~((odd << 1) - (odd >> 15));                // the halves of odd values: all ones
    }
    return any != 0;
}
// value, if it is one of these, else 0
__device__ __forceinline__ float wide_odd(float x) { return __builtin_fabsf(x) < __builtin_inff() ? 0.f : x; }

// S^T of NB 32-row K blocks from `k` on, K reads DEEP products ahead; TWO: K's second fp16 terms
// are at `k2`.
template <int D, int NB, int DEEP, bool TWO>
__device__ __forceinline__ void wide_scores(const lds_u8* k, const lds_u8* k2, const WideAddr<D>& ad, const f16x8 (&q)[D / 16], f32x16 (&s)[NB]) {
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int b = 0; b < NB; ++b) s[b] = f32x16{};
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
        if (TWO)
#pragma unroll
            for (int b = 0; b < NB; ++b) s[b] = mfma_32x32x16(lds_row8(k2 + b * 64 * D, ad.k(i)), q[i], s[b]);
#pragma unroll
        for (int b = 0; b < NB; ++b) s[b] = mfma_32x32x16(lds_row8(k + b * 64 * D, ad.k(i)), q[i], s[b]);
    }
    feed_mfma<NB * D / 16 * (TWO ? 2 : 1), 1, DEEP>();
    __builtin_amdgcn_sched_barrier(0);
}

// The weights of NB blocks of scores, exp2(s qs - m) with m = the lazy maximum times qs, less
// WIDE_OFF; their part of the sum l, and the rescale of what is there.
template <int D, int NB>
__device__ __forceinline__ void wide_weights(const f32x16 (&s)[NB], float qs, float& m, float& l, f32x16 (&o)[D / 32], f16x8 (&p)[NB][2]) {
    float top = s[0][0];
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int v = 0; v < 16; ++v) top = fmaxf(top, s[b][v]);
    top = halves_max(top);
    if (__any(__builtin_fmaf(top, qs, -m) > WIDE_OFF + WIDE_SLACK)) {   // also at the first one: m = -inf
        const float to = fmaxf(m, __builtin_fmaf(top, qs, -WIDE_OFF)), f = to == m ? 1.f : fast_exp2(m - to);
        m = to;
        l *= f;
#pragma unroll
        for (int db = 0; db < D / 32; ++db) o[db] *= f;
    }
    const float base = m == -__builtin_inff() ? 0.f : m;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int v = 0; v < 16; ++v) {
            const float e = fast_exp2(__builtin_fmaf(s[b][v], qs, -base));
            l += e;
            p[b][v / 8][v % 8] = (_Float16)e;
        }
}

// A barrier that waits for this wave's LDS reads and all but the last N of its loads to LDS.
// (__syncthreads would wait for every load.)
template <int N> __device__ __forceinline__ void barrier_but() {
    static_assert(N == 0 || N == 2 || N == 4, "loads per operand");
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (N == 0) asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if constexpr (N == 2) asm volatile("s_waitcnt vmcnt(2) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if constexpr (N == 4) asm volatile("s_waitcnt vmcnt(4) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

template <int N> __device__ __forceinline__ void wait_loads() {
    static_assert(N == 0 || N == 2 || N == 4, "loads per operand");
    if constexpr (N == 0) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if constexpr (N == 2) asm volatile("s_waitcnt vmcnt(2)" ::: "memory");
    if constexpr (N == 4) asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
}

// A tile of WIDE_BN fp16 rows (row_bytes apart; uniform) on its way to LDS, a quarter by each wave
// of a 4-wave group, 16 bytes per lane and load, zeros from out of range: the whole offset is in the
// vector operand, which the descriptor's range check covers by its documentation. (With the rows in
// the scalar operand a short tile relies on a check of the sum, which MI355X makes; no slower so:
// one prompt of 16384 tokens 2.06 ms with either.) Load i of a wave covers
// rows (wave N + i) ROWS + lane / (D/8); its lanes fetch the chunks that swz() puts in their
// places, which are those of load 0 with another XOR.
constexpr int WIDE_BN = 64;
template <int D> struct WideFetch {
    static constexpr int TILE = WIDE_BN * 2 * D, N = TILE / 1024 / 4, ROWS = 1024 / (2 * D);
    int wave;
    uint32_t row_bytes, at, chunk;
    __device__ __forceinline__ WideFetch(int w, int lane, uint32_t bytes) : wave(w), row_bytes(bytes) {
        const uint32_t row = (uint32_t)(w * N * ROWS + lane / (D / 8));
        at = row * bytes;
        chunk = (uint32_t)((lane % (D / 8)) ^ swz<D>((int)row)) << 4;
    }
    __device__ __forceinline__ void operator()(__amdgpu_buffer_rsrc_t r, lds_u8* to) const {
#pragma unroll
        for (int i = 0; i < N; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(r, to + (wave * N + i) * 1024, 16,
                                                     at + (uint32_t)(i * ROWS) * row_bytes + (chunk ^ (uint32_t)((D == 128 ? i : 2 * i) << 4)), 0, 0, 0);
    }
};

// One pass over the fp16 K/V tiles t0 .. t1 - 1 (t0 < t1) of a 4-wave group, 32 query rows to a
// wave. K is fetched a tile ahead and V during its tile's scores (fetch_k(t, to), fetch_v(t, to));
// mask(t, s) takes what a row does not see out of the scores, hides(t) is whether it does so for
// any row of the group: V is then cleaned, and *odd set where that took something out. LDS: K of
// two tiles, V of one. Three work-groups fit a CU (D = 128: 168 registers, 48 KB) and cover what
// a wave waits for.
template <int D, int DEEP, class FK, class FV, class HD, class MK>
__device__ __forceinline__ void wide_walk(lds_u8* lds, const WideAddr<D>& ad0, const f16x8 (&q)[D / 16], int t0, int t1, float qs,
                                          FK&& fetch_k, FV&& fetch_v, HD&& hides, MK&& mask, lds_int* odd, float& m, float& l, f32x16 (&o)[D / 32]) {
    constexpr int TILE = WideFetch<D>::TILE, NB = WIDE_BN / 32, N = WideFetch<D>::N;
    lds_u8* vt = lds + 2 * TILE;
    fetch_k(t0, lds);
    for (int t = t0, cur = 0; t < t1; ++t, cur ^= TILE) {
        barrier_but<0>();                                   // K has arrived; V of the last tile is read
        const WideAddr<D> ad = ad0.fresh();
        fetch_v(t, vt);
        const bool more = t + 1 < t1;
        if (more) fetch_k(t + 1, lds + (cur ^ TILE));
        f32x16 s[NB];
        wide_scores<D, NB, DEEP, false>(lds + cur, nullptr, ad, q, s);
        mask(t, s);
        f16x8 p[NB][2];
        wide_weights<D, NB>(s, qs, m, l, o, p);
        if (hides(t)) {                                     // every wave what it fetched itself
            if (more) wait_loads<N>();
            else wait_loads<0>();
            lds_u8* to = vt + (int)threadIdx.x / 64 * (N * 1024) + (int)__lane_id() * 16;
            bool any = false;
#pragma unroll 1
            for (int i = 0; i < N; ++i, to += 1024) {
                u32x4 x = __builtin_bit_cast(u32x4, lds_row8(to, 0u));
                if (wide_clean(x)) {
                    any = true;
                    *reinterpret_cast<lds_f16x8*>(to) = __builtin_bit_cast(f16x8, x);
                }
            }
            if (any) *odd = 1;
        }
        if (more) barrier_but<N>();                         // V has arrived, K of the next tile may not have
        else barrier_but<0>();
        wide_values<D, NB>(vt, ad, p, o);
    }
}

} // namespace va
