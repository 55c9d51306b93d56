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

// The running maximum that weights are relative to follows lazily: weights start at
// 2^WIDE_OFF (fp16 keeps their digits down to 2^-14, and some to 2^-24) and may grow by
// 2^WIDE_SLACK before sums and output are rescaled, which a wave then rarely does.
constexpr float WIDE_OFF = 4.f, WIDE_SLACK = 8.f;

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

// S^T of one 32-row K block at `k` (its first row's LDS address).
template <int D>
__device__ __forceinline__ f32x16 wide_scores(const lds_u8* k, const WideAddr<D>& ad, const f16x8 (&q)[D / 16]) {
    f32x16 s = {};
#pragma unroll
    for (int i = 0; i < D / 16; ++i) s = mfma_32x32x16(lds_row8(k, ad.k(i)), q[i], s);
    return s;
}

// O^T += V^T P^T over one 32-row V block at `v`; p: its S^T registers as fp16.
template <int D>
__device__ __forceinline__ void wide_values(lds_u8* v, const WideAddr<D>& ad, const f16x8 (&p)[2], f32x16 (&o)[D / 32]) {
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int db = 0; db < D / 32; ++db) {
            const uint32_t at = (uint32_t)(t * 16 * 2 * D);
            o[db] = mfma_32x32x16(lds_tr8(v, ad.v(db, 0) + at, ad.v(db, 1) + at), p[t], o[db]);
        }
}

} // namespace va
