// va_pack.hpp — the symmetric per-group quantizer and packer of a lane's consecutive
// elements, shared by the quantizer and the cache writes (va_quant.hip, va_rope.hip).
#pragma once
#include "va_device.hpp"

namespace va {

template <int BITS> struct QLim;
template <> struct QLim<8> { static constexpr int value = 127; };
template <> struct QLim<4> { static constexpr int value = 7; };
template <> struct QLim<3> { static constexpr int value = 3; };

// Written once and not read back by the kernel: a non-temporal store (append f16
// 26.0 -> 20.4 us, quantize q8 112.7 -> 105.5 in the sizes above, dequantize q8 66.6
// -> 47.9, against plain stores).
template <class T>
__device__ __forceinline__ void stream_store(T* p, T v) { __builtin_nontemporal_store(v, p); }

// Codes of E values against the group scale sh (its fp16 value): bit-exact with
// clamp(rint(x / sh)), a non-finite quotient giving 0. x * rcp(sh) is within 2^-22 of the
// IEEE quotient, relatively. A quotient of lim + 1 or more clamps whichever side of a
// boundary it lands; below, |quotient| < 128, so the two differ by less than 2^-15:
// where no value lies within 2^-14 of a rounding boundary (twice that; and none is NaN or
// infinite), rounding it gives the same code; otherwise the wave divides.
template <int BITS, int E>
__device__ __forceinline__ void quant_codes(const float (&x)[E], float sh, int (&code)[E]) {
    constexpr int lim = QLim<BITS>::value;
    const float r = __builtin_amdgcn_rcpf(sh);
    float n[E], far = 0.f, any = 0.f;              // largest distance to the code; NaN if one is
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const float y = x[i] * r;
        n[i] = __builtin_rintf(y);
        const float d = __builtin_fabsf(y - n[i]);
        far = fmaxf(far, d);
        any += d;
    }
    if (__builtin_amdgcn_ballot_w64(!(far < 0.5f - 0x1p-14f && any < (float)E)) != 0) {
        asm volatile("");                          // kept a branch: the divisions are not computed ahead of it
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const float t = x[i] / sh;
            n[i] = __builtin_isfinite(t) ? __builtin_rintf(t) : 0.f;
        }
    }
#pragma unroll
    for (int i = 0; i < E; ++i) code[i] = (int)__builtin_amdgcn_fmed3f(n[i], (float)-lim, (float)lim);
}

// The fp16 scale of a group from its largest |x|.
template <int BITS>
__device__ __forceinline__ uint16_t quant_scale(float amax) {
    return f2h_rne(amax > 0.f ? amax / (float)QLim<BITS>::value : 1.f);
}

// Pack the lane's E codes and write its share of the group's bytes, the lane's
// elements starting `e` elements into the 4-byte aligned stream at dst. q3: E codes
// are 12 or 24 bits; the four 24-bit values of 32 elements make three words, word k
// from values k and k + 1.
template <int BITS, int E>
__device__ __forceinline__ void pack_store(const int (&code)[E], uint8_t* dst, size_t e, bool on) {
    if constexpr (BITS == 8) {
        uint32_t w[E / 4];
#pragma unroll
        for (int k = 0; k < E / 4; ++k)
            w[k] = ((uint32_t)code[4 * k] & 0xFFu) | ((uint32_t)code[4 * k + 1] & 0xFFu) << 8 |
                   ((uint32_t)code[4 * k + 2] & 0xFFu) << 16 | (uint32_t)code[4 * k + 3] << 24;
        if (!on) return;
        uint32_t* d = reinterpret_cast<uint32_t*>(dst + e);
#pragma unroll
        for (int k = 0; k < E / 4; ++k) stream_store(d + k, w[k]);
    } else if constexpr (BITS == 4) {             // element i: byte i/2, low nibble when i even
        uint32_t w = 0;
#pragma unroll
        for (int i = 0; i < E; ++i) w |= (uint32_t)(code[i] + 8) << (4 * i);
        if (!on) return;
        if constexpr (E == 8) stream_store(reinterpret_cast<uint32_t*>(dst + e / 2), w);
        else stream_store(reinterpret_cast<uint16_t*>(dst + e / 2), (uint16_t)w);
    } else {                                       // element i: bits [3i, 3i+3), little endian
        uint32_t w = 0;
#pragma unroll
        for (int i = 0; i < E; ++i) w |= (uint32_t)(code[i] + 4) << (3 * i);
        constexpr int SPAN = 32 / E;               // lanes of 32 elements
        const int l = (int)(threadIdx.x & (SPAN - 1));
        uint32_t next;                             // the next 24-bit value of the same 32 elements
        if constexpr (E == 4) {                    // pairs of lanes make a value, in the even lane
            w |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)w, DPP_QP_XOR1, 0xF, 0xF, true) << 12;
            next = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)w, 0x102 /* row_shl:2 */, 0xF, 0xF, true);
        } else {
            next = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)w, 0x101 /* row_shl:1 */, 0xF, 0xF, true);
        }
        const int k = E == 4 ? l >> 1 : l;
        if (!on || k == 3 || (E == 4 && (l & 1))) return;
        stream_store(reinterpret_cast<uint32_t*>(dst) + (e / 32) * 3 + k, (w & 0xFFFFFFu) >> (8 * k) | next << (24 - 8 * k));
    }
}

} // namespace va
