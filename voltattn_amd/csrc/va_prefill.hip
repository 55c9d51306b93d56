// va_prefill.hip — causal attention of whole prompts, packed one behind the other
// (va_prefill): row i of a sequence of n tokens attends its rows 0..i,
//   o_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp2((q_i.k_j - m_i) * log2(e)/sqrt(D)).
//
// A work-group of 4 waves takes 128 consecutive rows of one sequence and query head
// (32 per wave, as the columns of va_wide.hpp's tiles) and walks the K/V rows up to
// its own last one in tiles of 64, one pass with a running maximum and sum. Scores,
// statistics and the output are held in fp32; the weights p are rounded to fp16 (RNE)
// for the second product, each off by at most 2^-11 of itself (down to 2^-24 of the row's
// largest, see WIDE_OFF), independently of each other, which adds to the output about
// the error of its own rounding to fp16 (together 1.3 to 1.4 times that).
//
// The matrix cores bound it: one prompt of 16384 tokens (Hq 32, Hkv 8, D 128) 1.96 ms, 1121
// TFLOP/s of the products that the mask leaves, where a plain 8192^3 fp16 product reaches 1465;
// the exponentials between the products take the rest. Twelve prompts of up to 4001 tokens 330 us
// (half-empty diagonal tiles, 1.11 of the products, besides), five of up to 261 12.3 us (latency). 128 rows to a work-group
// read K and V half as often as 64; three work-groups to a CU cover each other's softmax. The
// row tiles are begun from the batch's last: of one prompt the longest first, so that short ones
// fill the tail; of several, whose order is the caller's, prompt by prompt from the last one.
#include "va_wide.hpp"
#include "va_kernels.hpp"

namespace va {

constexpr int PF_BM = 128;         // query rows per work-group

// Rows [begin, begin + n) of the packed batch; keys: whether they are a sequence (the
// rows before the first and behind the last sequence are in none, and get zeros).
struct PrefillSpan {
    int begin, n, tile;
    bool keys;
};

// The spans are the rows between consecutive bounds 0, cu[0], .., cu[B], total (each
// limited to what lies between its predecessor and total). Item `item` of all their
// tiles of PF_BM rows; false behind the last one. Every wave scans by itself.
__device__ __forceinline__ bool prefill_span(const int32_t* __restrict__ cu, int B, int total, int item, PrefillSpan& sp) {
    const int lane = (int)__lane_id();
    int before = 0, prev = 0;                               // tiles and bound ahead of this round's first span
    for (int i0 = 0; i0 <= B + 1; i0 += 64) {
        const int i = i0 + lane;
        int e = i <= B ? cu[i] : total;
        e = max(0, min(e, total));
        e = max(prev, wave_scan_max(e));                    // bounds never fall back
        const int b = __builtin_amdgcn_update_dpp(prev, e, 0x138, 0xF, 0xF, false);   // wave shift right by one
        const int tiles = i <= B + 1 ? (e - b + PF_BM - 1) / PF_BM : 0;
        const int upto = before + wave_scan(tiles);
        const uint64_t hit = __ballot(upto > item);
        if (hit) {
            const int l = __builtin_ctzll(hit);
            sp.begin = __builtin_amdgcn_readlane(b, l);
            sp.n = __builtin_amdgcn_readlane(e, l) - sp.begin;
            sp.tile = item - (__builtin_amdgcn_readlane(upto, l) - __builtin_amdgcn_readlane(tiles, l));
            sp.keys = i0 + l >= 1 && i0 + l <= B;
            return true;
        }
        before = __builtin_amdgcn_readlane(upto, 63);
        prev = __builtin_amdgcn_readlane(e, 63);
    }
    return false;
}

template <int D>
__global__ __launch_bounds__(256, 3) void prefill_causal(PrefillArgs a) {
    constexpr int KS = D / 16, DB = D / 32;
    __shared__ __align__(1024) uint8_t lds[3 * WideFetch<D>::TILE + 4];
    lds_int* odd = (lds_int*)((lds_u8*)lds + 3 * WideFetch<D>::TILE);   // infinite or NaN values were left out

    const int lane = (int)__lane_id(), wave = uniform((int)threadIdx.x >> 6), half = lane >> 5;
    const int item = (int)(a.items - 1 - blockIdx.x / (unsigned)a.hq);
    const int hh = (int)(blockIdx.x % (unsigned)a.hq);
    const int head = (a.hq & 7) == 0 ? (hh & 7) * (a.hq >> 3) + (hh >> 3) : hh;
    PrefillSpan sp;
    if (!prefill_span(a.cu, a.B, a.total, item, sp)) return;

    const int r0 = sp.tile * PF_BM, row = r0 + wave * 32 + (lane & 31);
    const bool live = row < sp.n;
    uint16_t* out = a.out + ((size_t)(sp.begin + row) * a.hq + head) * D + 4 * half;
    if (!sp.keys) {
        if (live)
            for (int d = 0; d < D; d += 8) *reinterpret_cast<u32x2*>(out + d) = u32x2{0u, 0u};
        return;
    }
    f16x8 q[KS];
    {
        const uint16_t* qp = a.q + (size_t)(sp.begin + min(row, sp.n - 1)) * a.q_row + (size_t)head * a.q_head + 8 * half;
#pragma unroll
        for (int s = 0; s < KS; ++s) q[s] = *reinterpret_cast<const f16x8*>(qp + 16 * s);
    }
    const int hk = head / a.group;
    const uint16_t* kp = a.k + (size_t)sp.begin * a.k_row + (size_t)hk * a.k_head;
    const uint16_t* vp = a.v + (size_t)sp.begin * a.v_row + (size_t)hk * a.v_head;
    WideAddr<D> ad;
    ad.init(lane);
    const WideFetch<D> load_k(wave, lane, (uint32_t)a.k_row * 2u), load_v(wave, lane, (uint32_t)a.v_row * 2u);
    auto tile = [&](const WideFetch<D>& load, const uint16_t* rows, long long stride, int t, lds_u8* to) {
        const int j0 = t * WIDE_BN, n = min(WIDE_BN, sp.n - j0);
        load(make_rsrc(rows + (size_t)j0 * stride, (uint32_t)(((n - 1) * (size_t)stride + D) * 2)), to);
    };
    if (threadIdx.x == 0) *odd = 0;
    f32x16 o[DB] = {};
    float m = -__builtin_inff(), l = 0.f;
    wide_walk<D, 4>((lds_u8*)lds, ad, q, 0, (min(r0 + PF_BM, sp.n) + WIDE_BN - 1) / WIDE_BN, a.qscale,
        [&](int t, lds_u8* to) { tile(load_k, kp, a.k_row, t, to); }, [&](int t, lds_u8* to) { tile(load_v, vp, a.v_row, t, to); },
        [&](int t) { return t * WIDE_BN + WIDE_BN - 1 > r0; },
        [&](int t, f32x16 (&s)[WIDE_BN / 32]) {
            if (t * WIDE_BN + WIDE_BN - 1 <= r0 + wave * 32) return;    // no key is behind a row of the wave
            const int last = row - t * WIDE_BN - 4 * half;
#pragma unroll
            for (int b = 0; b < WIDE_BN / 32; ++b)
#pragma unroll
                for (int v = 0; v < 16; ++v)
                    s[b][v] = 32 * b + 8 * (v / 4) + v % 4 > last ? -__builtin_inff() : s[b][v];
        }, odd, m, l, o);
    l = halves_sum(l);
    if (!live) return;
    if (*odd)                                               // of the tiles from the block's first row's on
#pragma unroll 1
        for (int j = r0; j <= row; ++j)
#pragma unroll
            for (int d = 0; d < D / 8; ++d) {
                const f16x4 x = *reinterpret_cast<const f16x4*>(vp + (size_t)j * a.v_row + 8 * d + 4 * half);
#pragma unroll
                for (int i = 0; i < 4; ++i) o[d / 4][4 * (d % 4) + i] += wide_odd((float)x[i]);
            }
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
}

long long prefill_items(int total, int B) { return (long long)total / PF_BM + B + 2; }   // every span's last tile may be a part

hipError_t launch_prefill(int D, const PrefillArgs& args, hipStream_t stream) {
    PrefillArgs a = args;
    a.items = (int)prefill_items(a.total, a.B);
    const dim3 grid((unsigned)a.items * (unsigned)a.hq), block(256);
    if (D == 128) hipLaunchKernelGGL((prefill_causal<128>), grid, block, 0, stream, a);
    else hipLaunchKernelGGL((prefill_causal<64>), grid, block, 0, stream, a);
    return hipGetLastError();
}

} // namespace va
