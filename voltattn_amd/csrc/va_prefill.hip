// va_prefill.hip — causal attention of whole prompts, packed one behind the other
// (va_prefill): row i of a sequence of n tokens attends its rows 0..i,
//   o_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp2((q_i.k_j - m_i) * log2(e)/sqrt(D)).
//
// A work-group of 4 waves takes 128 consecutive rows of one sequence and query head
// (32 per wave, as the columns of va_wide.hpp's tiles) and walks the K/V rows up to
// its own last one in tiles of 64, one pass with a running maximum and sum. Scores,
// statistics and the output are held in fp32; the weights p are rounded to fp16 (RNE)
// for the second product, an error of 2^-12 of each weight, independent between
// weights, so that of the output stays below its own rounding to fp16.
#include "va_wide.hpp"
#include "va_kernels.hpp"

namespace va {

constexpr int PF_BM = 128;         // query rows per work-group
constexpr int PF_BN = 64;          // K/V rows per tile

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

// 16 bytes per lane to LDS, lane l's at `to` + 16 l; zeros where the offset is out of range.
__device__ __forceinline__ void fetch_lds(__amdgpu_buffer_rsrc_t r, lds_u8* to, uint32_t off, uint32_t soff) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, to, 16, off, sgpr(soff), 0, 0);
}

// A barrier that waits for this wave's LDS reads and all but the last N of its loads to LDS.
// (__syncthreads would wait for every load.)
template <int N> __device__ __forceinline__ void barrier_but() {
    static_assert(N == 0 || N == 2 || N == 4, "loads per operand");
    if constexpr (N == 0) asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if constexpr (N == 2) asm volatile("s_waitcnt vmcnt(2) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if constexpr (N == 4) asm volatile("s_waitcnt vmcnt(4) lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

template <int D>
__global__ __launch_bounds__(256, 3) void prefill_causal(PrefillArgs a) {
    constexpr int KS = D / 16, DB = D / 32;
    constexpr int TILE = PF_BN * 2 * D;                     // bytes of a K (or V) tile
    constexpr int RPI = 1024 / (2 * D);                     // rows that one wave's 16-byte load covers
    constexpr int LPW = TILE / 1024 / 4;                    // loads per wave and tile
    __shared__ __align__(1024) uint8_t lds[3 * TILE];       // K of two tiles, V of one

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
    // Load i of the wave covers rows (wave LPW + i) RPI + lane / (D/8); its lanes fetch the chunks
    // that swz() puts in their places: those of load 0 with another XOR.
    const int lr = wave * LPW * RPI + lane / (D / 8);
    const uint32_t kr = (uint32_t)lr * (uint32_t)a.k_row * 2u, vr = (uint32_t)lr * (uint32_t)a.v_row * 2u;
    const uint32_t lc = (uint32_t)((lane % (D / 8)) ^ swz<D>(lr));
    WideAddr<D> ad0;
    ad0.init(lane);
    lds_u8* kt = (lds_u8*)lds;
    lds_u8* vt = kt + 2 * TILE;
    // Loads go straight to LDS (4 per wave and operand); a wave waits for its own, the barrier
    // behind the wait for everybody's. K is fetched a tile ahead, V during its tile's scores.
    auto fetch = [&](const uint16_t* rows, long long stride, uint32_t lane_row, int j0, lds_u8* to) {
        const int n = min(PF_BN, sp.n - j0);
        const __amdgpu_buffer_rsrc_t r = make_rsrc(rows + (size_t)j0 * stride, (uint32_t)(((n - 1) * (size_t)stride + D) * 2));
#pragma unroll
        for (int i = 0; i < LPW; ++i)
            fetch_lds(r, to + (wave * LPW + i) * 1024, lane_row + ((lc ^ (uint32_t)(D == 128 ? i : 2 * i)) << 4), (uint32_t)(i * RPI * 2) * (uint32_t)stride);
    };

    f32x16 o[DB] = {};
    float m = -__builtin_inff(), l = 0.f;                   // m: in raw scores
    const int last = min(r0 + PF_BM, sp.n);                 // keys that the work-group needs
    fetch(kp, a.k_row, kr, 0, kt);
    for (int j0 = 0, odd = 0; j0 < last; j0 += PF_BN, odd ^= TILE) {
        barrier_but<0>();                                   // K has arrived; V of the last tile is read
        const WideAddr<D> ad = ad0.fresh();
        fetch(vp, a.v_row, vr, j0, vt);
        const bool more = j0 + PF_BN < last;
        if (more) fetch(kp, a.k_row, kr, j0 + PF_BN, kt + (odd ^ TILE));
        __builtin_amdgcn_sched_barrier(0);
        f32x16 s[PF_BN / 32] = {};
#pragma unroll
        for (int i = 0; i < KS; ++i)
#pragma unroll
            for (int b = 0; b < PF_BN / 32; ++b) s[b] = mfma_32x32x16(lds_row8(kt + odd + b * 64 * D, ad.k(i)), q[i], s[b]);
        feed_mfma<PF_BN / 32 * KS, 1, 4>();
        __builtin_amdgcn_sched_barrier(0);
        if (j0 + PF_BN - 1 > r0 + wave * 32) {              // keys behind some row of the wave
#pragma unroll
            for (int b = 0; b < PF_BN / 32; ++b)
#pragma unroll
                for (int v = 0; v < 16; ++v)
                    if (j0 + 32 * b + 8 * (v / 4) + 4 * half + v % 4 > row) s[b][v] = -__builtin_inff();
        }
        float top = s[0][0];
#pragma unroll
        for (int b = 0; b < PF_BN / 32; ++b)
#pragma unroll
            for (int v = 0; v < 16; ++v) top = fmaxf(top, s[b][v]);
        top = halves_max(top);
        if (__any((top - m) * a.qscale > WIDE_SLACK)) {     // also at the first tile: m = -inf
            const float to = fmaxf(m, top), f = to == m ? 1.f : fast_exp2((m - to) * a.qscale);
            m = to;
            l *= f;
#pragma unroll
            for (int db = 0; db < DB; ++db) o[db] *= f;
        }
        const float base = m == -__builtin_inff() ? 0.f : m * a.qscale - WIDE_OFF;
        f16x8 p[PF_BN / 32][2];
#pragma unroll
        for (int b = 0; b < PF_BN / 32; ++b)
#pragma unroll
            for (int v = 0; v < 16; ++v) {
                const float e = fast_exp2(__builtin_fmaf(s[b][v], a.qscale, -base));
                l += e;
                p[b][v / 8][v % 8] = (_Float16)e;
            }
        __builtin_amdgcn_sched_barrier(0);
        if (more) barrier_but<LPW>();                       // V has arrived, K of the next tile may not have
        else barrier_but<0>();
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int b = 0; b < PF_BN / 32; ++b) wide_values<D>(vt + b * 64 * D, ad, p[b], o);
        feed_mfma<PF_BN / 32 * 2 * DB, 2, 4>();
    }
    l = halves_sum(l);
    if (!live) return;
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
