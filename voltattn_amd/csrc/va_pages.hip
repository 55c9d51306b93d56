// va_pages.hip — the page pool's bookkeeping and row moves: va_compact_kv,
// va_fork_pages and va_resize_pages.
//
// The pool's state is refs[num_pages], how many sequences hold each page: a page is
// free when its count is 0, and pages are handed out lowest id first, so the result
// depends on nothing but the arguments. A sequence of n positions holds the first
// ceil(n / page_rows) entries of its block-table row; entries behind them are -1. Ids
// outside the pool are carried along and never counted, read or written.
#include "va_device.hpp"
#include "va_kernels.hpp"

namespace va {

constexpr int PLAN_T = 1024;          // threads of the planning work-group
constexpr int PLAN_IDS = 8;           // page counts that one of its threads looks at at once

__device__ __forceinline__ int pages_of(int n, int page_rows) { return n <= 0 ? 0 : (n - 1) / page_rows + 1; }
__device__ __forceinline__ bool in_pool(const PageArgs& a, int id) { return id >= 0 && id < a.num_pages; }

// Inclusive sum over the work-group's threads; total: of all. `s`: a word per wave.
template <int THREADS>
__device__ __forceinline__ int block_scan(int x, int* s, int& total) {
    const int wave = (int)threadIdx.x >> 6;
    const int upto = wave_scan(x);
    __syncthreads();
    if ((threadIdx.x & 63) == 63) s[wave] = upto;
    __syncthreads();
    int before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) {
        if (w < wave) before += s[w];
        total += s[w];
    }
    return before + upto;
}

// How many of parents[0 .. n) are `p`, by the lanes of one wave.
__device__ __forceinline__ int count_parents(const int32_t* parents, int n, int p) {
    int kids = 0;
    for (int c0 = 0; c0 < n; c0 += 64) {
        const int c = c0 + (int)__lane_id();
        kids += __popcll(__ballot(c < n && parents[c] == p));
    }
    return kids;
}

// A child's block-table row and length, by one wave. The entry of a page that it needs of
// its own (a later child's copy of the partly filled last page) is -2.
__device__ __forceinline__ void fork_child(const PageArgs& a, int c) {
    const int p = a.parents[c], lane = (int)__lane_id();
    const bool has = p >= 0 && p < a.B;
    const int cap = a.max_pages * a.page_rows;
    const int len = has ? max(0, min(a.lens[p], cap)) : 0;
    const int own = pages_of(len, a.page_rows), full = len / a.page_rows;
    const bool later = has && count_parents(a.parents, c, p) > 0;
    const int32_t* from = a.table + (size_t)(has ? p : 0) * a.max_pages;
    int32_t* to = a.new_table + (size_t)c * a.max_pages;
    for (int i = lane; i < a.max_pages; i += 64) {
        int id = i < own ? from[i] : -1;
        if (later && i == full && in_pool(a, id)) id = -2;          // i < own here: the page in part
        to[i] = id;
    }
    if (lane == 0) a.new_lens[c] = len;
}
// The counts of a parent's pages: every child more holds the full ones, the first child
// keeps the last one, and without children all are given up.
__device__ __forceinline__ void fork_parent(const PageArgs& a, int p) {
    const int cap = a.max_pages * a.page_rows;
    const int len = max(0, min(a.lens[p], cap));
    const int own = pages_of(len, a.page_rows), full = len / a.page_rows;
    const int kids = count_parents(a.parents, a.children, p);
    const int32_t* from = a.table + (size_t)p * a.max_pages;
    for (int i = (int)__lane_id(); i < own; i += 64) {
        const int id = from[i], more = (i < full ? kids : min(kids, 1)) - 1;
        if (more != 0 && in_pool(a, id)) atomicAdd(a.refs + id, more);
    }
}
// Sequence b's entries given up and asked for, by one wave.
__device__ __forceinline__ void resize_row(const PageArgs& a, int b) {
    const int cap = a.max_pages * a.page_rows;
    const int n0 = pages_of(min(a.lens[b], cap), a.page_rows), n1 = pages_of(min(a.after[b], cap), a.page_rows);
    int32_t* row = a.new_table + (size_t)b * a.max_pages;
    for (int i = min(n0, n1) + (int)__lane_id(); i < max(n0, n1); i += 64) {
        if (i < n0) {
            const int id = row[i];
            if (in_pool(a, id)) atomicAdd(a.refs + id, -1);
        }
        row[i] = -1;
    }
}
// The pages that row b of new_table asks for: `first` and how many.
template <bool FORK>
__device__ __forceinline__ int asked(const PageArgs& a, int b, int& first) {
    const int cap = a.max_pages * a.page_rows;
    if (FORK) {
        const int len = a.new_lens[b];
        first = len / a.page_rows;
        return first < a.max_pages && a.new_table[(size_t)b * a.max_pages + first] == -2;
    }
    first = pages_of(min(a.lens[b], cap), a.page_rows);
    return max(0, pages_of(min(a.after[b], cap), a.page_rows) - first);
}

// Rows and counts of a large batch, a wave to a sequence: children, then parents.
template <bool FORK>
__global__ __launch_bounds__(256) void pages_rows(PageArgs a) {
    const int i = (int)blockIdx.x * 4 + ((int)threadIdx.x >> 6);
    if (FORK) {
        if (i < a.children) fork_child(a, i);
        else if (i < a.children + a.B) fork_parent(a, i - a.children);
    } else if (i < a.B) {
        resize_row(a, i);
    }
}

// Hands out the lowest free pages, in (sequence, index) order: one work-group. ALL: it
// also does pages_rows' part first. Counts changed by this launch's atomics are read from
// the coherence point, never from a line cached before.
template <bool FORK, bool ALL>
__global__ __launch_bounds__(PLAN_T) void pages_take(PageArgs a) {
    __shared__ int s_scan[PLAN_T / 64];
    __shared__ int s_upto[PLAN_T];
    const int tid = (int)threadIdx.x, wave = tid >> 6;
    if (ALL) {
        if (FORK) {
            for (int c = wave; c < a.children; c += PLAN_T / 64) fork_child(a, c);
            for (int p = wave; p < a.B; p += PLAN_T / 64) fork_parent(a, p);
        } else {
            for (int b = wave; b < a.B; b += PLAN_T / 64) resize_row(a, b);
        }
        __threadfence();
        __syncthreads();
    }
    const int rows = FORK ? a.children : a.B;
    int cursor = 0, missing = 0;                            // every page below cursor is taken
    for (int b0 = 0; b0 < rows; b0 += PLAN_T) {
        const int b = b0 + tid;
        int first = 0, total;
        const int need = b < rows ? asked<FORK>(a, b, first) : 0;
        const int upto = block_scan<PLAN_T>(need, s_scan, total);
        s_upto[tid] = upto;
        __syncthreads();
        int got = 0;                                        // of these sequences' requests
        while (got < total && cursor < a.num_pages) {
            const int id0 = cursor + tid * PLAN_IDS;
            int n = 0, found;
            uint32_t free = 0;
#pragma unroll
            for (int k = 0; k < PLAN_IDS; ++k)
                if (id0 + k < a.num_pages && (int)load_dev(reinterpret_cast<const unsigned*>(a.refs) + id0 + k) == 0) {
                    free |= 1u << k;
                    ++n;
                }
            int rank = got + block_scan<PLAN_T>(n, s_scan, found) - n;
            for (; free && rank < total; free &= free - 1, ++rank) {
                const int id = id0 + __builtin_ctz(free);
                int lo = 0, hi = PLAN_T - 1;                // the sequence whose requests end behind `rank`
                while (lo < hi) {
                    const int mid = (lo + hi) >> 1;
                    if (s_upto[mid] > rank) hi = mid; else lo = mid + 1;
                }
                int at;
                asked<FORK>(a, b0 + lo, at);
                at += rank - (lo ? s_upto[lo - 1] : 0);
                a.new_table[(size_t)(b0 + lo) * a.max_pages + at] = id;
                store_dev(reinterpret_cast<unsigned*>(a.refs) + id, 1u);
            }
            const bool more = got + found < total;
            got = min(total, got + found);
            if (more) cursor += PLAN_T * PLAN_IDS;
            __threadfence();
            __syncthreads();
        }
        missing += total - got;
        if (FORK && need && upto > got) a.new_table[(size_t)b * a.max_pages + first] = -1;
        __syncthreads();                                    // s_upto is read
    }
    if (tid == 0 && a.missing) *a.missing = missing;
}

// Copies `bytes` from src to dst (one work-group), in U-byte words.
template <typename U>
__device__ __forceinline__ void copy_words(const uint8_t* src, uint8_t* dst, size_t bytes) {
    const U* s = reinterpret_cast<const U*>(src);
    U* d = reinterpret_cast<U*>(dst);
    const size_t n = bytes / sizeof(U);
    size_t i = threadIdx.x;
    for (; i + 3 * 256 < n; i += 4 * 256) {
        U x[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = s[i + 256 * k];
#pragma unroll
        for (int k = 0; k < 4; ++k) d[i + 256 * k] = x[k];
    }
    for (; i < n; i += 256) d[i] = s[i];
}
__device__ __forceinline__ void copy_any(const uint8_t* src, uint8_t* dst, size_t bytes) {
    const uint64_t all = (uint64_t)(uintptr_t)src | (uint64_t)(uintptr_t)dst | bytes;
    if (!(all & 15)) copy_words<u32x4>(src, dst, bytes);
    else if (!(all & 3)) copy_words<uint32_t>(src, dst, bytes);
    else copy_words<uint16_t>(src, dst, bytes);
}

// The rows in use of every page that pages_take gave to a later child, from its parent's.
__global__ __launch_bounds__(256) void fork_copy(PageArgs a) {
    const int hk = (int)blockIdx.x % a.hkv, c = (int)blockIdx.x / a.hkv;
    const int p = a.parents[c];
    if (p < 0 || p >= a.B) return;
    const int len = a.new_lens[c], last = len / a.page_rows, rest = len - last * a.page_rows;
    if (rest == 0) return;
    const int from = a.table[(size_t)p * a.max_pages + last], to = a.new_table[(size_t)c * a.max_pages + last];
    if (from == to || !in_pool(a, from) || !in_pool(a, to)) return;
    const size_t fr = ((size_t)from * a.hkv + hk) * a.page_rows, tr = ((size_t)to * a.hkv + hk) * a.page_rows;
    uint8_t* pool = blockIdx.y == 0 ? a.k : a.v;
    copy_any(pool + fr * a.row_bytes, pool + tr * a.row_bytes, (size_t)rest * a.row_bytes);
    if (a.scale_bytes) {
        uint8_t* sp = blockIdx.y == 0 ? a.sk : a.sv;
        copy_any(sp + fr * a.scale_bytes, sp + tr * a.scale_bytes, (size_t)rest * a.scale_bytes);
    }
}

// ------------------------------------------------------------ compaction --
constexpr int COMPACT_MAX = 64;       // kept rows per sequence

// Pool row of position p of sequence b and K/V head hk, or -1.
__device__ __forceinline__ long long pool_row(const PageArgs& a, int b, int hk, long long p) {
    if (p < 0 || p >= (long long)a.max_pages * a.page_rows) return -1;
    const int pi = (int)p / a.page_rows, id = a.table[(size_t)b * a.max_pages + pi];
    return in_pool(a, id) ? ((long long)id * a.hkv + hk) * a.page_rows + ((int)p - pi * a.page_rows) : -1;
}

// One (sequence, K/V head) and tensor: every kept row is in registers before the first
// one is written, so any order and repetition of `keep` is a plain gather. U: the words
// that rows are moved in, MAXW of them to a row at most.
template <typename U, int MAXW>
__global__ __launch_bounds__(256) void compact_rows(PageArgs a) {
    constexpr int PER = COMPACT_MAX * MAXW / 256;
    __shared__ long long s_from[COMPACT_MAX], s_to[COMPACT_MAX];
    const int hk = (int)blockIdx.x % a.hkv, b = (int)blockIdx.x / a.hkv, tid = (int)threadIdx.x;
    const int n = max(0, min(a.counts[b], a.n));
    if (n == 0) return;
    if (tid < n) {
        const long long base = a.lens[b];
        const int k = a.keep[(size_t)b * a.n + tid];
        s_from[tid] = base < 0 || k < 0 ? -1 : pool_row(a, b, hk, base + k);
        s_to[tid] = base < 0 ? -1 : pool_row(a, b, hk, base + tid);
    }
    __syncthreads();
    uint8_t* pool = blockIdx.y == 0 ? a.k : a.v;
    const int w = a.row_bytes / (int)sizeof(U), ng = a.scale_bytes / 2;
    U x[PER];
    uint16_t sc = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int at = i * 256 + tid, r = at / w;
        if (r < n && s_from[r] >= 0) x[i] = reinterpret_cast<const U*>(pool + s_from[r] * a.row_bytes)[at - r * w];
    }
    uint16_t* sp = reinterpret_cast<uint16_t*>(blockIdx.y == 0 ? a.sk : a.sv);
    const int sr = ng ? tid / ng : n;                       // at most 4 scales a row: one per thread
    if (sr < n && s_from[sr] >= 0) sc = sp[s_from[sr] * ng + (tid - sr * ng)];
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");        // this wave's loads have arrived,
    __syncthreads();                                        // and every other's
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int at = i * 256 + tid, r = at / w;
        if (r < n && s_from[r] >= 0 && s_to[r] >= 0) reinterpret_cast<U*>(pool + s_to[r] * a.row_bytes)[at - r * w] = x[i];
    }
    if (sr < n && s_from[sr] >= 0 && s_to[sr] >= 0) sp[s_to[sr] * ng + (tid - sr * ng)] = sc;
}

hipError_t launch_compact(const PageArgs& a, hipStream_t stream) {
    const dim3 grid((unsigned)((size_t)a.B * a.hkv), 2), block(256);
    if (a.wide) hipLaunchKernelGGL((compact_rows<u32x4, 16>), grid, block, 0, stream, a);
    else hipLaunchKernelGGL((compact_rows<uint32_t, 32>), grid, block, 0, stream, a);
    return hipGetLastError();
}

// One launch plans a small batch; a large one's rows are dealt over the device first.
static bool plan_in_one(const PageArgs& a, int rows) { return rows <= 128 && (long long)rows * a.max_pages <= 1 << 15; }

hipError_t launch_resize(const PageArgs& a, hipStream_t stream) {
    if (plan_in_one(a, a.B)) {
        hipLaunchKernelGGL((pages_take<false, true>), dim3(1), dim3(PLAN_T), 0, stream, a);
        return hipGetLastError();
    }
    hipLaunchKernelGGL((pages_rows<false>), dim3((unsigned)(a.B + 3) / 4), dim3(256), 0, stream, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((pages_take<false, false>), dim3(1), dim3(PLAN_T), 0, stream, a);
    return hipGetLastError();
}

hipError_t launch_fork(const PageArgs& a, hipStream_t stream) {
    hipError_t e;
    if (plan_in_one(a, a.children + a.B)) {
        hipLaunchKernelGGL((pages_take<true, true>), dim3(1), dim3(PLAN_T), 0, stream, a);
        e = hipGetLastError();
    } else {
        hipLaunchKernelGGL((pages_rows<true>), dim3((unsigned)(a.children + a.B + 3) / 4), dim3(256), 0, stream, a);
        e = hipGetLastError();
        if (e != hipSuccess) return e;
        hipLaunchKernelGGL((pages_take<true, false>), dim3(1), dim3(PLAN_T), 0, stream, a);
        e = hipGetLastError();
    }
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(fork_copy, dim3((unsigned)((size_t)a.children * a.hkv), 2), dim3(256), 0, stream, a);
    return hipGetLastError();
}

} // namespace va
