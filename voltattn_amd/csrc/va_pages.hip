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
constexpr int PLAN_ONE = 32;          // sequences (parents and children) that it plans by itself at most

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

// A child's block-table row and length, by one wave; true, and the entry, if it needs a page
// of its own there (a later child's copy of the partly filled last page): the entry is -1. NOTE:
// its length is then left as its complement for the next launch, which looks for no id, since any id
// outside the pool may be a parent's.
template <bool NOTE>
__device__ __forceinline__ bool fork_child(const PageArgs& a, const int32_t* parents, const int32_t* lens, int c, int& full) {
    const int p = parents[c], lane = (int)__lane_id();
    const bool has = p >= 0 && p < a.B;
    const int cap = a.max_pages * a.page_rows;
    const int len = has ? max(0, min(lens[p], cap)) : 0, own = pages_of(len, a.page_rows);
    full = len / a.page_rows;
    const bool later = has && count_parents(parents, c, p) > 0;
    const int32_t* from = a.table + (size_t)(has ? p : 0) * a.max_pages;
    int32_t* to = a.new_table + (size_t)c * a.max_pages;
    bool asks = false;
    for (int i = lane; i < a.max_pages; i += 64) {
        int id = i < own ? from[i] : -1;
        if (later && i == full && in_pool(a, id)) {         // i < own here: the page in part
            id = -1;
            asks = true;
        }
        to[i] = id;
    }
    asks = __any(asks);
    if (lane == 0) a.new_lens[c] = NOTE && asks ? ~len : len;
    return asks;
}
// The counts of a parent's pages: every child more holds the full ones, the first child
// keeps the last one, and without children all are given up.
template <int SCOPE>
__device__ __forceinline__ void fork_parent(const PageArgs& a, const int32_t* parents, const int32_t* lens, int p) {
    const int cap = a.max_pages * a.page_rows;
    const int len = max(0, min(lens[p], cap));
    const int own = pages_of(len, a.page_rows), full = len / a.page_rows;
    const int kids = count_parents(parents, a.children, p);
    const int32_t* from = a.table + (size_t)p * a.max_pages;
    for (int i = (int)__lane_id(); i < own; i += 64) {
        const int id = from[i], more = (i < full ? kids : min(kids, 1)) - 1;
        if (more != 0 && in_pool(a, id)) __hip_atomic_fetch_add(a.refs + id, more, __ATOMIC_RELAXED, SCOPE);
    }
}
// Sequence b's entries given up and asked for, by one wave; how many are asked for.
template <int SCOPE>
__device__ __forceinline__ int resize_row(const PageArgs& a, int b, int before, int after, int& first) {
    const int cap = a.max_pages * a.page_rows;
    const int n0 = pages_of(min(before, cap), a.page_rows), n1 = pages_of(min(after, cap), a.page_rows);
    int32_t* row = a.new_table + (size_t)b * a.max_pages;
    for (int i = min(n0, n1) + (int)__lane_id(); i < max(n0, n1); i += 64) {
        if (i < n0) {
            const int id = row[i];
            if (in_pool(a, id)) __hip_atomic_fetch_add(a.refs + id, -1, __ATOMIC_RELAXED, SCOPE);
        }
        row[i] = -1;
    }
    first = n0;
    return max(0, n1 - n0);
}

// Rows and counts of a large batch, a wave to a sequence: children, then parents.
template <bool FORK>
__global__ __launch_bounds__(256) void pages_rows(PageArgs a) {
    const int i = (int)blockIdx.x * 4 + ((int)threadIdx.x >> 6);
    int first;
    if (FORK) {
        if (i < a.children) (void)fork_child<true>(a, a.parents, a.lens, i, first);
        else if (i < a.children + a.B) fork_parent<__HIP_MEMORY_SCOPE_AGENT>(a, a.parents, a.lens, i - a.children);
    } else if (i < a.B) {
        (void)resize_row<__HIP_MEMORY_SCOPE_AGENT>(a, i, a.lens[i], a.after[i], first);
    }
}

// Hands out the lowest free pages, in (sequence, index) order: one work-group, which a round
// looks through PLAN_T * PLAN_IDS counts, lists the free ids and deals them to the sequences, a
// wave to each. ALL: it also does pages_rows' part first, every sequence's chain of loads at once.
template <bool FORK, bool ALL>
__global__ __launch_bounds__(PLAN_T) void pages_take(PageArgs a) {
    constexpr int WAVES = PLAN_T / 64;
    __shared__ int s_scan[WAVES];
    __shared__ int s_upto[PLAN_T], s_first[PLAN_T], s_need[ALL ? PLAN_ONE : 1], s_in[ALL ? 2 * PLAN_ONE : 1];
    __shared__ int s_free[PLAN_T * PLAN_IDS];
    const int tid = (int)threadIdx.x, wave = uniform(tid >> 6), lane = tid & 63;
    const int rows = FORK ? a.children : a.B;
    if constexpr (ALL) {                                    // at most PLAN_ONE sequences
        int* in0 = s_in;                                    // parents, or lengths before
        int* in1 = s_in + PLAN_ONE;                         // lengths, or lengths after
        if (tid < rows) in0[tid] = FORK ? a.parents[tid] : a.lens[tid];
        else if (tid >= PLAN_ONE && tid < PLAN_ONE + a.B) in1[tid - PLAN_ONE] = (FORK ? a.lens : a.after)[tid - PLAN_ONE];
        __syncthreads();
        for (int i = wave; i < rows + (FORK ? a.B : 0); i += WAVES) {
            int first = 0, need = 0;
            if (FORK && i >= rows) {
                fork_parent<__HIP_MEMORY_SCOPE_WORKGROUP>(a, in0, in1, i - rows);
                continue;
            }
            if (FORK) need = fork_child<false>(a, in0, in1, i, first);
            else need = resize_row<__HIP_MEMORY_SCOPE_WORKGROUP>(a, i, in0[i], in1[i], first);
            if (lane == 0) {
                s_first[i] = first;
                s_need[i] = need;
            }
        }
        // the counts are read below, for the first time in this launch, when all are changed
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
    }
    int cursor = 0, missing = 0;                            // every page below cursor is taken
    for (int b0 = 0; b0 < rows; b0 += PLAN_T) {
        const int b = b0 + tid;
        int need = 0, total;
        if (b < rows) {
            if constexpr (ALL) {
                need = s_need[b];
            } else {
                const int cap = a.max_pages * a.page_rows;
                int first;
                if (FORK) {
                    int len = a.new_lens[b];
                    need = len < 0;
                    if (need) a.new_lens[b] = len = ~len;
                    first = len / a.page_rows;
                } else {
                    first = pages_of(min(a.lens[b], cap), a.page_rows);
                    need = max(0, pages_of(min(a.after[b], cap), a.page_rows) - first);
                }
                s_first[tid] = first;
            }
        }
        const int upto = block_scan<PLAN_T>(need, s_scan, total);
        s_upto[tid] = upto;
        int got = 0;                                        // of these sequences' requests
        while (got < total && cursor < a.num_pages) {
            const int id0 = cursor + tid * PLAN_IDS;
            int n = 0, found;
            uint32_t free = 0;
            const __amdgpu_buffer_rsrc_t r = make_rsrc(a.refs + cursor, (uint32_t)min(a.num_pages - cursor, PLAN_T * PLAN_IDS) * 4u);
#pragma unroll
            for (int k = 0; k < PLAN_IDS; k += 4) {
                const u32x4 c = __builtin_amdgcn_raw_buffer_load_b128(r, (uint32_t)(tid * PLAN_IDS + k) * 4u, 0, 0);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (c[e] == 0 && id0 + k + e < a.num_pages) {
                        free |= 1u << (k + e);
                        ++n;
                    }
            }
            int rank = block_scan<PLAN_T>(n, s_scan, found) - n;   // among this round's
            for (; free && got + rank < total; free &= free - 1, ++rank) {
                const int id = id0 + __builtin_ctz(free);
                s_free[rank] = id;
                a.refs[id] = 1;
            }
            __syncthreads();
            const int end = min(total, got + found);
            for (int j = wave; j < min(PLAN_T, rows - b0); j += WAVES) {
                const int lo = j ? s_upto[j - 1] : 0, hi = min(s_upto[j], end);
                for (int k = max(lo, got) + lane; k < hi; k += 64)
                    a.new_table[(size_t)(b0 + j) * a.max_pages + s_first[j] + (k - lo)] = s_free[k - got];
            }
            if (got + found < total) cursor += PLAN_T * PLAN_IDS;
            got = end;
            __syncthreads();                                // s_free is read
        }
        missing += total - got;
        __syncthreads();                                    // s_upto and s_first are read
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
        if (r < n && s_from[r] >= 0 && s_to[r] >= 0) __builtin_nontemporal_store(x[i], reinterpret_cast<U*>(pool + s_to[r] * a.row_bytes) + (at - r * w));
    }
    if (sr < n && s_from[sr] >= 0 && s_to[sr] >= 0) sp[s_to[sr] * ng + (tid - sr * ng)] = sc;
}

hipError_t launch_compact(const PageArgs& a, hipStream_t stream) {
    const dim3 grid((unsigned)((size_t)a.B * a.hkv), 2), block(256);
    if (a.wide) hipLaunchKernelGGL((compact_rows<u32x4, 16>), grid, block, 0, stream, a);
    else hipLaunchKernelGGL((compact_rows<uint32_t, 32>), grid, block, 0, stream, a);
    return hipGetLastError();
}

// One launch plans a small batch; a large one's rows are dealt over the device first. One launch :
// two, us a call: a resize of 16 sequences 3.8 : 4.7, 32 4.6 : 5.1, 48 5.5 : 5.1, 128 9.3 : 6.0, about
// the same for tables of 8 to 4096 columns. A fork writes whole rows of the table (with a 2 us reset of the
// counts): 8 sequences into 8 9.9 : 10.2 with 256 columns, 13.2 : 12.4 with 1024; 16 into 16 10.2 : 10.0
// with 64, 11.3 : 10.6 with 256; 64 into 64 16.7 : 11.3 with 64.
static bool plan_in_one(const PageArgs& a, int rows, bool whole_rows) {
    return rows <= PLAN_ONE && (!whole_rows || (long long)rows * a.max_pages <= 1 << 12);
}

hipError_t launch_resize(const PageArgs& a, hipStream_t stream) {
    if (plan_in_one(a, a.B, false)) {
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
    if (plan_in_one(a, a.children + a.B, true)) {
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
