// Page tables, slots and positions of a step from the requests' lengths (gfx950).
//
// Integers only, a few bytes a request and row: bound by latency (64 requests of one row
// 5.4 us, 256 of 8500 rows 9.4; a small launch takes 2).  One workgroup
// does the whole step: the requests' sums (rows, pages given back, pages taken)
// are three scans over LDS, then the pages move (a thread a page), then the rows
// are mapped (a thread a row), each finding its request by bisection of the sums.
// The stack of free pages is also what carries a page from the request that gives
// it back to the one that takes it: pushes, a barrier, pops.
#pragma once

#include "krk_common.h"

namespace krk {

struct PageStepParams {
    int32_t* lens;
    const int32_t *keep, *fresh, *labels;
    int32_t* table;
    int64_t table_row;
    int32_t *free_pages, *free_count;
    int32_t *starts, *keys, *slots, *positions, *owner;
    int B, rows, pages, shift, width;
};

constexpr int kPageThreads = 1024;
constexpr int kPageWaves = kPageThreads / 64;

__host__ __device__ constexpr size_t page_step_lds_bytes(int B) { return (size_t)(5 * B + 4) * sizeof(int); }

// Sum over the lanes up to this one.
__device__ __forceinline__ int wave_scan(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, true);  // row_shr 1, 2, 4, 8
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);  // lane 15 of each row to rows 1 and 3
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);  // lane 31 to the upper half
    return v;
}

// What comes before this thread's v in the workgroup; the sum of all to *total.
__device__ __forceinline__ int block_scan(int v, int* scratch, int* total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int in = wave_scan(v);
    __syncthreads();  // the scratch is free again
    if (lane == 63) scratch[wave] = in;
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kPageWaves; ++w) {
        before += w < wave ? scratch[w] : 0;
        all += scratch[w];
    }
    *total = all;
    return before + in - v;
}

// The last i of n with first[i] <= x (first ascends, first[0] <= x).
__device__ __forceinline__ int owner_of(const int* first, int n, int x) {
    int lo = 0;
    while (n > 1) {
        const int half = n >> 1;
        if (first[lo + half] <= x) lo += half;
        n -= half;
    }
    return lo;
}

// N rows of the step, r, r + apart, ...: starts and keys as the step leaves them.  Side by
// side, as each is a chain of reads (requests' sums, table, label): 8500 rows of 256
// requests in one workgroup took 9 us one after the other, four at a time 6.
template <int N>
__device__ __forceinline__ void map_rows(const PageStepParams& p, const int* starts, const int* keys, int r, int apart) {
    const int total = starts[p.B];
    int b[N], pos[N], page[N], who[N];
#pragma unroll
    for (int i = 0; i < N; ++i) b[i] = 0;
    for (int n = p.B; n > 1; n -= n >> 1) {  // as owner_of
#pragma unroll
        for (int i = 0; i < N; ++i) b[i] += starts[b[i] + (n >> 1)] <= r + i * apart ? n >> 1 : 0;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
        pos[i] = r + i * apart < total ? keys[b[i]] - (starts[b[i] + 1] - (r + i * apart)) : -1;
        const int at = pos[i] < 0 ? 0 : pos[i] >> p.shift;
        page[i] = p.table[(int64_t)b[i] * p.table_row + at];
        who[i] = p.labels ? p.labels[b[i]] : b[i];
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int row = r + i * apart;
        if (row >= p.rows) break;
        const bool ok = pos[i] >= 0 && (unsigned)page[i] < (unsigned)p.pages;
        p.slots[row] = ok ? (page[i] << p.shift) + (pos[i] & ((1 << p.shift) - 1)) : -1;
        p.positions[row] = ok ? pos[i] : -1;
        p.owner[row] = ok ? who[i] : -1;
    }
}

// ROWS: the rows too (else page_rows_kernel behind it).
template <bool ROWS>
__global__ void __launch_bounds__(kPageThreads) page_step_kernel(PageStepParams p) {
    extern __shared__ __align__(16) unsigned char lds[];
    __shared__ int scratch[kPageWaves];
    int* starts = reinterpret_cast<int*>(lds);  // [B + 1] sums of new rows, at most p.rows
    int* keys = starts + p.B + 1;    // [B]
    int* held = keys + p.B;          // [B] pages that stay
    int* given = held + p.B;         // [B + 1] sums of pages given back
    int* taken = given + p.B + 1;    // [B + 1] sums of pages wanted
    const int page = 1 << p.shift;
    const int per = (p.B + kPageThreads - 1) / kPageThreads;  // requests of a thread, in order
    const int b0 = (int)threadIdx.x * per, b1 = b0 + per < p.B ? b0 + per : p.B;
    const int full = p.width << p.shift;
    const bool managed = p.free_pages;
    int count = managed ? *p.free_count : 0;
    count = count < 0 ? 0 : count > p.pages ? p.pages : count;

    auto cut_of = [&](int b, int* old) {
        int n = p.lens[b];
        n = n < 0 ? 0 : n > full ? full : n;
        *old = n;
        if (!p.keep) return n;
        const int k = p.keep[b] > 0 ? p.keep[b] : 0;
        return k < n ? k : n;
    };
    // More rows than a step has are as good as one more: sums stay below 2^31.
    auto fresh_of = [&](int b) {
        const int n = p.fresh[b];
        return n < 0 ? 0 : n > p.rows ? p.rows + 1 : n;
    };
    int rows = 0, back = 0;
    for (int b = b0; b < b1; ++b) {
        int old;
        const int cut = cut_of(b, &old);
        held[b] = (cut + page - 1) >> p.shift;
        rows += fresh_of(b);
        back += managed ? ((old + page - 1) >> p.shift) - held[b] : 0;
    }
    int all_rows, all_back, all_wanted;
    int row = block_scan(rows, scratch, &all_rows);
    int gave = block_scan(back, scratch, &all_back);
    const int first_row = row;
    int want = 0;
    for (int b = b0; b < b1; ++b) {
        int old;
        const int cut = cut_of(b, &old), n = fresh_of(b);
        starts[b] = row < p.rows ? row : p.rows;
        given[b] = gave;
        row += n;
        gave += managed ? ((old + page - 1) >> p.shift) - held[b] : 0;
        const bool fits = n > 0 && row <= p.rows && n <= full - cut;
        want += fits && managed ? ((cut + n + page - 1) >> p.shift) - held[b] : 0;
    }
    int take = block_scan(want, scratch, &all_wanted);
    // Lengths that no step left may give back more pages than there are (B * width, so
    // the sum with count could pass 2^31): those behind the stack's end are lost.
    const int top = all_back < p.pages - count ? count + all_back : p.pages;
    row = first_row;
    for (int b = b0; b < b1; ++b) {
        int old;
        const int cut = cut_of(b, &old), n = fresh_of(b);
        row += n;
        const bool fits = n > 0 && row <= p.rows && n <= full - cut;
        const int need = fits && managed ? ((cut + n + page - 1) >> p.shift) - held[b] : 0;
        const bool ok = fits && (need == 0 || take + need <= top);
        taken[b] = take;
        take += need;
        const int len = ok ? cut + n : cut;
        keys[b] = ok || n == 0 ? len : 0;
        p.lens[b] = len;
    }
    if (threadIdx.x == 0) {
        starts[p.B] = all_rows < p.rows ? all_rows : p.rows;
        given[p.B] = all_back;
        taken[p.B] = all_wanted;
    }
    __syncthreads();
    if (managed) {
        for (int i = threadIdx.x; i < top - count; i += kPageThreads) {
            const int b = owner_of(given, p.B, i);
            p.free_pages[top - 1 - i] = p.table[(int64_t)b * p.table_row + held[b] + i - given[b]];
        }
        __syncthreads();
        // What the requests in order take, up to the first that no longer fits.
        for (int i = threadIdx.x; i < all_wanted; i += kPageThreads) {
            const int b = owner_of(taken, p.B, i);
            if (taken[b + 1] <= top) p.table[(int64_t)b * p.table_row + held[b] + i - taken[b]] = p.free_pages[top - 1 - i];
        }
        if (threadIdx.x == 0) {
            int used = all_wanted;
            if (used > top) used = taken[owner_of(taken, p.B, top)];
            *p.free_count = top - used;
        }
        __syncthreads();
    }
    for (int b = threadIdx.x; b <= p.B; b += kPageThreads) {
        p.starts[b] = starts[b];
        if (b < p.B) p.keys[b] = keys[b];
    }
    if constexpr (ROWS)
        for (int r = threadIdx.x; r < p.rows; r += 4 * kPageThreads) map_rows<4>(p, starts, keys, r, kPageThreads);
}

__global__ void __launch_bounds__(256) page_rows_kernel(PageStepParams p) {
    const int r = (int)(blockIdx.x * 256 + threadIdx.x);
    if (r < p.rows) map_rows<1>(p, p.starts, p.keys, r, 0);
}

}  // namespace krk
