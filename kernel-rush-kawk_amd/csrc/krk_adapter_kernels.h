// Low-rank adapters of many rows beside a shared projection (gfx950):
//
//   h = x A_i^T        [rows, slices * rank], fp32, summed over ranges of K
//   out = y + s_i h B_i^T
//
// Rows are the columns of v_mfma_f32_16x16x32_bf16, in tiles of 16 (few rows) or 64;
// the rows of a factor are its rows.  A tile's rows of one adapter are taken together
// (their first row leads them), those of the others masked where results are stored.
//
// Bound by reading A, B and y once (2 bytes a value): a rank of 16 makes 16 flops a
// byte of x or y.
#pragma once

#include "krk_attn_common.h"

namespace krk {

constexpr int kAdapterSlices = 4;
constexpr int kAdapterThreads = 256;
constexpr int kAdapterWaves = kAdapterThreads / 64;
constexpr int kAdapterTiles = 4;      // of 16 rows of A that a workgroup takes
// Ranges of K at most, of few rows and of many (870 rows of 9728, a call: 24 us in 8, 22
// in 12, 19.5 in 16; few rows are no faster in 16).
constexpr int kAdapterFewSplits = 8, kAdapterManySplits = 16;
constexpr int kAdapterFewStep = 128, kAdapterManyStep = 128;  // of K: of a wave, of a workgroup
constexpr int kAdapterCols = 64;      // of y that a wave takes

struct AdapterParams {
    const uint16_t* x;
    int64_t ldx;
    const uint16_t* a;
    int64_t a_adapter, a_row;
    const uint16_t* b;
    int64_t b_adapter, b_row;
    const float* scale;
    const int32_t* index;
    const uint16_t* y;
    int64_t ldy;
    uint16_t* out;
    int64_t ldo;
    float* h;      // [splits][rows][HN]
    int rows, N, K, rank, HN, adapters, splits, slices;
    uint16_t* joined;  // [rows][2 HN] of tiles of 64 rows
    int slots;     // workgroups of a tile of rows that share its adapters
    int same;      // out is y: rows without an adapter stay
    int first[kAdapterSlices];       // first column of a slice
    int width[kAdapterSlices];
    int block[kAdapterSlices + 1];   // first block of columns of a slice
};

// The rows of a tile of 16 * MT, adapter by adapter; lane i knows row i's.  Of a tile's
// adapters each of `slots` blocks takes every slots-th, so that rows of many adapters do
// not wait for one another.  All tiles' first slots come first: workgroups go to the
// shader engines in a fixed order, and with idle ones in every other place half of the
// CUs stayed idle (4096 rows of 9728: 40 us and 28).
template <int MT>
struct RowSets {
    static constexpr int TR = 16 * MT;
    int row0, id;     // id: of row0 + lane % TR, -1 for none
    int skip, slots;
    uint64_t todo;    // bit i: row0 + i
    __device__ __forceinline__ RowSets(const AdapterParams& p, int tile, int slot) {
        const int i = (threadIdx.x & 63) % TR;
        slots = p.slots;
        skip = slot;
        row0 = TR * tile;
        const bool in = row0 + i < p.rows;
        id = p.index[in ? row0 + i : p.rows - 1];
        id = id >= 0 && id < p.adapters ? id : -1;
        todo = bits(in);
    }
    static __device__ __forceinline__ uint64_t bits(bool x) {
        const uint64_t b = __ballot(x);
        return TR == 64 ? b : b & ((1ull << (TR & 63)) - 1);
    }
    // The slot's next adapter and its rows (bits); false: none left.
    __device__ __forceinline__ bool next(int* which, uint64_t* rows) {
        for (; todo; --skip) {
            *which = __builtin_amdgcn_readlane(id, __builtin_ctzll(todo));
            *rows = bits(id == *which) & todo;
            todo &= ~*rows;
            if (skip == 0) {
                skip = slots - 1;
                return true;
            }
        }
        return false;
    }
};

// h of 16 rows, 64 rows of A and one range of K.  The waves take 128 of K in turn, all
// of their loads in flight at once, and meet in LDS.  Bound by latency: 32 rows of 2560
// over 16 adapters 6 us, 4.6 with one row.
__global__ void __launch_bounds__(kAdapterThreads, 2) adapter_shrink_kernel(AdapterParams p) {
    constexpr int U = kAdapterFewStep / 32;
    __shared__ f32x4 lds[kAdapterWaves][kAdapterTiles][64];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n16 = lane & 15, q4 = lane >> 4;
    const int n0 = 16 * kAdapterTiles * blockIdx.z;
    const int steps = (p.K + kAdapterFewStep - 1) / kAdapterFewStep;
    const int c0 = (int)((int64_t)steps * blockIdx.x / p.splits), c1 = (int)((int64_t)steps * (blockIdx.x + 1) / p.splits);
    const int tiles = (p.rows + 15) / 16;
    RowSets<1> sets(p, blockIdx.y % tiles, blockIdx.y / tiles);
    const int row = sets.row0 + n16;
    const uint16_t* x = p.x + (int64_t)(row < p.rows ? row : p.rows - 1) * p.ldx + 8 * q4;
    const u32x4 zero = {0, 0, 0, 0};
    int id;
    uint64_t rows;
    while (sets.next(&id, &rows)) {
        if (id < 0) continue;
        const uint16_t* a[kAdapterTiles];
#pragma unroll
        for (int t = 0; t < kAdapterTiles; ++t) {
            const int n = n0 + 16 * t + n16;
            a[t] = p.a + id * p.a_adapter + (n < p.HN ? n : p.HN - 1) * p.a_row + 8 * q4;
        }
        f32x4 acc[kAdapterTiles];
#pragma unroll
        for (int t = 0; t < kAdapterTiles; ++t) acc[t] = f32x4{0, 0, 0, 0};
        for (int c = c0 + wave; c < c1; c += kAdapterWaves) {
            u32x4 xf[U], af[U][kAdapterTiles];
            const int k0 = kAdapterFewStep * c;
            if (k0 + kAdapterFewStep <= p.K) {
#pragma unroll
                for (int s = 0; s < U; ++s) {
                    xf[s] = load_cached16(x + k0 + 32 * s);
#pragma unroll
                    for (int t = 0; t < kAdapterTiles; ++t) af[s][t] = load_cached16(a[t] + k0 + 32 * s);
                }
            } else {  // zeros behind K, in place of the rows' first values
#pragma unroll
                for (int s = 0; s < U; ++s) {
                    const bool in = k0 + 32 * s + 8 * q4 < p.K;
                    const int k = in ? k0 + 32 * s : -8 * q4;
                    const u32x4 v = load_cached16(x + k);
                    xf[s] = in ? v : zero;
#pragma unroll
                    for (int t = 0; t < kAdapterTiles; ++t) {
                        const u32x4 w = load_cached16(a[t] + k);
                        af[s][t] = in ? w : zero;
                    }
                }
            }
#pragma unroll
            for (int s = 0; s < U; ++s)
#pragma unroll
                for (int t = 0; t < kAdapterTiles; ++t) acc[t] = mfma16(af[s][t], xf[s], acc[t]);
        }
        __syncthreads();
#pragma unroll
        for (int t = 0; t < kAdapterTiles; ++t) lds[wave][t][lane] = acc[t];
        __syncthreads();
        f32x4 sum = lds[0][wave][lane];
#pragma unroll
        for (int w = 1; w < kAdapterWaves; ++w) sum += lds[w][wave][lane];
        const int n = n0 + 16 * wave + 4 * q4;
        if (n < p.HN && (rows >> n16 & 1))
            *reinterpret_cast<f32x4*>(p.h + ((int64_t)blockIdx.x * p.rows + row) * p.HN + n) = sum;
    }
}

// The same of 64 rows: x and A come through LDS by DMA, 256 bytes of a row at a time,
// in a ring of two steps; each wave takes 16 of the rows.  (Straight into operands a
// load takes 64 bytes each of 16 rows: rows whose length is a multiple of 1 KB then
// meet in a few sets of the L1, and 4096 rows of 9728 took 43 us.)  Chunks of 16 bytes
// of a row are permuted with the row's low bits, against bank conflicts.  The tiles of a
// range of K lie side by side on one XCD or two, which keep to that part of every A.
__global__ void __launch_bounds__(kAdapterThreads, 2) adapter_shrink64_kernel(AdapterParams p) {
    constexpr int ROWS = 64, CH = kAdapterManyStep / 8;  // chunks of a row and step
    constexpr int DMAS = ROWS / 4 / kAdapterWaves;       // of 4 rows, of x and of A, per wave and step
    constexpr uint32_t HALF = ROWS * kAdapterManyStep * 2;
    __shared__ __align__(16) unsigned char lds[2][2][HALF];  // [step][x, A]
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n16 = lane & 15, q4 = lane >> 4;
    const int n0 = 16 * kAdapterTiles * blockIdx.z;
    const int steps = (p.K + kAdapterManyStep - 1) / kAdapterManyStep;
    const int tiles = (p.rows + ROWS - 1) / ROWS;
    const int block = xcd_block(blockIdx.x, tiles * p.splits), range = block / tiles;
    const int c0 = (int)((int64_t)steps * range / p.splits), c1 = (int)((int64_t)steps * (range + 1) / p.splits);
    RowSets<4> sets(p, block - range * tiles, blockIdx.y);
    int id;
    uint64_t rows;
    while (sets.next(&id, &rows)) {
        if (id < 0) continue;
        // This lane's share of a step: 16 bytes of a row of each of its DMAs.
        const uint16_t *xs[DMAS], *as[DMAS];
        int chunk[DMAS];
#pragma unroll
        for (int i = 0; i < DMAS; ++i) {
            const int r = 4 * (wave + kAdapterWaves * i) + lane / CH;
            chunk[i] = 8 * ((lane % CH) ^ (r & (CH - 1)));
            const int row = sets.row0 + r, n = n0 + r;
            xs[i] = p.x + (int64_t)(row < p.rows ? row : p.rows - 1) * p.ldx;
            as[i] = p.a + id * p.a_adapter + (n < p.HN ? n : p.HN - 1) * p.a_row;
        }
        auto fetch = [&](int c) {
#pragma unroll
            for (int i = 0; i < DMAS; ++i) {
                // Behind K the row's first values, which are not used.
                const int k = kAdapterManyStep * c + chunk[i], at = k < p.K ? k : 0;
                dma_row(xs[i] + at, lds[c & 1][0] + 1024 * (wave + kAdapterWaves * i));
                dma_row(as[i] + at, lds[c & 1][1] + 1024 * (wave + kAdapterWaves * i));
            }
        };
        f32x4 acc[kAdapterTiles];
#pragma unroll
        for (int t = 0; t < kAdapterTiles; ++t) acc[t] = f32x4{0, 0, 0, 0};
        if (c0 < c1) fetch(c0);
        for (int c = c0; c < c1; ++c) {
            if (c + 1 < c1) fetch(c + 1);
            vm_wait_stages<2 * DMAS>(c + 1 < c1 ? 1 : 0);
            bare_barrier();  // step c is here
            const int left = p.K - kAdapterManyStep * c;
#pragma unroll
            for (int s = 0; s < kAdapterManyStep / 32; ++s) {
                const int at = 16 * ((4 * s + q4) ^ n16);  // rows 16 t + n16: their low bits are n16
                u32x4 xf = *reinterpret_cast<const u32x4*>(lds[c & 1][0] + (16 * wave + n16) * kAdapterManyStep * 2 + at);
                u32x4 af[kAdapterTiles];
#pragma unroll
                for (int t = 0; t < kAdapterTiles; ++t)
                    af[t] = *reinterpret_cast<const u32x4*>(lds[c & 1][1] + (16 * t + n16) * kAdapterManyStep * 2 + at);
                if (left < kAdapterManyStep && 32 * s + 8 * q4 >= left) {
                    xf = u32x4{0, 0, 0, 0};
#pragma unroll
                    for (int t = 0; t < kAdapterTiles; ++t) af[t] = u32x4{0, 0, 0, 0};
                }
#pragma unroll
                for (int t = 0; t < kAdapterTiles; ++t) acc[t] = mfma16(af[t], xf, acc[t]);
            }
            lds_wait();
            bare_barrier();  // and free again
        }
        const int row = sets.row0 + 16 * wave + n16;
        if (rows >> (16 * wave + n16) & 1) {
#pragma unroll
            for (int t = 0; t < kAdapterTiles; ++t) {
                const int n = n0 + 16 * t + 4 * q4;
                if (n < p.HN) *reinterpret_cast<f32x4*>(p.h + ((int64_t)range * p.rows + row) * p.HN + n) = acc[t];
            }
        }
    }
}

__device__ __forceinline__ float silu_mul(float g, float u) { return g / (1.0f + expf(-g)) * u; }

// h of a row as the second product takes it: of each slice `rank` values to the upper 8
// bits of their mantissa, then what is left of them.
struct SplitH {
    uint2 hi, lo;
    __device__ __forceinline__ explicit SplitH(const f32x4& v) {
        hi.x = pack_bf16(v[0], v[1]);
        hi.y = pack_bf16(v[2], v[3]);
        lo.x = pack_bf16(rest(v[0], hi.x << 16), rest(v[1], hi.x & 0xffff0000u));
        lo.y = pack_bf16(rest(v[2], hi.y << 16), rest(v[3], hi.y & 0xffff0000u));
    }
    static __device__ __forceinline__ float rest(float x, uint32_t top) {  // of an infinity nothing (not a NaN)
        const float d = x - __uint_as_float(top);
        return d == d ? d : 0.0f;
    }
};

// Four values of h of a row, scaled: the sums over the ranges of K, in order.
template <int SPLITS>
__device__ __forceinline__ f32x4 sum_h(const AdapterParams& p, int row, int j) {
    const int id = p.index[row];
    f32x4 v = {0, 0, 0, 0};
    if (id < 0 || id >= p.adapters) return v;
    const float* h = p.h + (int64_t)row * p.HN + j;
    const int64_t next = (int64_t)p.rows * p.HN;
    f32x4 x[SPLITS];
    // All at once: behind the last range it is read again, and left out of the sum.
#pragma unroll
    for (int k = 0; k < SPLITS; ++k) x[k] = *reinterpret_cast<const f32x4*>(h + (k < p.splits ? k : p.splits - 1) * next);
#pragma unroll
    for (int k = 0; k < SPLITS; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = k < p.splits ? v[e] + x[k][e] : v[e];
    return v * (p.scale ? p.scale[id] : 1.0f);
}

// Tiles of 64 rows: h is put together once, not by every block of columns (4096 rows of
// 2560 columns, rank 64, 8 ranges: each of 10 blocks would read 131 KB a tile).
// SPLITS: ranges of K at most.
template <int SPLITS>
__global__ void __launch_bounds__(256) adapter_join_kernel(AdapterParams p) {
    const int q = p.HN / 4;
    const int e = (int)(blockIdx.x * 256 + threadIdx.x);  // rows * q <= 2^25
    const int row = e / q, j = 4 * (e - row * q);
    if (row >= p.rows) return;
    const SplitH h(sum_h<SPLITS>(p, row, j));
    const int slice = j / p.rank;
    uint16_t* to = p.joined + (int64_t)row * 2 * p.HN + slice * p.rank + j;
    *reinterpret_cast<uint2*>(to) = h.hi;
    *reinterpret_cast<uint2*>(to + p.rank) = h.lo;
}

// Bytes of h of a row in LDS: 16 more put rows on other banks.
__host__ __device__ constexpr int adapter_row_bytes(int rank) { return 4 * rank + 16; }

// 256 columns of y of one slice (with SILU: of gate and of up) and 16 * MT rows, a wave
// 64 of the columns.  Of a tile of 16 columns lane group q gets four; tiles are
// interleaved so that those of two are 8 neighbours, 16 bytes beside the next group's:
// row i of tile t is column 32 (t >> 1) + 8 (i >> 2) + 4 (t & 1) + (i & 3).  Blocks of
// columns change fastest, so that rows are read and written whole.  An adapter's B (of
// the first 32 of its rank) and y are on their way before h is put together (or, JOINED,
// copied as adapter_join_kernel left it).  h comes through LDS, once for the four waves
// (each wave's own loads, in two steps: 4096 rows of 2560 columns 22.6 us, now 19).
template <int MT, bool SILU, bool JOINED>
__global__ void __launch_bounds__(kAdapterThreads, 2) adapter_expand_kernel(AdapterParams p) {
    constexpr int PARTS = SILU ? 2 : 1, TR = 16 * MT;
    extern __shared__ __align__(16) unsigned char lds[];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n16 = lane & 15, q4 = lane >> 4;
    const int tiles = (p.rows + TR - 1) / TR;
    RowSets<MT> sets(p, blockIdx.y % tiles, blockIdx.y / tiles);
    int id;
    uint64_t rows;
    bool more = sets.next(&id, &rows);
    if (!more) return;
    // The block's columns: slices begin blocks of their own.
    int block = blockIdx.x, slice = 0;
#pragma unroll
    for (int s = 1; s < kAdapterSlices; ++s) slice = !SILU && s < p.slices && block >= p.block[s] ? s : slice;
    block -= SILU ? 0 : p.block[slice];
    const int at = kAdapterCols * (kAdapterWaves * block + wave);
    int col[PARTS], part[PARTS];
    col[0] = (SILU ? 0 : p.first[slice]) + at;
    part[0] = slice * p.rank;
    if constexpr (SILU) {
        col[1] = p.N / 2 + at;
        part[1] = (p.slices - 1) * p.rank;
    }
    const int n = (SILU ? p.N / 2 : p.width[slice]) - at;  // columns left, none where <= 0
    const int r8 = p.rank / 8;
    auto has = [&](int i) { return MT == 1 || ((rows >> (16 * i)) & 0xffff) != 0; };
    // Two chunks of 8 columns of a row.
    auto mine = [&](int i, int k) { return 8 * q4 + 32 * k < n && (rows >> (16 * i + n16) & 1); };

    u32x4 y[PARTS][MT][2], bf[PARTS][4];
    // Eight values a lane of B's rows, of step s of 32.
    auto load_b = [&](int u, int s) {
        const int g = 4 * s + q4;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const int c = 32 * (t >> 1) + 8 * (n16 >> 2) + 4 * (t & 1) + (n16 & 3);
            const uint16_t* b = p.b + id * p.b_adapter + (int64_t)(col[u] + (c < n ? c : n - 1)) * p.b_row;
            bf[u][t] = g < r8 ? load_cached16(b + 8 * g) : u32x4{0, 0, 0, 0};
        }
    };
    auto load = [&]() {
        if (id >= 0) {
#pragma unroll
            for (int u = 0; u < PARTS; ++u) load_b(u, 0);
        } else if (p.same) {
            return;
        }
#pragma unroll
        for (int i = 0; i < MT; ++i)
            if (has(i)) {
#pragma unroll
                for (int k = 0; k < 2; ++k)
#pragma unroll
                    for (int u = 0; u < PARTS; ++u)
                        if (mine(i, k)) y[u][i][k] = load_cached16(p.y + (int64_t)(sets.row0 + 16 * i + n16) * p.ldy + col[u] + 8 * q4 + 32 * k);
            }
    };
    if (n > 0) load();

    const int pitch = adapter_row_bytes(p.rank);
    if constexpr (JOINED) {
        const int r4 = p.rank / 4;  // 16 bytes each of a row's h, both parts
        for (int e = threadIdx.x; e < PARTS * TR * r4; e += kAdapterThreads) {
            const int u = PARTS > 1 && e >= TR * r4;
            const int i = (e - u * TR * r4) / r4, j = e - u * TR * r4 - i * r4;
            const int row = sets.row0 + i < p.rows ? sets.row0 + i : p.rows - 1;
            *reinterpret_cast<u32x4*>(lds + (u * TR + i) * pitch + 16 * j) =
                load_cached16(p.joined + (int64_t)row * 2 * p.HN + 2 * part[PARTS > 1 ? u : 0] + 8 * j);
        }
        __syncthreads();
    } else {
        const int r4 = p.rank / 4;
        for (int e = threadIdx.x; e < PARTS * TR * r4; e += kAdapterThreads) {
            const int u = PARTS > 1 && e >= TR * r4;
            const int i = (e - u * TR * r4) / r4, j = 4 * (e - u * TR * r4 - i * r4);
            const SplitH h(sum_h<kAdapterFewSplits>(p, sets.row0 + i < p.rows ? sets.row0 + i : p.rows - 1, part[PARTS > 1 ? u : 0] + j));
            unsigned char* to = lds + (u * TR + i) * pitch + 2 * j;
            *reinterpret_cast<uint2*>(to) = h.hi;
            *reinterpret_cast<uint2*>(to + 2 * p.rank) = h.lo;
        }
        __syncthreads();
    }
    if (n <= 0) return;
    for (;;) {
        f32x4 acc[PARTS][MT][4];
#pragma unroll
        for (int u = 0; u < PARTS; ++u)
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int t = 0; t < 4; ++t) acc[u][i][t] = f32x4{-0.0f, -0.0f, -0.0f, -0.0f};  // y + -0 is y, -0 too
        if (id >= 0) {
#pragma unroll
            for (int u = 0; u < PARTS; ++u) {
                for (int s = 0; 4 * s < r8; ++s) {
                    if (s) load_b(u, s);
                    const int g = 4 * s + q4;
#pragma unroll
                    for (int i = 0; i < MT; ++i) {
                        if (!has(i)) continue;
                        const unsigned char* h = lds + (u * TR + 16 * i + n16) * pitch;
                        u32x4 hi = {0, 0, 0, 0}, lo = {0, 0, 0, 0};
                        if (g < r8) {
                            hi = *reinterpret_cast<const u32x4*>(h + 16 * g);
                            lo = *reinterpret_cast<const u32x4*>(h + 2 * p.rank + 16 * g);
                        }
#pragma unroll
                        for (int t = 0; t < 4; ++t) acc[u][i][t] = mfma16(bf[u][t], lo, acc[u][i][t]);
#pragma unroll
                        for (int t = 0; t < 4; ++t) acc[u][i][t] = mfma16(bf[u][t], hi, acc[u][i][t]);
                    }
                }
            }
        }
        if (id >= 0 || !p.same) {
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    if (!mine(i, k)) continue;
                    float z[PARTS][8];
#pragma unroll
                    for (int u = 0; u < PARTS; ++u)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            z[u][2 * e] = bf16_to_f32(y[u][i][k][e] & 0xffffu) + acc[u][i][2 * k + (e >> 1)][2 * (e & 1)];
                            z[u][2 * e + 1] = __uint_as_float(y[u][i][k][e] & 0xffff0000u) + acc[u][i][2 * k + (e >> 1)][2 * (e & 1) + 1];
                        }
                    u32x4 o;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if constexpr (SILU) o[e] = pack_bf16(silu_mul(z[0][2 * e], z[1][2 * e]), silu_mul(z[0][2 * e + 1], z[1][2 * e + 1]));
                        else o[e] = pack_bf16(z[0][2 * e], z[0][2 * e + 1]);
                    }
                    *reinterpret_cast<u32x4*>(p.out + (int64_t)(sets.row0 + 16 * i + n16) * p.ldo + col[0] + 8 * q4 + 32 * k) = o;
                }
        }
        if (!sets.next(&id, &rows)) break;
        load();
    }
}

}  // namespace krk
