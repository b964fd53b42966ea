// Low-rank adapters of many rows beside a shared projection (gfx950):
//
//   h = x A_i^T        [rows, slices * rank], fp32, summed over ranges of K
//   out = y + s_i h B_i^T
//
// Rows are taken 16 at a time, as the columns of v_mfma_f32_16x16x32_bf16; the rows
// of a factor are its rows.  Rows of one adapter among the 16 are taken together
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
constexpr int kAdapterChunk = 128;    // of K that a wave takes at a time
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
    int by_row;    // a workgroup per row (that leads) instead of per 16 rows
    int same;      // out is y: rows without an adapter stay
    int first[kAdapterSlices];       // first column of a slice
    int width[kAdapterSlices];
    int group[kAdapterSlices + 1];   // first group of 64 columns of a slice
};

// The rows of a tile, adapter by adapter.
struct RowSets {
    int row0, id;     // id: of this lane's row (lane & 15), -1 for none
    uint32_t todo;
    __device__ __forceinline__ RowSets(const AdapterParams& p, int block) {
        const int n16 = threadIdx.x & 15;
        row0 = (p.by_row ? block & ~15 : 16 * block);
        const bool in = row0 + n16 < p.rows;
        id = p.index[in ? row0 + n16 : p.rows - 1];
        id = id >= 0 && id < p.adapters ? id : -1;
        todo = (uint32_t)__ballot(in) & 0xffffu;
        if (p.by_row) {  // this block's row, if it leads
            const int j = block & 15;
            const uint32_t same = (uint32_t)__ballot(in && id == __builtin_amdgcn_readlane(id, j)) & 0xffffu;
            todo = __builtin_ctz(same) == j ? same : 0;
        }
    }
    // The next adapter and its rows (bits); false: none left.
    __device__ __forceinline__ bool next(int* which, uint32_t* rows) {
        if (!todo) return false;
        *which = __builtin_amdgcn_readlane(id, __builtin_ctz(todo));
        *rows = (uint32_t)__ballot(id == *which) & todo;
        todo &= ~*rows;
        return true;
    }
};

// h of 16 rows, 64 rows of A and one range of K.  The waves take 128 of K in turn
// and meet in LDS.
__global__ void __launch_bounds__(kAdapterThreads) adapter_shrink_kernel(AdapterParams p) {
    __shared__ f32x4 lds[kAdapterWaves][kAdapterTiles][64];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n16 = lane & 15, q4 = lane >> 4;
    const int n0 = 16 * kAdapterTiles * blockIdx.z;
    const int chunks = (p.K + kAdapterChunk - 1) / kAdapterChunk;
    const int c0 = (int)((int64_t)chunks * blockIdx.y / p.splits), c1 = (int)((int64_t)chunks * (blockIdx.y + 1) / p.splits);
    RowSets sets(p, blockIdx.x);
    const int mine = sets.row0 + n16 < p.rows ? sets.row0 + n16 : p.rows - 1;
    const uint16_t* x = p.x + (int64_t)mine * p.ldx + 8 * q4;
    const u32x4 zero = {0, 0, 0, 0};
    int id;
    uint32_t rows;
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
#pragma unroll
            for (int s = 0; s < kAdapterChunk / 32; ++s) {
                const int k = c * kAdapterChunk + 32 * s;
                const bool in = k + 8 * q4 < p.K;
                const u32x4 xf = in ? load_cached16(x + k) : zero;
#pragma unroll
                for (int t = 0; t < kAdapterTiles; ++t)
                    acc[t] = mfma16(in ? load_cached16(a[t] + k) : zero, xf, acc[t]);
            }
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
            *reinterpret_cast<f32x4*>(p.h + ((int64_t)blockIdx.y * p.rows + sets.row0 + n16) * p.HN + n) = sum;
    }
}

// The 64 columns of a group: their first, how many, and the slice.
struct ColumnGroup {
    int col, n, slice;
    __device__ __forceinline__ ColumnGroup(const AdapterParams& p, int g) {
        slice = 0;
#pragma unroll
        for (int s = 1; s < kAdapterSlices; ++s) slice = s < p.slices && g >= p.group[s] ? s : slice;
        const int at = kAdapterCols * (g - p.group[slice]);
        col = p.first[slice] + at;
        n = p.width[slice] - at;
    }
};

__device__ __forceinline__ float silu_mul(float g, float u) { return g / (1.0f + expf(-g)) * u; }

// 64 columns of y (with SILU: of gate and of up) of 16 rows a wave.  Of a tile of 16
// columns lane group q gets four; the four tiles are interleaved so that they are 16
// neighbours: row i of tile t is column 16 (i >> 2) + 4 t + (i & 3).
template <bool SILU>
__global__ void __launch_bounds__(kAdapterThreads) adapter_expand_kernel(AdapterParams p) {
    constexpr int PARTS = SILU ? 2 : 1;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n16 = lane & 15, q4 = lane >> 4;
    const int g = (int)blockIdx.y * kAdapterWaves + wave;
    const int half = p.N / 2;
    int col[PARTS], n, slice[PARTS];
    if constexpr (SILU) {
        col[0] = kAdapterCols * g;
        col[1] = half + col[0];
        n = half - col[0];
        slice[0] = 0;
        slice[1] = p.slices - 1;
    } else {
        if (g >= p.group[p.slices]) return;
        const ColumnGroup c(p, g);
        col[0] = c.col;
        n = c.n;
        slice[0] = c.slice;
    }
    if (n <= 0) return;
    RowSets sets(p, blockIdx.x);
    const int mine = sets.row0 + n16 < p.rows ? sets.row0 + n16 : p.rows - 1;
    const int r8 = p.rank / 8;
    int id;
    uint32_t rows;
    while (sets.next(&id, &rows)) {
        if (id < 0 && p.same) continue;
        f32x4 acc[PARTS][4];
#pragma unroll
        for (int u = 0; u < PARTS; ++u)
#pragma unroll
            for (int t = 0; t < 4; ++t) acc[u][t] = f32x4{-0.0f, -0.0f, -0.0f, -0.0f};  // y + -0 is y, -0 too
        if (id >= 0) {
            const float scale = p.scale ? p.scale[id] : 1.0f;
#pragma unroll
            for (int u = 0; u < PARTS; ++u) {
                const uint16_t* b[4];
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    const int c = 16 * (n16 >> 2) + 4 * t + (n16 & 3);
                    b[t] = p.b + id * p.b_adapter + (int64_t)(col[u] + (c < n ? c : n - 1)) * p.b_row;
                }
                // Eight values of h a lane and step: all of them in 2 * r8 groups, as the
                // upper 8 bits of their mantissa, then the rest of it.
                const float* h = p.h + (int64_t)mine * p.HN + slice[u] * p.rank;
                for (int s = 0; s < 2 * r8; s += 4) {
                    const int at = s + q4;
                    const bool in = at < 2 * r8, low = at >= r8;
                    const int j = in ? 8 * (low ? at - r8 : at) : 0;
                    float v[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] = 0.0f;
                    for (int k = 0; k < p.splits; ++k) {
                        const float* hk = h + (int64_t)k * p.rows * p.HN + j;
                        const f32x4 lo = *reinterpret_cast<const f32x4*>(hk), up = *reinterpret_cast<const f32x4*>(hk + 4);
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            v[e] += lo[e];
                            v[4 + e] += up[e];
                        }
                    }
                    u32x4 hf;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float v0 = v[2 * e] * scale, v1 = v[2 * e + 1] * scale;
                        const uint32_t w = pack_bf16(v0, v1);
                        const float d0 = v0 - bf16_to_f32(w & 0xffffu), d1 = v1 - __uint_as_float(w & 0xffff0000u);
                        // Of an infinity nothing is left (not a NaN).
                        hf[e] = low ? pack_bf16(d0 == d0 ? d0 : 0.0f, d1 == d1 ? d1 : 0.0f) : w;
                        hf[e] = in ? hf[e] : 0;
                    }
#pragma unroll
                    for (int t = 0; t < 4; ++t) {
                        const u32x4 bf = in ? load_cached16(b[t] + j) : u32x4{0, 0, 0, 0};
                        acc[u][t] = mfma16(bf, hf, acc[u][t]);
                    }
                }
            }
        }
        // 16 columns of a row: two chunks of 8.
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int c = 16 * q4 + 8 * i;
            if (c >= n || !(rows >> n16 & 1)) continue;
            float z[PARTS][8];
#pragma unroll
            for (int u = 0; u < PARTS; ++u) {
                const u32x4 y = load_cached16(p.y + (int64_t)mine * p.ldy + col[u] + c);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    z[u][2 * e] = bf16_to_f32(y[e] & 0xffffu) + acc[u][2 * i + (e >> 1)][2 * (e & 1)];
                    z[u][2 * e + 1] = __uint_as_float(y[e] & 0xffff0000u) + acc[u][2 * i + (e >> 1)][2 * (e & 1) + 1];
                }
            }
            u32x4 o;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if constexpr (SILU) o[e] = pack_bf16(silu_mul(z[0][2 * e], z[1][2 * e]), silu_mul(z[0][2 * e + 1], z[1][2 * e + 1]));
                else o[e] = pack_bf16(z[0][2 * e], z[0][2 * e + 1]);
            }
            *reinterpret_cast<u32x4*>(p.out + (int64_t)mine * p.ldo + col[0] + c) = o;
        }
    }
}

}  // namespace krk
