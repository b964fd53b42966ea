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
constexpr int kAdapterSplits = 8;     // ranges of K at most
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
    int by_row;    // a workgroup per row (that leads) instead of per tile of rows
    int same;      // out is y: rows without an adapter stay
    int first[kAdapterSlices];       // first column of a slice
    int width[kAdapterSlices];
    int block[kAdapterSlices + 1];   // first block of columns of a slice
};

// The rows of a tile of 16 * MT, adapter by adapter; lane i knows row i's.
template <int MT>
struct RowSets {
    static constexpr int TR = 16 * MT;
    int row0, id;     // id: of row0 + lane % TR, -1 for none
    uint64_t todo;    // bit i: row0 + i
    __device__ __forceinline__ RowSets(const AdapterParams& p, int block) {
        const int i = (threadIdx.x & 63) % TR;
        row0 = p.by_row ? block & ~(TR - 1) : TR * block;
        const bool in = row0 + i < p.rows;
        id = p.index[in ? row0 + i : p.rows - 1];
        id = id >= 0 && id < p.adapters ? id : -1;
        todo = bits(in);
        if (p.by_row) {  // this block's row, if it leads
            const int j = block & (TR - 1);
            const uint64_t same = bits(in && id == __builtin_amdgcn_readlane(id, j));
            todo = __builtin_ctzll(same) == j ? same : 0;
        }
    }
    static __device__ __forceinline__ uint64_t bits(bool x) {
        const uint64_t b = __ballot(x);
        return TR == 64 ? b : b & ((1ull << (TR & 63)) - 1);
    }
    // The next adapter and its rows (bits); false: none left.
    __device__ __forceinline__ bool next(int* which, uint64_t* rows) {
        if (!todo) return false;
        *which = __builtin_amdgcn_readlane(id, __builtin_ctzll(todo));
        *rows = bits(id == *which) & todo;
        todo &= ~*rows;
        return true;
    }
};

// h of 16 * MT rows, 64 rows of A and one range of K.  The waves take U * 32 of K in
// turn, all of their loads in flight at once, and meet in LDS.
template <int MT, int U>
__global__ void __launch_bounds__(kAdapterThreads, 2) adapter_shrink_kernel(AdapterParams p) {
    __shared__ f32x4 lds[kAdapterWaves][MT][kAdapterTiles][64];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n16 = lane & 15, q4 = lane >> 4;
    const int n0 = 16 * kAdapterTiles * blockIdx.z;
    const int chunks = (p.K + 32 * U - 1) / (32 * U);
    const int c0 = (int)((int64_t)chunks * blockIdx.y / p.splits), c1 = (int)((int64_t)chunks * (blockIdx.y + 1) / p.splits);
    RowSets<MT> sets(p, blockIdx.x);
    const uint16_t* x[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const int row = sets.row0 + 16 * i + n16;
        x[i] = p.x + (int64_t)(row < p.rows ? row : p.rows - 1) * p.ldx + 8 * q4;
    }
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
        f32x4 acc[MT][kAdapterTiles];
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int t = 0; t < kAdapterTiles; ++t) acc[i][t] = f32x4{0, 0, 0, 0};
        for (int c = c0 + wave; c < c1; c += kAdapterWaves) {
            u32x4 xf[U][MT], af[U][kAdapterTiles];
#pragma unroll
            for (int s = 0; s < U; ++s) {
                const int k = 32 * (c * U + s);
                const bool in = k + 8 * q4 < p.K;
#pragma unroll
                for (int i = 0; i < MT; ++i) xf[s][i] = in ? load_cached16(x[i] + k) : zero;
#pragma unroll
                for (int t = 0; t < kAdapterTiles; ++t) af[s][t] = in ? load_cached16(a[t] + k) : zero;
            }
#pragma unroll
            for (int s = 0; s < U; ++s)
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int t = 0; t < kAdapterTiles; ++t) acc[i][t] = mfma16(af[s][t], xf[s][i], acc[i][t]);
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int t = 0; t < kAdapterTiles; ++t) lds[wave][i][t][lane] = acc[i][t];
        __syncthreads();
        const int n = n0 + 16 * wave + 4 * q4;
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            f32x4 sum = lds[0][i][wave][lane];
#pragma unroll
            for (int w = 1; w < kAdapterWaves; ++w) sum += lds[w][i][wave][lane];
            if (n < p.HN && (rows >> (16 * i + n16) & 1))
                *reinterpret_cast<f32x4*>(p.h + ((int64_t)blockIdx.y * p.rows + sets.row0 + 16 * i + n16) * p.HN + n) = sum;
        }
    }
}

__device__ __forceinline__ float silu_mul(float g, float u) { return g / (1.0f + expf(-g)) * u; }

// Bytes of h of a row in LDS: its values' upper 8 bits of mantissa, what is left of
// them, and 16 bytes that put rows on other banks.
__host__ __device__ constexpr int adapter_row_bytes(int rank) { return 4 * rank + 16; }

// 256 columns of y of one slice (with SILU: of gate and of up) and 16 * MT rows, a wave
// 64 of the columns.  Of a tile of 16 columns lane group q gets four; the four tiles
// are interleaved so that they are 16 neighbours: row i of tile t is column 16 (i >> 2)
// + 4 t + (i & 3).
template <int MT, bool SILU>
__global__ void __launch_bounds__(kAdapterThreads, 2) adapter_expand_kernel(AdapterParams p) {
    constexpr int PARTS = SILU ? 2 : 1, TR = 16 * MT;
    extern __shared__ __align__(16) unsigned char lds[];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n16 = lane & 15, q4 = lane >> 4;
    RowSets<MT> sets(p, blockIdx.x);
    if (!sets.todo) return;
    // The block's columns: slices begin blocks of their own.
    int block = blockIdx.y, slice = 0;
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
    const int n = (SILU ? p.N / 2 : p.width[slice]) - at;  // columns left
    // h, scaled, into LDS: rows whose sums over the ranges of K are taken in order.
    const int r8 = p.rank / 8, r4 = p.rank / 4, pitch = adapter_row_bytes(p.rank);
    for (int e = threadIdx.x; e < PARTS * TR * r4; e += kAdapterThreads) {
        const int u = PARTS > 1 && e >= TR * r4;
        const int i = (e - u * TR * r4) / r4, j = 4 * (e - u * TR * r4 - i * r4);
        const int row = sets.row0 + i < p.rows ? sets.row0 + i : p.rows - 1;
        const int id = p.index[row];
        f32x4 v = {0, 0, 0, 0};
        if (id >= 0 && id < p.adapters) {
            const float* h = p.h + (int64_t)row * p.HN + part[PARTS > 1 ? u : 0] + j;
            const int64_t next = (int64_t)p.rows * p.HN;
            f32x4 x[kAdapterSplits];
#pragma unroll
            for (int k = 0; k < kAdapterSplits; ++k)
                if (k < p.splits) x[k] = *reinterpret_cast<const f32x4*>(h + k * next);
#pragma unroll
            for (int k = 0; k < kAdapterSplits; ++k)
                if (k < p.splits) v += x[k];
            v *= p.scale ? p.scale[id] : 1.0f;
        }
        uint2 hi, lo;
        hi.x = pack_bf16(v[0], v[1]);
        hi.y = pack_bf16(v[2], v[3]);
        auto rest = [](float x, uint32_t top) {  // of an infinity nothing is left (not a NaN)
            const float d = x - __uint_as_float(top);
            return d == d ? d : 0.0f;
        };
        lo.x = pack_bf16(rest(v[0], hi.x << 16), rest(v[1], hi.x & 0xffff0000u));
        lo.y = pack_bf16(rest(v[2], hi.y << 16), rest(v[3], hi.y & 0xffff0000u));
        unsigned char* to = lds + (u * TR + i) * pitch + 2 * j;
        *reinterpret_cast<uint2*>(to) = hi;
        *reinterpret_cast<uint2*>(to + 2 * p.rank) = lo;
    }
    __syncthreads();
    if (n <= 0) return;
    int id;
    uint64_t rows;
    while (sets.next(&id, &rows)) {
        if (id < 0 && p.same) continue;
        // 16 columns of a row: two chunks of 8.
        u32x4 y[PARTS][MT][2];
        bool mine[MT][2];
        int row[MT];
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            row[i] = sets.row0 + 16 * i + n16;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int c = 16 * q4 + 8 * k;
                mine[i][k] = c < n && (rows >> (16 * i + n16) & 1);
#pragma unroll
                for (int u = 0; u < PARTS; ++u)
                    if (mine[i][k]) y[u][i][k] = load_cached16(p.y + (int64_t)row[i] * p.ldy + col[u] + c);
            }
        }
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
                const uint16_t* b[4];
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    const int c = 16 * (n16 >> 2) + 4 * t + (n16 & 3);
                    b[t] = p.b + id * p.b_adapter + (int64_t)(col[u] + (c < n ? c : n - 1)) * p.b_row;
                }
                const unsigned char* h = lds + (u * TR + n16) * pitch;
                // 8 values a lane and step, of 2 * rank: upper bits first.
                for (int s = 0; s < 2 * r8; s += 4) {
                    const int g = s + q4;
                    const bool in = g < 2 * r8;
                    const int j = 8 * (g >= r8 ? g - r8 : g);
                    u32x4 bf[4];
#pragma unroll
                    for (int t = 0; t < 4; ++t) bf[t] = in ? load_cached16(b[t] + j) : u32x4{0, 0, 0, 0};
#pragma unroll
                    for (int i = 0; i < MT; ++i) {
                        const u32x4 hf = in ? *reinterpret_cast<const u32x4*>(h + 16 * i * pitch + 16 * g) : u32x4{0, 0, 0, 0};
#pragma unroll
                        for (int t = 0; t < 4; ++t) acc[u][i][t] = mfma16(bf[t], hf, acc[u][i][t]);
                    }
                }
            }
        }
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                if (!mine[i][k]) continue;
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
                *reinterpret_cast<u32x4*>(p.out + (int64_t)row[i] * p.ldo + col[0] + 16 * q4 + 8 * k) = o;
            }
    }
}

}  // namespace krk
