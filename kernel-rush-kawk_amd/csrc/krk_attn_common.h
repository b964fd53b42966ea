// Shared pieces of the cache-attention kernels (gfx950): the operands as the
// kernels take them, what a row sees, and fragment helpers.
//
// Rows.  A key/value head h serves G = heads / kv_heads query heads, so its
// products have R * G rows per sequence: row j is new row j / G of the
// sequence with query head h * G + j % G.
//
// Products.  Both run as S^T = K Q^T and O^T = V^T P^T on v_mfma_f32_16x16x32_bf16,
// with the row as the column (lane & 15) of either result: a row's maximum,
// sum and rescaling factor then live in the lane that needs them.  Of 32 keys
// k0.., lane group q = lane >> 4 takes keys 8q .. 8q + 7 as the k-slots of the
// second product; the first product's two 16-key tiles are therefore filled
// with keys 8 (r >> 2) + (r & 3) and those + 4, which leaves lane (n, q) with
// the scores of row n against exactly keys 8q .. 8q + 7.  The weights go from
// one product to the next without leaving their lane.
#pragma once

#include "krk_common.h"
#include "krk_sync.h"

namespace krk {

constexpr int kPadding = 0x7fffffff;  // RowSight::lo of a row without a slot
constexpr float kNegInf = -__builtin_inff();

struct CacheView {
    const uint16_t* p;
    int64_t seq, slot, head;
};

struct AttnParams {
    const uint16_t* q;
    int64_t q_row;
    CacheView k, v, kp, vp;
    const int32_t* lens;
    const int64_t* tree;
    uint16_t* out;
    int64_t out_row;
    float* lse;
    const float* scores;
    int64_t sc_seq, sc_head;
    float* scores_out;
    int64_t so_seq, so_head;
    float* part;   // [splits + prefix_splits][rows][D] unnormalised outputs
    float2* ml;    // [splits + prefix_splits][rows] running maximum (of q.k) and sum
    float2* stat;  // [rows] final maximum and 1 / sum (scored calls)
    float scale;   // of q.k
    float c;       // scale * log2(e)
    int B, R, heads, kv_heads, G, RG, capacity, window, sinks, prefix;
    int splits, prefix_splits;          // key ranges
    int row_tiles, prefix_row_tiles;    // tiles of a sequence's rows; of all sequences' rows
};

// Which positions a row sees: t <= hi with (t >= lo or t < sinks), and from
// `first` on (tree masks) those whose bit is set.  Padding: lo = kPadding, hi = -1.
struct RowSight {
    int lo, hi;
    int first;       // position of the sequence's first new row (tree)
    uint64_t bits;   // of the new rows, 0 without tree masks
};

__device__ __forceinline__ int seq_len(const AttnParams& p, int b) {
    const int n = p.lens[b];
    return n < 0 ? 0 : n > p.capacity ? p.capacity : n;
}

// Row r of sequence b, whose cache holds len keys.
__device__ __forceinline__ RowSight row_sight(const AttnParams& p, int b, int r, int len) {
    RowSight s;
    const int slot = len - p.R + r;
    s.first = p.prefix + len - p.R;
    s.bits = 0;
    int pos = p.prefix + slot;
    s.hi = pos;
    if (p.tree) {
        const uint64_t all = p.R >= 64 ? ~0ull : (1ull << p.R) - 1;
        s.bits = (uint64_t)p.tree[(int64_t)b * p.R + r] & all;
        pos = s.first + __popcll(s.bits) - 1;
        s.hi = s.first - 1;
    }
    const int lo = p.window ? pos - p.window + 1 : 0;
    s.lo = lo > 0 ? lo : 0;
    if (slot < 0) {
        s.hi = -1;
        s.lo = kPadding;
        s.bits = 0;
    }
    return s;
}

__device__ __forceinline__ bool sees(const RowSight& s, int t, int sinks) {
    bool ok = t <= s.hi && (t >= s.lo || t < sinks);
    if (s.bits) {
        const unsigned d = (unsigned)(t - s.first);
        ok = ok || (d < 64 && ((s.bits >> d) & 1));
    }
    return ok;
}

// Wait until every load this wave issued has returned.
__device__ __forceinline__ void drain_loads() {
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    vm_wait<0>();
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
}

__device__ __forceinline__ float exp2_raw(float v) { return __builtin_amdgcn_exp2f(v); }

// Maximum / sum over the four lanes n, n + 16, n + 32, n + 48 that hold a row.
__device__ __forceinline__ float row_max(float v) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float row_sum(float v) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}
__device__ __forceinline__ int row_min_i(int v) {
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) {
        const int o = __shfl_xor(v, s);
        v = o < v ? o : v;
    }
    return __builtin_amdgcn_readfirstlane(v);
}
__device__ __forceinline__ int row_max_i(int v) {
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) {
        const int o = __shfl_xor(v, s);
        v = o > v ? o : v;
    }
    return __builtin_amdgcn_readfirstlane(v);
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    bf16x2 v;
    v[0] = (__bf16)lo;
    v[1] = (__bf16)hi;
    return __builtin_bit_cast(uint32_t, v);
}

// The key of 32 that row r of 16-key tile t holds (see the top).
__device__ __forceinline__ int tile_key(int t, int r) { return 8 * (r >> 2) + 4 * t + (r & 3); }

// 32 keys as operands of S^T = K Q^T: two 16-key tiles of D / 32 k-steps.
template <int D>
struct KeyFrag {
    u32x4 f[2][D / 32];
    // keys kb .. kb + 31 of the run at `base`; those from `limit` (>= 1) on
    // re-read the last one.
    __device__ __forceinline__ void load(const uint16_t* base, int64_t slot, int kb, int limit, int lane) {
        const int r = lane & 15, q = lane >> 4;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            int key = kb + tile_key(t, r);
            key = key < limit ? key : limit - 1;
            const uint16_t* row = base + (int64_t)key * slot + 8 * q;
#pragma unroll
            for (int s = 0; s < D / 32; ++s) f[t][s] = load_cached16(row + 32 * s);
        }
    }
};

// 32 keys' values as operands of O^T = V^T P^T.  Lane (r, q) reads elements
// [VD r, VD r + VD) of keys 8q .. 8q + 7, VD = D / 16: whole rows, 16 lanes
// each.  Paired over adjacent keys (one v_perm_b32 per pair), element j of each
// is the lane's operand for the 16 outputs d = VD r + j: no trip through LDS.
template <int D>
struct ValueFrag {
    static constexpr int VD = D / 16;
    static constexpr int W = VD / 2;  // dwords of a key in a lane
    uint32_t f[8][W];
    __device__ __forceinline__ void load(const uint16_t* base, int64_t slot, int kb, int limit, int lane) {
        const int r = lane & 15, q = lane >> 4;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            int key = kb + 8 * q + i;
            key = key < limit ? key : limit - 1;
            const uint16_t* row = base + (int64_t)key * slot + VD * r;
            if constexpr (VD == 8) {
                const u32x4 x = load_cached16(row);
#pragma unroll
                for (int w = 0; w < 4; ++w) f[i][w] = x[w];
            } else {
                const uint2 x = *reinterpret_cast<const uint2*>(row);
                f[i][0] = x.x;
                f[i][1] = x.y;
            }
        }
    }
    // Operand of outputs d = VD r + j.
    __device__ __forceinline__ bf16x8 operand(int j) const {
        u32x4 x;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            x[i] = __builtin_amdgcn_perm(f[2 * i + 1][j >> 1], f[2 * i][j >> 1], (j & 1) ? 0x07060302u : 0x05040100u);
        return __builtin_bit_cast(bf16x8, x);
    }
    // Whether this lane holds an infinity or a NaN.
    __device__ __forceinline__ bool odd() const {
        typedef __attribute__((ext_vector_type(2))) unsigned short u16x2;
        u16x2 m = {0, 0};
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int w = 0; w < W; ++w)
                m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, f[i][w] & 0x7f807f80u));
        return m[0] == 0x7f80 || m[1] == 0x7f80;
    }
};

__device__ __forceinline__ f32x4 mfma16(const u32x4& a, const u32x4& b, const f32x4& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma16(const bf16x8& a, const bf16x8& b, const f32x4& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// O^T += V^T P^T where values among the 32 keys are infinite or NaN; bit i of
// vis says that the lane's row sees key 8q + i.  A zero weight times an infinity
// would reach rows that do not see it, so the products run on the finite values
// alone, and a count of the visible infinities and NaNs of each output (a
// product of zeros and ones) adds them.
template <int D, int MT>
__device__ __forceinline__ void add_odd_values(f32x4 (&acc)[MT][D / 16], const ValueFrag<D>& v, const bf16x8 (&hi)[MT],
                                               const bf16x8 (&lo)[MT], const uint32_t (&vis)[MT]) {
    const float special[3] = {__builtin_inff(), -__builtin_inff(), __builtin_nanf("")};
#pragma unroll
    for (int j = 0; j < D / 16; ++j) {
        const u32x4 x = __builtin_bit_cast(u32x4, v.operand(j));
        u32x4 fin, kind[3];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t keep = 0, k0 = 0, k1 = 0, k2 = 0;
#pragma unroll
            for (int h = 0; h < 32; h += 16) {
                const uint32_t e = (x[i] >> h) & 0xffffu;
                const uint32_t one = 0x3f80u << h;
                const bool f = (e & 0x7f80u) != 0x7f80u;
                keep |= f ? e << h : 0u;
                k0 |= e == 0x7f80u ? one : 0u;
                k1 |= e == 0xff80u ? one : 0u;
                k2 |= !f && (e & 0x7fu) ? one : 0u;
            }
            fin[i] = keep;
            kind[0][i] = k0;
            kind[1][i] = k1;
            kind[2][i] = k2;
        }
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            u32x4 ones;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                ones[e] = ((vis[i] >> (2 * e)) & 1 ? 0x3f80u : 0u) | ((vis[i] >> (2 * e + 1)) & 1 ? 0x3f800000u : 0u);
            const bf16x8 a = __builtin_bit_cast(bf16x8, fin);
            acc[i][j] = mfma16(a, hi[i], mfma16(a, lo[i], acc[i][j]));
#pragma unroll
            for (int s = 0; s < 3; ++s) {
                const f32x4 n = mfma16(kind[s], ones, f32x4{0, 0, 0, 0});
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[i][j][e] += n[e] > 0.0f ? special[s] : 0.0f;
            }
            __builtin_amdgcn_sched_barrier(0);  // one tile's temporaries at a time
        }
    }
}

}  // namespace krk
