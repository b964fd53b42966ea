// Cache attention for many rows of a head (prompts, large batches over a
// shared prefix): one workgroup per tile of 32 * W rows, K and V through LDS.
//
// Bound by the matrix pipe, the exponentials and LDS alike: 64 keys of a wave's
// 32 rows are 1.05 MFLOP (1030 cycles of a SIMD's MFMA at head size 128), 32 KB
// of LDS reads (a quarter of 1030 cycles of what a CU's LDS delivers), and 2048
// weights at about 30 VALU cycles per 64 of them.
//
// Work split.  W waves (4 or 8), each with 32 rows of its own, all reading the
// same 64-key steps of K and V from LDS; two waves per SIMD, so that one's
// softmax runs under the other's products.  S^T = K Q^T and O^T = V^T P^T on
// v_mfma_f32_32x32x16_bf16, the row in the column (lane & 31) of either; the key
// order of a step's second product is the one the first leaves in its lanes, so
// weights stay in their lane.  V's operand comes transposed out of LDS
// (ds_read_b64_tr_b16).
//
// Steps are pipelined: the scores of step j + 1 (MFMA) run with the weights of
// step j (VALU), then step j's products with V with the maxima of step j + 1.
// The running maximum moves only when a row's grows by more than 2^8 (the
// weights stay below 2^8 then, which costs no precision), so O is rescaled a
// few times a row instead of every step.
//
// LDS: rings of three 64-key steps of K and two of V (80 KB at head size 128:
// two workgroups a CU), filled by DMA, one barrier a step.  16-byte chunks of a
// row are permuted with the row's low bits, so that neither kind of read meets
// bank conflicts.
//
// Weights are rounded to bf16 for the product with V (their sum is not): with
// 8 bits of mantissa each, the error of a weighted mean of many values is that
// of the final rounding again.
#pragma once

#include "krk_attn_common.h"

namespace krk {

typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(4))) short s16x4;
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

constexpr int kTileStep = 64;
constexpr int kTileKRing = 3, kTileVRing = 2;

template <int D>
constexpr size_t tile_lds_bytes() {
    return (size_t)(kTileKRing + kTileVRing) * kTileStep * D * 2;
}

__device__ __forceinline__ f32x16 mfma32(const bf16x8& a, const bf16x8& b, const f32x16& c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

template <int D, int W>
struct TileKernel {
    static constexpr int KS = D / 16;  // k-steps of S^T
    static constexpr int DT = D / 32;  // 32-wide tiles of O^T
    static constexpr int CH = D / 8;   // 16-byte chunks of a row
    static constexpr int ROWS_PER_DMA = 64 / CH;
    static constexpr int DMAS = kTileStep / ROWS_PER_DMA / W;  // of K, or of V, per wave and step
    static constexpr int STEP_BYTES = kTileStep * D * 2;

    // Chunk permutations: K reads take 16 (8) rows of one chunk at a time, V
    // reads 4 (2) rows of 4 chunks.
    static __device__ __forceinline__ int k_swizzle(int row) { return row & (CH - 1); }
    static __device__ __forceinline__ int v_swizzle(int row) { return 4 * (row & (CH / 4 - 1)); }

    // This wave's share of keys kb .. kb + 63 into `to`: off[i] is the lane's
    // place from the step's first key; keys from `limit` on read the last one
    // again.
    template <bool V>
    static __device__ __forceinline__ int chunk_of(int i, int wave, int lane) {
        const int row = (wave + W * i) * ROWS_PER_DMA + lane / CH;
        return (lane % CH) ^ (V ? v_swizzle(row) : k_swizzle(row));
    }
    template <bool V>
    static __device__ __forceinline__ void fetch(const uint16_t* base, int64_t slot, const int64_t (&off)[DMAS], int kb,
                                                 int limit, unsigned char* to, int wave, int lane) {
        const uint16_t* step = base + (int64_t)kb * slot;
#pragma unroll
        for (int i = 0; i < DMAS; ++i) {
            const int idx = wave + W * i;
            const uint16_t* from = step + off[i];
            if (kb + kTileStep > limit) {
                const int key = kb + idx * ROWS_PER_DMA + lane / CH;
                from = base + (int64_t)(key < limit ? key : limit - 1) * slot + 8 * chunk_of<V>(i, wave, lane);
            }
            dma_row(from, to + idx * 1024);
        }
    }

    static __device__ __forceinline__ bf16x8 k_operand(const unsigned char* at, int off) {
        return *reinterpret_cast<const bf16x8*>(at + off);
    }
    // Two transposed reads: keys k .. k + 3 and k + 8 .. k + 11 of this lane's d.
    static __device__ __forceinline__ bf16x8 v_operand(const unsigned char* at) {
        const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)at);
        const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(at + 8 * D * 2));
        typedef __attribute__((ext_vector_type(8))) short s16x8;
        const s16x8 x = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
        return __builtin_bit_cast(bf16x8, x);
    }
};

// The key (of 64) behind score register i of 32-key tile kt in lane group g.
__device__ __forceinline__ int tile32_key(int kt, int i, int g) { return 32 * kt + 8 * (i >> 2) + 4 * g + (i & 3); }

__device__ __forceinline__ bool odd_bf16x8(const bf16x8& v) {
    const u32x4 x = __builtin_bit_cast(u32x4, v);
    bool odd = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) odd = odd || (x[i] & 0x7f80u) == 0x7f80u || (x[i] & 0x7f800000u) == 0x7f800000u;
    return odd;
}

template <int D, int W>
__global__ void __launch_bounds__(64 * W, 8 / W) attn_tile_kernel(AttnParams p) {
    using T = TileKernel<D, W>;
    constexpr int KS = T::KS, DT = T::DT;
    constexpr int TR = 32 * W;
    extern __shared__ __align__(16) unsigned char lds[];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n32 = lane & 31, g2 = lane >> 5;
    const Task task = task_of<TR>(p, blockIdx.x);
    const int limit = task.limit;

    const int my_row = task.row0 + wave * 32 + n32;
    const TaskRow mine = task_row(p, task, my_row);
    const RowSight sight = mine.sight;
    bf16x8 qf[KS];
    Reach reach;  // of this wave's rows
    Reach block;  // of the workgroup's
    reach.add(sight, my_row < task.rows);
    {
        const uint16_t* qr = p.q + ((int64_t)mine.b * p.R + mine.r) * p.q_row + (int64_t)mine.head * D + 8 * g2;
#pragma unroll
        for (int s = 0; s < KS; ++s) qf[s] = __builtin_bit_cast(bf16x8, load_cached16(qr + 16 * s));
    }
    reach.join_lanes();
    {
        int* x = reinterpret_cast<int*>(lds);
        if (lane == 0) {
            x[4 * wave] = reach.lo_min;
            x[4 * wave + 1] = reach.hi_max;
            x[4 * wave + 2] = reach.lo_max;
            x[4 * wave + 3] = reach.hi_min;
        }
        __syncthreads();
#pragma unroll
        for (int w = 0; w < W; ++w) {
            block.lo_min = x[4 * w] < block.lo_min ? x[4 * w] : block.lo_min;
            block.hi_max = x[4 * w + 1] > block.hi_max ? x[4 * w + 1] : block.hi_max;
            block.lo_max = x[4 * w + 2] > block.lo_max ? x[4 * w + 2] : block.lo_max;
            block.hi_min = x[4 * w + 3] < block.hi_min ? x[4 * w + 3] : block.hi_min;
        }
        block.lo_min = __builtin_amdgcn_readfirstlane(block.lo_min);
        block.hi_max = __builtin_amdgcn_readfirstlane(block.hi_max);
        block.lo_max = __builtin_amdgcn_readfirstlane(block.lo_max);
        block.hi_min = __builtin_amdgcn_readfirstlane(block.hi_min);
        __syncthreads();
    }
    const KeySteps<kTileStep> steps(p, task, block);
    const int t0 = steps.t0, t1 = steps.t1;

    unsigned char* kring = lds;
    unsigned char* vring = lds + kTileKRing * T::STEP_BYTES;
    auto k_at = [&](int t) { return kring + (unsigned)t % kTileKRing * T::STEP_BYTES; };
    auto v_at = [&](int t) { return vring + (unsigned)t % kTileVRing * T::STEP_BYTES; };
    int64_t k_off[T::DMAS], v_off_in[T::DMAS];
#pragma unroll
    for (int i = 0; i < T::DMAS; ++i) {
        const int row = (wave + W * i) * T::ROWS_PER_DMA + lane / T::CH;
        k_off[i] = row * task.k_slot + 8 * T::template chunk_of<false>(i, wave, lane);
        v_off_in[i] = row * task.v_slot + 8 * T::template chunk_of<true>(i, wave, lane);
    }
    auto fetch_k = [&](int t) { T::template fetch<false>(task.k, task.k_slot, k_off, steps.key(t), limit, k_at(t), wave, lane); };
    auto fetch_v = [&](int t) { T::template fetch<true>(task.v, task.v_slot, v_off_in, steps.key(t), limit, v_at(t), wave, lane); };

    // This lane's places in a step's K and V.
    const int k_row = n32 * D * 2;
    const int k_xor = g2 ^ T::k_swizzle(n32);
    const int j4 = (lane & 15) >> 2;
    int v_off[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d) {
        const int key = 4 * g2 + j4;
        const int chunk = (4 * d + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) ^ T::v_swizzle(key);
        v_off[d] = key * D * 2 + chunk * 16 + (lane & 1) * 8;
    }

    f32x16 o[DT], s[2];
    float m = kNegInf, mc = 0.0f, l = 0.0f;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[d][e] = 0.0f;

    // Scores of a step into x.
    auto scores = [&](int t, f32x16 (&x)[2]) {
        const unsigned char* kb = k_at(t) + k_row;
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
            for (int e = 0; e < 16; ++e) x[kt][e] = 0.0f;
        // Two k-steps' operands are read ahead, no more: the compiler would
        // read all of them at once and spill q.
        bf16x8 a[2][2];
        auto read = [&](int ks) {
#pragma unroll
            for (int kt = 0; kt < 2; ++kt) a[ks & 1][kt] = T::k_operand(kb, 32 * kt * D * 2 + ((2 * ks) ^ k_xor) * 16);
        };
        read(0);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            if (ks + 1 < KS) read(ks + 1);
#pragma unroll
            for (int kt = 0; kt < 2; ++kt) x[kt] = mfma32(a[ks & 1][kt], qf[ks], x[kt]);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    // No weight for what the row does not see.  Steps that every row of the
    // wave sees whole skip this.
    const int hi = sight.hi < task.seg + limit - 1 ? sight.hi : task.seg + limit - 1;
    auto seen_whole = [&](const Reach& r, int kb) {
        const int pos = task.seg + kb;
        return kb + kTileStep <= limit && pos + kTileStep - 1 <= r.hi_min && (pos >= r.lo_max || pos + kTileStep <= p.sinks);
    };
    auto hide = [&](int t, f32x16 (&x)[2]) {
        const int kb = steps.key(t);
        if (seen_whole(reach, kb)) return;
        uint32_t vis = 0;  // bit e: the key of register e
        if (p.tree) {
#pragma unroll 1
            for (int e = 0; e < 32; ++e) {
                const int key = kb + tile32_key(e >> 4, e & 15, g2);
                vis |= (key < limit && sees(sight, task.seg + key, p.sinks)) ? 1u << e : 0u;
            }
        } else {
            const int from = task.seg + kb + 4 * g2;
#pragma unroll
            for (int e = 0; e < 32; ++e) {
                const int t_e = from + tile32_key(e >> 4, e & 15, 0);
                const bool ok = (t_e <= hi) & ((t_e >= sight.lo) | (t_e < p.sinks));
                vis |= ok ? 1u << e : 0u;
            }
        }
#pragma unroll
        for (int e = 0; e < 32; ++e) x[e >> 4][e & 15] = (vis >> e) & 1 ? x[e >> 4][e & 15] : kNegInf;
    };
    auto maximum = [&](const f32x16 (&x)[2]) {
        float v = fmaxf(x[0][0], x[1][0]);
#pragma unroll
        for (int e = 1; e < 16; ++e) v = fmaxf(fmaxf(v, x[0][e]), x[1][e]);
        const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    };
    const float slack = fminf(8.0f / p.c, 1e30f);
    auto raise = [&](float mx) {
        if (__any(mx > m + slack)) {
            const float mn = fmaxf(m, mx);
            const float ms = mn == kNegInf ? 0.0f : mn;
            const float alpha = exp2_raw((m - ms) * p.c);
            m = mn;
            mc = ms * p.c;
            l *= alpha;
#pragma unroll
            for (int d = 0; d < DT; ++d) o[d] *= alpha;
        }
    };
    // Weights of a step, rounded to bf16 as the operand of the second product.
    auto weigh = [&](const f32x16 (&x)[2], u32x4 (&w)[4]) {
        float sum[2] = {0.0f, 0.0f};
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
            const float a = exp2_raw(__builtin_fmaf(x[e >> 4][e & 15], p.c, -mc));
            const float b = exp2_raw(__builtin_fmaf(x[e >> 4][(e & 15) + 1], p.c, -mc));
            sum[0] += a;
            sum[1] += b;
            w[e >> 3][(e & 7) >> 1] = pack_bf16(a, b);
        }
        l += sum[0] + sum[1];
    };
    auto products = [&](int t, const u32x4 (&w)[4]) {
        const unsigned char* vb = v_at(t);
#pragma unroll
        for (int ks = 0; ks < 4; ++ks)
#pragma unroll
            for (int d = 0; d < DT; ++d)
                o[d] = mfma32(T::v_operand(vb + v_off[d] + 16 * ks * D * 2), __builtin_bit_cast(bf16x8, w[ks]), o[d]);
    };
    // A step that some row of the workgroup does not see whole may hold
    // infinities or NaNs that only some rows see.  Each wave then zeroes those
    // among the values it fetched; they are added behind the last step.
    bool any_odd = false;
    auto tame = [&](int t) {
        unsigned char* at = v_at(t);
#pragma unroll
        for (int i = 0; i < T::DMAS; ++i) {
            u32x4* x = reinterpret_cast<u32x4*>(at + (wave + W * i) * 1024 + lane * 16);
            const u32x4 v = *x;
            if (__any(odd_bf16x8(__builtin_bit_cast(bf16x8, v)))) {
                *x = finite_bf16x8(v);
                any_odd = true;
            }
        }
    };

    if (t0 < t1) {
        // K two steps ahead of the scores, V one ahead of its products.
        const int two = t0 + 1 < t1, three = t0 + 2 < t1;
        fetch_k(t0);
        if (two) fetch_k(t0 + 1);
        fetch_v(t0);
        if (three) fetch_k(t0 + 2);
        vm_wait_stages<T::DMAS>(1 + two + three);  // K of the first step has landed
        bare_barrier();
        scores(t0, s);
        hide(t0, s);
        raise(maximum(s));
        for (int t = t0; t < t1; ++t) {
            // K of step t + 1 and V of step t have landed (K of step t + 2,
            // issued after them, may not have), and every wave is through with
            // the slots that the next DMAs fill.
            vm_wait_stages<T::DMAS>(t + 2 < t1);
            if (!seen_whole(block, steps.key(t))) tame(t);
            lds_wait();
            bare_barrier();
            if (t + 1 < t1) fetch_v(t + 1);
            if (t + 3 < t1) fetch_k(t + 3);
            f32x16 nx[2];
            const bool more = t + 1 < t1;
            if (more) scores(t + 1, nx);
            u32x4 w[4];
            weigh(s, w);
            __builtin_amdgcn_sched_barrier(0);
            products(t, w);
            if (more) {
                s[0] = nx[0];
                s[1] = nx[1];
                hide(t + 1, s);
                raise(maximum(s));
            }
        }
        int* flags = reinterpret_cast<int*>(lds);
        __syncthreads();
        if (lane == 0) flags[wave] = any_odd;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < W; ++w) any_odd = any_odd || flags[w];
        if (any_odd) {  // the infinities and NaNs left out above: rare, so key by key
#pragma unroll 1
            for (int t = t0; t < t1; ++t) {
                const int kb = steps.key(t);
                if (seen_whole(block, kb)) continue;
#pragma unroll 1
                for (int key = kb; key < kb + kTileStep && key < limit; ++key) {
                    const bool ok = sees(sight, task.seg + key, p.sinks);
                    const uint16_t* vr = task.v + (int64_t)key * task.v_slot + 4 * g2;
#pragma unroll
                    for (int d = 0; d < DT; ++d)
#pragma unroll
                        for (int e = 0; e < 16; e += 4) {
                            const uint2 x = *reinterpret_cast<const uint2*>(vr + 32 * d + 2 * e);
                            const uint32_t y[4] = {x.x << 16, x.x & 0xffff0000u, x.y << 16, x.y & 0xffff0000u};
#pragma unroll
                            for (int k = 0; k < 4; ++k)
                                o[d][e + k] += ok && (y[k] & 0x7f800000u) == 0x7f800000u ? __uint_as_float(y[k]) : 0.0f;
                        }
                }
            }
        }
    }

    // Each wave owns its rows: straight from its registers.
    const int64_t all_rows = (int64_t)p.B * p.kv_heads * p.RG;
    const bool last = p.splits + p.prefix_splits == 1;
    const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(l), __float_as_uint(l), false, false);
    float L = __uint_as_float(both[0]) + __uint_as_float(both[1]);
    if (sight.lo == kPadding) {  // unmasked in the steps that its neighbours see whole
        L = 0.0f;
        m = kNegInf;
    }
    if (my_row >= task.rows) return;
    const int64_t at = (int64_t)mine.b * p.R + mine.r;
    const int64_t g = ((int64_t)mine.b * p.kv_heads + task.h) * p.RG + (int64_t)mine.r * p.G + (mine.head - task.h * p.G);
    const float inv = L == 0.0f ? 0.0f : last ? 1.0f / L : 1.0f;
    if (g2 == 0) {
        if (!last) p.ml[(int64_t)task.part * all_rows + g] = make_float2(m, L);
        if (last && p.lse) p.lse[at * p.heads + mine.head] = L == 0.0f ? kNegInf : m * p.scale + logf(L);
        if (last && p.stat) p.stat[g] = make_float2(m == kNegInf ? 0.0f : m, inv);
    }
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
            f32x4 y;
#pragma unroll
            for (int k = 0; k < 4; ++k) y[k] = L == 0.0f ? 0.0f : o[d][e + k] * inv;
            const int col = 32 * d + 2 * e + 4 * g2;
            if (last)
                *reinterpret_cast<uint2*>(p.out + at * p.out_row + (int64_t)mine.head * D + col) =
                    make_uint2(pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3]));
            else
                *reinterpret_cast<f32x4*>(p.part + ((int64_t)task.part * all_rows + g) * D + col) = y;
        }
}

}  // namespace krk
