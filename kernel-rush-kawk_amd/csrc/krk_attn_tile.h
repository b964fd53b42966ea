// Cache attention for many rows of a head (prompts, batches over a shared
// prefix): one workgroup per tile of 128 rows, K and V through LDS.
//
// Bound by the matrix pipe, LDS and the vector pipe alike: 64 keys of a wave's 32
// rows are 1024 cycles of its SIMD's matrix pipe at head size 128 (1.05 MFLOP), 32 KB
// of LDS reads, 1030 cycles for a CU's four waves (the keys' own 32 KB come on
// top), and 1260 cycles of the vector pipe for the 2048 weights, their maxima and
// what goes with them (counted).  Two waves of a SIMD need 4200 cycles for a step
// each, the first loads and the last stores included: 840-880 TFLOP/s of an 8192-row
// prompt with a window of 2048, at the 2.1 GHz that the clock falls to under it.
//
// Work split.  Four waves, each with 32 rows of its own, all reading the same
// 64-key steps of K and V from LDS.  S^T = K Q^T and O^T = V^T P^T on
// v_mfma_f32_32x32x16_bf16, the row in the column (lane & 31) of either; the key
// order of a step's second product is the one the first leaves in its lanes, so
// weights stay in their lane.  V's operand comes transposed out of LDS
// (ds_read_b64_tr_b16).  Two workgroups share a CU (80 KB of LDS and up to 256
// registers a lane each) and run apart: 8 waves in one workgroup, four of them
// half a step behind, need half the DMAs but were 20% slower (5.6M GPU cycles
// against 4.6M), as one half's weights wait for LDS and issue slots under the
// other's products.  64 rows a wave would halve the LDS reads, but their
// registers spill.
//
// The running maximum moves only when a row's grows by more than 2^8 (the
// weights stay below 2^8 then, which costs no precision), so O is rescaled a
// few times a row instead of every step.
//
// LDS: rings of three 64-key steps of K and two of V, filled by DMA, one
// barrier a step.  16-byte chunks of a row are permuted with the row's low
// bits, so that neither kind of read meets bank conflicts.
//
// Weights are rounded to one bf16 for the product with V; their sum is not.  A
// choice: with two parts, as the split kernel has them, the products take half as
// many matrix instructions again (8192-row prompt 279 -> 366 us, 64 sequences over
// 32768 shared keys 92 -> 101, 32 scored rows over 2 x 16000 keys 67 -> 73).  Each
// weight is off by up to 2^-8 of itself, so an output by up to 2^-8 of sum p |v|
// before its own rounding, whether its row sees many keys or few: measured, 0.0021
// of the outputs' norm for rows of many keys and 0.0017-0.0020 for rows of 2 to 32
// (rounding the exact result: 0.0017).  The sum of the rounded weights in its place
// would help rows whose weight lies on a few keys (0.0019 -> 0.0017, the others
// alike) and costs 3%.
#pragma once

#include <type_traits>

#include "krk_attn_common.h"

namespace krk {

typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(4))) short s16x4;
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

constexpr int kTileStep = 64;
constexpr int kTileWaves = 4;
constexpr int kTileThreads = 64 * kTileWaves;
constexpr int kTileRows = 32 * kTileWaves;
constexpr int kTileKRing = 3, kTileVRing = 2;  // steps in LDS

template <int D>
constexpr size_t tile_lds_bytes() {
    return (size_t)(kTileKRing + kTileVRing) * kTileStep * D * 2;
}

// One 1 KB DMA into LDS, lane l's 16 bytes from src to dst + 16 l (as dma_row).
// In assembly, because around the builtin the compiler waits for every DMA in
// flight before a transposed LDS read, and a step then lasts as long as the
// fetch that it started; the waits here are vm_wait_stages' alone.
__device__ __forceinline__ void dma_row_quiet(const uint16_t* src, uint32_t dst) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" : : "v"(src), "s"(dst) : "memory", "m0");
}

__device__ __forceinline__ f32x16 mfma32(const bf16x8& a, const bf16x8& b, const f32x16& c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

template <int D>
struct TileKernel {
    static constexpr int KS = D / 16;  // k-steps of S^T
    static constexpr int DT = D / 32;  // 32-wide tiles of O^T
    static constexpr int CH = D / 8;   // 16-byte chunks of a row
    static constexpr int ROWS_PER_DMA = 64 / CH;
    static constexpr int DMAS = kTileStep / ROWS_PER_DMA / kTileWaves;  // of K, or of V, per wave and step
    static constexpr int STEP_BYTES = kTileStep * D * 2;

    // Chunk permutations: K reads take 16 (8) rows of one chunk at a time, V
    // reads 4 (2) rows of 4 chunks.
    static __device__ __forceinline__ int k_swizzle(int row) { return row & (CH - 1); }
    static __device__ __forceinline__ int v_swizzle(int row) { return 4 * (row & (CH / 4 - 1)); }

    // This wave's share of keys kb .. kb + 63 into `to`: lane offsets from the
    // step's first key; keys from `limit` on read the last one again.
    template <bool V>
    static __device__ __forceinline__ void offsets(int64_t slot, int wave, int lane, int64_t (&off)[DMAS]) {
#pragma unroll
        for (int i = 0; i < DMAS; ++i) {
            const int row = (wave + kTileWaves * i) * ROWS_PER_DMA + lane / CH;
            off[i] = row * slot + 8 * ((lane % CH) ^ (V ? v_swizzle(row) : k_swizzle(row)));
        }
    }
    // Fetches a task's steps in order: this wave's share of a step's 64 rows.
    // Places advance instead of being worked out: a wave's scalar instructions
    // are on its path (this and the like took 2.5% off the cycles).
    struct Stream {
        const uint16_t* from;  // the step's first row
        int t;
        uint32_t to;  // its slot in the ring
        __device__ __forceinline__ Stream(const uint16_t* base, int64_t slot, const KeySteps<kTileStep>& steps)
            : from(base + (int64_t)steps.key(steps.t0) * slot), t(steps.t0), to(0) {}
        template <int RING>
        __device__ __forceinline__ void fetch(int64_t slot, const int64_t (&off)[DMAS], const KeySteps<kTileStep>& steps, int t_full,
                                              int limit, uint32_t ring, int wave, int lane) {
            const uint32_t dst = ring + to + wave * 1024;
            if (t < t_full) {
#pragma unroll
                for (int i = 0; i < DMAS; ++i) dma_row_quiet(from + off[i], dst + kTileWaves * i * 1024);
            } else {  // rows from the limit on read the last one again
                const int kb = steps.key(t);
#pragma unroll
                for (int i = 0; i < DMAS; ++i) {
                    const int over = kb + (wave + kTileWaves * i) * ROWS_PER_DMA + lane / CH - (limit - 1);
                    dma_row_quiet(from + off[i] - (over > 0 ? over : 0) * slot, dst + kTileWaves * i * 1024);
                }
            }
            if (t < steps.t1 - 1) {
                from += kTileStep * slot;
                ++t;
                if (t == steps.sink_steps) from += (int64_t)(steps.from - kTileStep * t) * slot;
            }
            to += STEP_BYTES;
            to = to == (uint32_t)RING * STEP_BYTES ? 0u : to;
        }
    };

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

// Issue order of the next N MFMAs and of LDS reads for later ones, EACH behind
// an MFMA.  Left alone the compiler reads each operand right before its MFMA
// and waits.
template <int N, int EACH>
__device__ __forceinline__ void read_ahead() {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        if (EACH) __builtin_amdgcn_sched_group_barrier(0x100, EACH, 0);
    }
}

template <int D>
__global__ void __launch_bounds__(kTileThreads, 2) attn_tile_kernel(AttnParams p) {
    using T = TileKernel<D>;
    constexpr int KS = T::KS, DT = T::DT;
    extern __shared__ __align__(16) unsigned char lds[];
    const Task task = task_of(p, blockIdx.x, kTileRows, kTileRows);
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n32 = lane & 31, g2 = lane >> 5;
    const int limit = task.limit;

    const int my_row = task.row0 + wave * 32 + n32;
    const TaskRow mine = task_row(p, task, my_row);
    const RowSight sight = mine.sight(p);
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
        for (int w = 0; w < kTileWaves; ++w) {
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
    const uint32_t lds_base = (uint32_t)(uintptr_t)(lds_s16x4*)lds;

    // The next fetches of K and of V: where from, where to.  Behind the last
    // step it is fetched again, into slots that nothing reads any more: every
    // step then has the same number of DMAs in flight.
    int64_t k_off[T::DMAS], v_from[T::DMAS];
    T::template offsets<false>(task.k_slot, wave, lane, k_off);
    T::template offsets<true>(task.v_slot, wave, lane, v_from);
    typename T::Stream k_next(task.k, task.k_slot, steps), v_next(task.v, task.v_slot, steps);
    const int t_full = steps.key(t1 - 1) + kTileStep <= limit ? t1 : t1 - 1;  // steps from here on pass the limit
    auto fetch_k = [&]() { k_next.template fetch<kTileKRing>(task.k_slot, k_off, steps, t_full, limit, lds_base, wave, lane); };
    auto fetch_v = [&]() {
        v_next.template fetch<kTileVRing>(task.v_slot, v_from, steps, t_full, limit, lds_base + kTileKRing * T::STEP_BYTES, wave, lane);
    };
    // The slots that the next scores and products read.
    uint32_t k_read = 0, v_read = 0;
    auto turn = [](uint32_t& slot, int ring) {
        slot += T::STEP_BYTES;
        slot = slot == (uint32_t)ring * T::STEP_BYTES ? 0u : slot;
    };

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
    float m = kNegInf, l = 0.0f;
    float ref = 0.0f;  // m, or 0 before the row has seen a key
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[d][e] = 0.0f;

    // Scores of a step: first those of its first 32 keys, whose maximum is then
    // taken under the others' products.
    auto scores = [&]() {
        const unsigned char* kb = kring + k_read + k_row;
        turn(k_read, kTileKRing);
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
#pragma unroll
            for (int e = 0; e < 16; ++e) s[kt][e] = 0.0f;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
                s[kt] = mfma32(T::k_operand(kb, 32 * kt * D * 2 + ((2 * ks) ^ k_xor) * 16), qf[ks], s[kt]);
        }
    };
    // No weight for what the row does not see (not called for steps that every
    // row of the wave sees whole).
    const int hi = sight.hi < task.seg + limit - 1 ? sight.hi : task.seg + limit - 1;
    // The steps that every row of a wave, or of the workgroup, sees whole.
    struct Steps {
        int from, n;
        __device__ __forceinline__ bool has(int t) const { return (unsigned)(t - from) < (unsigned)n; }
    };
    auto whole_steps = [&](const Reach& r) {
        Steps x;
        const int end = r.hi_min - task.seg < limit ? r.hi_min - task.seg + 1 : limit;
        const int low = r.lo_max - task.seg - steps.from;
        x.from = steps.sink_steps + (low > 0 ? (low + kTileStep - 1) / kTileStep : 0);
        const int n = steps.sink_steps + (end > steps.from ? (end - steps.from) / kTileStep : 0) - x.from;
        x.n = n > 0 ? n : 0;
        return x;
    };
    const Steps mine_whole = whole_steps(reach), all_whole = whole_steps(block);
    auto hide = [&](int t) {
        const int kb = steps.key(t);
        const int from = task.seg + kb + 4 * g2;
        if (!p.tree) {
            const int top = hi - from, low = sight.lo - from, sink = p.sinks - from;
#pragma unroll
            for (int e = 0; e < 32; ++e) {
                const int k = tile32_key(e >> 4, e & 15, 0);
                const bool ok = (k <= top) & ((k >= low) | (k < sink));
                s[e >> 4][e & 15] = ok ? s[e >> 4][e & 15] : kNegInf;
            }
            return;
        }
        uint32_t vis = 0;  // bit e: the key of register e
#pragma unroll 1
        for (int e = 0; e < 32; ++e) {
            const int k = tile32_key(e >> 4, e & 15, 0) + 4 * g2;
            vis |= (kb + k < limit && sees(sight, task.seg + kb + k, p.sinks)) ? 1u << e : 0u;
        }
#pragma unroll
        for (int e = 0; e < 32; ++e) s[e >> 4][e & 15] = (vis >> e) & 1 ? s[e >> 4][e & 15] : kNegInf;
    };
    auto highest = [&](int kt) {
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = fmaxf(fmaxf(s[kt][3 * e], s[kt][3 * e + 1]), s[kt][3 * e + 2]);
        v[0] = fmaxf(fmaxf(v[0], s[kt][12]), s[kt][13]);
        v[1] = fmaxf(fmaxf(v[1], s[kt][14]), s[kt][15]);
        return fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3]));
    };
    const float slack = fminf(8.0f / p.c, 1e30f);
    auto raise = [&](float v) {
        const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        const float mx = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
        if (__any(mx > m + slack)) {
            const float mn = fmaxf(m, mx);
            ref = mn == kNegInf ? 0.0f : mn;
            const float alpha = exp2_raw((m - ref) * p.c);
            m = mn;
            l *= alpha;
#pragma unroll
            for (int d = 0; d < DT; ++d) o[d] *= alpha;
        }
    };
    // Its weights, rounded to bf16 as the operand of the second product.  The
    // difference first: one fma of s * c - m * c would be 2% faster, but its m * c is
    // rounded, and at scores of 10^9 that turns weights of 1 into 0 or infinity.
    u32x4 w[4];
    auto weigh = [&]() {
        float sum[2] = {0.0f, 0.0f};
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
            const float a = exp2_raw((s[e >> 4][e & 15] - ref) * p.c);
            const float b = exp2_raw((s[e >> 4][(e & 15) + 1] - ref) * p.c);
            sum[0] += a;
            sum[1] += b;
            w[e >> 3][(e & 7) >> 1] = pack_bf16(a, b);
        }
        l += sum[0] + sum[1];
        asm volatile("" : "+v"(l));  // the sums here, not behind the products
    };
    auto v_at = [&](int ks, int d) { return T::v_operand(vring + v_read + v_off[d] + 16 * ks * D * 2); };
    // A step that some row of the workgroup does not see whole may hold
    // infinities or NaNs that only some rows see.  Each wave then zeroes those
    // among the values it fetched; they are added behind the last step.
    bool any_odd = false;
    auto tame = [&](uint32_t slot) {
        unsigned char* at = vring + slot;
#pragma unroll 1
        for (int i = 0; i < T::DMAS; ++i) {
            u32x4* x = reinterpret_cast<u32x4*>(at + (wave + kTileWaves * i) * 1024 + lane * 16);
            const u32x4 v = *x;
            if (__any(odd_bf16x8(__builtin_bit_cast(bf16x8, v)))) {
                *x = finite_bf16x8(v);
                any_odd = true;
            }
        }
    };

    if (t0 < t1) {
        // A step's maximum, behind its scores.
        auto settle = [&](int t, float first) {
            if (!mine_whole.has(t)) {
                hide(t);
                first = highest(0);
            }
            raise(fmaxf(first, highest(1)));
        };
        // The products with V, and the next step's scores where there is one.
        auto multiply = [&](const bf16x8 (&first)[DT], auto more) {
#pragma unroll
            for (int ks = 0; ks < 4; ++ks)
#pragma unroll
                for (int d = 0; d < DT; ++d)
                    o[d] = mfma32(ks ? v_at(ks, d) : first[d], __builtin_bit_cast(bf16x8, w[ks]), o[d]);
            turn(v_read, kTileVRing);
            float top = 0.0f;
            if constexpr (decltype(more)::value) {
                scores();
                top = highest(0);
                read_ahead<4 * DT, 2>();
                read_ahead<KS, 1>();
                read_ahead<KS, 0>();
            } else {
                read_ahead<3 * DT, 2>();
                read_ahead<DT, 0>();
            }
            __builtin_amdgcn_sched_barrier(0);
            return top;
        };
        // K two steps ahead of the scores, V one ahead of its products.
        fetch_k();
        fetch_k();
        fetch_v();
        fetch_k();
        vm_wait_stages<T::DMAS>(3);  // K of the first step has landed
        // q has landed as well; said here, or the compiler waits for it in the
        // loop, and with it for the DMAs just issued.
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) asm volatile("" : "+v"(qf[ks]));
        bare_barrier();
        scores();
        settle(t0, highest(0));
        auto step = [&](int t, auto more) {
            // K of step t + 1 and V of step t have landed (K of step t + 2,
            // fetched behind them, may not have), and every wave is through
            // with the slots that the next DMAs fill.
            vm_wait_stages<T::DMAS>(1);
            if (!all_whole.has(t)) tame(v_read);
            lds_wait();
            bare_barrier();
            bf16x8 first[DT];
#pragma unroll
            for (int d = 0; d < DT; ++d) first[d] = v_at(0, d);
            fetch_v();
            fetch_k();
            weigh();
            // The other workgroup's wave of this SIMD leaves the matrix pipe
            // to the one that is at its products (3% fewer cycles).
            __builtin_amdgcn_s_setprio(1);
            __builtin_amdgcn_sched_barrier(0);
            const float top = multiply(first, more);
            if constexpr (decltype(more)::value) settle(t + 1, top);
            __builtin_amdgcn_s_setprio(0);
        };
        for (int t = t0; t < t1 - 1; ++t) step(t, std::true_type{});
        step(t1 - 1, std::false_type{});
        vm_wait_stages<T::DMAS>(0);
        // Behind the wave's output rows below.
        int* flags = reinterpret_cast<int*>(lds + tile_lds_bytes<D>() - 64);
        __syncthreads();
        if (lane == 0) flags[wave] = any_odd;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kTileWaves; ++w) any_odd = any_odd || flags[w];
        if (any_odd) {  // the infinities and NaNs left out above: rare, so key by key
#pragma unroll 1
            for (int t = t0; t < t1; ++t) {
                const int kb = steps.key(t);
                if (all_whole.has(t)) continue;
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
                                o[d][e + k] += ok ? odd_or_zero(y[k]) : 0.0f;
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
    const bool live = my_row < task.rows;
    const int64_t at = (int64_t)mine.b * p.R + mine.r;
    const int64_t g = ((int64_t)mine.b * p.kv_heads + task.h) * p.RG + (int64_t)mine.r * p.G + (mine.head - task.h * p.G);
    const bool none = L == 0.0f;
    const float inv = none ? 0.0f : 1.0f / L;
    if (live && g2 == 0) {
        if (!last) p.ml[(int64_t)task.part * all_rows + g] = make_float2(m, L);
        if (last && p.lse) p.lse[at * p.heads + mine.head] = none ? kNegInf : m * p.scale + logf(L);
        if (last && p.stat) p.stat[g] = make_float2(m == kNegInf ? 0.0f : m, inv);
    }
    if (!last) {
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int e = 0; e < 16; e += 4)
                if (live)
                    *reinterpret_cast<f32x4*>(p.part + ((int64_t)task.part * all_rows + g) * D + 32 * d + 2 * e + 4 * g2) =
                        none ? f32x4{0, 0, 0, 0} : f32x4{o[d][e], o[d][e + 1], o[d][e + 2], o[d][e + 3]};
        return;
    }
    // Through LDS, so that a store covers whole rows of a head instead of 16
    // bytes of 32 rows.
    constexpr int ROW = D * 2 + 16;
    unsigned char* mine_lds = lds + wave * 32 * ROW;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int e = 0; e < 16; e += 4)
            *reinterpret_cast<uint2*>(mine_lds + n32 * ROW + (32 * d + 2 * e + 4 * g2) * 2) =
                none ? make_uint2(0u, 0u)
                     : make_uint2(pack_bf16(o[d][e] * inv, o[d][e + 1] * inv), pack_bf16(o[d][e + 2] * inv, o[d][e + 3] * inv));
    lds_wait();
    const int64_t to = live ? at * p.out_row + (int64_t)mine.head * D : -1;
    constexpr int CH = T::CH;
#pragma unroll
    for (int i = 0; i < 32 * CH / 64; ++i) {
        const int row = i * (64 / CH) + lane / CH;
        const int lo = __shfl((int)to, row), up = __shfl((int)(to >> 32), row);
        const int64_t off = ((int64_t)up << 32) | (uint32_t)lo;
        const u32x4 y = *reinterpret_cast<const u32x4*>(mine_lds + row * ROW + (lane % CH) * 16);
        if (off >= 0) *reinterpret_cast<u32x4*>(p.out + off + 8 * (lane % CH)) = y;
    }
}

}  // namespace krk
