// Cache eviction by accumulated attention weight (gfx950): which slots stay,
// then the move.
//
// Selection: one workgroup per sequence and head.  The highest scores come
// from a radix select (11 + 11 + 10 bits of an order-preserving key, a
// histogram in LDS each), which reads the scores three times from L2, then two
// passes over contiguous runs of slots per wave: one counts, one writes the
// kept slots in order.  The histograms' integer atomics commute, so the result
// does not depend on their order.
//
// Move: bound by reading and writing the kept rows once.  Slots keep their
// order, so row i comes from a slot >= i.
#pragma once

#include "krk_attn_common.h"

namespace krk {

struct EvictParams {
    CacheView k, v;
    uint16_t *ko, *vo;
    int64_t ko_seq, ko_slot, ko_head, vo_seq, vo_slot, vo_head;
    const float* scores;
    int64_t sc_seq, sc_head;
    float* scores_out;
    int64_t so_seq, so_head;
    const int32_t* lens;
    int32_t* lens_out;
    int32_t* keep;
    int B, kv_heads, capacity, budget, sinks, recent;
};

// Larger scores get larger keys: NaN above +inf, -0 as +0.
__device__ __forceinline__ uint32_t score_key(float s) {
    const uint32_t u = __float_as_uint(s);
    if ((u & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
    if (u == 0x80000000u) return 0x80000000u;
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int kEvictThreads = 1024;
constexpr int kEvictWaves = kEvictThreads / 64;

__global__ void __launch_bounds__(kEvictThreads) evict_select_kernel(EvictParams p) {
    __shared__ uint32_t hist[2048];
    __shared__ uint32_t wave_sum[kEvictWaves];
    __shared__ uint32_t found[2];  // the digit, and how many are still wanted of it
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const int h = blockIdx.x, b = blockIdx.y;
    int len = p.lens[b];
    len = len < 0 ? 0 : len > p.capacity ? p.capacity : len;
    int32_t* keep = p.keep + ((int64_t)b * p.kv_heads + h) * p.budget;
    if (len <= p.budget) {
        for (int i = t; i < p.budget; i += kEvictThreads) keep[i] = i < len ? i : -1;
        return;
    }
    const float* sc = p.scores + (int64_t)b * p.sc_seq + (int64_t)h * p.sc_head;
    const int lo = p.sinks, hi = len - p.recent;  // the slots that compete
    uint32_t want = (uint32_t)(p.budget - p.sinks - p.recent);
    uint32_t prefix = 0;  // the digits found so far, from the top
    int shift = 32;
    // After the loop `prefix` is the key of the last slot that stays, and
    // `want` how many slots of exactly that key do.
    if (want > 0) {
        for (int pass = 0; pass < 3; ++pass) {
            const int bits = pass < 2 ? 11 : 10;
            const int above = shift;
            shift -= bits;
            for (int i = t; i < 2048; i += kEvictThreads) hist[i] = 0;
            __syncthreads();
            for (int i = lo + t; i < hi; i += kEvictThreads) {
                const uint32_t key = score_key(sc[i]);
                if (pass == 0 || (key >> above) == (prefix >> above))
                    atomicAdd(&hist[(key >> shift) & ((1u << bits) - 1)], 1u);
            }
            __syncthreads();
            // Thread t holds digits 2047 - 2t and the one below it: a scan over
            // threads counts from the largest digit down.
            const uint32_t a = hist[2047 - 2 * t], c = hist[2046 - 2 * t];
            uint32_t sum = a + c;
#pragma unroll
            for (int s = 1; s < 64; s <<= 1) {
                const uint32_t o = __shfl_up(sum, s);
                if (lane >= s) sum += o;
            }
            if (lane == 63) wave_sum[wave] = sum;
            __syncthreads();
            uint32_t before = sum - a - c;
            for (int w = 0; w < wave; ++w) before += wave_sum[w];
            if (before < want && want <= before + a) {
                found[0] = 2047 - 2 * t;
                found[1] = want - before;
            } else if (before + a < want && want <= before + a + c) {
                found[0] = 2046 - 2 * t;
                found[1] = want - before - a;
            }
            __syncthreads();
            prefix |= found[0] << shift;
            want = found[1];
            __syncthreads();
        }
    }
    const bool any = p.budget - p.sinks - p.recent > 0;
    // Each wave's run of slots; of the keys equal to the last one that stays,
    // those of the first slots are taken.
    const int per = ((len + kEvictWaves - 1) / kEvictWaves + 63) & ~63;
    const int w0 = wave * per < len ? wave * per : len;
    const int w1 = w0 + per < len ? w0 + per : len;
    uint32_t sure = 0, equal = 0;
    for (int i = w0; i < w1; i += 64) {
        const int s = i + lane;
        bool take = s < len && (s < lo || s >= hi), eq = false;
        if (any && s >= lo && s < hi) {
            const uint32_t key = score_key(sc[s]);
            take = key > prefix;
            eq = key == prefix;
        }
        sure += __popcll(__ballot(take));
        equal += __popcll(__ballot(eq));
    }
    if (lane == 0) {
        hist[wave] = sure;
        hist[64 + wave] = equal;
    }
    __syncthreads();
    uint32_t at = 0, eq_before = 0;
    for (int w = 0; w < wave; ++w) {
        at += hist[w];
        eq_before += hist[64 + w];
    }
    at += eq_before < want ? eq_before : want;
    const uint64_t below = (1ull << lane) - 1;
    for (int i = w0; i < w1; i += 64) {
        const int s = i + lane;
        bool take = s < len && (s < lo || s >= hi), eq = false;
        if (any && s >= lo && s < hi) {
            const uint32_t key = score_key(sc[s]);
            take = key > prefix;
            eq = key == prefix;
        }
        const uint64_t eqs = __ballot(eq);
        if (eq) take = eq_before + __popcll(eqs & below) < want;
        eq_before += __popcll(eqs);
        const uint64_t takes = __ballot(take);
        if (take) keep[at + __popcll(takes & below)] = s;
        at += __popcll(takes);
    }
}

// Kept rows to another cache: D / 8 lanes a row, K and V.
template <int D>
__global__ void __launch_bounds__(256) evict_copy_kernel(EvictParams p) {
    constexpr int L = D / 8;
    const int h = blockIdx.y, b = blockIdx.z;
    const int c = threadIdx.x % L;
    int len = p.lens[b];
    len = len < 0 ? 0 : len > p.capacity ? p.capacity : len;
    const int n = len < p.budget ? len : p.budget;
    const int i = blockIdx.x * (256 / L) + threadIdx.x / L;
    // lens_out may be lens: the minimum is the same of either.
    if (h == 0 && blockIdx.x == 0 && threadIdx.x == 0) p.lens_out[b] = n;
    if (i >= n) return;
    const int s = p.keep[((int64_t)b * p.kv_heads + h) * p.budget + i];
    const u32x4 k = load_stream16(p.k.p + (int64_t)b * p.k.seq + (int64_t)s * p.k.slot + (int64_t)h * p.k.head + 8 * c);
    const u32x4 v = load_stream16(p.v.p + (int64_t)b * p.v.seq + (int64_t)s * p.v.slot + (int64_t)h * p.v.head + 8 * c);
    *reinterpret_cast<u32x4*>(p.ko + (int64_t)b * p.ko_seq + (int64_t)i * p.ko_slot + (int64_t)h * p.ko_head + 8 * c) = k;
    *reinterpret_cast<u32x4*>(p.vo + (int64_t)b * p.vo_seq + (int64_t)i * p.vo_slot + (int64_t)h * p.vo_head + 8 * c) = v;
    if (c == 0)
        p.scores_out[(int64_t)b * p.so_seq + (int64_t)h * p.so_head + i] =
            p.scores[(int64_t)b * p.sc_seq + (int64_t)h * p.sc_head + s];
}

// The same within one cache.  A workgroup owns a slice of every row (32
// elements of K or of V, or the scores) and goes through the rows in order, a
// batch at a time: all of a batch's loads have returned before its first
// store.  Row i's source is a slot >= i and sources ascend, so a batch's
// stores, to rows below the next batch's first, never touch a later source.
template <int D>
__global__ void __launch_bounds__(256) evict_move_kernel(EvictParams p) {
    constexpr int U = 8;  // rows of a thread in a batch
    const int h = blockIdx.y, b = blockIdx.z;
    const int slice = blockIdx.x;
    const int n = p.budget;
    // lens_out may be lens, so only the thread that writes it reads it; the
    // rest goes by the last kept slot, which is -1 (fewer slots than the
    // budget) or n - 1 (the slots 0 .. n - 1) where nothing moves.
    if (h == 0 && slice == 0 && threadIdx.x == 0) {
        const int len = p.lens[b];
        p.lens_out[b] = len < 0 ? 0 : len < n ? len : n;
    }
    const int32_t* keep = p.keep + ((int64_t)b * p.kv_heads + h) * p.budget;
    if (keep[n - 1] < n) return;
    if (slice == 2 * (D / 32)) {
        float* to = p.scores_out + (int64_t)b * p.so_seq + (int64_t)h * p.so_head;
        for (int i0 = 0; i0 < n; i0 += 256 * U) {
            float x[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int i = i0 + 256 * u + threadIdx.x;
                x[u] = to[keep[i < n ? i : n - 1]];
            }
            drain_loads();
            __syncthreads();
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int i = i0 + 256 * u + threadIdx.x;
                if (i < n) to[i] = x[u];
            }
        }
        return;
    }
    const bool is_v = slice >= D / 32;
    const int64_t slot = is_v ? p.vo_slot : p.ko_slot;
    uint16_t* to = (is_v ? p.vo + (int64_t)b * p.vo_seq + (int64_t)h * p.vo_head
                         : p.ko + (int64_t)b * p.ko_seq + (int64_t)h * p.ko_head) +
                   32 * (is_v ? slice - D / 32 : slice) + 8 * (threadIdx.x & 3);
    const int j = threadIdx.x >> 2;
    for (int i0 = 0; i0 < n; i0 += 64 * U) {
        u32x4 x[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + 64 * u + j;
            x[u] = load_cached16(to + (int64_t)keep[i < n ? i : n - 1] * slot);
        }
        drain_loads();
        __syncthreads();
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + 64 * u + j;
            if (i < n) *reinterpret_cast<u32x4*>(to + (int64_t)i * slot) = x[u];
        }
    }
}

}  // namespace krk
