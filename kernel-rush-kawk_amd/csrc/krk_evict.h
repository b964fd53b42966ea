// Cache eviction by accumulated attention weight (gfx950): which slots stay,
// then the move.
//
// Selection: one workgroup per sequence and head; each wave has a run of slots
// next to each other.  The highest scores come from a radix select (11 + 11 + 10
// bits of an order-preserving key, histograms in LDS), then two passes, one to
// count, one to write the kept slots in order.  Up to 36864 slots the keys stay
// in registers and the scores are read once; a longer cache reads them for each
// of the five passes.  The histograms' integer atomics commute, so the result
// does not depend on their order.  Bound by latency, the LDS atomics and the
// vector pipe of the B * kv_heads CUs that have a workgroup.
//
// Move: bound by reading and writing the kept rows once (a launch of its own:
// copied by the selecting workgroup, 512 rows of 8 heads took 6 us instead of 3).  Slots keep their
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

// PER: keys a lane holds, for caches of up to 1024 * PER slots (code and time
// grow with it); 0: none, any length.
template <int PER>
__global__ void __launch_bounds__(kEvictThreads) evict_select_kernel(EvictParams p) {
    // Few keys: one histogram.  Many: each quarter of the waves has its own, as
    // heavy-tailed scores crowd into some 80 of the first digits.
    constexpr int COPIES = PER > 0 && PER <= 4 ? 1 : 4;
    __shared__ uint32_t hist[COPIES][2048];
    __shared__ uint32_t wave_sum[kEvictWaves];
    __shared__ uint32_t counts[2][kEvictWaves];
    __shared__ uint32_t found[2];  // the digit, and how many are still wanted of it
    const int t = threadIdx.x, lane = t & 63;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int h = blockIdx.x, b = blockIdx.y;
    int len = p.lens[b];
    len = len < 0 ? 0 : len > p.capacity ? p.capacity : len;
    int32_t* keep = p.keep + ((int64_t)b * p.kv_heads + h) * p.budget;
    if (len <= p.budget) {
        for (int i = t; i < p.budget; i += kEvictThreads) keep[i] = i < len ? i : -1;
        return;
    }
    // The first and the last slots stay; those between them compete.
    const int lo = p.sinks, hi = len - p.recent;
    const int chosen = p.budget - p.sinks - p.recent;
    for (int i = t; i < p.sinks; i += kEvictThreads) keep[i] = i;
    for (int i = t; i < p.recent; i += kEvictThreads) keep[p.budget - p.recent + i] = hi + i;
    if (chosen == 0) return;

    const float* sc = p.scores + (int64_t)b * p.sc_seq + (int64_t)h * p.sc_head;
    // This wave's run: slots w0 + 64 i + lane.  Keys of competing slots are at
    // least 0x007fffff (-infinity's); 0 stands for a slot that does not compete.
    const int rounds = (hi - lo + kEvictThreads - 1) / kEvictThreads;
    const int w0 = lo + wave * rounds * 64 + lane;
    auto key_of = [&](int s, float v) { return s < hi ? score_key(v) : 0u; };
    uint32_t held[PER > 0 ? PER : 1];
    if constexpr (PER > 0) {
        float v[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int s = w0 + 64 * i;
            v[i] = i < rounds ? sc[s < hi ? s : hi - 1] : 0.0f;
        }
#pragma unroll
        for (int i = 0; i < PER; ++i) held[i] = i < rounds ? key_of(w0 + 64 * i, v[i]) : 0u;
    }
    // fn(slot, key) for this lane's slots, in order.
    auto each = [&](auto fn) {
        if constexpr (PER > 0) {
#pragma unroll
            for (int i = 0; i < PER; ++i)
                if (i < rounds) fn(w0 + 64 * i, held[i]);
        } else {
            for (int i = 0; i < rounds; ++i) {
                const int s = w0 + 64 * i;
                fn(s, key_of(s, sc[s < hi ? s : hi - 1]));
            }
        }
    };
    // `last` becomes the key of the last slot that stays, `want` how many slots
    // of exactly that key do.
    uint32_t want = (uint32_t)chosen, last = 0;
#pragma unroll
    for (int pass = 0; pass < 3; ++pass) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
        const uint32_t digits = pass < 2 ? 2047 : 1023;
        for (int i = t; i < COPIES * 2048; i += kEvictThreads) (&hist[0][0])[i] = 0;
        __syncthreads();
        uint32_t* mine = hist[wave % COPIES];
        each([&](int, uint32_t key) {
            if (pass == 0 ? key != 0 : (key ^ last) >> (pass == 1 ? 21 : 10) == 0) atomicAdd(&mine[(key >> shift) & digits], 1u);
        });
        __syncthreads();
        // Thread t holds digits 2047 - 2t and the one below it: a scan over
        // threads counts from the largest digit down.
        uint32_t a = 0, c = 0;
#pragma unroll
        for (int k = 0; k < COPIES; ++k) {
            a += hist[k][2047 - 2 * t];
            c += hist[k][2046 - 2 * t];
        }
        uint32_t sum = a + c;
#pragma unroll
        for (int s = 1; s < 64; s <<= 1) {
            const uint32_t o = __shfl_up(sum, s);
            if (lane >= s) sum += o;
        }
        if (lane == 63) wave_sum[wave] = sum;
        __syncthreads();
        uint32_t before = sum - a - c;
#pragma unroll
        for (int w = 0; w < kEvictWaves; ++w) before += w < wave ? wave_sum[w] : 0;
        if (before < want && want <= before + a) {
            found[0] = 2047 - 2 * t;
            found[1] = want - before;
        } else if (before + a < want && want <= before + a + c) {
            found[0] = 2046 - 2 * t;
            found[1] = want - before - a;
        }
        __syncthreads();
        last |= found[0] << shift;
        want = found[1];
    }
    // Of the keys equal to the last one that stays, those of the first slots
    // are taken.
    uint32_t above = 0, equal = 0;
    each([&](int, uint32_t key) {
        above += __popcll(__ballot(key > last));
        equal += __popcll(__ballot(key == last));
    });
    if (lane == 0) {
        counts[0][wave] = above;
        counts[1][wave] = equal;
    }
    __syncthreads();
    uint32_t at = p.sinks, eq_before = 0;
#pragma unroll
    for (int w = 0; w < kEvictWaves; ++w) {
        at += w < wave ? counts[0][w] : 0;
        eq_before += w < wave ? counts[1][w] : 0;
    }
    at += eq_before < want ? eq_before : want;
    const uint64_t below = (1ull << lane) - 1;
    each([&](int s, uint32_t key) {
        const uint64_t eqs = __ballot(key == last);
        const bool take = key > last || (key == last && eq_before + __popcll(eqs & below) < want);
        eq_before += __popcll(eqs);
        const uint64_t takes = __ballot(take);
        if (take) keep[at + __popcll(takes & below)] = s;
        at += __popcll(takes);
    });
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
