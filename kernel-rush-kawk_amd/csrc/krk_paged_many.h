// Attention over pages for requests of many rows (chunks of prompts): 128 rows of a
// head a workgroup, K and V through LDS.
//
// Bound by the matrix pipe, LDS and the vector pipe alike (2048 rows over 16384 keys
// 490 to 520 us, 990 to 1050 TFLOP/s; the matrix pipe is busy half of the time), as the contiguous caches'
// tile kernel is, whose fragments and orders of issue these are: four waves, each with 32
// rows of its own, all reading the same 64-key steps from LDS; S^T = K Q^T and O^T = V^T
// P^T on v_mfma_f32_32x32x16_bf16, weights staying in their lane; rings of three steps of
// K and two of V, filled by DMA, one barrier a step; two workgroups a CU.  Weights are
// rounded to one bf16 for the product with V (their sum is not).  A choice: with two parts
// the products take half as many matrix instructions again (the chunk above 493 -> 658 us,
// two chunks beside 48 decoding requests 278 -> 315, a prompt of 4096 rows 147 -> 190), and
// the relative error against 64 bits, of which bf16 results alone make 0.00164 to 0.00167,
// is 0.00170 and 0.00183 with one.
//
// Pages.  A DMA copies 1 KB, 4 or 8 keys of a head, which lie in one page.  Its page
// number is the same for the whole wave: a scalar load, issued behind the DMAs of the
// step before it and there before that step's products.
#pragma once

#include "krk_attn_tile.h"
#include "krk_paged_attn.h"

namespace krk {

static_assert(kTileThreads == kPagedThreads, "one workgroup size");

// Scalar registers are what this kernel is short of: with too many of them alive the
// compiler gives up the order of issue that the products are written in.  What follows
// from a value that went through here is worked out where it is used.
template <typename I>
__device__ __forceinline__ I here(I x) {
    asm volatile("" : "+s"(x));
    return x;
}

// What a job's streams of K and V have in common.
struct PageWalk {
    typedef __attribute__((address_space(4))) const int32_t const_i32;
    const const_i32* table;  // of the request, through the scalar cache
    unsigned last_page;      // of the pool
    int shift, end, t1;
    __device__ __forceinline__ PageWalk(const PagedParams& p, const Job& j, int end_, int t1_)
        : table(reinterpret_cast<const const_i32*>(reinterpret_cast<uint64_t>(p.table + (int64_t)j.b * p.table_row))),
          last_page((unsigned)p.pages - 1), shift(p.shift), end(end_), t1(t1_) {}
    __device__ __forceinline__ int in_page(int key) const { return key & ((1 << shift) - 1); }
};

// Fetches a job's 64-key steps of K or V in order into a ring in LDS, this wave's share
// of them: keys RPD * (wave + 4 * i) .. of a step, i = 0 .. DMAS - 1.  Behind the range's
// last step that step is fetched again, into slots that nothing reads any more: every
// step then has the same number of DMAs in flight.
template <int D, bool V>
struct PageStream {
    using T = TileKernel<D>;
    static constexpr int DMAS = T::DMAS, RPD = T::ROWS_PER_DMA, APART = RPD * kTileWaves;
    uint64_t at;        // of the wave's first key in page 0, for a step that begins a page
    uint32_t page, slot;  // bytes
    uint32_t to, lane_off;
    int t;
    unsigned id[DMAS];  // page numbers of step t (of pages of 64 slots and more: id[0])

    // The first of the keys that DMA i of a step fetches; behind the end the last keys again.
    __device__ __forceinline__ int first_key(const PageWalk& w, int kb, int i, int wave) const {
        const int g = kb + RPD * wave + APART * i, last = (w.end - 1) & ~(RPD - 1);
        return g < last ? g : last;
    }
    __device__ __forceinline__ void numbers(PageWalk w, const KeySpan<kTileStep>& span, int wave) {
        w.shift = here(w.shift);
        const int kb = span.key(t);
        if (kb + kTileStep <= w.end) {
            const auto* from = w.table + (kb >> w.shift);
            if (w.shift >= 6) {
                id[0] = (unsigned)from[0];
            } else {
#pragma unroll
                for (int i = 0; i < DMAS; ++i) id[i] = (unsigned)from[(RPD * wave + APART * i) >> w.shift];
            }
        } else {
#pragma unroll
            for (int i = 0; i < DMAS; ++i) id[i] = (unsigned)w.table[first_key(w, kb, i, wave) >> w.shift];
        }
    }
    __device__ __forceinline__ PageStream(const PagedParams& p, const PageView& v, const Job& j, const PageWalk& w,
                                          const KeySpan<kTileStep>& span, int t0, int wave, int lane) {
        page = (uint32_t)v.page * 2;
        slot = (uint32_t)v.slot * 2;
        at = reinterpret_cast<uint64_t>(v.p + (int64_t)j.h * v.head) + (uint64_t)w.in_page(RPD * wave) * slot;
        t = t0;
        to = 0;
        const int l = lane / T::CH;
        // The permutation of a row's chunks goes by its low bits, which are the lane's.
        const int row = RPD * wave + l;
        lane_off = (uint32_t)l * slot + 16 * ((lane % T::CH) ^ (V ? T::v_swizzle(row) : T::k_swizzle(row)));
        numbers(w, span, wave);
    }
    __device__ __forceinline__ uint64_t page_at(const PageWalk& w, int i) const {
        return (uint64_t)(id[i] < w.last_page ? id[i] : w.last_page) * page;
    }
    template <int RING>
    __device__ __forceinline__ void fetch(PageWalk w, const KeySpan<kTileStep>& span, uint32_t ring, int wave, int lane) {
        w.shift = here(w.shift);
        const uint32_t slot = here(this->slot);
        const uint32_t dst = ring + to + wave * 1024;
        const int kb = span.key(t);
        if (kb + kTileStep <= w.end) {
            if (w.shift >= 6) {  // the step lies in one page
                const uint64_t from = at + page_at(w, 0) + (uint64_t)w.in_page(kb) * slot;
#pragma unroll
                for (int i = 0; i < DMAS; ++i) dma(from + i * APART * slot, lane_off, dst + kTileWaves * i * 1024);
            } else {  // it begins one
#pragma unroll
                for (int i = 0; i < DMAS; ++i)
                    dma(at + page_at(w, i) + (uint32_t)w.in_page(APART * i) * slot, lane_off, dst + kTileWaves * i * 1024);
            }
        } else {  // keys from the end on: the last one again
#pragma unroll
            for (int i = 0; i < DMAS; ++i) {
                const int g = first_key(w, kb, i, wave);
                const int over = g + lane / T::CH - (w.end - 1);
                dma(at + page_at(w, i) + ((int64_t)w.in_page(g) - w.in_page(RPD * wave)) * (int64_t)slot,
                    lane_off - (over > 0 ? over : 0) * slot, dst + kTileWaves * i * 1024);
            }
        }
        t = t < w.t1 - 1 ? t + 1 : t;
        numbers(w, span, wave);
        to += T::STEP_BYTES;
        to = to == (uint32_t)RING * T::STEP_BYTES ? 0u : to;
    }
    // One 1 KB DMA into LDS, lane l's 16 bytes from base + off to dst + 16 l.  In
    // assembly, because around the builtin the compiler waits for every DMA in flight
    // before a transposed LDS read; the waits here are vm_wait_stages' alone.
    static __device__ __forceinline__ void dma(uint64_t base, uint32_t off, uint32_t dst) {
        asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" : : "v"(off), "s"(base), "s"(dst) : "memory", "m0");
    }
};

// A job in the lanes of a vector register, and the kernel's arguments read where they
// are used: neither takes scalar registers while the products run.
struct ParkedJob {
    int v = 0;
    __device__ __forceinline__ explicit ParkedJob(const Job& j) {
        put(0, j.b), put(1, j.h), put(2, j.tile), put(3, j.row0), put(4, j.part), put(5, j.parts), put(6, j.slot);
        put(7, j.req.row), put(8, j.req.n), put(9, j.req.len);
    }
    __device__ __forceinline__ Job job() const {
        Job j;
        j.b = get(0), j.h = get(1), j.tile = get(2), j.row0 = get(3), j.part = get(4), j.parts = get(5), j.slot = get(6);
        j.req = {get(7), get(8), get(9)};
        return j;
    }
    __device__ __forceinline__ void put(unsigned i, int x) { v = (threadIdx.x & 63) == i ? x : v; }
    __device__ __forceinline__ int get(int i) const { return __builtin_amdgcn_readlane(v, i); }
};
__device__ __forceinline__ PagedParams kernel_params() {
    typedef __attribute__((address_space(4))) const PagedParams arguments;
    auto at = reinterpret_cast<uint64_t>(__builtin_amdgcn_kernarg_segment_ptr());
    asm("" : "+s"(at));  // not what an earlier call returned
    PagedParams p;
    __builtin_memcpy(&p, reinterpret_cast<arguments*>(at), sizeof p);
    return p;
}

template <int D>
__device__ __forceinline__ void many_rows(const PagedParams& p, const ParkedJob& parked, unsigned char* lds) {
    const Job early = parked.job();
    using T = TileKernel<D>;
    constexpr int KS = T::KS, DT = T::DT;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n32 = lane & 31, g2 = lane >> 5;
    const int rows = early.req.n * p.G;
    const int pos0 = early.req.len - early.req.n;
    auto clamped = [&](int row) { return row < rows ? row : rows - 1; };
    // Positions of the first and last row of the tile and of this wave's rows.
    const int wave0 = early.row0 + 32 * wave;
    auto position = [&](int row) { return pos0 + __builtin_amdgcn_readfirstlane(quotient(clamped(row), p.G, p.inv_G)); };
    const int wave_first = position(wave0), wave_last = position(wave0 + 31);
    const int tile_first = position(early.row0), tile_last = position(early.row0 + kTileRows - 1);
    const KeySpan<kTileStep> span(p, early.req.len, tile_first, tile_last);
    const int t0 = (int)((int64_t)span.steps * early.part / early.parts), t1 = (int)((int64_t)span.steps * (early.part + 1) / early.parts);
    const int my_row = wave0 + n32;
    const TileRow mine(p, early, clamped(my_row));
    const int64_t at = early.req.row + mine.r;

    bf16x8 qf[KS];
    {
        const uint16_t* qr = p.q + at * p.q_row + (int64_t)mine.head * D + 8 * g2;
#pragma unroll
        for (int s = 0; s < KS; ++s) qf[s] = __builtin_bit_cast(bf16x8, load_cached16(qr + 16 * s));
    }
    unsigned char* kring = lds;
    unsigned char* vring = lds + kTileKRing * T::STEP_BYTES;
    const uint32_t lds_base = (uint32_t)(uintptr_t)(lds_s16x4*)lds;
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
    // The steps behind the sinks that all rows from position first to last see whole.
    struct Steps {
        int from, n;
        __device__ __forceinline__ bool has(int t) const { return (unsigned)(t - from) < (unsigned)n; }
    };
    auto whole_steps = [&](int first, int last) {
        Steps x;
        const int end = first + 1 < span.end ? first + 1 : span.end;
        const int lo = p.window && last >= p.window ? last - p.window + 1 - span.from : 0;
        x.from = span.sink_steps + (lo > 0 ? (lo + kTileStep - 1) / kTileStep : 0);
        const int n = span.sink_steps + (end > span.from ? (end - span.from) / kTileStep : 0) - x.from;
        x.n = n > 0 ? n : 0;
        return x;
    };
    const Steps mine_whole = whole_steps(wave_first, wave_last), all_whole = whole_steps(tile_first, tile_last);
    // No weight for what the row does not see.
    const int hi = mine.pos < span.end - 1 ? mine.pos : span.end - 1;
    auto hide = [&](int t) {
        const int from = span.key(t) + 4 * g2;
        const int top = hi - from, low = mine.lo - from, sink = p.sinks - from;
#pragma unroll
        for (int e = 0; e < 32; ++e) {
            const int k = tile32_key(e >> 4, e & 15, 0);
            const bool ok = (k <= top) & ((k >= low) | (k < sink));
            s[e >> 4][e & 15] = ok ? s[e >> 4][e & 15] : kNegInf;
        }
    };
    auto highest = [&](int kt) {
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = fmaxf(fmaxf(s[kt][3 * e], s[kt][3 * e + 1]), s[kt][3 * e + 2]);
        v[0] = fmaxf(fmaxf(v[0], s[kt][12]), s[kt][13]);
        v[1] = fmaxf(fmaxf(v[1], s[kt][14]), s[kt][15]);
        return fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3]));
    };
    // The running maximum moves only when a row's grows by more than 2^8 (weights
    // stay below 2^8 then, which costs no precision): O is rescaled a few times a row.
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
    // difference first: s * c - m * c in one fma would be off where scores are large.
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
    // A step that some row of the workgroup does not see whole may hold infinities or
    // NaNs that only some rows see.  Each wave then zeroes those among the values it
    // fetched; they are added behind the last step.
    bool any_odd = false;
    auto tame = [&](uint32_t slot) {
        unsigned char* x0 = vring + slot;
#pragma unroll 1
        for (int i = 0; i < T::DMAS; ++i) {
            u32x4* x = reinterpret_cast<u32x4*>(x0 + (wave + kTileWaves * i) * 1024 + lane * 16);
            const u32x4 v = *x;
            if (__any(odd_bf16x8(__builtin_bit_cast(bf16x8, v)))) {
                *x = finite_bf16x8(v);
                any_odd = true;
            }
        }
    };

    if (t0 < t1) {
        const PageWalk walk(p, early, span.end, t1);
        PageStream<D, false> k_next(p, p.k, early, walk, span, t0, wave, lane);
        PageStream<D, true> v_next(p, p.v, early, walk, span, t0, wave, lane);
        auto fetch_k = [&]() { k_next.template fetch<kTileKRing>(walk, span, lds_base, wave, lane); };
        auto fetch_v = [&]() { v_next.template fetch<kTileVRing>(walk, span, lds_base + kTileKRing * T::STEP_BYTES, wave, lane); };
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
            // K of step t + 1 and V of step t have landed (K of step t + 2, fetched
            // behind them, may not have), and every wave is through with the slots that
            // the next DMAs fill.
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
            // The page numbers are here: with scalar loads under way every read of LDS
            // below would have to wait for all of them.
            lds_wait();
            // The other workgroup's wave of this SIMD leaves the matrix pipe to the
            // one that is at its products.
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
        for (int i = 0; i < kTileWaves; ++i) any_odd = any_odd || flags[i];
        if (any_odd) {  // the infinities and NaNs left out above: rare, so key by key
            const PagedParams p = kernel_params();
            const PagedRun vr(p, p.v, parked.job(), span.end);
#pragma unroll 1
            for (int t = t0; t < t1; ++t) {
                const int kb = span.key(t);
                if (all_whole.has(t)) continue;
#pragma unroll 1
                for (int key = kb; key < kb + kTileStep && key < span.end; ++key) {
                    const bool ok = row_sees(mine.pos, mine.lo, p.sinks, key);
                    const uint16_t* x0 = vr.row(key, vr.page_of(key)) + 4 * g2;
#pragma unroll
                    for (int d = 0; d < DT; ++d)
#pragma unroll
                        for (int e = 0; e < 16; e += 4) {
                            const uint2 x = *reinterpret_cast<const uint2*>(x0 + 32 * d + 2 * e);
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
    const PagedParams late = kernel_params();
    const Job job = parked.job();
    const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(l), __float_as_uint(l), false, false);
    const float L = __uint_as_float(both[0]) + __uint_as_float(both[1]);
    const bool live = my_row < rows;
    const bool none = L == 0.0f;
    if (job.parts > 1) {  // for a workgroup of this launch, maybe on another XCD
        const int64_t g = job.slot + (int64_t)job.part * kTileRows + 32 * wave + n32;
        if (!live) return;
        if (g2 == 0) put_agent(late.ml + g, make_float2(m, L));
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int e = 0; e < 16; e += 4)
                put_agent(late.part + g * D + 32 * d + 2 * e + 4 * g2, f32x4{o[d][e], o[d][e + 1], o[d][e + 2], o[d][e + 3]});
        return;
    }
    const float inv = none ? 0.0f : 1.0f / L;
    if (live && g2 == 0 && late.lse) late.lse[at * late.heads + mine.head] = none ? kNegInf : m * late.scale + logf(L);
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
    const int64_t to = live ? at * late.out_row + (int64_t)mine.head * D : -1;
    constexpr int CH = T::CH;
#pragma unroll
    for (int i = 0; i < 32 * CH / 64; ++i) {
        const int row = i * (64 / CH) + lane / CH;
        const int low = __shfl((int)to, row), up = __shfl((int)(to >> 32), row);
        const int64_t off = ((int64_t)up << 32) | (uint32_t)low;
        const u32x4 y = *reinterpret_cast<const u32x4*>(mine_lds + row * ROW + (lane % CH) * 16);
        if (off >= 0) *reinterpret_cast<u32x4*>(late.out + off + 8 * (lane % CH)) = y;
    }
}

// MANY: requests of many rows too (else no request of the call can have as many).
template <int D, bool MANY>
__global__ void __launch_bounds__(kPagedThreads, 2) paged_attn_kernel(PagedParams p) {
    extern __shared__ __align__(16) unsigned char lds[];
    const Job first = p.planned ? planned_job(p, (int)blockIdx.x) : job_of(p, (int)blockIdx.x);
    if (first.tile < 0) return;
    const ParkedJob parked(first);
    // Each kind of job with arguments of its own: what they have in common would else
    // be worked out for all of them ahead of the branch, and stay in registers.
    if (MANY && first.tile == kTileRows) {
        many_rows<D>(kernel_params(), parked, lds);
    } else if (first.tile == 16) {
        few_rows<D, 1>(kernel_params(), parked.job(), lds);
    } else {
        few_rows<D, 2>(kernel_params(), parked.job(), lds);
    }
    const Job job = parked.job();
    if (job.parts == 1) return;
    join_ranges<D>(kernel_params(), job, lds);
}

}  // namespace krk
