// Cache attention for few rows (decode, draft trees, batches over a shared
// prefix): key ranges split over workgroups, and what joins them.
//
// Bound by reading K and V once (4 * D bytes a key and key/value head): with
// at most 64 rows of a head, the products are at most 64 flops a byte.
//
// Work split.  A workgroup takes TR = 16 * MT rows of one key/value head and one
// range of the keys those rows see, its four waves 32 keys at a time in turn
// (16 KB of K and V at head size 128, adjacent waves adjacent keys).  Waves
// keep their own running maximum, sum and O and meet in LDS once, at the end.
// K's registers are reloaded for the next 32 keys as soon as the scores are
// taken, V's as soon as the products are, so a wave has loads in flight all
// the time and a CU holds 2-3 such workgroups at MT = 1.  Short calls are
// latency: of 25000 cycles of a workgroup with 3 steps a wave (draft trees), the
// first loads (addresses of cold pages) take 7000, a step 2700, the merge 3000.
//
// The rows of the shared prefix are those of all sequences together, so it is
// read once per TR rows of the batch instead of once per sequence.
//
// Weights go into the second product as two bf16 parts (p = hi + lo, 16 bits of
// mantissa): the matrix pipe has the time, and the sums then carry fp32's
// weights to within 2^-17.
#pragma once

#include "krk_attn_common.h"
#include "krk_epilogue.h"

namespace krk {

constexpr int kSplitWaves = 4;
constexpr int kSplitThreads = 64 * kSplitWaves;

template <int D, int MT>
constexpr size_t split_lds_bytes() {
    return (size_t)kSplitWaves * 16 * MT * ((D + 4) * sizeof(float) + sizeof(float2));
}

// Four outputs of a row over some of its key ranges, and their maximum and sum.
struct Joined {
    float M = kNegInf, L = 0.0f;
    f32x4 o = {0, 0, 0, 0};
    __device__ __forceinline__ void add(const AttnParams& p, float m, float l, const f32x4& x) {
        const float mn = fmaxf(M, m);
        const float ms = mn == kNegInf ? 0.0f : mn;
        const float f0 = exp2_raw((M - ms) * p.c), f1 = exp2_raw((m - ms) * p.c);
        L = L * f0 + f1 * l;
        o = o * f0 + f1 * x;
        M = mn;
    }
};

// Joins key ranges from, from + step, ... of row `row` (of all rows); kJoin
// loads are in flight at a time.  AGENT: they were written by this launch, so
// each is a round trip beyond this XCD's L2.
constexpr int kJoin = 8;
template <int D, bool AGENT>
__device__ __forceinline__ Joined join_ranges(const AttnParams& p, int64_t row, int d, int from, int step) {
    const int64_t all_rows = (int64_t)p.B * p.kv_heads * p.RG;
    const int n = p.splits + p.prefix_splits;
    Joined y;
    for (int s0 = from; s0 < n; s0 += kJoin * step) {
        float2 ml[kJoin];
        f32x4 x[kJoin];
#pragma unroll
        for (int s = 0; s < kJoin; ++s) {
            const int at = s0 + s * step;
            const int64_t g = (at < n ? at : s0) * all_rows + row;
            ml[s] = AGENT ? get_agent(p.ml + g) : p.ml[g];
            x[s] = AGENT ? get_agent(p.part + g * D + d) : *reinterpret_cast<const f32x4*>(p.part + g * D + d);
        }
#pragma unroll
        for (int s = 0; s < kJoin; ++s)
            if (s0 + s * step < n) y.add(p, ml[s].x, ml[s].y, x[s]);
    }
    return y;
}

// JOIN: the prefix's ranges were taken by an earlier launch and this workgroup's
// is all of the own cache; it joins them.
template <int D, int MT, bool JOIN>
__device__ __forceinline__ void split_task(const AttnParams& p, const Task& task, unsigned char* lds) {
    constexpr int TR = 16 * MT;
    constexpr int KS = D / 32;
    constexpr int VD = D / 16;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n16 = lane & 15, q4 = lane >> 4;

    const int limit = task.limit;

    // This lane's rows, and their q.  Loads first: what the rows see is worked
    // out while the first keys are on their way.
    TaskRow rows[MT];
    RowSight sight[MT];
    u32x4 qf[MT][KS];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        rows[i] = task_row(p, task, task.row0 + 16 * i + n16);
        const uint16_t* qr = p.q + ((int64_t)rows[i].b * p.R + rows[i].r) * p.q_row + (int64_t)rows[i].head * D + 8 * q4;
#pragma unroll
        for (int s = 0; s < KS; ++s) qf[i][s] = load_cached16(qr + 32 * s);
    }
    Reach reach;
    auto see = [&]() {
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            sight[i] = rows[i].sight(p);
            reach.add(sight[i], task.row0 + 16 * i + n16 < task.rows);
        }
        reach.join_lanes();
    };
    const bool late = task.shared && p.window;
    if (late) see();
    const KeySteps<32> steps(p, task, late ? reach : reach_at_most(p, task));
    KeyFrag<D> kf;
    ValueFrag<D> vf;
    const int t1 = steps.t1;
    int t = steps.t0 + wave;
    if (t < t1) {
        kf.load(task.k, task.k_slot, steps.key(t), limit, lane);
        vf.load(task.v, task.v_slot, steps.key(t), limit, lane);
    }
    if (!late) see();

    // Of the merge at the end: this thread's outputs of rows i * ROWS + ...
    constexpr int PER_ROW = D / 4, ROWS = kSplitThreads / PER_ROW;
    const int d = 4 * (threadIdx.x % PER_ROW);
    const int64_t all_rows = (int64_t)p.B * p.kv_heads * p.RG;
    Joined shared[JOIN ? TR / ROWS : 1];
    if constexpr (JOIN) {  // under the first keys' loads
#pragma unroll
        for (int i = 0; i < TR / ROWS; ++i) {
            const int row = task.row0 + i * ROWS + threadIdx.x / PER_ROW;
            if (row < task.rows)
                shared[i] = join_ranges<D, false>(p, ((int64_t)task.b0 * p.kv_heads + task.h) * p.RG + row, d, p.splits, 1);
        }
    }

    f32x4 acc[MT][VD];
    float m[MT], l[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        m[i] = kNegInf;
        l[i] = 0.0f;
#pragma unroll
        for (int j = 0; j < VD; ++j) acc[i][j] = f32x4{0, 0, 0, 0};
    }

    // An infinity or a NaN times a zero weight would reach rows that do not see
    // it: the products run on zeros in their place, and the rows that see them
    // get them behind the last step.
    bool any_odd = false;
    for (; t < t1; t += kSplitWaves) {
        const int kb = steps.key(t);
        const int next = t + kSplitWaves;
        f32x4 s[MT][2];
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                s[i][u] = f32x4{0, 0, 0, 0};
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) s[i][u] = mfma16(kf.f[u][ks], qf[i][ks], s[i][u]);
            }
        if (next < t1) kf.load(task.k, task.k_slot, steps.key(next), limit, lane);

        // What each row does not see gets no weight.  Steps that every row
        // sees whole skip this.
        const int pos = task.seg + kb;
        const bool whole = kb + 32 <= limit && pos + 31 <= reach.hi_min && (pos >= reach.lo_max || pos + 32 <= p.sinks);
        if (!whole) {
#pragma unroll
            for (int i = 0; i < MT; ++i) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int key = kb + 8 * q4 + e;
                    const bool ok = key < limit && sees(sight[i], task.seg + key, p.sinks);
                    s[i][e >> 2][e & 3] = ok ? s[i][e >> 2][e & 3] : kNegInf;
                }
            }
        }
        if (p.raw) {
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                const int row = task.row0 + 16 * i + n16;
                if (row < task.rows) {
                    float* to = p.raw + (((int64_t)task.b0 * p.kv_heads + task.h) * p.RG + row) * p.raw_row + kb + 8 * q4;
                    *reinterpret_cast<f32x4*>(to) = s[i][0];
                    *reinterpret_cast<f32x4*>(to + 4) = s[i][1];
                }
            }
        }
        bf16x8 hi[MT], lo[MT];
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            float mx = s[i][0][0];
#pragma unroll
            for (int e = 1; e < 8; ++e) mx = fmaxf(mx, s[i][e >> 2][e & 3]);
            const float mn = fmaxf(m[i], row_max(mx));
            const float ms = mn == kNegInf ? 0.0f : mn;  // nothing seen yet: weights exp2(-inf) = 0
            const float alpha = exp2_raw((m[i] - ms) * p.c);
            m[i] = mn;
            float w[8], sum = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                w[e] = exp2_raw((s[i][e >> 2][e & 3] - ms) * p.c);
                sum += w[e];
            }
            l[i] = l[i] * alpha + sum;
            u32x4 ph, pl;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                ph[e] = pack_bf16(w[2 * e], w[2 * e + 1]);
                const uint32_t x = ph[e];
                pl[e] = pack_bf16(w[2 * e] - bf16_to_f32(x & 0xffffu), w[2 * e + 1] - __uint_as_float(x & 0xffff0000u));
            }
            hi[i] = __builtin_bit_cast(bf16x8, ph);
            lo[i] = __builtin_bit_cast(bf16x8, pl);
            if (__any(alpha != 1.0f)) {
#pragma unroll
                for (int j = 0; j < VD; ++j) acc[i][j] *= alpha;
            }
        }
        if (__any(vf.odd())) {
            vf.tame();
            any_odd = true;
        }
#pragma unroll
        for (int j = 0; j < VD; ++j) {
            const bf16x8 a = vf.operand(j);
#pragma unroll
            for (int i = 0; i < MT; ++i) acc[i][j] = mfma16(a, hi[i], mfma16(a, lo[i], acc[i][j]));
        }
        if (next < t1) vf.load(task.v, task.v_slot, steps.key(next), limit, lane);
    }

    if (any_odd) {  // rare, so key by key
#pragma unroll 1
        for (t = steps.t0 + wave; t < t1; t += kSplitWaves) {
#pragma unroll 1
            for (int key = steps.key(t); key < steps.key(t) + 32 && key < limit; ++key) {
                const uint16_t* vr = task.v + (int64_t)key * task.v_slot + 4 * q4 * VD;
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int j = 0; j < VD; j += 2) {
                        const uint32_t x = *reinterpret_cast<const uint32_t*>(vr + e * VD + j);
#pragma unroll
                        for (int i = 0; i < MT; ++i) {
                            const bool ok = sees(sight[i], task.seg + key, p.sinks);
                            acc[i][j][e] += ok ? odd_or_zero(x << 16) : 0.0f;
                            acc[i][j + 1][e] += ok ? odd_or_zero(x & 0xffff0000u) : 0.0f;
                        }
                    }
            }
        }
    }

    // The waves meet: O as [wave][row][D + 4] (rows 4 banks apart), maxima and
    // sums behind.
    constexpr int LD = D + 4;
    float* lo_o = reinterpret_cast<float*>(lds);
    float2* lo_ml = reinterpret_cast<float2*>(lds + (size_t)kSplitWaves * TR * LD * sizeof(float));
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        if (sight[i].lo == kPadding) {  // unmasked in the steps that its neighbours see whole
            m[i] = kNegInf;
            l[i] = 0.0f;
#pragma unroll
            for (int j = 0; j < VD; ++j) acc[i][j] = f32x4{0, 0, 0, 0};
        }
        const float ls = row_sum(l[i]);
        if (q4 == 0) lo_ml[wave * TR + 16 * i + n16] = make_float2(m[i], ls);
        float* o = lo_o + ((size_t)wave * TR + 16 * i + n16) * LD;
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int j = 0; j < VD; j += 4)
                *reinterpret_cast<f32x4*>(o + (4 * q4 + e) * VD + j) =
                    f32x4{acc[i][j][e], acc[i][j + 1][e], acc[i][j + 2][e], acc[i][j + 3][e]};
    }
    __syncthreads();
    const bool last = p.splits + p.prefix_splits == 1;
#pragma unroll
    for (int i = 0; i < TR / ROWS; ++i) {  // unrolled: one after the other, each waits 800 cycles for LDS
        const int n = i * ROWS + threadIdx.x / PER_ROW;
        const int row = task.row0 + n;
        float mw[kSplitWaves], M = kNegInf, L = 0.0f;
#pragma unroll
        for (int w = 0; w < kSplitWaves; ++w) {
            mw[w] = lo_ml[w * TR + n].x;
            M = fmaxf(M, mw[w]);
        }
        const float ms = M == kNegInf ? 0.0f : M;
        f32x4 o = {0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < kSplitWaves; ++w) {
            const float f = exp2_raw((mw[w] - ms) * p.c);
            L += f * lo_ml[w * TR + n].y;
            o += f * *reinterpret_cast<const f32x4*>(lo_o + ((size_t)w * TR + n) * LD + d);
        }
        if (row < task.rows) {
            const int b = task.shared ? row / p.RG : task.b0;
            const int j = task.shared ? row - b * p.RG : row;
            const int64_t g = (int64_t)task.part * all_rows + ((int64_t)b * p.kv_heads + task.h) * p.RG + j;
            if constexpr (JOIN) {
                shared[i].add(p, M, L, o);
                finish_row(p, b, task.h, j, D, d, shared[i].o, shared[i].M, shared[i].L);
            } else if (last) {
                finish_row(p, b, task.h, j, D, d, o, M, L);
            } else if (p.ctr) {  // for a workgroup of this launch, maybe on another XCD
                put_agent(p.part + g * D + d, o);
                if (d == 0) put_agent(p.ml + g, make_float2(M, L));
            } else {
                *reinterpret_cast<f32x4*>(p.part + g * D + d) = o;
                if (d == 0) p.ml[g] = make_float2(M, L);
            }
        }
    }
}

// Joins all rows of (b, h) with the whole workgroup: every four outputs of a
// row are one thread's, or (few rows) several threads', each with every
// groups-th range, which then meet in LDS in order.  The ranges a thread takes
// and the order they are added in follow from the shape alone, so the result
// does not depend on which range finished first.
template <int D>
__device__ __forceinline__ void join_rows(const AttnParams& p, int b, int h, unsigned char* lds) {
    const int64_t first = ((int64_t)b * p.kv_heads + h) * p.RG;
    const int units = p.RG * (D / 4);
    int groups = 1;
    while (2 * groups * units <= kSplitThreads && groups < 8) groups *= 2;
    const int g = groups > 1 ? threadIdx.x / units : 0;
    if (groups > 1) {
        const int e = threadIdx.x - g * units;
        const int j = e / (D / 4), d = 4 * (e % (D / 4));
        Joined y;
        if (g < groups) y = join_ranges<D, true>(p, first + j, d, g, groups);
        f32x4* lo = reinterpret_cast<f32x4*>(lds);
        float2* lml = reinterpret_cast<float2*>(lds + kSplitThreads * sizeof(f32x4));
        __syncthreads();
        lo[threadIdx.x] = y.o;
        lml[threadIdx.x] = make_float2(y.M, y.L);
        __syncthreads();
        if (g == 0) {
            for (int k = 1; k < groups; ++k) y.add(p, lml[e + k * units].x, lml[e + k * units].y, lo[e + k * units]);
            finish_row(p, b, h, j, D, d, y.o, y.M, y.L);
        }
        return;
    }
    for (int e = threadIdx.x; e < units; e += kSplitThreads) {
        const int j = e / (D / 4), d = 4 * (e % (D / 4));
        const Joined y = join_ranges<D, true>(p, first + j, d, 0, 1);
        finish_row(p, b, h, j, D, d, y.o, y.M, y.L);
    }
}

// MTO 16-row tiles of a sequence's own rows per workgroup, MTP of the rows over
// a shared prefix, in one launch.  Where partial results are joined here (no
// prefix), the workgroup that finishes last for a sequence and head does it: no
// second launch (one decode row over 1000 keys: 13.3 us a call in two launches,
// 9.1 in one).
template <int D, int MTO, int MTP, bool JOIN>
__global__ void __launch_bounds__(kSplitThreads, 2) attn_split_kernel(AttnParams p) {
    extern __shared__ __align__(16) unsigned char lds[];
    __shared__ int last;
    const Task task = task_of(p, blockIdx.x, 16 * MTO, 16 * MTP);
    if (MTO == MTP || !task.shared) split_task<D, MTO, JOIN>(p, task, lds);
    else split_task<D, MTP, false>(p, task, lds);
    if (JOIN || !p.ctr) return;
    drain_memory();
    __syncthreads();
    uint32_t* ctr = p.ctr + (int64_t)task.b0 * p.kv_heads + task.h;
    if (threadIdx.x == 0) {
        const uint32_t before = __hip_atomic_fetch_add(ctr, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        last = before == (uint32_t)(p.row_tiles * p.splits) - 1;
    }
    __syncthreads();
    if (!last) return;
    join_rows<D>(p, task.b0, task.h, lds);
    if (threadIdx.x == 0) __hip_atomic_store(ctr, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Joins the key ranges in a launch of its own: D / 4 threads a row and group
// of ranges, kGroups groups that meet in LDS in order.
constexpr int kGroups = 4;
template <int D>
__global__ void __launch_bounds__(256) attn_join_kernel(AttnParams p) {
    constexpr int T = D / 4;                      // threads of a row and group
    constexpr int ROWS = 256 / T / kGroups;       // of a workgroup
    __shared__ f32x4 lo[256];
    __shared__ float2 lml[256];
    const int64_t all_rows = (int64_t)p.B * p.kv_heads * p.RG;
    const int t = threadIdx.x % T, g = threadIdx.x / T % kGroups;
    const int64_t row = (int64_t)blockIdx.x * ROWS + threadIdx.x / (T * kGroups);
    const bool live = row < all_rows;
    Joined y;
    if (live) y = join_ranges<D, false>(p, row, 4 * t, g, kGroups);
    lo[threadIdx.x] = y.o;
    lml[threadIdx.x] = make_float2(y.M, y.L);
    __syncthreads();
    if (!live || g) return;
#pragma unroll
    for (int k = 1; k < kGroups; ++k) y.add(p, lml[threadIdx.x + k * T].x, lml[threadIdx.x + k * T].y, lo[threadIdx.x + k * T]);
    const int64_t bh = row / p.RG;
    finish_row(p, (int)(bh / p.kv_heads), (int)(bh % p.kv_heads), (int)(row - bh * p.RG), D, 4 * t, y.o, y.M, y.L);
}

// Adds the keys' weights to their scores from the kept q.k: 4 keys a thread.
// 8 bytes a key and row (write, read) against a second read of K at 2 * D.
__global__ void __launch_bounds__(256) attn_weights_raw_kernel(AttnParams p) {
    const int h = blockIdx.y, b = blockIdx.z;
    const int len = seq_len(p, b);
    const int key = 4 * ((int)blockIdx.x * 256 + (int)threadIdx.x);
    if (key >= len) return;
    const int64_t first = ((int64_t)b * p.kv_heads + h) * p.RG;
    f32x4 w = {0, 0, 0, 0};
#pragma unroll 4
    for (int j = 0; j < p.RG; ++j) {
        const f32x4 s = *reinterpret_cast<const f32x4*>(p.raw + (first + j) * p.raw_row + key);
        const float2 st = p.stat[first + j];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float x = exp2_raw((s[e] - st.x) * p.c) * st.y;
            w[e] += s[e] == kNegInf || st.y == 0.0f ? 0.0f : x;  // hidden, or the row sees nothing
        }
    }
    const float* was = p.scores + (int64_t)b * p.sc_seq + (int64_t)h * p.sc_head + key;
    float* to = p.scores_out + (int64_t)b * p.so_seq + (int64_t)h * p.so_head + key;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (key + e < len) to[e] = was[e] + w[e];
}

// Adds the keys' weights to their scores where q.k was not kept: a wave per 32
// keys of a sequence and head, whose K stays in registers, over all R * G rows
// in order (no atomics).  The rows come 32 at a time through LDS, shared by the
// four waves, the next 32 loading meanwhile.  Bound by reading K once more and
// by the weights themselves (20 VALU cycles a wave and 64 of them): 26 us for 32
// rows over 2 x 16000 keys.  All rows, also those that see none of the 32 keys: 2.7
// ms for a prompt of 8192 rows, whose attention takes 0.56 ms (0.28 with a window of
// 2048).
constexpr int kWeightRows = 32;
template <int D>
__global__ void __launch_bounds__(256, 4) attn_weights_kernel(AttnParams p) {
    constexpr int KS = D / 32;
    constexpr int LDQ = D * 2 + 16;  // bytes of a row in LDS: rows 4 banks apart
    constexpr int CH = D / 8, PARTS = kWeightRows * CH / 256;
    __shared__ __align__(16) unsigned char lq[kWeightRows * LDQ];
    __shared__ float2 lst[kWeightRows];
    const int lane = threadIdx.x & 63;
    const int n16 = lane & 15, q4 = lane >> 4;
    const int h = blockIdx.y, b = blockIdx.z;
    const int len = seq_len(p, b);
    if (128 * (int)blockIdx.x >= len) return;  // the whole workgroup
    const int kb = 32 * ((int)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6));
    const uint16_t* base = p.k.p + (int64_t)b * p.k.seq + (int64_t)h * p.k.head;
    KeyFrag<D> kf;
    kf.load(base, p.k.slot, kb, len, lane);
    // Which rows see what, from the first live row and the last.
    const int live_from = len - p.R > 0 ? len - p.R : 0;  // slot of the first row that has one
    const int hi_min = p.tree ? live_from - 1 : live_from;
    const int lo_max = p.window && len > p.window ? len - p.window : 0;
    const bool whole = kb + 32 <= len && kb + 31 <= hi_min && (kb >= lo_max || kb + 32 <= p.sinks);

    float w[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = 0.0f;
    const float2* stat = p.stat + ((int64_t)b * p.kv_heads + h) * p.RG;
    const uint16_t* qbase = p.q + (int64_t)b * p.R * p.q_row + (int64_t)h * p.G * D;
    u32x4 part[PARTS];
    float2 st;
    auto fetch = [&](int row0) {
#pragma unroll
        for (int i = 0; i < PARTS; ++i) {
            const int e = i * 256 + threadIdx.x;
            int j = row0 + e / CH;
            j = j < p.RG ? j : p.RG - 1;
            const int r = j / p.G;
            part[i] = load_cached16(qbase + (int64_t)r * p.q_row + (int64_t)(j - r * p.G) * D + 8 * (e % CH));
        }
        const int j = row0 + (int)threadIdx.x;  // the first 32 threads
        // Behind the last row: exp2(-infinity) times 0.
        st = j < p.RG && threadIdx.x < kWeightRows ? stat[j] : make_float2(__builtin_inff(), 0.0f);
    };
    fetch(0);
    for (int row0 = 0; row0 < p.RG; row0 += kWeightRows) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < PARTS; ++i) {
            const int e = i * 256 + threadIdx.x;
            *reinterpret_cast<u32x4*>(lq + e / CH * LDQ + e % CH * 16) = part[i];
        }
        if (threadIdx.x < kWeightRows) lst[threadIdx.x] = st;
        __syncthreads();
        if (row0 + kWeightRows < p.RG) fetch(row0 + kWeightRows);
        for (int i0 = 0; i0 < kWeightRows && row0 + i0 < p.RG; i0 += 16) {
            f32x4 s[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) s[u] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                const u32x4 q = *reinterpret_cast<const u32x4*>(lq + (i0 + n16) * LDQ + 64 * ks + 16 * q4);
#pragma unroll
                for (int u = 0; u < 2; ++u) s[u] = mfma16(kf.f[u][ks], q, s[u]);
            }
            const float2 now = lst[i0 + n16];
            if (whole) {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    w[e] = __builtin_fmaf(exp2_raw((s[e >> 2][e & 3] - now.x) * p.c), now.y, w[e]);
            } else {
                const int j = row0 + i0 + n16;
                const int r = (j < p.RG ? j : p.RG - 1) / p.G;
                const RowSight sight = row_sight(p, r, len, tree_bits(p, b, r));
                // A row that sees nothing (or is none) adds nothing, whatever its q.
                const bool adds = now.y != 0.0f;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int key = kb + 8 * q4 + e;
                    const float x = exp2_raw((s[e >> 2][e & 3] - now.x) * p.c) * now.y;
                    w[e] += adds && key < len && sees(sight, key, p.sinks) ? x : 0.0f;
                }
            }
        }
    }
    // Sum over the 16 rows in the lanes; lane n16 = e of each group keeps key e.
    float mine = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        float x = w[e];
        x += partner<8>(x);
        x += partner<4>(x);
        x += partner<2>(x);
        x += partner<1>(x);
        mine = n16 == e ? x : mine;
    }
    const int key = kb + 8 * q4 + n16;
    if (n16 < 8 && key < len) {
        const float was = p.scores[(int64_t)b * p.sc_seq + (int64_t)h * p.sc_head + key];
        p.scores_out[(int64_t)b * p.so_seq + (int64_t)h * p.so_head + key] = was + mine;
    }
}

}  // namespace krk
