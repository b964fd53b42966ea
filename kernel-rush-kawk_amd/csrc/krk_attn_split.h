// Cache attention for few rows (decode, draft trees, batches over a shared
// prefix): key ranges split over workgroups, joined by a second kernel.
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
// the time and a CU holds 2-3 such workgroups at MT = 1.
//
// The rows of the shared prefix are those of all sequences together, so it is
// read once per TR rows of the batch instead of once per sequence.
//
// Weights go into the second product as two bf16 parts (p = hi + lo, 16 bits of
// mantissa): the matrix pipe has the time, and the sums then carry fp32's
// weights to within 2^-17.
#pragma once

#include "krk_attn_common.h"

namespace krk {

constexpr int kSplitWaves = 4;
constexpr int kSplitThreads = 64 * kSplitWaves;

template <int D, int MT>
constexpr size_t split_lds_bytes() {
    return (size_t)kSplitWaves * 16 * MT * ((D + 4) * sizeof(float) + sizeof(float2));
}

template <int D, int MT>
__global__ void __launch_bounds__(kSplitThreads, MT == 1 ? 2 : 1) attn_split_kernel(AttnParams p) {
    constexpr int TR = 16 * MT;
    constexpr int KS = D / 32;
    constexpr int VD = D / 16;
    extern __shared__ __align__(16) unsigned char lds[];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n16 = lane & 15, q4 = lane >> 4;

    const Task task = task_of<TR>(p, blockIdx.x);
    const int limit = task.limit;

    // This lane's rows: what they see, and their q.
    RowSight sight[MT];
    u32x4 qf[MT][KS];
    Reach reach;
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const int row = task.row0 + 16 * i + n16;
        const TaskRow x = task_row(p, task, row);
        sight[i] = x.sight;
        reach.add(x.sight, row < task.rows);
        const uint16_t* qr = p.q + ((int64_t)x.b * p.R + x.r) * p.q_row + (int64_t)x.head * D + 8 * q4;
#pragma unroll
        for (int s = 0; s < KS; ++s) qf[i][s] = load_cached16(qr + 32 * s);
    }
    reach.join_lanes();
    const KeySteps<32> steps(p, task, reach);

    f32x4 acc[MT][VD];
    float m[MT], l[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        m[i] = kNegInf;
        l[i] = 0.0f;
#pragma unroll
        for (int j = 0; j < VD; ++j) acc[i][j] = f32x4{0, 0, 0, 0};
    }

    KeyFrag<D> kf;
    ValueFrag<D> vf;
    const int t1 = steps.t1;
    int t = steps.t0 + wave;
    if (t < t1) {
        kf.load(task.k, task.k_slot, steps.key(t), limit, lane);
        vf.load(task.v, task.v_slot, steps.key(t), limit, lane);
    }
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
        uint32_t vis[MT];
#pragma unroll
        for (int i = 0; i < MT; ++i) vis[i] = 0xff;
        if (!whole) {
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                vis[i] = 0;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int key = kb + 8 * q4 + e;
                    const bool ok = key < limit && sees(sight[i], task.seg + key, p.sinks);
                    vis[i] |= ok ? 1u << e : 0u;
                    s[i][e >> 2][e & 3] = ok ? s[i][e >> 2][e & 3] : kNegInf;
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
            add_odd_values<D, MT>(acc, vf, hi, lo, vis);
        } else {
#pragma unroll
            for (int j = 0; j < VD; ++j) {
                const bf16x8 a = vf.operand(j);
#pragma unroll
                for (int i = 0; i < MT; ++i) acc[i][j] = mfma16(a, hi[i], mfma16(a, lo[i], acc[i][j]));
            }
        }
        if (next < t1) vf.load(task.v, task.v_slot, steps.key(next), limit, lane);
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
    const int64_t all_rows = (int64_t)p.B * p.kv_heads * p.RG;
    const bool last = p.splits + p.prefix_splits == 1;
    constexpr int PER_ROW = D / 4;
    for (int e = threadIdx.x; e < TR * PER_ROW; e += kSplitThreads) {
        const int n = e / PER_ROW, d = 4 * (e % PER_ROW);
        const int row = task.row0 + n;
        if (row >= task.rows) break;  // rows grow with e
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
        const int b = task.shared ? row / p.RG : task.b0;
        const int j = task.shared ? row - b * p.RG : row;
        const int64_t g = ((int64_t)b * p.kv_heads + task.h) * p.RG + j;
        if (last) {
            const int r = j / p.G;
            const int head = task.h * p.G + (j - r * p.G);
            const float inv = L == 0.0f ? 0.0f : 1.0f / L;
            if (L == 0.0f) o = f32x4{0, 0, 0, 0};
            const int64_t at = (int64_t)b * p.R + r;
            *reinterpret_cast<uint2*>(p.out + at * p.out_row + (int64_t)head * D + d) =
                make_uint2(pack_bf16(o[0] * inv, o[1] * inv), pack_bf16(o[2] * inv, o[3] * inv));
            if (d == 0) {
                if (p.lse) p.lse[at * p.heads + head] = L == 0.0f ? kNegInf : M * p.scale + logf(L);
                if (p.stat) p.stat[g] = make_float2(ms, inv);
            }
        } else {
            *reinterpret_cast<f32x4*>(p.part + ((int64_t)task.part * all_rows + g) * D + d) = o;
            if (d == 0) p.ml[(int64_t)task.part * all_rows + g] = make_float2(M, L);
        }
    }
}

// Joins the key ranges: a wave per row.  Ranges in order, so the result does
// not depend on which finished first.
template <int D>
__global__ void __launch_bounds__(256) attn_join_kernel(AttnParams p) {
    const int lane = threadIdx.x & 63;
    const int64_t all_rows = (int64_t)p.B * p.kv_heads * p.RG;
    const int64_t g = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (g >= all_rows) return;
    const int n = p.splits + p.prefix_splits;
    float M = kNegInf;
    for (int s = lane; s < n; s += 64) M = fmaxf(M, p.ml[s * all_rows + g].x);
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) M = fmaxf(M, __shfl_xor(M, s));
    const float ms = M == kNegInf ? 0.0f : M;
    float L = 0.0f, o[D / 64];
#pragma unroll
    for (int e = 0; e < D / 64; ++e) o[e] = 0.0f;
    for (int s0 = 0; s0 < n; s0 += 64) {
        float f = 0.0f, part_l = 0.0f;
        if (s0 + lane < n) {
            const float2 ml = p.ml[(s0 + lane) * all_rows + g];
            f = exp2_raw((ml.x - ms) * p.c);
            part_l = f * ml.y;
        }
        const int cnt = n - s0 < 64 ? n - s0 : 64;
#pragma unroll 4
        for (int s = 0; s < cnt; ++s) {
            const float fs = __shfl(f, s);
            L += __shfl(part_l, s);
            const float* q = p.part + ((int64_t)(s0 + s) * all_rows + g) * D + lane * (D / 64);
            if constexpr (D == 128) {
                const float2 x = *reinterpret_cast<const float2*>(q);
                o[0] = __builtin_fmaf(fs, x.x, o[0]);
                o[1] = __builtin_fmaf(fs, x.y, o[1]);
            } else {
                o[0] = __builtin_fmaf(fs, *q, o[0]);
            }
        }
    }
    const int64_t bh = g / p.RG;
    const int j = (int)(g - bh * p.RG);
    const int b = (int)(bh / p.kv_heads), h = (int)(bh - (int64_t)b * p.kv_heads);
    const int r = j / p.G;
    const int head = h * p.G + (j - r * p.G);
    const int64_t at = (int64_t)b * p.R + r;
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
    if (L == 0.0f) o[0] = o[D / 64 - 1] = 0.0f;
    uint16_t* y = p.out + at * p.out_row + (int64_t)head * D + lane * (D / 64);
    if constexpr (D == 128)
        *reinterpret_cast<uint32_t*>(y) = pack_bf16(o[0] * inv, o[1] * inv);
    else
        *y = (uint16_t)f32_to_bf16(o[0] * inv);
    if (lane == 0) {
        if (p.lse) p.lse[at * p.heads + head] = L == 0.0f ? kNegInf : M * p.scale + logf(L);
        if (p.stat) p.stat[g] = make_float2(ms, inv);
    }
}

// Adds the keys' weights to their scores: a wave per 32 keys of a sequence
// and head, over all R * G rows; no atomics, rows in order.
template <int D>
__global__ void __launch_bounds__(256) attn_weights_kernel(AttnParams p) {
    constexpr int KS = D / 32;
    const int lane = threadIdx.x & 63;
    const int n16 = lane & 15, q4 = lane >> 4;
    const int h = blockIdx.y, b = blockIdx.z;
    const int len = seq_len(p, b);
    const int kb = 32 * ((int)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6));
    if (kb >= len) return;
    KeyFrag<D> kf;
    kf.load(p.k.p + (int64_t)b * p.k.seq + (int64_t)h * p.k.head, p.k.slot, kb, len, lane);
    const float2* stat = p.stat + ((int64_t)b * p.kv_heads + h) * p.RG;
    float w[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = 0.0f;
    for (int row0 = 0; row0 < p.RG; row0 += 16) {
        const int row = row0 + n16;
        const int j = row < p.RG ? row : p.RG - 1;
        const int r = j / p.G;
        const RowSight sight = row_sight(p, b, r, len);
        const uint16_t* qr = p.q + ((int64_t)b * p.R + r) * p.q_row + (int64_t)(h * p.G + (j - r * p.G)) * D + 8 * q4;
        const float2 st = stat[j];
        f32x4 s[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) s[u] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const u32x4 qf = load_cached16(qr + 32 * ks);
#pragma unroll
            for (int u = 0; u < 2; ++u) s[u] = mfma16(kf.f[u][ks], qf, s[u]);
        }
        const bool live = row < p.RG;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int key = kb + 8 * q4 + e;
            const float x = exp2_raw((s[e >> 2][e & 3] - st.x) * p.c) * st.y;
            w[e] += live && key < len && sees(sight, key, p.sinks) ? x : 0.0f;
        }
    }
    // Sum over the 16 rows in the lanes; lane n16 = e of each group keeps key e.
    float mine = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        float x = w[e];
#pragma unroll
        for (int s = 1; s < 16; s <<= 1) x += __shfl_xor(x, s);
        mine = n16 == e ? x : mine;
    }
    const int key = kb + 8 * q4 + n16;
    if (n16 < 8 && key < len) {
        const float was = p.scores[(int64_t)b * p.sc_seq + (int64_t)h * p.sc_head + key];
        p.scores_out[(int64_t)b * p.so_seq + (int64_t)h * p.so_head + key] = was + mine;
    }
}

}  // namespace krk
