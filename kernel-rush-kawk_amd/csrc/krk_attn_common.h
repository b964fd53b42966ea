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
    float* raw;    // [rows][raw_row] scores q.k of a scored call that keeps them, else null
    uint32_t* ctr; // [B][kv_heads] finished workgroups, null where the join has a launch of its own
    int64_t raw_row;
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
    int last;        // the highest position it may see; with tree masks that of bit 63, set or not
    int first;       // position of bit 0 (tree); before the cache where the first rows have no slot
    uint64_t bits;   // of the new rows, 0 without tree masks
};

__device__ __forceinline__ int seq_len(const AttnParams& p, int b) {
    const int n = p.lens[b];
    return n < 0 ? 0 : n > p.capacity ? p.capacity : n;
}

// The tree masks of row r of sequence b.
__device__ __forceinline__ uint64_t tree_bits(const AttnParams& p, int b, int r) {
    return p.tree ? (uint64_t)p.tree[(int64_t)b * p.R + r] : 0;
}

// Row r of a sequence whose cache holds len keys.
__device__ __forceinline__ RowSight row_sight(const AttnParams& p, int r, int len, uint64_t bits) {
    RowSight s;
    const int slot = len - p.R + r;
    s.first = p.prefix + len - p.R;
    s.bits = 0;
    int pos = p.prefix + slot;
    s.hi = pos;
    if (p.tree) {
        s.bits = p.R < 64 ? bits & ((1ull << p.R) - 1) : bits;
        const int none = p.R - len;  // the first rows, which have no slot
        if (none > 0) s.bits = none < 64 ? s.bits >> none << none : 0;
        const int cached = p.prefix + (none > 0 ? 0 : -none);
        pos = cached + __popcll(s.bits) - 1;
        s.hi = cached - 1;
    }
    s.last = p.tree ? s.first + 63 : s.hi;
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
    const unsigned d = (unsigned)(t - s.first);
    const bool node = d < 64 && ((s.bits >> (d & 63)) & 1);
    return (t <= s.hi && (t >= s.lo || t < sinks)) || node;
}

// Partial results cross XCDs, whose L2s are not coherent with each other:
// agent-scope relaxed accesses, ordered by a drain before the counter moves.
__device__ __forceinline__ void put_agent(float2* p, float2 v) {
    __hip_atomic_store(reinterpret_cast<uint64_t*>(p), __builtin_bit_cast(uint64_t, v), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 get_agent(const float2* p) {
    return __builtin_bit_cast(float2, __hip_atomic_load(reinterpret_cast<const uint64_t*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
}
__device__ __forceinline__ void put_agent(float* p, const f32x4& v) {
    put_agent(reinterpret_cast<float2*>(p), make_float2(v[0], v[1]));
    put_agent(reinterpret_cast<float2*>(p) + 1, make_float2(v[2], v[3]));
}
__device__ __forceinline__ f32x4 get_agent(const float* p) {
    const float2 a = get_agent(reinterpret_cast<const float2*>(p)), b = get_agent(reinterpret_cast<const float2*>(p) + 1);
    return f32x4{a.x, a.y, b.x, b.y};
}

// Wait until every load this wave issued has returned.
__device__ __forceinline__ void drain_loads() {
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    vm_wait<0>();
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
}

__device__ __forceinline__ float exp2_raw(float v) { return __builtin_amdgcn_exp2f(v); }

// A workgroup's share: a tile of rows of a key/value head against one range of the
// keys of a run (a sequence's own cache, or the shared prefix).
struct Task {
    bool shared;
    int h, b0;          // head; sequence (own cache)
    int rows, row0;     // rows of the run's row list, and the task's first
    int sp, nsp, part;  // key range, of how many, and its place among the partial results
    int seg, limit;     // position of the run's first key; its keys
    const uint16_t *k, *v;
    int64_t k_slot, v_slot;
};

// Heads change fastest: with 8 heads each XCD (workgroups go to them round
// robin) keeps to one head's keys.  Later row tiles, which see more keys, go
// first.
__device__ __forceinline__ Task task_of(const AttnParams& p, int id, int own_rows, int prefix_rows) {
    Task t;
    const int nprefix = p.prefix_row_tiles * p.kv_heads * p.prefix_splits;
    t.shared = id < nprefix;
    if (!t.shared) id -= nprefix;
    t.h = id % p.kv_heads;
    id /= p.kv_heads;
    t.b0 = 0;
    int tile;
    if (t.shared) {
        tile = id % p.prefix_row_tiles;
        t.sp = id / p.prefix_row_tiles;
        t.nsp = p.prefix_splits;
        t.part = p.splits + t.sp;
        t.rows = p.B * p.RG;
        t.seg = 0;
        t.limit = p.prefix;
    } else {
        tile = p.row_tiles - 1 - id % p.row_tiles;
        id /= p.row_tiles;
        t.b0 = id % p.B;
        t.sp = id / p.B;
        t.nsp = p.splits;
        t.part = t.sp;
        t.rows = p.RG;
        t.seg = p.prefix;
        t.limit = seq_len(p, t.b0);
    }
    t.row0 = tile * (t.shared ? prefix_rows : own_rows);
    const CacheView& k = t.shared ? p.kp : p.k;
    const CacheView& v = t.shared ? p.vp : p.v;
    t.k = k.p + (t.shared ? 0 : (int64_t)t.b0 * k.seq) + (int64_t)t.h * k.head;
    t.v = v.p + (t.shared ? 0 : (int64_t)t.b0 * v.seq) + (int64_t)t.h * v.head;
    t.k_slot = k.slot;
    t.v_slot = v.slot;
    return t;
}

// Row `row` of a task's list (the last one again behind its end), and what it
// takes to say what the row sees.
struct TaskRow {
    int b, r, head, len;
    uint64_t bits;
    __device__ __forceinline__ RowSight sight(const AttnParams& p) const { return row_sight(p, r, len, bits); }
};
__device__ __forceinline__ TaskRow task_row(const AttnParams& p, const Task& t, int row) {
    TaskRow x;
    const int j = row < t.rows ? row : t.rows - 1;
    x.b = t.shared ? j / p.RG : t.b0;
    const int jj = t.shared ? j - x.b * p.RG : j;
    x.r = jj / p.G;
    x.head = t.h * p.G + (jj - x.r * p.G);
    x.len = t.shared ? seq_len(p, x.b) : t.limit;
    x.bits = tree_bits(p, x.b, x.r);
    return x;
}

// What a set of rows sees at most (lo_min .. hi_max) and all of them see (from
// lo_max to hi_min), over the lanes of a wave.  Without a window a sequence's
// steps reach its last key, whatever its tree masks hold: kept scores are then
// written for every key.
struct Reach {
    int lo_min = 0x7fffffff, hi_max = -1, lo_max = 0, hi_min = 0x7fffffff;
    __device__ __forceinline__ void add(const RowSight& s, bool live) {
        if (live && s.lo != kPadding) {
            lo_min = s.lo < lo_min ? s.lo : lo_min;
            lo_max = s.lo > lo_max ? s.lo : lo_max;
            hi_max = s.last > hi_max ? s.last : hi_max;
            hi_min = s.hi < hi_min ? s.hi : hi_min;
        }
    }
    __device__ __forceinline__ void join_lanes() {
        lo_min = wave_min_i(lo_min);
        lo_max = -wave_min_i(-lo_max);
        hi_max = -wave_min_i(-hi_max);
        hi_min = wave_min_i(hi_min);
    }
    template <int CTRL>
    __device__ static __forceinline__ int dpp_min(int v) {
        const int o = __builtin_amdgcn_update_dpp(0, v, CTRL, 0xF, 0xF, false);
        return o < v ? o : v;
    }
    __device__ static __forceinline__ int wave_min_i(int v) {
        v = dpp_min<0xB1>(v);   // lane ^ 1
        v = dpp_min<0x4E>(v);   // lane ^ 2
        v = dpp_min<0x141>(v);  // mirrored in 8
        v = dpp_min<0x140>(v);  // mirrored in 16
        const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        v = (int)a[0] < (int)a[1] ? (int)a[0] : (int)a[1];
        const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        v = (int)b[0] < (int)b[1] ? (int)b[0] : (int)b[1];
        return __builtin_amdgcn_readfirstlane(v);
    }
};

// The same from the lengths alone, of all of a task's rows; not for a shared
// prefix with a window, where it takes every sequence's.
__device__ __forceinline__ Reach reach_at_most(const AttnParams& p, const Task& t) {
    Reach r;
    const int first = t.limit - p.R > 0 ? t.limit - p.R : 0;  // slot of the first row that has one
    r.hi_max = t.seg + t.limit - 1;
    // A row with tree masks may lie one position before the first.
    const int lo = p.window ? t.seg + first - (p.tree ? 1 : 0) - p.window + 1 : 0;
    r.lo_min = lo > 0 ? lo : 0;
    return r;
}

// A task's keys in steps of STEP: those that hold sinks, then from the first
// key that some row's window holds to the last that some row sees.  The task
// takes steps t0 .. t1 - 1.
template <int STEP>
struct KeySteps {
    int from, sink_steps, t0, t1;
    __device__ __forceinline__ KeySteps(const AttnParams& p, const Task& t, const Reach& r) {
        int end = r.hi_max + 1 - t.seg;
        end = end < t.limit ? end : t.limit;
        end = end > 0 ? end : 0;
        from = r.lo_min - t.seg;
        from = from > 0 ? (from < end ? from & ~(STEP - 1) : end) : 0;
        int nsink = p.sinks - t.seg;
        nsink = nsink > 0 ? (nsink < end ? nsink : end) : 0;
        sink_steps = (nsink + STEP - 1) / STEP;
        if (STEP * sink_steps >= from) {
            from = 0;
            sink_steps = 0;
        }
        const int steps = sink_steps + (end > from ? (end - from + STEP - 1) / STEP : 0);
        t0 = (int)((int64_t)steps * t.sp / t.nsp);
        t1 = (int)((int64_t)steps * (t.sp + 1) / t.nsp);
    }
    __device__ __forceinline__ int key(int t) const { return t < sink_steps ? STEP * t : from + STEP * (t - sink_steps); }
};

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
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    bf16x2 v;
    v[0] = (__bf16)lo;
    v[1] = (__bf16)hi;
    return __builtin_bit_cast(uint32_t, v);
}

// The key of 32 that row r of 16-key tile t holds (see the top).
__device__ __forceinline__ int tile_key(int t, int r) { return 8 * (r >> 2) + 4 * t + (r & 3); }

// Two bf16 values with zeros for infinities and NaNs.
__device__ __forceinline__ uint32_t finite_bf16x2(uint32_t w) {
    return ((w & 0x7f80u) != 0x7f80u ? w & 0xffffu : 0u) | ((w & 0x7f800000u) != 0x7f800000u ? w & 0xffff0000u : 0u);
}
// An infinity or NaN given as an fp32's bits, else 0.
__device__ __forceinline__ float odd_or_zero(uint32_t f32_bits) {
    return (f32_bits & 0x7f800000u) == 0x7f800000u ? __uint_as_float(f32_bits) : 0.0f;
}

// Four finished outputs of row j of (b, h), and with d = 0 what else is kept
// of the row: M the maximum of q.k (-infinity: the row sees nothing), L the sum.
__device__ __forceinline__ void finish_row(const AttnParams& p, int b, int h, int j, int D, int d, const f32x4& o, float M, float L) {
    const int r = j / p.G;
    const int head = h * p.G + (j - r * p.G);
    const int64_t at = (int64_t)b * p.R + r;
    const bool none = L == 0.0f;
    const float inv = none ? 0.0f : 1.0f / L;
    *reinterpret_cast<uint2*>(p.out + at * p.out_row + (int64_t)head * D + d) =
        none ? make_uint2(0u, 0u) : make_uint2(pack_bf16(o[0] * inv, o[1] * inv), pack_bf16(o[2] * inv, o[3] * inv));
    if (d == 0) {
        if (p.lse) p.lse[at * p.heads + head] = none ? kNegInf : M * p.scale + logf(L);
        if (p.stat) p.stat[((int64_t)b * p.kv_heads + h) * p.RG + j] = make_float2(M == kNegInf ? 0.0f : M, inv);
    }
}

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
    typedef __attribute__((ext_vector_type(W))) uint32_t vec;
    vec f[8];
    __device__ __forceinline__ void load(const uint16_t* base, int64_t slot, int kb, int limit, int lane) {
        const int r = lane & 15, q = lane >> 4;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            int key = kb + 8 * q + i;
            key = key < limit ? key : limit - 1;
            f[i] = __builtin_nontemporal_load(reinterpret_cast<const vec*>(base + (int64_t)key * slot + VD * r));
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
    // Infinities and NaNs to zero.
    __device__ __forceinline__ void tame() {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const vec e = f[i] & 0x7f807f80u;
            vec keep;
#pragma unroll
            for (int w = 0; w < W; ++w)
                keep[w] = ((e[w] & 0xffffu) != 0x7f80u ? 0xffffu : 0u) | ((e[w] >> 16) != 0x7f80u ? 0xffff0000u : 0u);
            f[i] &= keep;
        }
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

__device__ __forceinline__ u32x4 finite_bf16x8(const u32x4& x) {
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = finite_bf16x2(x[i]);
    return r;
}

}  // namespace krk
