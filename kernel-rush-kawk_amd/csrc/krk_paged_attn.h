// Attention of many requests' new rows over their pages (gfx950): how a call is
// cut into jobs, and the kernel for requests of few rows.
//
// Rows.  A key/value head h serves G = heads / kv_heads query heads, so request b's
// products have n * G rows per key/value head: row j is its new row j / G with
// query head h * G + j % G.
//
// Jobs.  A call's lengths are on the device, so each workgroup works out from them
// which job its number stands for: a lane takes one request in 64 of them (in order),
// and a scan over the wave finds the request.  Every wave does so for itself: no
// barrier, no launch in front, nothing kept from call to call.
//
// Products, key order and the treatment of infinities and NaNs in masked places are
// those of the contiguous caches' kernels.
#pragma once

#include "krk_attn_common.h"
#include "krk_page_step.h"

namespace krk {

struct PageView {
    const uint16_t* p;
    int64_t page, slot, head;
};

struct PagedParams {
    const uint16_t* q;
    int64_t q_row;
    PageView k, v;
    const int32_t* table;
    int64_t table_row;
    const int32_t *starts, *keys;
    uint16_t* out;
    int64_t out_row;
    float* lse;
    float scale;  // of q.k
    float c;      // scale * log2(e)
    int B, rows, heads, kv_heads, G, pages, shift, width, window, sinks;
};

// A request: its first row, rows and keys, whatever the arrays hold.
struct Request {
    int row, n, len;
};
__device__ __forceinline__ Request request(const PagedParams& p, int b) {
    Request x;
    const int full = p.width << p.shift;
    int s0 = p.starts[b], s1 = p.starts[b + 1], len = p.keys[b];
    s0 = s0 < 0 ? 0 : s0 > p.rows ? p.rows : s0;
    s1 = s1 < s0 ? s0 : s1 > p.rows ? p.rows : s1;
    x.row = s0;
    x.n = s1 - s0;
    x.len = len < 0 ? 0 : len > full ? full : len;
    return x;
}

constexpr int kFewThreads = 256;
constexpr int kFewWaves = kFewThreads / 64;

// A tile of a request's rows of one key/value head.
struct Job {
    int b, h, tile;
    Request req;
};

// The job that `id` stands for; tile < 0: none.
__device__ __forceinline__ Job job_of(const PagedParams& p, int id) {
    const int lane = threadIdx.x & 63;
    const int per = (p.B + 63) / 64;
    const int b0 = lane * per, b1 = b0 + per < p.B ? b0 + per : p.B;
    int mine = 0;
    for (int b = b0; b < b1; ++b) mine += (request(p, b).n * p.G + 15) / 16 * p.kv_heads;
    const int end = wave_scan(mine);
    int left = id - (end - mine);
    const uint64_t who = __ballot(left >= 0 && left < mine);
    Job j;
    j.tile = -1;
    if (!who) return j;
    const int src = __ffsll((unsigned long long)who) - 1;
    int b = b0;
    Request r = {0, 0, 0};
    if (lane == src)
        for (; b < b1; ++b) {
            r = request(p, b);
            const int jobs = (r.n * p.G + 15) / 16 * p.kv_heads;
            if (left < jobs) break;
            left -= jobs;
        }
    left = __builtin_amdgcn_readlane(left, src);
    j.b = __builtin_amdgcn_readlane(b, src);
    j.req.row = __builtin_amdgcn_readlane(r.row, src);
    j.req.n = __builtin_amdgcn_readlane(r.n, src);
    j.req.len = __builtin_amdgcn_readlane(r.len, src);
    j.h = left % p.kv_heads;
    j.tile = left / p.kv_heads;
    return j;
}

// The keys that a tile of rows sees, of one request: rows at positions first .. last
// (first may be negative: rows without a key), in steps of STEP keys: those that
// hold sinks, then from the first key that some row's window holds to the last
// row's own.
template <int STEP>
struct KeySpan {
    int end;            // keys behind the last that a row sees
    int hi_min, lo_max; // every row sees the keys from lo_max (and the sinks) to hi_min
    int from, sink_steps, steps;
    __device__ __forceinline__ KeySpan(const PagedParams& p, int len, int first, int last) {
        end = last + 1 < len ? last + 1 : len;
        end = end > 0 ? end : 0;
        hi_min = first;
        lo_max = p.window && last >= p.window ? last - p.window + 1 : 0;
        from = p.window && first >= p.window ? first - p.window + 1 : 0;
        from = from < end ? from & ~(STEP - 1) : end;
        sink_steps = ((p.sinks < end ? p.sinks : end) + STEP - 1) / STEP;
        if (STEP * sink_steps >= from) {
            from = 0;
            sink_steps = 0;
        }
        steps = sink_steps + (end - from + STEP - 1) / STEP;
    }
    __device__ __forceinline__ int key(int t) const { return t < sink_steps ? STEP * t : from + STEP * (t - sink_steps); }
    // Whether every row sees the whole step at key kb.
    __device__ __forceinline__ bool whole(int kb, int sinks) const {
        return kb + STEP <= end && kb + STEP - 1 <= hi_min && (kb >= lo_max || kb + STEP <= sinks);
    }
};

__device__ __forceinline__ bool row_sees(int pos, int lo, int sinks, int t) { return t <= pos && (t >= lo || t < sinks); }

// A request's keys or values of one head, through its table row.  Keys from `end`
// (>= 1) on read the last one again, page numbers outside the pool another page.
struct PagedRun {
    const uint16_t* base;  // of the head
    const int32_t* table;  // of the request
    int64_t page;
    int slot, shift, end;
    unsigned last_page;    // of the pool
    __device__ __forceinline__ PagedRun(const PagedParams& p, const PageView& v, const Job& j, int end_)
        : base(v.p + (int64_t)j.h * v.head), table(p.table + (int64_t)j.b * p.table_row), page(v.page), slot((int)v.slot),
          shift(p.shift), end(end_), last_page((unsigned)p.pages - 1) {}
    // Eight keys from a multiple of eight lie in one page: the page number of key g's.
    __device__ __forceinline__ unsigned page_of(int g) const {
        const int at = g < end ? g : end - 1;
        const unsigned n = (unsigned)table[at >> shift];
        return n < last_page ? n : last_page;
    }
    // Row of key `key`, whose eight keys' page number is n.
    __device__ __forceinline__ const uint16_t* row(int key, unsigned n) const {
        const int at = key < end ? key : end - 1;
        return base + (int64_t)n * page + (int64_t)(at & ((1 << shift) - 1)) * slot;
    }
};

template <int D>
constexpr size_t few_lds_bytes() {
    return (size_t)kFewWaves * 16 * ((D + 4) * sizeof(float) + sizeof(float2));
}

// Requests of few rows: 16 rows of a head and all of the keys they see, the four
// waves 32 keys at a time in turn.  Waves keep their own running maximum, sum and O
// and meet in LDS once, at the end.  Bound by reading K and V once a tile (4 * D
// bytes a key).  Weights go into the second product as two bf16 parts (p = hi + lo,
// 16 bits of mantissa).
template <int D>
__global__ void __launch_bounds__(kFewThreads, 2) paged_attn_kernel(PagedParams p) {
    extern __shared__ __align__(16) unsigned char lds[];
    constexpr int KS = D / 32;
    constexpr int VD = D / 16;
    const Job job = job_of(p, (int)blockIdx.x);
    if (job.tile < 0) return;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n16 = lane & 15, q4 = lane >> 4;
    const int rows = job.req.n * p.G, row0 = 16 * job.tile;
    const int pos0 = job.req.len - job.req.n;  // of the request's first row
    const int last_row = row0 + 15 < rows ? row0 + 15 : rows - 1;
    const KeySpan<32> span(p, job.req.len, pos0 + row0 / p.G, pos0 + last_row / p.G);
    const PagedRun kr(p, p.k, job, span.end), vr(p, p.v, job, span.end);

    // This lane's row (the last one again behind the end).
    const int mine = row0 + n16 < rows ? row0 + n16 : rows - 1;
    const int r = mine / p.G;
    const int head = job.h * p.G + (mine - r * p.G);
    const int pos = pos0 + r;
    const int lo = p.window && pos >= p.window ? pos - p.window + 1 : 0;
    u32x4 qf[KS];
    {
        const uint16_t* qr = p.q + (int64_t)(job.req.row + r) * p.q_row + (int64_t)head * D + 8 * q4;
#pragma unroll
        for (int s = 0; s < KS; ++s) qf[s] = load_cached16(qr + 32 * s);
    }
    f32x4 acc[VD];
    float m = kNegInf, l = 0.0f;
#pragma unroll
    for (int j = 0; j < VD; ++j) acc[j] = f32x4{0, 0, 0, 0};
    bool any_odd = false;
    for (int t = wave; t < span.steps; t += kFewWaves) {
        const int kb = span.key(t);
        KeyFrag<D> kf;
        ValueFrag<D> vf;
        {
            const int group = kb + 8 * (n16 >> 2);
            const unsigned page = kr.page_of(group);
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const uint16_t* x = kr.row(kb + tile_key(u, n16), page) + 8 * q4;
#pragma unroll
                for (int s = 0; s < KS; ++s) kf.f[u][s] = load_cached16(x + 32 * s);
            }
            const unsigned vpage = vr.page_of(kb + 8 * q4);
#pragma unroll
            for (int i = 0; i < 8; ++i)
                vf.f[i] = __builtin_nontemporal_load(
                    reinterpret_cast<const typename ValueFrag<D>::vec*>(vr.row(kb + 8 * q4 + i, vpage) + VD * n16));
        }
        f32x4 s[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            s[u] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) s[u] = mfma16(kf.f[u][ks], qf[ks], s[u]);
        }
        if (!span.whole(kb, p.sinks)) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int key = kb + 8 * q4 + e;
                s[e >> 2][e & 3] = row_sees(pos, lo, p.sinks, key) ? s[e >> 2][e & 3] : kNegInf;
            }
        }
        float mx = s[0][0];
#pragma unroll
        for (int e = 1; e < 8; ++e) mx = fmaxf(mx, s[e >> 2][e & 3]);
        const float mn = fmaxf(m, row_max(mx));
        const float ms = mn == kNegInf ? 0.0f : mn;  // nothing seen yet: weights exp2(-inf) = 0
        const float alpha = exp2_raw((m - ms) * p.c);
        m = mn;
        float w[8], sum = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            w[e] = exp2_raw((s[e >> 2][e & 3] - ms) * p.c);
            sum += w[e];
        }
        l = l * alpha + sum;
        u32x4 ph, pl;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            ph[e] = pack_bf16(w[2 * e], w[2 * e + 1]);
            const uint32_t x = ph[e];
            pl[e] = pack_bf16(w[2 * e] - bf16_to_f32(x & 0xffffu), w[2 * e + 1] - __uint_as_float(x & 0xffff0000u));
        }
        const bf16x8 hi = __builtin_bit_cast(bf16x8, ph), low = __builtin_bit_cast(bf16x8, pl);
#pragma unroll
        for (int j = 0; j < VD; ++j) acc[j] *= alpha;
        // An infinity or a NaN times a zero weight would reach rows that do not see
        // it: the products run on zeros in their place, and the rows that see them
        // get them behind the last step.
        if (__any(vf.odd())) {
            vf.tame();
            any_odd = true;
        }
#pragma unroll
        for (int j = 0; j < VD; ++j) {
            const bf16x8 a = vf.operand(j);
            acc[j] = mfma16(a, hi, mfma16(a, low, acc[j]));
        }
    }
    if (any_odd) {  // rare, so key by key
#pragma unroll 1
        for (int t = wave; t < span.steps; t += kFewWaves) {
            const int kb = span.key(t);
#pragma unroll 1
            for (int key = kb; key < kb + 32 && key < span.end; ++key) {
                const uint16_t* x = vr.row(key, vr.page_of(key)) + 4 * q4 * VD;
                const bool ok = row_sees(pos, lo, p.sinks, key);
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int j = 0; j < VD; j += 2) {
                        const uint32_t y = *reinterpret_cast<const uint32_t*>(x + e * VD + j);
                        acc[j][e] += ok ? odd_or_zero(y << 16) : 0.0f;
                        acc[j + 1][e] += ok ? odd_or_zero(y & 0xffff0000u) : 0.0f;
                    }
            }
        }
    }

    // The waves meet: O as [wave][row][D + 4] (rows 4 banks apart), maxima and
    // sums behind.
    constexpr int LD = D + 4;
    float* lo_o = reinterpret_cast<float*>(lds);
    float2* lo_ml = reinterpret_cast<float2*>(lds + (size_t)kFewWaves * 16 * LD * sizeof(float));
    const float ls = row_sum(l);
    if (q4 == 0) lo_ml[wave * 16 + n16] = make_float2(m, ls);
    float* o = lo_o + (wave * 16 + n16) * LD;
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int j = 0; j < VD; j += 4)
            *reinterpret_cast<f32x4*>(o + (4 * q4 + e) * VD + j) = f32x4{acc[j][e], acc[j + 1][e], acc[j + 2][e], acc[j + 3][e]};
    __syncthreads();
    constexpr int PER_ROW = D / 4, ROWS = kFewThreads / PER_ROW;
    const int d = 4 * (threadIdx.x % PER_ROW);
#pragma unroll
    for (int i = 0; i < 16 / ROWS; ++i) {
        const int n = i * ROWS + threadIdx.x / PER_ROW;
        if (row0 + n >= rows) continue;
        float mw[kFewWaves], M = kNegInf, L = 0.0f;
#pragma unroll
        for (int w = 0; w < kFewWaves; ++w) {
            mw[w] = lo_ml[w * 16 + n].x;
            M = fmaxf(M, mw[w]);
        }
        const float ms = M == kNegInf ? 0.0f : M;
        f32x4 x = {0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < kFewWaves; ++w) {
            const float f = exp2_raw((mw[w] - ms) * p.c);
            L += f * lo_ml[w * 16 + n].y;
            x += f * *reinterpret_cast<const f32x4*>(lo_o + (w * 16 + n) * LD + d);
        }
        const int rr = (row0 + n) / p.G;
        const int64_t at = job.req.row + rr;
        const int hd = job.h * p.G + (row0 + n - rr * p.G);
        const bool none = L == 0.0f;
        const float inv = none ? 0.0f : 1.0f / L;
        *reinterpret_cast<uint2*>(p.out + at * p.out_row + (int64_t)hd * D + d) =
            none ? make_uint2(0u, 0u) : make_uint2(pack_bf16(x[0] * inv, x[1] * inv), pack_bf16(x[2] * inv, x[3] * inv));
        if (d == 0 && p.lse) p.lse[at * p.heads + hd] = none ? kNegInf : M * p.scale + logf(L);
    }
}

}  // namespace krk
