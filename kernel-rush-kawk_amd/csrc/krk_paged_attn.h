// Attention of many requests' new rows over their pages (gfx950): which job each
// workgroup has (how a call is cut into them: krk_paged_cut.h), and the jobs of requests
// of few rows.
//
// Rows.  A key/value head h serves G = heads / kv_heads query heads, so request b's
// products have n * G rows per key/value head: row j is its new row j / G with
// query head h * G + j % G.
//
// Jobs.  A job is a tile of a request's rows of one head against one range of the
// keys they see.  A call's lengths are on the device, so each wave works out from them
// which job its workgroup's number stands for, a lane a request: no barrier, no launch
// in front, nothing kept from call to call (1.6 us; more than 64 requests are planned by
// a launch in front).  Keys are cut by
// length: into ranges that cost about what one of kTarget workgroups would take of
// all of the call's work, so a long request beside short ones does not work on alone.
// The workgroup that finishes the last range of a tile joins them, in order (many ranges
// of many rows: group by group, and the groups then).
//
// Products, key order and the treatment of infinities and NaNs in masked places are
// those of the contiguous caches' kernels.
#pragma once

#include <type_traits>

#include "krk_attn_common.h"
#include "krk_epilogue.h"
#include "krk_page_step.h"
#include "krk_paged_cut.h"

namespace krk {

__device__ __forceinline__ float wave_total(float v) {
    v += partner<1>(v);
    v += partner<2>(v);
    v += partner<4>(v);
    v += partner<8>(v);
    return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(row_sum(v))));
}

// A tile of a request's rows of one key/value head, against one range of its keys.
struct Job {
    int b, h, tile;     // tile: rows of a tile; < 0: no job
    int row0;           // first row of the tile, of the head's row list
    int part, parts;    // range, of how many
    int slot;           // of parts > 1: row of the tile's first range's results
    Request req;
    // The counter of range `part`: each has 16 rows of results at least.
    __device__ __forceinline__ int counter(int part) const { return (slot + part * tile) >> 4; }
    // place: of a request's jobs.  Heads change fastest, then ranges, then tiles, those
    // that see more keys first.
    __device__ __forceinline__ void at(const PagedParams& p, const Tiling& t, int place, int slot0) {
        const int over_heads = __builtin_amdgcn_readfirstlane(quotient(place, p.kv_heads, p.inv_kv));
        h = place - over_heads * p.kv_heads;
        const int over_parts = __builtin_amdgcn_readfirstlane(quotient(over_heads, parts, __builtin_amdgcn_rcpf((float)parts)));
        part = over_heads - over_parts * parts;
        const int nth = t.tiles - 1 - over_parts;
        tile = 1 << t.shift;
        row0 = nth << t.shift;
        slot = slot0 + ((nth * p.kv_heads + h) * parts << t.shift);
    }
};

__device__ __forceinline__ Job job_of(const PagedParams& p, int id) {
    const int lane = threadIdx.x & 63;
    Request r = request(p, lane < p.B ? lane : p.B - 1);
    if (lane >= p.B) r.n = 0;
    const Tiling t = tiling(p, r);
    const float share = wave_total(cost_of(t)) * (float)p.kv_heads * (1.0f / kTarget);
    Ranges ranges(share);
    int parts, jobs, upto_many, upto_few, all_many, all_few;
    auto count = [&]() {
        parts = ranges.parts(t);
        jobs = t.tiles * p.kv_heads * parts;
        upto_many = wave_scan(t.many ? jobs : 0);
        upto_few = wave_scan(t.many ? 0 : jobs);
        all_many = __builtin_amdgcn_readlane(upto_many, 63);
        all_few = __builtin_amdgcn_readlane(upto_few, 63);
    };
    count();
    if (all_many + all_few > kTarget && all_few) {
        ranges.cut_anew(share, all_many + all_few);
        count();
    }
    const Nth nth(id, all_many, all_few, 8);
    const int left = nth.n - (t.many ? upto_many : upto_few) + jobs;
    const uint64_t who = __ballot(t.many == nth.many && left >= 0 && left < jobs);
    Job j;
    j.tile = -1;
    // More rows than the call has, as starts do not ascend: the jobs' bounds would not hold.
    if (!who || __builtin_amdgcn_readlane(wave_scan(r.n), 63) > p.rows) return j;
    const int src = __ffsll((unsigned long long)who) - 1;
    const int rows = parts > 1 ? jobs << t.shift : 0;
    const int slot0 = wave_scan(rows) - rows;
    j.b = src;
    j.req.row = __builtin_amdgcn_readlane(r.row, src);
    j.req.n = __builtin_amdgcn_readlane(r.n, src);
    j.req.len = __builtin_amdgcn_readlane(r.len, src);
    j.parts = __builtin_amdgcn_readlane(parts, src);
    j.at(p, tiling(p, j.req), __builtin_amdgcn_readlane(left, src), __builtin_amdgcn_readlane(slot0, src));
    return j;
}

// More requests: a launch in front, of one workgroup, lists the tiles' ranges in the order
// of the jobs; a job is a head of one of them.  (Each wave for itself, with four requests
// a lane: 4.0 us a job instead of 1.6 at 256 requests.)
constexpr int kPlanThreads = 1024;
__host__ __device__ constexpr size_t plan_lds_bytes(int B) { return (size_t)(3 * B + 2) * sizeof(int); }

__global__ void __launch_bounds__(kPlanThreads) paged_plan_kernel(PagedParams p) {
    extern __shared__ __align__(16) unsigned char lds[];
    __shared__ int scratch[kPageWaves];
    __shared__ float costs[kPageWaves];
    int* first_many = reinterpret_cast<int*>(lds);  // [B + 1] ranges of earlier requests, by kind
    int* first_few = first_many + p.B + 1;
    int* first_row = first_few + p.B + 1;           // [B] rows of results of earlier requests
    const int per = (p.B + kPlanThreads - 1) / kPlanThreads;
    const int b0 = (int)threadIdx.x * per, b1 = b0 + per < p.B ? b0 + per : p.B;
    float cost = 0.0f;
    int all_rows = 0;
    for (int b = b0; b < b1; ++b) {
        const Request r = request(p, b);
        all_rows += r.n;
        cost += cost_of(tiling(p, r));
    }
    cost = wave_total(cost);
    if ((threadIdx.x & 63) == 0) costs[threadIdx.x >> 6] = cost;
    int total;
    block_scan(all_rows, scratch, &total);
    float share = 0.0f;
    for (int w = 0; w < kPageWaves; ++w) share += costs[w];
    share *= (float)p.kv_heads * (1.0f / kTarget);
    Ranges ranges(share);
    int many, few, rows, all_many, all_few;
    auto count = [&]() {
        many = few = rows = 0;
        for (int b = b0; b < b1; ++b) {
            const Tiling t = tiling(p, request(p, b));
            const int parts = ranges.parts(t), n = t.tiles * parts;
            many += t.many ? n : 0;
            few += t.many ? 0 : n;
            rows += parts > 1 ? n * p.kv_heads << t.shift : 0;
        }
        many = block_scan(many, scratch, &all_many);
        few = block_scan(few, scratch, &all_few);
    };
    count();
    if ((all_many + all_few) * p.kv_heads > kTarget && all_few) {
        ranges.cut_anew(share, (all_many + all_few) * p.kv_heads);
        count();
    }
    int unused;
    rows = block_scan(rows, scratch, &unused);
    for (int b = b0; b < b1; ++b) {
        const Tiling t = tiling(p, request(p, b));
        const int parts = ranges.parts(t), n = t.tiles * parts;
        first_many[b] = many;
        first_few[b] = few;
        first_row[b] = rows;
        many += t.many ? n : 0;
        few += t.many ? 0 : n;
        rows += parts > 1 ? n * p.kv_heads << t.shift : 0;
    }
    __syncthreads();
    // More rows than the call has, as starts do not ascend: no job.
    const int n = total > p.rows ? 0 : all_many + all_few;
    if (threadIdx.x == 0) *p.planned = n;
    int block = 8;  // blocks of 256 jobs
    while (block > 0 && (p.kv_heads << block) > 256) --block;
    for (int e = threadIdx.x; e < n; e += kPlanThreads) {
        const Nth nth(e, all_many, all_few, block);
        const int* first = nth.many ? first_many : first_few;
        const int b = owner_of(first, p.B, nth.n);
        const Tiling t = tiling(p, request(p, b));
        const int parts = ranges.parts(t), place = nth.n - first[b];
        const int tile = quotient(place, parts, __builtin_amdgcn_rcpf((float)parts)), part = place - tile * parts;
        PlannedRange x;
        x.b = b;
        x.row0 = (t.tiles - 1 - tile) << t.shift;
        x.parts_part = parts << 16 | part;
        x.slot = first_row[b] + ((t.tiles - 1 - tile) * p.kv_heads * parts << t.shift);
        p.plan[e] = x;
    }
}

__device__ __forceinline__ Job planned_job(const PagedParams& p, int id) {
    Job j;
    j.tile = -1;
    const int e = __builtin_amdgcn_readfirstlane(quotient(id, p.kv_heads, p.inv_kv));
    if (e >= *p.planned) return j;
    const PlannedRange x = p.plan[e];
    j.b = __builtin_amdgcn_readfirstlane(x.b);
    j.row0 = __builtin_amdgcn_readfirstlane(x.row0);
    const int pp = __builtin_amdgcn_readfirstlane(x.parts_part);
    j.parts = pp >> 16;
    j.part = pp & 0xffff;
    const Request r = request(p, j.b);
    j.req = {__builtin_amdgcn_readfirstlane(r.row), __builtin_amdgcn_readfirstlane(r.n), __builtin_amdgcn_readfirstlane(r.len)};
    j.h = id - e * p.kv_heads;
    const int shift = tiling(p, j.req).shift;
    j.tile = 1 << shift;
    j.slot = __builtin_amdgcn_readfirstlane(x.slot) + (j.h * j.parts << shift);
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

// Where the rows of a tile are.
struct TileRow {
    int r, head, pos, lo;  // row of the request, query head, position and the first key of its window
    __device__ __forceinline__ TileRow(const PagedParams& p, const Job& j, int row) {
        r = quotient(row, p.G, p.inv_G);
        head = j.h * p.G + (row - r * p.G);
        pos = j.req.len - j.req.n + r;
        lo = p.window && pos >= p.window ? pos - p.window + 1 : 0;
    }
};

// Four finished outputs of a tile's row, and with d = 0 the log of its sum: M the
// maximum of q.k (-infinity: the row sees nothing), L the sum.
__device__ __forceinline__ void finish_row(const PagedParams& p, const Job& j, int row, int D, int d, const f32x4& o, float M, float L) {
    const TileRow t(p, j, row);
    const int64_t at = j.req.row + t.r;
    const bool none = L == 0.0f;
    const float inv = none ? 0.0f : 1.0f / L;
    *reinterpret_cast<uint2*>(p.out + at * p.out_row + (int64_t)t.head * D + d) =
        none ? make_uint2(0u, 0u) : make_uint2(pack_bf16(o[0] * inv, o[1] * inv), pack_bf16(o[2] * inv, o[3] * inv));
    if (d == 0 && p.lse) p.lse[at * p.heads + t.head] = none ? kNegInf : M * p.scale + logf(L);
}

// Outputs of one row over several ranges, put together.
struct Merged {
    float M = kNegInf, L = 0.0f;
    f32x4 o = {0, 0, 0, 0};
    __device__ __forceinline__ void add(float c, float m, float l, const f32x4& x) {
        const float mn = fmaxf(M, m);
        const float ms = mn == kNegInf ? 0.0f : mn;
        const float f0 = exp2_raw((M - ms) * c), f1 = exp2_raw((m - ms) * c);
        L = L * f0 + f1 * l;
        o = o * f0 + f1 * x;
        M = mn;
    }
};

// Which ranges of a tile are joined: part, part + apart, ... (`parts` of them); into the
// tile's results, or (`again`) into the first one's place, to be joined with others.
struct Joined {
    int part, apart, parts;
    bool again;
};
// Joins them with the whole workgroup: every four outputs of a row are one thread's, or
// (few rows) several threads', each with every groups-th range, which then meet in LDS
// in order: the result does not depend on which range finished first.  A thread has loads of up to kJoinUnits of its outputs and kJoinParts ranges in
// flight at a time, as each is a round trip beyond this XCD's L2.
constexpr int kJoinUnits = 4, kJoinParts = 4, kJoinAlone = 8;
template <int D>
__device__ __forceinline__ void join_tile(const PagedParams& p, const Job& j, const Joined& of, unsigned char* lds) {
    const int left = j.req.n * p.G - j.row0;
    const int units = (left < j.tile ? left : j.tile) * (D / 4);
    auto place = [&](int nth, int e) { return j.slot + (int64_t)(of.part + nth * of.apart) * j.tile + e / (D / 4); };
    // Outputs first, first + kPagedThreads, ... (of `units`), over ranges from, from + step, ...
    auto join = [&](Merged (&y)[kJoinUnits], int first, int from, int step) {
        for (int s0 = from; s0 < of.parts; s0 += kJoinParts * step) {
            float2 ml[kJoinUnits][kJoinParts];
            f32x4 x[kJoinUnits][kJoinParts];
#pragma unroll
            for (int u = 0; u < kJoinUnits; ++u) {
                const int e = first + u * kPagedThreads;
                if (u && e >= units) break;
#pragma unroll
                for (int s = 0; s < kJoinParts; ++s) {
                    const int at = s0 + s * step;
                    const int64_t g = place(at < of.parts ? at : s0, e);
                    ml[u][s] = get_agent(p.ml + g);
                    x[u][s] = get_agent(p.part + g * D + 4 * (e % (D / 4)));
                }
            }
#pragma unroll
            for (int u = 0; u < kJoinUnits; ++u) {
                if (u && first + u * kPagedThreads >= units) break;
#pragma unroll
                for (int s = 0; s < kJoinParts; ++s)
                    if (s0 + s * step < of.parts) y[u].add(p.c, ml[u][s].x, ml[u][s].y, x[u][s]);
            }
        }
    };
    auto finish = [&](const Merged& y, int e) {
        if (of.again) {  // read by this thread alone, and its row's maximum and sum by this wave alone
            const int64_t g = place(0, e);
            put_agent(p.part + g * D + 4 * (e % (D / 4)), y.o);
            if (e % (D / 4) == 0) put_agent(p.ml + g, make_float2(y.M, y.L));
        } else {
            finish_row(p, j, j.row0 + e / (D / 4), D, 4 * (e % (D / 4)), y.o, y.M, y.L);
        }
    };
    int groups = 1;
    while (2 * groups * units <= kPagedThreads && groups < 8) groups *= 2;
    if (groups > 1) {
        const int g = threadIdx.x / units, e = threadIdx.x - g * units;
        Merged y[kJoinUnits];
        if (g < groups) join(y, e, g, groups);
        f32x4* lo = reinterpret_cast<f32x4*>(lds);
        float2* lml = reinterpret_cast<float2*>(lds + kPagedThreads * sizeof(f32x4));
        __syncthreads();
        lo[threadIdx.x] = y[0].o;
        lml[threadIdx.x] = make_float2(y[0].M, y[0].L);
        __syncthreads();
        if (g == 0) {
            for (int k = 1; k < groups; ++k) y[0].add(p.c, lml[e + k * units].x, lml[e + k * units].y, lo[e + k * units]);
            finish(y[0], e);
        }
        return;
    }
    for (int e = threadIdx.x; e < units; e += kJoinUnits * kPagedThreads) {
        Merged y[kJoinUnits];
        join(y, e, 0, 1);
#pragma unroll
        for (int u = 0; u < kJoinUnits; ++u)
            if (e + u * kPagedThreads < units) finish(y[u], e + u * kPagedThreads);
    }
}

template <int D>
constexpr size_t few_lds_bytes() {
    return (size_t)kPagedWaves * 32 * ((D + 4) * sizeof(float) + sizeof(float2));
}

// Jobs of few rows: 16 * MT rows of a head against one range of keys, the four waves 32
// keys at a time in turn.  Waves keep their own running maximum, sum and O and meet in
// LDS once, at the end.  Bound by reading K and V once a tile (4 * D bytes a key; 64
// requests of 300 to 16000 keys 383 to 392 us, 5.7 TB/s; one of 1000 keys 8 us, latency), so
// a wave's loads run ahead: K's registers are loaded again as soon as the scores are
// taken, V's as soon as the products are, and the page numbers of the step behind
// those are on their way meanwhile.  Weights go into the second product as bf16 parts,
// three of up to 16 rows: all 24 bits of them, nearly under the time of the reads (one
// request of 1000 keys 8.0 us, with two parts 7.9; 64 of 300 to 16000 keys 392 and 389;
// with two, 1.4 outputs in 1000 of the one request were not the bf16 nearest to the exact
// value, now 0.2).  Two of 32 rows, 16 bits: a third would cost 8 drafts of 16 rows 7%
// (32.4 -> 34.6 us) for 0.7 outputs in 1000.
template <int D, int MT>
__device__ __forceinline__ void few_rows(const PagedParams& p, const Job& job, unsigned char* lds) {
    constexpr int TR = 16 * MT;
    constexpr int KS = D / 32;
    constexpr int VD = D / 16;
    constexpr int PARTS = MT == 1 ? 3 : 2;  // of a weight
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n16 = lane & 15, q4 = lane >> 4;
    const int rows = job.req.n * p.G, row0 = job.row0;
    const int pos0 = job.req.len - job.req.n;  // of the request's first row
    const int last_row = row0 + TR - 1 < rows ? row0 + TR - 1 : rows - 1;
    auto position = [&](int row) { return pos0 + __builtin_amdgcn_readfirstlane(quotient(row, p.G, p.inv_G)); };
    const KeySpan<32> span(p, job.req.len, position(row0), position(last_row));
    const PagedRun kr(p, p.k, job, span.end), vr(p, p.v, job, span.end);
    const int t1 = (int)((int64_t)span.steps * (job.part + 1) / job.parts);
    int t = (int)((int64_t)span.steps * job.part / job.parts) + wave;

    KeyFrag<D> kf;
    ValueFrag<D> vf;
    auto load_k = [&](int kb, unsigned page) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const uint16_t* x = kr.row(kb + tile_key(u, n16), page) + 8 * q4;
#pragma unroll
            for (int s = 0; s < KS; ++s) kf.f[u][s] = load_cached16(x + 32 * s);
        }
    };
    auto load_v = [&](int kb, unsigned page) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            vf.f[i] = __builtin_nontemporal_load(
                reinterpret_cast<const typename ValueFrag<D>::vec*>(vr.row(kb + 8 * q4 + i, page) + VD * n16));
    };
    // Page numbers of the keys that this lane loads of the wave's next step and of the
    // one behind it (behind the range: of some step in it).
    auto k_page = [&](int t) { return kr.page_of(span.key(t < t1 ? t : t1 - 1) + 8 * (n16 >> 2)); };
    auto v_page = [&](int t) { return vr.page_of(span.key(t < t1 ? t : t1 - 1) + 8 * q4); };
    unsigned kp = 0, vp = 0;
    if (t < t1) {
        const unsigned kp0 = k_page(t), vp0 = v_page(t);
        kp = k_page(t + kPagedWaves);
        vp = v_page(t + kPagedWaves);
        load_k(span.key(t), kp0);
        load_v(span.key(t), vp0);
    }
    const int t_first = t;

    // This lane's rows (the last one again behind the end), and their q.
    u32x4 qf[MT][KS];
    int pos[MT], lo[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const int row = row0 + 16 * i + n16;
        const TileRow x(p, job, row < rows ? row : rows - 1);
        pos[i] = x.pos;
        lo[i] = x.lo;
        const uint16_t* qr = p.q + (int64_t)(job.req.row + x.r) * p.q_row + (int64_t)x.head * D + 8 * q4;
#pragma unroll
        for (int s = 0; s < KS; ++s) qf[i][s] = load_cached16(qr + 32 * s);
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
    // The last step without the loads for a next one, in code of its own: where loads may
    // have been left out the compiler waits as if they had, for V before it takes the
    // scores (8 drafts of 16 rows: 34.3 -> 32.5 us).
    auto step = [&](int t, auto more) {
        constexpr bool MORE = decltype(more)::value;
        const int kb = span.key(t);
        const int next = t + kPagedWaves;
        unsigned kp2 = 0, vp2 = 0;
        if constexpr (MORE) {
            kp2 = k_page(next + kPagedWaves);
            vp2 = v_page(next + kPagedWaves);
        }
        f32x4 s[MT][2];
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                s[i][u] = f32x4{0, 0, 0, 0};
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) s[i][u] = mfma16(kf.f[u][ks], qf[i][ks], s[i][u]);
            }
        if constexpr (MORE) load_k(span.key(next), kp);
        // What each row does not see gets no weight.
        if (!span.whole(kb, p.sinks)) {
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int key = kb + 8 * q4 + e;
                    s[i][e >> 2][e & 3] = row_sees(pos[i], lo[i], p.sinks, key) ? s[i][e >> 2][e & 3] : kNegInf;
                }
        }
        bf16x8 weight[MT][PARTS];
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
#pragma unroll
            for (int n = 0; n < PARTS; ++n) {
                u32x4 x;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    x[e] = pack_bf16(w[2 * e], w[2 * e + 1]);
                    const uint32_t y = x[e];
                    w[2 * e] -= bf16_to_f32(y & 0xffffu);  // what is left, exactly
                    w[2 * e + 1] -= __uint_as_float(y & 0xffff0000u);
                }
                weight[i][n] = __builtin_bit_cast(bf16x8, x);
            }
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
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int n = PARTS - 1; n >= 0; --n) acc[i][j] = mfma16(a, weight[i][n], acc[i][j]);
        }
        if constexpr (MORE) load_v(span.key(next), vp);
        kp = kp2;
        vp = vp2;
    };
    for (; t + kPagedWaves < t1; t += kPagedWaves) step(t, std::true_type{});
    if (t < t1) step(t, std::false_type{});
    if (any_odd) {  // rare, so key by key
#pragma unroll 1
        for (t = t_first; t < t1; t += kPagedWaves) {
            const int kb = span.key(t);
#pragma unroll 1
            for (int key = kb; key < kb + 32 && key < span.end; ++key) {
                const uint16_t* x = vr.row(key, vr.page_of(key)) + 4 * q4 * VD;
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int j = 0; j < VD; j += 2) {
                        const uint32_t y = *reinterpret_cast<const uint32_t*>(x + e * VD + j);
#pragma unroll
                        for (int i = 0; i < MT; ++i) {
                            const bool ok = row_sees(pos[i], lo[i], p.sinks, key);
                            acc[i][j][e] += ok ? odd_or_zero(y << 16) : 0.0f;
                            acc[i][j + 1][e] += ok ? odd_or_zero(y & 0xffff0000u) : 0.0f;
                        }
                    }
            }
        }
    }

    // The waves meet: O as [wave][row][D + 4] (rows 4 banks apart), maxima and
    // sums behind.
    constexpr int LD = D + 4;
    float* lo_o = reinterpret_cast<float*>(lds);
    float2* lo_ml = reinterpret_cast<float2*>(lds + (size_t)kPagedWaves * TR * LD * sizeof(float));
#pragma unroll
    for (int i = 0; i < MT; ++i) {
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
    constexpr int PER_ROW = D / 4, ROWS = kPagedThreads / PER_ROW;
    const int d = 4 * (threadIdx.x % PER_ROW);
#pragma unroll
    for (int i = 0; i < TR / ROWS; ++i) {
        const int n = i * ROWS + threadIdx.x / PER_ROW;
        float mw[kPagedWaves], M = kNegInf, L = 0.0f;
#pragma unroll
        for (int w = 0; w < kPagedWaves; ++w) {
            mw[w] = lo_ml[w * TR + n].x;
            M = fmaxf(M, mw[w]);
        }
        const float ms = M == kNegInf ? 0.0f : M;
        f32x4 x = {0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < kPagedWaves; ++w) {
            const float f = exp2_raw((mw[w] - ms) * p.c);
            L += f * lo_ml[w * TR + n].y;
            x += f * *reinterpret_cast<const f32x4*>(lo_o + ((size_t)w * TR + n) * LD + d);
        }
        if (row0 + n >= rows) continue;
        if (job.parts == 1) {
            finish_row(p, job, row0 + n, D, d, x, M, L);
        } else {  // for a workgroup of this launch, maybe on another XCD
            const int64_t g = job.slot + (int64_t)job.part * TR + n;
            put_agent(p.part + g * D + d, x);
            if (d == 0) put_agent(p.ml + g, make_float2(M, L));
        }
    }
}

// Whether this workgroup was the last of `all` at a counter.  (Through the front of lds,
// which nobody uses any more: the tile kernel's 80 KB are all that two workgroups of a
// CU can have.)
__device__ __forceinline__ bool last_of(const PagedParams& p, int counter, int all, unsigned char* lds) {
    int* last = reinterpret_cast<int*>(lds);
    drain_memory();
    __syncthreads();
    if (threadIdx.x == 0) {
        const uint32_t before = __hip_atomic_fetch_add(p.ctr + counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        *last = before == (uint32_t)all - 1;
        if (*last) __hip_atomic_store(p.ctr + counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    const bool yes = *last;
    __syncthreads();
    return yes;
}

// The ranges of a tile joined by the workgroups that finish last.  Many ranges of many
// rows would keep the last one busy by itself: about sqrt(parts) of them at a time are
// joined by the last of each such group, then those by the last group's (one request of
// 32 rows over 5200 keys, 21 ranges: 66 us, in two goes 58; 12 rows, 14 ranges: 22.5 and
// 19.7).
template <int D>
__device__ __forceinline__ void join_ranges(const PagedParams& p, const Job& job, unsigned char* lds) {
    int per = job.parts;
    if (job.parts > kJoinAlone && (job.req.n * p.G - job.row0) * (D / 4) > kPagedThreads / 2)
        for (per = 3; per * per < job.parts; ++per) {}
    const int group = job.part / per, groups = (job.parts + per - 1) / per;
    const int left = job.parts - group * per;
    Joined of = {group * per, 1, left < per ? left : per, groups > 1};
    int counter = job.counter(of.part);
    for (;;) {
        if (!last_of(p, counter, of.parts, lds)) return;
        join_tile<D>(p, job, of, lds);
        if (!of.again) return;
        of = {0, per, groups, false};
        counter = job.counter(1);  // no group begins there
    }
}

}  // namespace krk
