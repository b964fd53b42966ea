// How a call of attention over pages is cut into jobs: from the lengths on the device,
// and on the host the bounds of what they can come to (grid and workspace).  Arithmetic
// alone, no instructions of the GPU's but the reciprocal, so that a host program can
// replay it.
#pragma once

#include <stdint.h>

#include "krk_paged.h"

namespace krk {

struct PageView {
    const uint16_t* p;
    int64_t page, slot, head;
};

struct PlannedRange;
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
    int* planned;   // ranges that a launch in front listed: how many, and which (more than
    PlannedRange* plan;  // kLaneRequests requests)
    uint32_t* ctr;  // finished ranges of a tile
    float* part;    // [..][D] unnormalised outputs of ranges' rows
    float2* ml;     // [..] their running maximum (of q.k) and sum
    float scale;    // of q.k
    float c;        // scale * log2(e)
    int B, rows, heads, kv_heads, G, pages, shift, width, window, sinks;
    float inv_G, inv_kv;  // 1 / G, 1 / kv_heads
};

constexpr int kPagedThreads = 256;
constexpr int kPagedWaves = kPagedThreads / 64;

// Workgroups that the work is cut for: one a CU, though two run at once (for 512, ranges
// half as long: 4 drafts of 8 rows 19 -> 26 us, 100 rows over 16000 keys 84 -> 102, 500 over
// 4000 73 -> 77, 32 requests of 4000 keys 88 -> 95; two chunks beside 48 requests 278 -> 271).
constexpr int kTarget = 256;
constexpr int kFewPairs = 64;   // rows of a head that tiles of few rows (16 or 32) take
constexpr int kManyRows = 128;  // rows of a job of many
// Keys of a step of a workgroup, least steps of a range, and what a step costs, in us of
// one of two workgroups of a CU (of head size 128, and close enough for 64: many rows at 1.2
// or 3.0 change its mixed calls by 1 to 4%; only the proportion is of matter).
constexpr int kFewStep = 32 * kPagedWaves, kManyStep = 64;
constexpr int kFewLeast = 1, kManyLeast = 4;
// A tile of many steps has longer ranges at least, by one step for every kManyMore: each
// range's 64 KB is joined by one workgroup (one request of 32 rows over 5200 keys: 58 us
// in ranges of 4 steps, 48 of 6, 49 of 8; over 1000 keys of 20 rows 25, 27, 30).
constexpr int kManyMore = 32;
constexpr float kFewCost = 5.0f, kManyCost = 2.0f;
// Jobs that do not all run at once: where a share of the work is long, ranges of few
// rows are cut finer, into up to kRounds a workgroup of at least kGrain us each.
constexpr int kRounds = 4;
constexpr float kGrain = 25.0f;
// Tiles of more than one range have less than twice as many ranges as there are of the
// target's size.
constexpr int kFewSplits = 2 * kRounds * kTarget + 64, kManySplits = 2 * kTarget + 64;
// Counters of tiles, one for every 16 rows of results.  As many for every shape: they are
// at the front of a workspace that shapes may share, and partial results behind them.
constexpr size_t kCounterBytes = (size_t)(2 * kFewSplits + 8 * kManySplits) * sizeof(uint32_t);
static_assert(kCounterBytes % 256 == 0, "what follows is aligned");

// n / d by its reciprocal (off by one at most), then put right.
__device__ __forceinline__ int quotient(int n, int d, float inv) {
    int q = (int)((float)n * inv);
    const int r = n - q * d;
    return q + (r >= d) - (r < 0);
}

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

// How a request's rows of one head are cut: tiles of 1 << shift rows, over `steps` steps
// of keys at most.
struct Tiling {
    bool many;
    int shift, tiles, steps;
};
__device__ __forceinline__ Tiling tiling(const PagedParams& p, const Request& r) {
    Tiling t;
    const int rows = r.n * p.G;
    t.many = rows > kFewPairs;
    t.shift = t.many ? 7 : rows <= 16 ? 4 : 5;
    t.tiles = (rows + (1 << t.shift) - 1) >> t.shift;
    int keys = r.len;
    if (p.window) {
        const int of_tile = quotient(1 << t.shift, p.G, p.inv_G) + 2;  // positions of a tile's rows
        const int near = p.window + p.sinks + (r.n < of_tile ? r.n : of_tile) + kManyStep;
        keys = near < keys ? near : keys;
    }
    t.steps = t.many ? (keys + kManyStep - 1) / kManyStep : (keys + kFewStep - 1) / kFewStep;
    return t;
}

// How many steps a range has: all of a call's work over kTarget workgroups, and what
// follows from the jobs that this gives.
struct Ranges {
    int few, many;
    float inv_few, inv_many;
    // share: of a workgroup, in us.
    __device__ __forceinline__ explicit Ranges(float share) {
        few = at_least(share * (1.0f / kFewCost), kFewLeast);
        many = at_least(share * (1.0f / kManyCost), kManyLeast);
        inv_few = __builtin_amdgcn_rcpf((float)few);
        inv_many = __builtin_amdgcn_rcpf((float)many);
    }
    // A few jobs too many would run by themselves behind the others: either ranges that
    // long that all run at once, or, where they are long, short ones.
    __device__ __forceinline__ void cut_anew(float share, int jobs) {
        float rounds = floorf(share * (1.0f / kGrain));
        rounds = rounds > (float)kRounds ? (float)kRounds : rounds;
        few = rounds >= 2.0f ? at_least(share / (kFewCost * rounds), kFewLeast) : at_least((float)few * (float)jobs * (1.0f / kTarget), kFewLeast);
        inv_few = __builtin_amdgcn_rcpf((float)few);
    }
    static __device__ __forceinline__ int at_least(float steps, int least) {
        const int n = (int)fminf(steps, 1e9f) + 1;
        return n > least ? n : least;
    }
    __device__ __forceinline__ int parts(const Tiling& t) const {
        const int least = kManyLeast + t.steps / kManyMore;
        const bool longer = t.many && least > many;
        const int len = longer ? least : t.many ? many : few;
        const float inv = longer ? __builtin_amdgcn_rcpf((float)least) : t.many ? inv_many : inv_few;
        return t.steps > len ? (int)((float)(t.steps - 1) * inv) + 1 : 1;
    }
};
// In floating point: 2^18 tiles of 2^21 steps pass 31 bits, and the bounds of make_plan
// rest on the sum of these.
__device__ __forceinline__ float cost_of(const Tiling& t) { return (float)t.tiles * (float)t.steps * (t.many ? kManyCost : kFewCost); }

// The nth of `many` jobs of many rows and `few` of few, by its number in the call: blocks
// of 1 << block of the one, which keep the matrix pipe busy, and of the other, which read,
// in turn, so that a CU has one of each; then what is left of the many and of the few.
struct Nth {
    bool many;
    int n;
    __device__ __forceinline__ Nth(int id, int all_many, int all_few, int block) {
        const int both = (all_many < all_few ? all_many : all_few) >> block;
        many = !(id >> block & 1);
        n = (id >> (block + 1) << block) + (id & ((1 << block) - 1));
        if (id >= both << (block + 1)) {
            n = id - (both << block);
            many = n < all_many;
            n = many ? n : id - all_many;
        }
    }
};

// Calls of up to as many requests: each wave works its job out from the lengths, a lane
// a request.
constexpr int kLaneRequests = 64;

struct PlannedRange {
    int b, row0, parts_part, slot;  // parts << 16 | part; row of results of the tile's ranges of head 0
};

// Bounds for a shape, whatever its calls' lengths.
struct Plan {
    bool many;  // some request may have more than kFewPairs rows of a head
    int64_t blocks;
    size_t ctr, part, ml, plan, bytes;  // workspace: sizes of its parts and their sum
};

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

inline Plan make_plan(const krk_paged_shape& s) {
    Plan p{};
    const int64_t RG = (int64_t)s.rows * (s.heads / s.kv_heads);
    p.many = RG > kFewPairs;
    // A request with rows has up to two tiles where they are few, of 16 rows or more but
    // for the last; else tiles of 128.
    const int64_t live = s.B < s.rows ? s.B : s.rows;
    const int64_t tiles = s.kv_heads * (RG / kManyRows + (live < RG / 16 ? 2 * live : live + RG / 16));
    // Their key ranges: as many as the longest request could have, and those of tiles
    // that have several are limited.
    const int64_t keys = (int64_t)s.width * s.page_size;
    auto splits = [&](int64_t least, int64_t most) {
        const int64_t parts = ceil_div(keys, least);
        return parts < 2 ? 0 : tiles * parts < most ? tiles * parts : most;
    };
    const int64_t few = splits(kFewStep * kFewLeast, kFewSplits);
    const int64_t many = p.many ? splits(kManyStep * kManyLeast, kManySplits) : 0;
    p.blocks = tiles + few + many;
    const size_t rows = (size_t)(few * 32 + many * kManyRows);
    p.part = rows * s.head_dim * sizeof(float);
    p.ml = rows * sizeof(float2);
    if (s.B > kLaneRequests) p.plan = 256 + (size_t)ceil_div(p.blocks, s.kv_heads) * sizeof(PlannedRange);
    if (rows || p.plan) p.ctr = kCounterBytes;  // also where this shape counts nothing: they stay zero
    p.bytes = p.ctr + p.part + p.ml + p.plan;
    return p;
}

}  // namespace krk
