// How a call of attention over pages is cut into jobs, replayed on the host with the
// library's own arithmetic (csrc/krk_paged_cut.h): every job has to come up once, within
// the grid, the results' rows and the counters that the library provides.
#include <math.h>
#include <stddef.h>
#include <stdint.h>

#include <vector>

#define __host__
#define __device__
#define __forceinline__ inline
struct float2 {
    float x, y;
};
static inline float __builtin_amdgcn_rcpf(float x) { return 1.0f / x; }
#include "krk_paged_cut.h"

using namespace krk;

enum { BLOCKS, ROWS, COUNTERS, JOBS, USED, PAIRS, ROUNDS, FEW_PARTS, MANY_PARTS, WRONG, FIELDS };

// nudge: what the sum of the costs is multiplied with, as the GPU adds them in another order.
extern "C" int replay(const krk_paged_shape* s, const int32_t* starts, const int32_t* keys, float nudge, int64_t* out) {
    const Plan plan = make_plan(*s);
    PagedParams p{};
    p.starts = starts;
    p.keys = keys;
    p.B = s->B;
    p.rows = s->rows;
    p.heads = s->heads;
    p.kv_heads = s->kv_heads;
    p.G = s->heads / s->kv_heads;
    p.inv_G = 1.0f / (float)p.G;
    p.inv_kv = 1.0f / (float)s->kv_heads;
    p.width = s->width;
    p.window = s->window;
    p.sinks = s->sinks;
    while (1 << p.shift < s->page_size) ++p.shift;
    const bool lanes = s->B <= kLaneRequests;
    const int per_tile = lanes ? p.kv_heads : 1;  // the plan in front lists ranges, of which each head is a job

    std::vector<Tiling> t(s->B);
    float share = 0.0f;
    for (int b = 0; b < s->B; ++b) {
        t[b] = tiling(p, request(p, b));
        share += cost_of(t[b]);
    }
    share *= nudge * (float)p.kv_heads * (1.0f / kTarget);
    Ranges ranges(share);
    std::vector<int64_t> first(s->B), row(s->B);
    std::vector<int> parts(s->B);
    int64_t all[2], used;  // of few, of many
    auto count = [&]() {
        all[0] = all[1] = used = 0;
        for (int b = 0; b < s->B; ++b) {
            parts[b] = ranges.parts(t[b]);
            first[b] = all[t[b].many];
            row[b] = used;
            const int64_t n = (int64_t)t[b].tiles * per_tile * parts[b];
            all[t[b].many] += n;
            used += parts[b] > 1 ? (int64_t)t[b].tiles * p.kv_heads * parts[b] << t[b].shift : 0;
        }
    };
    count();
    out[ROUNDS] = 0;
    const int64_t heads = lanes ? 1 : p.kv_heads;
    if ((all[0] + all[1]) * heads > kTarget && all[0]) {
        ranges.cut_anew(share, (int)((all[0] + all[1]) * heads));
        count();
        out[ROUNDS] = share / kGrain >= 2.0f ? 2 : 1;
    }
    int block = 8;
    while (!lanes && block > 0 && (p.kv_heads << block) > 256) --block;
    const int64_t listed = all[0] + all[1];
    out[BLOCKS] = plan.blocks;
    out[ROWS] = (int64_t)(plan.ml / sizeof(float2));
    out[COUNTERS] = (int64_t)(plan.ctr / sizeof(uint32_t));
    out[JOBS] = listed * heads;
    out[USED] = used;
    out[PAIRS] = (all[0] < all[1] ? all[0] : all[1]) >> block;
    out[FEW_PARTS] = out[MANY_PARTS] = out[WRONG] = 0;
    for (int b = 0; b < s->B; ++b) {
        int64_t& most = out[t[b].many ? MANY_PARTS : FEW_PARTS];
        most = parts[b] > most && t[b].tiles ? parts[b] : most;
    }
    if (listed > plan.blocks) return 0;
    // Which ranges the numbers stand for: each of a request's tiles, heads and parts once.
    std::vector<unsigned char> seen(listed, 0);
    std::vector<int> of_kind[2];
    for (int b = 0; b < s->B; ++b)
        if (t[b].tiles) of_kind[t[b].many].push_back(b);
    for (int64_t e = 0; e < listed; ++e) {
        const Nth nth((int)e, (int)all[1], (int)all[0], block);
        const std::vector<int>& who = of_kind[nth.many];
        if (nth.n < 0 || nth.n >= all[nth.many]) {
            ++out[WRONG];
            continue;
        }
        size_t lo = 0, hi = who.size();
        while (hi - lo > 1) (first[who[(lo + hi) / 2]] <= nth.n ? lo : hi) = (lo + hi) / 2;
        const int b = who[lo], place = (int)(nth.n - first[b]);
        const int over_heads = quotient(place, per_tile, 1.0f / (float)per_tile), h = place - over_heads * per_tile;
        const int tile = quotient(over_heads, parts[b], __builtin_amdgcn_rcpf((float)parts[b])), part = over_heads - tile * parts[b];
        if (h < 0 || h >= per_tile || tile < 0 || tile >= t[b].tiles || part < 0 || part >= parts[b] || parts[b] > 0x7fff) {
            ++out[WRONG];
            continue;
        }
        const int64_t at = (nth.many ? 0 : all[1]) + first[b] + ((int64_t)tile * per_tile + h) * parts[b] + part;
        out[WRONG] += seen[at]++ != 0;
        if (parts[b] > 1) {
            const int64_t slot = row[b] + ((int64_t)(tile * p.kv_heads + (lanes ? h : p.kv_heads - 1)) * parts[b] << t[b].shift);
            const int64_t end = slot + ((int64_t)parts[b] << t[b].shift);
            out[WRONG] += end > out[ROWS] || (end - 1) >> 4 >= out[COUNTERS];
        }
    }
    return 0;
}
