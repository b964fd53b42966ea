// C ABI of the cache operators (declared in include/krk_attn.h): argument
// checks, how the work is cut, and stream-ordered launches.  Nothing here
// allocates, synchronises or touches device memory from the host, so every
// call is graph-capturable.
#include <hip/hip_runtime.h>
#include <stdarg.h>
#include <stdint.h>
#include <stdio.h>

#include <atomic>
#include <utility>

#include "krk_attn.h"
#include "krk_attn_split.h"
#include "krk_attn_tile.h"
#include "krk_evict.h"
#include "krk_rope.h"

namespace {

thread_local char g_err[512] = "";

int fail(int code, const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_err, sizeof g_err, fmt, ap);
    va_end(ap);
    return code;
}

constexpr int kCuCount = 256;  // MI355X: 8 XCDs x 32 CUs
constexpr int64_t kMaxStride = (int64_t)1 << 40;

inline int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline size_t align_up(size_t v, size_t a) { return (v + a - 1) / a * a; }

int hip_status(hipError_t e, const char* what) {
    if (e == hipSuccess) return KRK_ATTN_OK;
    return fail(KRK_ATTN_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
}

// Raise a kernel's dynamic-LDS limit on the current device, once per device
// and kernel.
hipError_t ensure_lds_limit(const void* fn, size_t bytes, std::atomic<uint64_t>& done) {
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess) return e;
    const uint64_t bit = dev < 64 ? (1ull << dev) : 0;
    if (bit && (done.load(std::memory_order_acquire) & bit)) return hipSuccess;
    e = hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e == hipSuccess && bit) done.fetch_or(bit, std::memory_order_acq_rel);
    return e;
}

// ------------------------------------------------------------------ checks
struct Span {
    uintptr_t a, b;
};
bool overlaps(const Span& x, const Span& y) { return x.a < y.b && y.a < x.b; }
Span span(const void* p, uint64_t elems, size_t size) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(p);
    return p ? Span{a, a + elems * size} : Span{0, 0};
}

// Whether no two elements of a written operand share memory: sorted by stride,
// each is at least the extent of those inside it.  (Strides of extents of one
// are 0.)
bool nested(const int64_t (&stride)[3], const int64_t (&n)[3], int64_t inner) {
    int at[3] = {0, 1, 2};
    for (int i = 0; i < 3; ++i)
        for (int j = i + 1; j < 3; ++j)
            if (stride[at[j]] < stride[at[i]]) std::swap(at[i], at[j]);
    for (int i : at) {
        if (n[i] > 1 && stride[i] < inner) return false;
        inner += (n[i] - 1) * stride[i];
    }
    return true;
}

// A cache of `seqs` sequences, `slots` keys, `heads` heads of `dim`.  Strides
// of extents of one are of no matter and set to 0.
int check_cache(const char* name, krk_cache& c, int64_t seqs, int64_t slots, int64_t heads, int dim, bool written,
                Span* out) {
    if (!c.p) return fail(KRK_ATTN_ERR_INVALID, "%s: null pointer", name);
    if (seqs == 1) c.seq = 0;
    if (slots == 1) c.slot = 0;
    if (heads == 1) c.head = 0;
    const int64_t st[3] = {c.seq, c.slot, c.head}, n[3] = {seqs, slots, heads};
    for (int i = 0; i < 3; ++i) {
        if (st[i] < 0 || st[i] > kMaxStride) return fail(KRK_ATTN_ERR_INVALID, "%s: stride %lld out of range", name, (long long)st[i]);
        if (written && n[i] > 1 && st[i] < dim)
            return fail(KRK_ATTN_ERR_INVALID, "%s is written: its strides must be at least head_dim=%d, got %lld", name, dim, (long long)st[i]);
        if (st[i] % 8) return fail(KRK_ATTN_ERR_ALIGN, "%s: strides must be multiples of 8 elements", name);
    }
    if (written && !nested(st, n, dim))
        return fail(KRK_ATTN_ERR_ALIAS, "%s is written: with strides of %lld, %lld and %lld its rows share memory", name, (long long)st[0], (long long)st[1], (long long)st[2]);
    if (reinterpret_cast<uintptr_t>(c.p) % 16) return fail(KRK_ATTN_ERR_ALIGN, "%s must be 16-byte aligned", name);
    *out = span(c.p, (uint64_t)((seqs - 1) * c.seq + (slots - 1) * c.slot + (heads - 1) * c.head + dim), 2);
    return KRK_ATTN_OK;
}

// Whether two written caches of one shape share memory.  Views whose spans meet
// (k and v side by side in one tensor) have to have the same strides; they are
// apart if no step from a row of one to a row of the other is shorter than a row.
// A step's part along the largest stride is one of the two multiples next to it,
// as what is left has to lie within the extent inside that stride.
bool apart(int64_t d, const int64_t (&stride)[3], const int64_t (&n)[3], int dim, int level = 0) {
    if (level == 3) return d <= -dim || d >= dim;
    const int64_t s = stride[level];
    if (s == 0) return apart(d, stride, n, dim, level + 1);
    int64_t q = d / s;
    if (q * s > d) --q;
    for (int64_t i = q; i <= q + 1; ++i)
        if (i > -n[level] && i < n[level] && !apart(d - i * s, stride, n, dim, level + 1)) return false;
    return true;
}
bool share_memory(const krk_cache& x, const Span& xs, const krk_cache& y, const Span& ys, int64_t seqs, int64_t slots, int64_t heads,
                  int dim) {
    if (!overlaps(xs, ys)) return false;
    if (x.seq != y.seq || x.slot != y.slot || x.head != y.head) return true;
    const intptr_t bytes = reinterpret_cast<intptr_t>(y.p) - reinterpret_cast<intptr_t>(x.p);
    int64_t stride[3] = {x.seq, x.slot, x.head}, n[3] = {seqs, slots, heads};
    for (int i = 0; i < 3; ++i)
        for (int j = i + 1; j < 3; ++j)
            if (stride[j] > stride[i]) {
                std::swap(stride[i], stride[j]);
                std::swap(n[i], n[j]);
            }
    return !apart(bytes / 2, stride, n, dim);
}

// [rows, cols] operand; one row's stride is of no matter and set to its length.
int check_rows(const char* name, const void* p, int64_t& row, int64_t rows, int64_t cols, Span* out) {
    if (rows == 1) row = cols;
    if (!p) return fail(KRK_ATTN_ERR_INVALID, "%s: null pointer", name);
    if (row < cols || row > kMaxStride) return fail(KRK_ATTN_ERR_INVALID, "%s: row stride %lld must be >= %lld", name, (long long)row, (long long)cols);
    if (row % 8) return fail(KRK_ATTN_ERR_ALIGN, "%s: the row stride must be a multiple of 8 elements", name);
    if (reinterpret_cast<uintptr_t>(p) % 16) return fail(KRK_ATTN_ERR_ALIGN, "%s must be 16-byte aligned", name);
    *out = span(p, (uint64_t)((rows - 1) * row + cols), 2);
    return KRK_ATTN_OK;
}

int check_scores(const char* name, const void* p, int64_t& seq, int64_t& head, int64_t seqs, int64_t heads, int64_t slots,
                 bool written, Span* out) {
    if (!p) return fail(KRK_ATTN_ERR_INVALID, "%s: null pointer", name);
    if (seqs == 1) seq = 0;
    if (heads == 1) head = 0;
    if (seq < 0 || head < 0 || seq > kMaxStride || head > kMaxStride)
        return fail(KRK_ATTN_ERR_INVALID, "%s: strides out of range", name);
    if (written && ((seqs > 1 && seq < slots) || (heads > 1 && head < slots)))
        return fail(KRK_ATTN_ERR_INVALID, "%s is written: its strides must be at least its %lld slots", name, (long long)slots);
    if (written && !nested({seq, head, 0}, {seqs, heads, 1}, slots))
        return fail(KRK_ATTN_ERR_ALIAS, "%s is written: with strides of %lld and %lld its rows share memory", name, (long long)seq, (long long)head);
    if (reinterpret_cast<uintptr_t>(p) % 4) return fail(KRK_ATTN_ERR_ALIGN, "%s must be 4-byte aligned", name);
    *out = span(p, (uint64_t)((seqs - 1) * seq + (heads - 1) * head + slots), 4);
    return KRK_ATTN_OK;
}

int check_layout(int B, int R, int heads, int kv_heads, int head_dim, int capacity) {
    if (B < 1 || R < 1 || kv_heads < 1 || heads < 1 || capacity < 1)
        return fail(KRK_ATTN_ERR_INVALID, "B=%d R=%d heads=%d kv_heads=%d capacity=%d must all be >= 1", B, R, heads, kv_heads, capacity);
    if (B > 65535 || kv_heads > 65535 || R > 65536) return fail(KRK_ATTN_ERR_INVALID, "B=%d, kv_heads=%d (most 65535) or R=%d (most 65536) too large", B, kv_heads, R);
    if (heads % kv_heads) return fail(KRK_ATTN_ERR_INVALID, "heads=%d must be a multiple of kv_heads=%d", heads, kv_heads);
    if (head_dim != 64 && head_dim != 128) return fail(KRK_ATTN_ERR_UNSUPPORTED, "head_dim=%d: this build has 64 and 128", head_dim);
    // Grids of up to 128 threads a row, or 256 a sequence and head, stay below 2^32 threads.
    if ((int64_t)B * R * heads >= ((int64_t)1 << 25)) return fail(KRK_ATTN_ERR_INVALID, "B * R * heads = %lld must be below 2^25", (long long)((int64_t)B * R * heads));
    if ((int64_t)B * kv_heads >= ((int64_t)1 << 23)) return fail(KRK_ATTN_ERR_INVALID, "B * kv_heads = %lld must be below 2^23", (long long)((int64_t)B * kv_heads));
    if (capacity >= 1 << 27) return fail(KRK_ATTN_ERR_INVALID, "capacity=%d must be below 2^27", capacity);
    return KRK_ATTN_OK;
}

int check_shape(const krk_attn_shape& s) {
    if (int rc = check_layout(s.B, s.R, s.heads, s.kv_heads, s.head_dim, s.capacity)) return rc;
    if (s.window >= 1 << 28 || s.sinks >= 1 << 28) return fail(KRK_ATTN_ERR_INVALID, "window=%d and sinks=%d must be below 2^28", s.window, s.sinks);
    if (s.window < 0 || s.sinks < 0 || s.prefix < 0) return fail(KRK_ATTN_ERR_INVALID, "window=%d, sinks=%d and prefix=%d must not be negative", s.window, s.sinks, s.prefix);
    if ((int64_t)s.prefix + s.capacity >= 1 << 27) return fail(KRK_ATTN_ERR_INVALID, "prefix + capacity must be below 2^27");
    if (s.sinks && !s.window) return fail(KRK_ATTN_ERR_INVALID, "sinks need a window");
    if (s.scored != 0 && s.scored != 1) return fail(KRK_ATTN_ERR_INVALID, "scored must be 0 or 1, got %d", s.scored);
    if (s.scored && s.prefix) return fail(KRK_ATTN_ERR_INVALID, "scores are not kept with a shared prefix");
    return KRK_ATTN_OK;
}

// -------------------------------------------------------------------- plan
// Rows of a workgroup: 16 or 32 on the split kernel (its waves share the rows
// and divide the keys), 128 on the tile kernel (the other way round).
struct Cut {
    int rows, tiles, splits;
};

struct Plan {
    Cut own, prefix;
    int64_t all_rows;
    bool join_in_kernel;
    bool join_prefix;  // the own caches' launch joins the prefix's ranges
    bool keep_raw;  // scored: q.k goes through the workspace instead of K being read again
    int64_t raw_row;
    size_t ctr, part, ml, stat, raw, bytes;  // workspace: sizes of its parts and their sum
};

// Key ranges of the tile kernel, where a range costs: its partial results are
// written and read at 8 * D bytes a row.  Measured, in us: 6 and 1.45 a step (D =
// 64: 1.05) for up to 512 workgroups, 4 for the join and the partial results at
// 3.5 TB/s.  s ranges then take 6 + T / s + 4 + C * s, least at sqrt(T / C), but
// not more than 512 workgroups, and not so many that only some CUs have two
// (3500 rows of 4 heads: 56 us in 2 ranges, 51 in 4; 2000 rows of 32 heads: 91 in
// one, 126 in 2; 100 rows of 32 heads over 4000 keys: 39 in 4, 33 in 8 and 16).
int tile_splits(int64_t rows, int64_t tiles, int64_t keys, int D) {
    const double T = (double)cdiv(keys, krk::kTileStep) * (D == 128 ? 1.45 : 1.05);
    const double C = (double)rows * D * 8 / 3.5e6;
    const int64_t full = 2 * kCuCount / tiles, half = kCuCount / tiles;
    const int64_t most = cdiv(keys, 4 * krk::kTileStep);
    int64_t s = (int64_t)__builtin_sqrt(T / C);
    s = s < full ? s : full;
    if (s < full && s > half) s = half;
    s = s < most ? s : most;
    return s > 1 && T / s + 4 + C * s < T ? (int)s : 1;
}

// `lists` row lists of `rows` rows each, over at most `keys` keys.  Key ranges of
// the split kernel: one workgroup per CU, which is enough to draw 6 TB/s (32
// sequences with windows of 4096 keys: 89 us in one range, 96 in two, 101 in six;
// of 2000 to 4000 keys: 80, 85 and 87).  But a step for every wave at least.  The
// lengths are not known here: the longest of many sequences takes as long as it
// would alone in as many ranges (32 of 1000 keys 24 us, with one of 32000 among them
// 372; 8 of 1000 12, with one of 32000 101), and a capacity far above the length
// costs ranges of one step (1000 keys in 1024 slots 9.0 us, in 4096 or more 11.3).
Cut make_cut(int64_t rows, int64_t lists, int64_t keys, int D) {
    Cut c;
    c.rows = rows <= 16 ? 16 : rows <= 64 ? 32 : krk::kTileRows;
    c.tiles = (int)cdiv(rows, c.rows);
    if (c.rows == krk::kTileRows) {
        c.splits = tile_splits(rows * lists, lists * c.tiles, keys, D);
        return c;
    }
    const int64_t want = cdiv(kCuCount, lists * c.tiles);
    const int64_t most = cdiv(keys, 32 * krk::kSplitWaves);
    c.splits = (int)(want < most ? want : most);
    return c;
}

Plan make_plan(const krk_attn_shape& s) {
    Plan p{};
    const int64_t RG = (int64_t)s.R * (s.heads / s.kv_heads);
    p.all_rows = RG * s.B * s.kv_heads;
    int64_t keys = s.capacity;
    if (s.window) {
        const int64_t G = s.heads / s.kv_heads, span = krk::kTileRows / G + 2;  // positions of a workgroup's rows
        const int64_t near = (int64_t)s.window + s.sinks + (s.R < span ? s.R : span) + 64;
        keys = near < keys ? near : keys;
    }
    if (s.prefix) p.prefix = make_cut(RG * s.B, s.kv_heads, s.prefix, s.head_dim);
    p.own = make_cut(RG, (int64_t)s.B * s.kv_heads, keys, s.head_dim);
    const int n = p.own.splits + p.prefix.splits;
    if (n > 1) {
        // One workgroup joins a sequence's head: up to 96 KB of partial results.
        // Not behind a prefix: the workgroup that finishes its last range would
        // join all sequences of its rows, one after the other (8 of them, 8 us).
        p.join_in_kernel = p.own.rows <= 32 && !s.prefix && RG * n * s.head_dim <= 24 << 10;
        // A launch of its own behind the prefix's anyway, in whole caches of up to 16
        // rows a head: it reads the prefix's ranges under its first keys' loads (64
        // sequences over 32768 shared keys: 91 us a call, 98 with a join behind).
        p.join_prefix = p.prefix.rows == krk::kTileRows && p.own.rows == 16 && p.own.splits == 1;
        p.part = align_up((size_t)n * p.all_rows * s.head_dim * sizeof(float), 256);
        p.ml = align_up((size_t)n * p.all_rows * sizeof(float2), 256);
    }
    if (s.scored) {
        p.stat = align_up((size_t)p.all_rows * sizeof(float2), 256);
        p.keep_raw = p.own.rows == 16 && s.window == 0;
        p.raw_row = (int64_t)align_up((size_t)s.capacity, 32);
        if (p.keep_raw) p.raw = align_up((size_t)p.all_rows * p.raw_row * sizeof(float), 256);
    }
    p.bytes = p.part + p.ml + p.stat + p.raw;
    // The counters have their place whether this shape uses them or not: shapes of one
    // B and kv_heads may then share a workspace without filling it again.
    if (p.bytes) p.ctr = align_up((size_t)s.B * s.kv_heads * sizeof(uint32_t), 256);
    p.bytes += p.ctr;
    return p;
}

// ---------------------------------------------------------------- launches
template <int D, int MTO, int MTP, bool JOIN = false>
int launch_split(const krk::AttnParams& p, int64_t blocks, hipStream_t stream) {
    static std::atomic<uint64_t> done{0};
    const void* fn = reinterpret_cast<const void*>(&krk::attn_split_kernel<D, MTO, MTP, JOIN>);
    const size_t shm = krk::split_lds_bytes<D, (MTO > MTP ? MTO : MTP)>();
    if (hipError_t e = ensure_lds_limit(fn, shm, done)) return hip_status(e, "attn_split_kernel LDS size");
    void* args[] = {(void*)&p};
    return hip_status(hipLaunchKernel(fn, dim3((unsigned)blocks), dim3(krk::kSplitThreads), args, shm, stream), "attn_split_kernel launch");
}

template <int D>
int launch_tile(const krk::AttnParams& p, int64_t blocks, hipStream_t stream) {
    static std::atomic<uint64_t> done{0};
    const void* fn = reinterpret_cast<const void*>(&krk::attn_tile_kernel<D>);
    const size_t lds = krk::tile_lds_bytes<D>();
    if (hipError_t e = ensure_lds_limit(fn, lds, done)) return hip_status(e, "attn_tile_kernel LDS size");
    void* args[] = {(void*)&p};
    return hip_status(hipLaunchKernel(fn, dim3((unsigned)blocks), dim3(krk::kTileThreads), args, lds, stream), "attn_tile_kernel launch");
}

template <int D>
int launch_attn(krk::AttnParams p, const Plan& plan, hipStream_t stream) {
    const int64_t own = (int64_t)plan.own.tiles * p.kv_heads * p.B * plan.own.splits;
    const int64_t shared = (int64_t)plan.prefix.tiles * p.kv_heads * plan.prefix.splits;
    void* args[] = {(void*)&p};
    int rc;
    if (plan.own.rows == krk::kTileRows) {
        rc = launch_tile<D>(p, own + shared, stream);
    } else if (plan.prefix.rows == krk::kTileRows) {
        // Two launches: one of both kinds of workgroups was no faster (they
        // share CUs at the register and LDS cost of the larger kind).
        rc = launch_tile<D>(p, shared, stream);
        krk::AttnParams o = p;
        o.prefix_row_tiles = 0;
        if (!rc) {
            if (plan.own.rows == 32) rc = launch_split<D, 2, 2>(o, own, stream);
            else if (plan.join_prefix) rc = launch_split<D, 1, 1, true>(o, own, stream);
            else rc = launch_split<D, 1, 1>(o, own, stream);
        }
    } else if (plan.own.rows == 32) {
        rc = launch_split<D, 2, 2>(p, own + shared, stream);
    } else if (plan.prefix.rows == 32) {
        rc = launch_split<D, 1, 2>(p, own + shared, stream);
    } else {
        rc = launch_split<D, 1, 1>(p, own + shared, stream);
    }
    if (rc) return rc;
    if (plan.own.splits + plan.prefix.splits > 1 && !plan.join_in_kernel && !plan.join_prefix) {
        const hipError_t e = hipLaunchKernel(reinterpret_cast<const void*>(&krk::attn_join_kernel<D>),
                                             dim3((unsigned)cdiv(plan.all_rows, 256 / (D / 4) / krk::kGroups)), dim3(256), args, 0, stream);
        if (int rc = hip_status(e, "attn_join_kernel launch")) return rc;
    }
    if (plan.keep_raw) {
        const hipError_t e = hipLaunchKernel(reinterpret_cast<const void*>(&krk::attn_weights_raw_kernel),
                                             dim3((unsigned)cdiv(p.capacity, 1024), p.kv_heads, p.B), dim3(256), args, 0, stream);
        if (int rc = hip_status(e, "attn_weights_raw_kernel launch")) return rc;
    } else if (p.stat) {
        const hipError_t e = hipLaunchKernel(reinterpret_cast<const void*>(&krk::attn_weights_kernel<D>),
                                             dim3((unsigned)cdiv(p.capacity, 128), p.kv_heads, p.B), dim3(256), args, 0, stream);
        if (int rc = hip_status(e, "attn_weights_kernel launch")) return rc;
    }
    return KRK_ATTN_OK;
}

// By how many keys a lane holds: time and code grow with it (1024 slots on the
// 36-key kernel: 13.7 us, on the 4-key one 7).
const void* select_kernel(int capacity) {
    if (capacity <= 4 * krk::kEvictThreads) return reinterpret_cast<const void*>(&krk::evict_select_kernel<4>);
    if (capacity <= 12 * krk::kEvictThreads) return reinterpret_cast<const void*>(&krk::evict_select_kernel<12>);
    if (capacity <= 36 * krk::kEvictThreads) return reinterpret_cast<const void*>(&krk::evict_select_kernel<36>);
    return reinterpret_cast<const void*>(&krk::evict_select_kernel<0>);
}

krk::CacheView view(const krk_cache& c) { return {static_cast<const uint16_t*>(c.p), c.seq, c.slot, c.head}; }

}  // namespace

extern "C" {

int krk_attn_abi_version(void) { return KRK_ATTN_ABI_VERSION; }

size_t krk_attn_struct_size(int which) {
    switch (which) {
        case 0: return sizeof(krk_attn_shape);
        case 1: return sizeof(krk_attn_args);
        case 2: return sizeof(krk_rope_args);
        case 3: return sizeof(krk_evict_args);
        case 4: return sizeof(krk_attn_plan_t);
        default: return 0;
    }
}

const char* krk_attn_last_error(void) { return g_err; }

int krk_attn_check(const krk_attn_shape* shape) {
    g_err[0] = '\0';
    if (!shape) return fail(KRK_ATTN_ERR_INVALID, "null shape");
    return check_shape(*shape);
}

size_t krk_attn_workspace_bytes(const krk_attn_shape* shape) {
    g_err[0] = '\0';
    if (!shape || check_shape(*shape)) return 0;
    return make_plan(*shape).bytes;
}

int krk_attn_plan(const krk_attn_shape* shape, krk_attn_plan_t* out) {
    g_err[0] = '\0';
    if (!shape || !out) return fail(KRK_ATTN_ERR_INVALID, "null argument");
    if (int rc = check_shape(*shape)) return rc;
    const Plan p = make_plan(*shape);
    *out = krk_attn_plan_t{p.own.rows, p.own.splits, p.prefix.rows, p.prefix.splits};
    return KRK_ATTN_OK;
}

int krk_attn_bf16(const krk_attn_shape* shape, const krk_attn_args* args, void* workspace, size_t workspace_bytes,
                  void* stream) {
    g_err[0] = '\0';
    if (!shape || !args) return fail(KRK_ATTN_ERR_INVALID, "null shape or args");
    const krk_attn_shape& s = *shape;
    krk_attn_args a = *args;
    if (int rc = check_shape(s)) return rc;
    if (a.prefix < 0 || a.prefix > s.prefix) return fail(KRK_ATTN_ERR_INVALID, "prefix=%d keys, the shape has 0 .. %d", a.prefix, s.prefix);
    // The kernels multiply by scale * log2(e).
    const float scale_log2 = (float)((double)a.scale * 1.4426950408889634);
    if (!(a.scale > 0.0f) || scale_log2 == __builtin_inff())
        return fail(KRK_ATTN_ERR_INVALID, "scale=%g must be positive and at most 2.3e38", (double)a.scale);
    if (!a.lens) return fail(KRK_ATTN_ERR_INVALID, "lens: null pointer");
    if (a.tree && (s.R > 64 || (s.window && s.window < s.R)))
        return fail(KRK_ATTN_ERR_INVALID, "tree masks need R <= 64 and a window of 0 or >= R, got R=%d window=%d", s.R, s.window);
    const int64_t M = (int64_t)s.B * s.R, cols = (int64_t)s.heads * s.head_dim;
    constexpr int kIn = 8;
    Span in[kIn] = {}, out, lse{}, sco{};
    if (int rc = check_rows("q", a.q, a.q_row, M, cols, &in[0])) return rc;
    if (int rc = check_rows("out", a.out, a.out_row, M, cols, &out)) return rc;
    if (int rc = check_cache("k", a.k, s.B, s.capacity, s.kv_heads, s.head_dim, false, &in[1])) return rc;
    if (int rc = check_cache("v", a.v, s.B, s.capacity, s.kv_heads, s.head_dim, false, &in[2])) return rc;
    if (a.prefix) {
        if (int rc = check_cache("prefix k", a.kp, 1, a.prefix, s.kv_heads, s.head_dim, false, &in[3])) return rc;
        if (int rc = check_cache("prefix v", a.vp, 1, a.prefix, s.kv_heads, s.head_dim, false, &in[4])) return rc;
    }
    if ((reinterpret_cast<uintptr_t>(a.lens) | reinterpret_cast<uintptr_t>(a.lse)) % 4 || reinterpret_cast<uintptr_t>(a.tree) % 8)
        return fail(KRK_ATTN_ERR_ALIGN, "lens and lse must be 4-byte aligned, tree 8-byte");
    in[5] = span(a.lens, s.B, 4);
    if (a.tree) in[6] = span(a.tree, M, 8);
    if (a.lse) lse = span(a.lse, M * s.heads, 4);
    if (s.scored) {
        if (int rc = check_scores("scores", a.scores, a.sc_seq, a.sc_head, s.B, s.kv_heads, s.capacity, false, &in[7])) return rc;
        if (int rc = check_scores("scores_out", a.scores_out, a.so_seq, a.so_head, s.B, s.kv_heads, s.capacity, true, &sco)) return rc;
    } else if (a.scores || a.scores_out) {
        return fail(KRK_ATTN_ERR_INVALID, "scores given, but the shape has scored = 0");
    }
    const Plan plan = make_plan(s);
    if (plan.bytes && (!workspace || workspace_bytes < plan.bytes))
        return fail(KRK_ATTN_ERR_WORKSPACE, "needs a workspace of %zu bytes, got %zu", plan.bytes, workspace ? workspace_bytes : (size_t)0);
    if (reinterpret_cast<uintptr_t>(workspace) % 16) return fail(KRK_ATTN_ERR_ALIGN, "workspace must be 16-byte aligned");
    const Span ws = plan.bytes ? span(workspace, plan.bytes, 1) : Span{0, 0};
    const Span outs[4] = {out, lse, sco, ws};
    const bool in_place = s.scored && a.scores == a.scores_out && a.sc_seq == a.so_seq && a.sc_head == a.so_head;
    for (int i = 0; i < 4; ++i) {
        for (int j = 0; j < kIn; ++j)
            if (overlaps(outs[i], in[j]) && !(i == 2 && j == 7 && in_place))
                return fail(KRK_ATTN_ERR_ALIAS, "out, lse, scores_out and the workspace may not share memory with the inputs (scores_out == scores aside)");
        for (int j = 0; j < i; ++j)
            if (overlaps(outs[i], outs[j])) return fail(KRK_ATTN_ERR_ALIAS, "out, lse, scores_out and the workspace may not overlap");
    }

    krk::AttnParams p{};
    p.q = static_cast<const uint16_t*>(a.q);
    p.q_row = a.q_row;
    p.k = view(a.k);
    p.v = view(a.v);
    if (a.prefix) {
        p.kp = view(a.kp);
        p.vp = view(a.vp);
    }
    p.lens = a.lens;
    p.tree = a.tree;
    p.out = static_cast<uint16_t*>(a.out);
    p.out_row = a.out_row;
    p.lse = a.lse;
    p.scores = a.scores;
    p.sc_seq = a.sc_seq;
    p.sc_head = a.sc_head;
    p.scores_out = a.scores_out;
    p.so_seq = a.so_seq;
    p.so_head = a.so_head;
    unsigned char* w = static_cast<unsigned char*>(workspace);
    auto take = [&](size_t n) {
        unsigned char* at = n ? w : nullptr;
        w += n;
        return at;
    };
    uint32_t* ctr = reinterpret_cast<uint32_t*>(take(plan.ctr));
    p.ctr = plan.join_in_kernel ? ctr : nullptr;
    p.part = reinterpret_cast<float*>(take(plan.part));
    p.ml = reinterpret_cast<float2*>(take(plan.ml));
    p.stat = reinterpret_cast<float2*>(take(plan.stat));
    p.raw = reinterpret_cast<float*>(take(plan.raw));
    p.raw_row = plan.raw_row;
    p.scale = a.scale;
    p.c = scale_log2;
    p.B = s.B;
    p.R = s.R;
    p.heads = s.heads;
    p.kv_heads = s.kv_heads;
    p.G = s.heads / s.kv_heads;
    p.RG = s.R * p.G;
    p.capacity = s.capacity;
    p.window = s.window;
    p.sinks = s.sinks;
    p.prefix = a.prefix;
    p.splits = plan.own.splits;
    p.prefix_splits = plan.prefix.splits;
    p.row_tiles = plan.own.tiles;
    p.prefix_row_tiles = plan.prefix.tiles;
    hipStream_t st = static_cast<hipStream_t>(stream);
    return s.head_dim == 128 ? launch_attn<128>(p, plan, st) : launch_attn<64>(p, plan, st);
}

int krk_qk_norm_rope_bf16(const krk_rope_args* args, void* stream) {
    g_err[0] = '\0';
    if (!args) return fail(KRK_ATTN_ERR_INVALID, "null args");
    krk_rope_args a = *args;
    if (int rc = check_layout(a.B, a.R, a.heads, a.kv_heads, a.head_dim, a.capacity)) return rc;
    const int64_t M = (int64_t)a.B * a.R;
    const int64_t all = a.heads + 2 * (int64_t)a.kv_heads;
    Span qkv, q, k, v;
    if (int rc = check_rows("qkv", a.qkv, a.qkv_row, M, all * a.head_dim, &qkv)) return rc;
    if (int rc = check_rows("q_out", a.q_out, a.q_row, M, (int64_t)a.heads * a.head_dim, &q)) return rc;
    if (int rc = check_cache("k", a.k, a.B, a.capacity, a.kv_heads, a.head_dim, true, &k)) return rc;
    if (int rc = check_cache("v", a.v, a.B, a.capacity, a.kv_heads, a.head_dim, true, &v)) return rc;
    if (!a.q_norm != !a.k_norm) return fail(KRK_ATTN_ERR_INVALID, "q_norm and k_norm come together");
    if (!a.lens || !a.table) return fail(KRK_ATTN_ERR_INVALID, "lens or table: null pointer");
    if (a.table_rows < 1) return fail(KRK_ATTN_ERR_INVALID, "table_rows=%d must be >= 1", a.table_rows);
    if (!(a.eps >= 0.0f) || a.eps == __builtin_inff()) return fail(KRK_ATTN_ERR_INVALID, "eps=%g must be finite and >= 0", (double)a.eps);
    if ((reinterpret_cast<uintptr_t>(a.q_norm) | reinterpret_cast<uintptr_t>(a.k_norm) | reinterpret_cast<uintptr_t>(a.table)) % 16)
        return fail(KRK_ATTN_ERR_ALIGN, "q_norm, k_norm and table must be 16-byte aligned");
    if ((reinterpret_cast<uintptr_t>(a.lens) | reinterpret_cast<uintptr_t>(a.positions)) % 4)
        return fail(KRK_ATTN_ERR_ALIGN, "lens and positions must be 4-byte aligned");
    const bool in_place = a.q_out == a.qkv && (M == 1 || a.q_row == a.qkv_row);
    const Span ins[5] = {span(a.q_norm, a.head_dim, 2), span(a.k_norm, a.head_dim, 2), span(a.table, (uint64_t)a.table_rows * a.head_dim, 4),
                         span(a.lens, a.B, 4), span(a.positions, M, 4)};
    bool bad = (overlaps(q, qkv) && !in_place) || overlaps(k, qkv) || overlaps(v, qkv) || overlaps(q, k) || overlaps(q, v) ||
               share_memory(a.k, k, a.v, v, a.B, a.capacity, a.kv_heads, a.head_dim);
    for (const Span& i : ins) bad = bad || overlaps(q, i) || overlaps(k, i) || overlaps(v, i);
    if (bad) return fail(KRK_ATTN_ERR_ALIAS, "q_out (unless it is qkv in place), k and v may not share memory with each other or the inputs");
    krk::RopeParams p{static_cast<const uint16_t*>(a.qkv), a.qkv_row, static_cast<const uint16_t*>(a.q_norm),
                      static_cast<const uint16_t*>(a.k_norm), a.eps, a.table, a.table_rows, a.positions, a.lens,
                      static_cast<uint16_t*>(a.q_out), a.q_row, static_cast<uint16_t*>(a.k.p), static_cast<uint16_t*>(a.v.p),
                      a.k.seq, a.k.slot, a.k.head, a.v.seq, a.v.slot, a.v.head, a.B, a.R, a.heads, a.kv_heads, a.capacity};
    const int64_t blocks = cdiv(M * all * (a.head_dim / 8), 256);
    void* kargs[] = {(void*)&p};
    const void* fn = a.head_dim == 128 ? reinterpret_cast<const void*>(&krk::qk_norm_rope_kernel<128>)
                                       : reinterpret_cast<const void*>(&krk::qk_norm_rope_kernel<64>);
    return hip_status(hipLaunchKernel(fn, dim3((unsigned)blocks), dim3(256), kargs, 0, static_cast<hipStream_t>(stream)),
                      "qk_norm_rope_kernel launch");
}

int krk_cache_evict_bf16(const krk_evict_args* args, void* stream) {
    g_err[0] = '\0';
    if (!args) return fail(KRK_ATTN_ERR_INVALID, "null args");
    krk_evict_args a = *args;
    if (int rc = check_layout(a.B, 1, a.kv_heads, a.kv_heads, a.head_dim, a.capacity)) return rc;
    if (a.budget < 1 || a.budget > a.capacity) return fail(KRK_ATTN_ERR_INVALID, "budget=%d must be 1 .. capacity=%d", a.budget, a.capacity);
    if (a.sinks < 0 || a.recent < 0 || (int64_t)a.sinks + a.recent > a.budget)
        return fail(KRK_ATTN_ERR_INVALID, "sinks=%d and recent=%d must be >= 0 and together at most budget=%d", a.sinks, a.recent, a.budget);
    if (!a.lens || !a.lens_out || !a.keep) return fail(KRK_ATTN_ERR_INVALID, "lens, lens_out or keep: null pointer");
    if ((reinterpret_cast<uintptr_t>(a.lens) | reinterpret_cast<uintptr_t>(a.lens_out) | reinterpret_cast<uintptr_t>(a.keep)) % 4)
        return fail(KRK_ATTN_ERR_ALIGN, "lens, lens_out and keep must be 4-byte aligned");
    const bool in_place = a.k_out.p == a.k.p;
    Span in[4], out[5];
    if (int rc = check_cache("k", a.k, a.B, a.capacity, a.kv_heads, a.head_dim, in_place, &in[0])) return rc;
    if (int rc = check_cache("v", a.v, a.B, a.capacity, a.kv_heads, a.head_dim, in_place, &in[1])) return rc;
    if (int rc = check_scores("scores", a.scores, a.sc_seq, a.sc_head, a.B, a.kv_heads, a.capacity, in_place, &in[2])) return rc;
    in[3] = span(a.lens, a.B, 4);
    const int64_t slots = in_place ? a.capacity : a.budget;
    // In place the inputs were checked as written, and the outputs have to equal them.
    if (int rc = check_cache("k_out", a.k_out, a.B, slots, a.kv_heads, a.head_dim, !in_place, &out[0])) return rc;
    if (int rc = check_cache("v_out", a.v_out, a.B, slots, a.kv_heads, a.head_dim, !in_place, &out[1])) return rc;
    if (int rc = check_scores("scores_out", a.scores_out, a.so_seq, a.so_head, a.B, a.kv_heads, slots, !in_place, &out[2])) return rc;
    out[3] = span(a.keep, (uint64_t)a.B * a.kv_heads * a.budget, 4);
    out[4] = span(a.lens_out, a.B, 4);
    if (a.k.p == a.v.p || a.k_out.p == a.v_out.p) return fail(KRK_ATTN_ERR_ALIAS, "k and v may not be one tensor");
    if (in_place) {
        const bool same = a.k.seq == a.k_out.seq && a.k.slot == a.k_out.slot && a.k.head == a.k_out.head && a.v.p == a.v_out.p &&
                          a.v.seq == a.v_out.seq && a.v.slot == a.v_out.slot && a.v.head == a.v_out.head &&
                          a.scores == a.scores_out && a.sc_seq == a.so_seq && a.sc_head == a.so_head;
        if (!same) return fail(KRK_ATTN_ERR_ALIAS, "in place, k_out, v_out and scores_out are k, v and scores with their strides");
    }
    // They may be interleaved views of one.
    if (share_memory(a.k_out, out[0], a.v_out, out[1], a.B, slots, a.kv_heads, a.head_dim))
        return fail(KRK_ATTN_ERR_ALIAS, "k_out and v_out may not share memory");
    for (int i = 0; i < 5; ++i)
        for (int j = 0; j < 4; ++j) {
            if (in_place && i < 3 && j < 3) continue;
            if (i == 4 && j == 3 && a.lens == a.lens_out) continue;
            if (overlaps(out[i], in[j])) return fail(KRK_ATTN_ERR_ALIAS, "the outputs may not share memory with the inputs (all in place, or lens_out == lens, aside)");
        }
    for (int i = 2; i < 5; ++i)
        for (int j = 0; j < i; ++j)
            if (overlaps(out[i], out[j])) return fail(KRK_ATTN_ERR_ALIAS, "the outputs may not overlap");
    krk::EvictParams p{view(a.k), view(a.v), static_cast<uint16_t*>(a.k_out.p), static_cast<uint16_t*>(a.v_out.p),
                       a.k_out.seq, a.k_out.slot, a.k_out.head, a.v_out.seq, a.v_out.slot, a.v_out.head,
                       a.scores, a.sc_seq, a.sc_head, a.scores_out, a.so_seq, a.so_head, a.lens, a.lens_out, a.keep,
                       a.B, a.kv_heads, a.capacity, a.budget, a.sinks, a.recent};
    hipStream_t st = static_cast<hipStream_t>(stream);
    void* kargs[] = {(void*)&p};
    const bool wide = a.head_dim == 128;
    const void* select = select_kernel(a.capacity);
    hipError_t e = hipLaunchKernel(select, dim3(a.kv_heads, a.B), dim3(krk::kEvictThreads), kargs, 0, st);
    if (int rc = hip_status(e, "evict_select_kernel launch")) return rc;
    const void* fn;
    dim3 grid;
    if (in_place) {
        fn = wide ? reinterpret_cast<const void*>(&krk::evict_move_kernel<128>) : reinterpret_cast<const void*>(&krk::evict_move_kernel<64>);
        grid = dim3(2 * (a.head_dim / 32) + 1, a.kv_heads, a.B);
    } else {
        fn = wide ? reinterpret_cast<const void*>(&krk::evict_copy_kernel<128>) : reinterpret_cast<const void*>(&krk::evict_copy_kernel<64>);
        grid = dim3((unsigned)cdiv(a.budget, 256 / (a.head_dim / 8)), a.kv_heads, a.B);
    }
    return hip_status(hipLaunchKernel(fn, grid, dim3(256), kargs, 0, st), "evict move launch");
}

}  // extern "C"
