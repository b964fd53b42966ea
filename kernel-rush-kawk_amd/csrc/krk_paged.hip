// C ABI of the paged cache (declared in include/krk_paged.h): argument checks, how
// the work is cut, and stream-ordered launches.  Nothing here allocates,
// synchronises or touches device memory from the host, so every call is
// graph-capturable.
#include "krk_host.h"
#include "krk_page_step.h"
#include "krk_paged.h"
#include "krk_paged_many.h"
#include "krk_rope.h"

namespace {

using krk::make_plan;
using krk::Plan;

constexpr int kMaxRequests = 4096, kMaxRows = 1 << 18;
// Rows that the one workgroup of a page step maps itself, four a thread at once; more
// have a launch of their own (8500 rows of 256 requests 9.4 us, 10.8 without).
constexpr int kStepRows = 4 * krk::kPageThreads;

// log2 of a page's slots, or a negative code.
int page_shift(int page_size) {
    for (int s = 3; s <= 12; ++s)
        if (page_size == 1 << s) return s;
    return fail(kErrInvalid, "page_size=%d must be a power of two, 8 .. 4096", page_size);
}

int check_pool(int pages, int page_size) {
    if (pages < 1 || (int64_t)pages * page_size >= (int64_t)1 << 31)
        return fail(kErrInvalid, "pages=%d of %d slots: needs 1 or more, and fewer than 2^31 slots", pages, page_size);
    return 0;
}

int check_step(int B, int rows, int page_size, int width) {
    if (B < 1 || B > kMaxRequests || rows < 1 || rows > kMaxRows)
        return fail(kErrInvalid, "B=%d must be 1 .. %d and rows=%d 1 .. %d", B, kMaxRequests, rows, kMaxRows);
    if (width < 1 || (int64_t)width * page_size >= 1 << 27 || (int64_t)B * width >= (int64_t)1 << 31)
        return fail(kErrInvalid, "width=%d: needs 1 or more, width * page_size below 2^27 and B * width below 2^31", width);
    return 0;
}

int check_table(const void* table, int64_t& row, int B, int width, Span* out) {
    if (B == 1) row = width;
    if (row < width || row > kMaxStride) return fail(kErrInvalid, "table: row stride %lld must be >= width=%d", (long long)row, width);
    return check_words("table", table, (uint64_t)((B - 1) * row + width), out);
}

// A pool of keys or values.  Strides of extents of one are of no matter and set to 0.
int check_pages(const char* name, krk_pages& c, int64_t pages, int64_t slots, int64_t heads, int dim, bool written, Span* out) {
    if (!c.p) return fail(kErrInvalid, "%s: null pointer", name);
    if (pages == 1) c.page = 0;
    if (heads == 1) c.head = 0;
    const int64_t st[3] = {c.page, c.slot, c.head}, n[3] = {pages, slots, heads};
    for (int i = 0; i < 3; ++i) {
        if (st[i] < 0 || st[i] >= (int64_t)1 << 31)
            return fail(kErrInvalid, "%s: stride %lld out of range (below 2^31)", name, (long long)st[i]);
        if (st[i] % 8) return fail(kErrAlign, "%s: strides must be multiples of 8 elements", name);
    }
    // Offsets among the 64 keys of a step are 32 bits of bytes.
    if (c.slot >= (int64_t)1 << 25) return fail(kErrInvalid, "%s: stride %lld from key to key out of range (below 2^25)", name, (long long)c.slot);
    if (written && !nested(st, n, dim))
        return fail(kErrAlias, "%s is written: with strides of %lld, %lld and %lld its rows share memory", name, (long long)st[0], (long long)st[1], (long long)st[2]);
    if (!aligned(c.p, 16)) return fail(kErrAlign, "%s must be 16-byte aligned", name);
    *out = span(c.p, (uint64_t)((pages - 1) * c.page + (slots - 1) * c.slot + (heads - 1) * c.head + dim), 2);
    return 0;
}

bool share_memory(const krk_pages& x, const Span& xs, const krk_pages& y, const Span& ys, int64_t pages, int64_t slots, int64_t heads,
                  int dim) {
    return share_memory(x.p, xs, {x.page, x.slot, x.head}, y.p, ys, {y.page, y.slot, y.head}, {pages, slots, heads}, dim);
}

int check_heads(int rows, int heads, int kv_heads, int head_dim) {
    if (heads < 1 || kv_heads < 1 || heads % kv_heads) return fail(kErrInvalid, "heads=%d must be a multiple of kv_heads=%d, both >= 1", heads, kv_heads);
    if (head_dim != 64 && head_dim != 128) return fail(kErrUnsupported, "head_dim=%d: this build has 64 and 128", head_dim);
    // The rotary embedding's grid: head_dim / 8 threads for each of up to 3 * heads heads
    // of a row, below 2^32 threads.
    if ((int64_t)rows * heads >= (int64_t)1 << 25) return fail(kErrInvalid, "rows * heads = %lld must be below 2^25", (long long)((int64_t)rows * heads));
    return 0;
}

int check_shape(const krk_paged_shape& s) {
    if (int rc = page_shift(s.page_size); rc < 0) return rc;
    if (int rc = check_step(s.B, s.rows, s.page_size, s.width)) return rc;
    if (int rc = check_heads(s.rows, s.heads, s.kv_heads, s.head_dim)) return rc;
    if (s.window < 0 || s.sinks < 0 || s.window >= 1 << 28 || s.sinks >= 1 << 28)
        return fail(kErrInvalid, "window=%d and sinks=%d must be 0 .. 2^28 - 1", s.window, s.sinks);
    if (s.sinks && !s.window) return fail(kErrInvalid, "sinks need a window");
    if (const int64_t blocks = make_plan(s).blocks; blocks * krk::kPagedThreads >= (int64_t)1 << 32)
        return fail(kErrInvalid, "%d rows of %d requests over %d heads take %lld workgroups: needs fewer than 2^32 threads in all", s.rows, s.B, s.kv_heads,
                    (long long)blocks);
    return 0;
}

template <int D, bool MANY>
int launch_attn(const krk::PagedParams& p, const Plan& plan, hipStream_t stream) {
    static std::atomic<uint64_t> done{0};
    const void* fn = reinterpret_cast<const void*>(&krk::paged_attn_kernel<D, MANY>);
    constexpr size_t few = krk::few_lds_bytes<D>(), many = krk::tile_lds_bytes<D>();
    constexpr size_t shm = MANY && many > few ? many : few;
    if (hipError_t e = ensure_lds_limit(fn, shm, done)) return hip_status(e, "paged_attn_kernel LDS size");
    void* args[] = {(void*)&p};
    if (p.planned) {
        const hipError_t e = hipLaunchKernel(reinterpret_cast<const void*>(&krk::paged_plan_kernel), dim3(1), dim3(krk::kPlanThreads), args,
                                             krk::plan_lds_bytes(p.B), stream);
        if (int rc = hip_status(e, "paged_plan_kernel launch")) return rc;
    }
    return hip_status(hipLaunchKernel(fn, dim3((unsigned)plan.blocks), dim3(krk::kPagedThreads), args, shm, stream), "paged_attn_kernel launch");
}

krk::PageView view(const krk_pages& c) { return {static_cast<const uint16_t*>(c.p), c.page, c.slot, c.head}; }

}  // namespace

extern "C" {

int krk_paged_abi_version(void) { return KRK_PAGED_ABI_VERSION; }

size_t krk_paged_struct_size(int which) {
    switch (which) {
        case 0: return sizeof(krk_page_step_args);
        case 1: return sizeof(krk_paged_rope_args);
        case 2: return sizeof(krk_paged_shape);
        case 3: return sizeof(krk_paged_attn_args);
        default: return 0;
    }
}

const char* krk_paged_last_error(void) { return g_err; }

int krk_page_step(const krk_page_step_args* args, void* stream) {
    g_err[0] = '\0';
    if (!args) return fail(kErrInvalid, "null args");
    krk_page_step_args a = *args;
    const int shift = page_shift(a.page_size);
    if (shift < 0) return shift;
    if (int rc = check_step(a.B, a.rows, a.page_size, a.width)) return rc;
    if (int rc = check_pool(a.pages, a.page_size)) return rc;
    if (!a.free_pages != !a.free_count) return fail(kErrInvalid, "free_pages and free_count come together");
    Span s[12] = {};
    if (int rc = check_words("lens", a.lens, a.B, &s[0])) return rc;
    if (int rc = check_table(a.table, a.table_row, a.B, a.width, &s[1])) return rc;
    if (int rc = check_words("starts", a.starts, a.B + 1, &s[2])) return rc;
    if (int rc = check_words("keys", a.keys, a.B, &s[3])) return rc;
    if (int rc = check_words("slots", a.slots, a.rows, &s[4])) return rc;
    if (int rc = check_words("positions", a.positions, a.rows, &s[5])) return rc;
    if (int rc = check_words("owner", a.owner, a.rows, &s[6])) return rc;
    if (a.free_pages) {
        if (int rc = check_words("free_pages", a.free_pages, a.pages, &s[7])) return rc;
        if (int rc = check_words("free_count", a.free_count, 1, &s[8])) return rc;
    }
    if (int rc = check_words("fresh", a.fresh, a.B, &s[9])) return rc;
    if (a.keep)
        if (int rc = check_words("keep", a.keep, a.B, &s[10])) return rc;
    if (a.labels)
        if (int rc = check_words("labels", a.labels, a.B, &s[11])) return rc;
    for (int i = 0; i < 9; ++i)
        for (int j = i + 1; j < 12; ++j)
            if (overlaps(s[i], s[j])) return fail(kErrAlias, "what a page step writes may not share memory with its other operands");
    krk::PageStepParams p{a.lens, a.keep, a.fresh, a.labels, a.table, a.table_row, a.free_pages, a.free_count,
                          a.starts, a.keys, a.slots, a.positions, a.owner, a.B, a.rows, a.pages, shift, a.width};
    hipStream_t st = static_cast<hipStream_t>(stream);
    void* kargs[] = {(void*)&p};
    const bool own_rows = a.rows <= kStepRows;
    const void* fn = own_rows ? reinterpret_cast<const void*>(&krk::page_step_kernel<true>)
                              : reinterpret_cast<const void*>(&krk::page_step_kernel<false>);
    static std::atomic<uint64_t> done[2];
    const size_t shm = krk::page_step_lds_bytes(a.B);
    if (hipError_t e = ensure_lds_limit(fn, krk::page_step_lds_bytes(kMaxRequests), done[own_rows])) return hip_status(e, "page_step_kernel LDS size");
    if (int rc = hip_status(hipLaunchKernel(fn, dim3(1), dim3(krk::kPageThreads), kargs, shm, st), "page_step_kernel launch")) return rc;
    if (own_rows) return 0;
    return hip_status(hipLaunchKernel(reinterpret_cast<const void*>(&krk::page_rows_kernel), dim3((unsigned)cdiv(a.rows, 256)), dim3(256), kargs, 0, st),
                      "page_rows_kernel launch");
}

int krk_paged_rope_bf16(const krk_paged_rope_args* args, void* stream) {
    g_err[0] = '\0';
    if (!args) return fail(kErrInvalid, "null args");
    krk_paged_rope_args a = *args;
    const int shift = page_shift(a.page_size);
    if (shift < 0) return shift;
    if (int rc = check_pool(a.pages, a.page_size)) return rc;
    if (a.rows < 1 || a.rows > kMaxRows) return fail(kErrInvalid, "rows=%d must be 1 .. %d", a.rows, kMaxRows);
    const int64_t all = a.heads + 2 * (int64_t)a.kv_heads;
    if (int rc = check_heads(a.rows, a.heads, a.kv_heads, a.head_dim)) return rc;
    Span qkv, q, k, v, in[5] = {};
    if (int rc = check_rows("qkv", a.qkv, a.qkv_row, a.rows, all * a.head_dim, &qkv)) return rc;
    if (int rc = check_rows("q_out", a.q_out, a.q_row, a.rows, (int64_t)a.heads * a.head_dim, &q)) return rc;
    if (int rc = check_pages("k", a.k, a.pages, a.page_size, a.kv_heads, a.head_dim, true, &k)) return rc;
    if (int rc = check_pages("v", a.v, a.pages, a.page_size, a.kv_heads, a.head_dim, true, &v)) return rc;
    if (!a.q_norm != !a.k_norm) return fail(kErrInvalid, "q_norm and k_norm come together");
    if (a.table_rows < 1) return fail(kErrInvalid, "table_rows=%d must be >= 1", a.table_rows);
    if (!(a.eps >= 0.0f) || a.eps == __builtin_inff()) return fail(kErrInvalid, "eps=%g must be finite and >= 0", (double)a.eps);
    if (int rc = check_words("table", a.table, (uint64_t)a.table_rows * a.head_dim, &in[0])) return rc;
    if (int rc = check_words("slots", a.slots, a.rows, &in[1])) return rc;
    if (int rc = check_words("positions", a.positions, a.rows, &in[2])) return rc;
    in[3] = span(a.q_norm, a.head_dim, 2);
    in[4] = span(a.k_norm, a.head_dim, 2);
    if (!aligned(a.q_norm, 16) || !aligned(a.k_norm, 16) || !aligned(a.table, 16))
        return fail(kErrAlign, "q_norm, k_norm and table must be 16-byte aligned");
    const bool in_place = a.q_out == a.qkv && (a.rows == 1 || a.q_row == a.qkv_row);
    bool bad = (overlaps(q, qkv) && !in_place) || overlaps(k, qkv) || overlaps(v, qkv) || overlaps(q, k) || overlaps(q, v) ||
               share_memory(a.k, k, a.v, v, a.pages, a.page_size, a.kv_heads, a.head_dim);
    for (const Span& i : in) bad = bad || overlaps(q, i) || overlaps(k, i) || overlaps(v, i);
    if (bad) return fail(kErrAlias, "q_out (unless it is qkv in place), k and v may not share memory with each other or the inputs");
    krk::RopeParams p{};
    p.qkv = static_cast<const uint16_t*>(a.qkv);
    p.qkv_row = a.qkv_row;
    p.q_norm = static_cast<const uint16_t*>(a.q_norm);
    p.k_norm = static_cast<const uint16_t*>(a.k_norm);
    p.eps = a.eps;
    p.table = a.table;
    p.table_rows = a.table_rows;
    p.positions = a.positions;
    p.q_out = static_cast<uint16_t*>(a.q_out);
    p.q_row = a.q_row;
    p.k = static_cast<uint16_t*>(a.k.p);
    p.v = static_cast<uint16_t*>(a.v.p);
    p.k_seq = a.k.page;
    p.k_slot = a.k.slot;
    p.k_head = a.k.head;
    p.v_seq = a.v.page;
    p.v_slot = a.v.slot;
    p.v_head = a.v.head;
    p.B = 1;
    p.R = a.rows;
    p.heads = a.heads;
    p.kv_heads = a.kv_heads;
    p.capacity = a.pages * a.page_size;
    p.slots = a.slots;
    p.shift = shift;
    void* kargs[] = {(void*)&p};
    const void* fn = a.head_dim == 128 ? reinterpret_cast<const void*>(&krk::qk_norm_rope_kernel<128, true>)
                                       : reinterpret_cast<const void*>(&krk::qk_norm_rope_kernel<64, true>);
    const int64_t blocks = cdiv(a.rows * all * (a.head_dim / 8), 256);
    return hip_status(hipLaunchKernel(fn, dim3((unsigned)blocks), dim3(256), kargs, 0, static_cast<hipStream_t>(stream)),
                      "qk_norm_rope_kernel launch");
}

int krk_paged_check(const krk_paged_shape* shape) {
    g_err[0] = '\0';
    if (!shape) return fail(kErrInvalid, "null shape");
    return check_shape(*shape);
}

size_t krk_paged_workspace_bytes(const krk_paged_shape* shape) {
    g_err[0] = '\0';
    if (!shape || check_shape(*shape)) return 0;
    return make_plan(*shape).bytes;
}

int krk_paged_attn_bf16(const krk_paged_shape* shape, const krk_paged_attn_args* args, void* workspace, size_t workspace_bytes,
                        void* stream) {
    g_err[0] = '\0';
    if (!shape || !args) return fail(kErrInvalid, "null shape or args");
    const krk_paged_shape& s = *shape;
    krk_paged_attn_args a = *args;
    if (int rc = check_shape(s)) return rc;
    if (int rc = check_pool(a.pages, s.page_size)) return rc;
    // The kernels multiply by scale * log2(e).
    const float scale_log2 = (float)((double)a.scale * 1.4426950408889634);
    if (!(a.scale > 0.0f) || scale_log2 == __builtin_inff())
        return fail(kErrInvalid, "scale=%g must be positive and at most 2.3e38", (double)a.scale);
    const int64_t cols = (int64_t)s.heads * s.head_dim;
    Span in[6] = {}, outs[3] = {};
    if (int rc = check_rows("q", a.q, a.q_row, s.rows, cols, &in[0])) return rc;
    if (int rc = check_rows("out", a.out, a.out_row, s.rows, cols, &outs[0])) return rc;
    if (int rc = check_pages("k", a.k, a.pages, s.page_size, s.kv_heads, s.head_dim, false, &in[1])) return rc;
    if (int rc = check_pages("v", a.v, a.pages, s.page_size, s.kv_heads, s.head_dim, false, &in[2])) return rc;
    if (int rc = check_table(a.table, a.table_row, s.B, s.width, &in[3])) return rc;
    if (int rc = check_words("starts", a.starts, s.B + 1, &in[4])) return rc;
    if (int rc = check_words("keys", a.keys, s.B, &in[5])) return rc;
    if (a.lse)
        if (int rc = check_words("lse", a.lse, (uint64_t)s.rows * s.heads, &outs[1])) return rc;
    const Plan plan = make_plan(s);
    if (plan.bytes && (!workspace || workspace_bytes < plan.bytes))
        return fail(kErrWorkspace, "needs a workspace of %zu bytes, got %zu", plan.bytes, workspace ? workspace_bytes : (size_t)0);
    if (!aligned(workspace, 16)) return fail(kErrAlign, "workspace must be 16-byte aligned");
    if (plan.bytes) outs[2] = span(workspace, plan.bytes, 1);
    for (int i = 0; i < 3; ++i) {
        for (const Span& x : in)
            if (overlaps(outs[i], x)) return fail(kErrAlias, "out, lse and the workspace may not share memory with the inputs");
        for (int j = 0; j < i; ++j)
            if (overlaps(outs[i], outs[j])) return fail(kErrAlias, "out, lse and the workspace may not overlap");
    }
    krk::PagedParams p{};
    p.q = static_cast<const uint16_t*>(a.q);
    p.q_row = a.q_row;
    p.k = view(a.k);
    p.v = view(a.v);
    p.table = a.table;
    p.table_row = a.table_row;
    p.starts = a.starts;
    p.keys = a.keys;
    p.out = static_cast<uint16_t*>(a.out);
    p.out_row = a.out_row;
    p.lse = a.lse;
    unsigned char* w = static_cast<unsigned char*>(workspace);
    p.ctr = reinterpret_cast<uint32_t*>(w);
    p.part = reinterpret_cast<float*>(w + plan.ctr);
    p.ml = reinterpret_cast<float2*>(w + plan.ctr + plan.part);
    if (plan.plan) {
        p.planned = reinterpret_cast<int*>(w + plan.ctr + plan.part + plan.ml);
        p.plan = reinterpret_cast<krk::PlannedRange*>(w + plan.ctr + plan.part + plan.ml + 256);
    }
    p.scale = a.scale;
    p.c = scale_log2;
    p.B = s.B;
    p.rows = s.rows;
    p.heads = s.heads;
    p.kv_heads = s.kv_heads;
    p.G = s.heads / s.kv_heads;
    p.inv_G = 1.0f / (float)p.G;
    p.inv_kv = 1.0f / (float)s.kv_heads;
    p.pages = a.pages;
    p.shift = page_shift(s.page_size);
    p.width = s.width;
    p.window = s.window;
    p.sinks = s.sinks;
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (s.head_dim == 128) return plan.many ? launch_attn<128, true>(p, plan, st) : launch_attn<128, false>(p, plan, st);
    return plan.many ? launch_attn<64, true>(p, plan, st) : launch_attn<64, false>(p, plan, st);
}

}  // extern "C"
