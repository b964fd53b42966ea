// C ABI of low-rank adapters (declared in include/krk_adapter.h): argument checks,
// how the work is cut, and stream-ordered launches.  Nothing here allocates,
// synchronises or touches device memory from the host, so every call is
// graph-capturable.
#include "krk_adapter.h"
#include "krk_adapter_kernels.h"
#include "krk_host.h"

namespace {

static_assert(KRK_ADAPTER_SLICES == krk::kAdapterSlices, "slices");
constexpr int kMaxRows = 1 << 18, kMaxSize = 1 << 20;

int check_shape(const krk_adapter_shape& s) {
    if (s.rows < 1 || s.rows > kMaxRows) return fail(kErrInvalid, "rows=%d must be 1 .. %d", s.rows, kMaxRows);
    if (s.K < 8 || s.K % 8 || s.K > kMaxSize || s.N < 8 || s.N % 8 || s.N > kMaxSize)
        return fail(kErrInvalid, "N=%d and K=%d must be multiples of 8, 8 .. %d", s.N, s.K, kMaxSize);
    if (s.rank < 8 || s.rank % 8 || s.rank > 128) return fail(kErrInvalid, "rank=%d must be a multiple of 8, 8 .. 128", s.rank);
    if (s.silu != 0 && s.silu != 1) return fail(kErrInvalid, "silu must be 0 or 1, got %d", s.silu);
    if (s.slices < 1 || s.slices > KRK_ADAPTER_SLICES) return fail(kErrInvalid, "slices=%d must be 1 .. %d", s.slices, KRK_ADAPTER_SLICES);
    int64_t sum = 0;
    for (int i = 0; i < s.slices; ++i) {
        if (s.widths[i] < 8 || s.widths[i] % 8) return fail(kErrInvalid, "slice %d of %d columns: needs a multiple of 8, 8 or more", i, s.widths[i]);
        sum += s.widths[i];
    }
    if (sum != s.N) return fail(kErrInvalid, "slices of %lld columns in all for N=%d", (long long)sum, s.N);
    if (s.silu && (s.N % 16 || s.slices > 2 || (s.slices == 2 && s.widths[0] != s.widths[1])))
        return fail(kErrInvalid, "silu needs N=%d a multiple of 16, and 1 slice or 2 equal ones", s.N);
    return 0;
}

struct Plan {
    bool many;              // tiles of 64 rows, else of 16
    int tiles, groups;      // of rows; of 64 rows of A
    int splits;             // ranges of K
    int shrink_slots, expand_slots;
    int col_blocks;
    size_t h, joined, bytes;  // workspace: sizes of its parts and their sum
};

constexpr int kFewRows = 256;
// Tiles of 16 that a workgroup of the second product takes of many rows: 32 rows read B
// half as often as 16 (4096 rows of 2560 columns, a call: 51 us, in 16 or 64 rows 53);
// with gate and up in registers 16 leave room for more workgroups (2048 rows: 57 us, 63).
template <bool SILU>
constexpr int kManyTiles = SILU ? 1 : 2;
// Workgroups that the slots of a tile's adapters may come to: those without one cost 9 ns
// each (64 rows of 4 runs, 38 blocks of columns: a workgroup for every row took 25 us).
constexpr int kSlotBlocks = 1024;

int slots(int64_t blocks, int rows) {
    const int64_t s = kSlotBlocks / blocks;
    return (int)(s < 1 ? 1 : s < rows ? s : rows);
}

Plan make_plan(const krk_adapter_shape& s) {
    Plan p{};
    p.many = s.rows > kFewRows;
    const int tile = p.many ? 64 : 16, most_sets = tile < s.rows ? tile : s.rows;
    p.tiles = (int)cdiv(s.rows, tile);
    p.groups = (int)cdiv((int64_t)s.slices * s.rank, 16 * krk::kAdapterTiles);
    // Few rows: a range each for two workgroups a CU, or more.  Many rows: at most three
    // workgroups for two CUs, since a tile of two requests has a second one that starts
    // where room is left (4096 rows of 9728, a call: 56.5 us in 8 ranges or 7, 53.9 in 6;
    // 1000 rows and narrower calls the same).
    const int64_t blocks = (int64_t)p.tiles * p.groups, few = cdiv(2 * kCuCount, blocks), many = 3 * kCuCount / 2 / blocks;
    const int64_t want = !p.many ? few : many > 0 ? many : 1;
    const int64_t most = p.many ? cdiv(s.K, 4 * krk::kAdapterManyStep) : cdiv(s.K, krk::kAdapterWaves * krk::kAdapterFewStep);
    p.splits = (int)(want < most ? want : most);
    const int limit = p.many ? krk::kAdapterManySplits : krk::kAdapterFewSplits;
    p.splits = p.splits < limit ? p.splits : limit;
    p.shrink_slots = slots((int64_t)p.tiles * p.groups * p.splits, most_sets);
    for (int i = 0; i < s.slices; ++i) p.col_blocks += (int)cdiv(s.widths[i], krk::kAdapterWaves * krk::kAdapterCols);
    if (s.silu) p.col_blocks = (int)cdiv(s.N / 2, krk::kAdapterWaves * krk::kAdapterCols);
    const int expand_tiles = p.many ? (int)cdiv(s.rows, 16 * (s.silu ? kManyTiles<true> : kManyTiles<false>)) : p.tiles;
    p.expand_slots = slots((int64_t)expand_tiles * p.col_blocks, most_sets);
    const size_t values = (size_t)s.rows * s.slices * s.rank;
    p.h = align_up(p.splits * values * sizeof(float), 256);
    p.joined = p.many ? align_up(2 * values * sizeof(uint16_t), 256) : 0;
    p.bytes = p.h + p.joined;
    return p;
}

int launch_shrink(krk::AdapterParams p, const Plan& plan, hipStream_t st) {
    p.slots = plan.shrink_slots;
    void* kargs[] = {(void*)&p};
    const void* fn = plan.many ? reinterpret_cast<const void*>(&krk::adapter_shrink64_kernel) : reinterpret_cast<const void*>(&krk::adapter_shrink_kernel);
    const dim3 grid = plan.many ? dim3(plan.splits * plan.tiles, p.slots, plan.groups) : dim3(plan.splits, plan.tiles * p.slots, plan.groups);
    const hipError_t e = hipLaunchKernel(fn, grid, dim3(krk::kAdapterThreads), kargs, 0, st);
    return hip_status(e, "adapter_shrink_kernel launch");
}

template <int MT, bool SILU, bool JOINED>
int launch_expand(krk::AdapterParams p, const Plan& plan, hipStream_t st) {
    p.slots = plan.expand_slots;
    void* kargs[] = {(void*)&p};
    const void* fn = reinterpret_cast<const void*>(&krk::adapter_expand_kernel<MT, SILU, JOINED>);
    static std::atomic<uint64_t> done{0};
    constexpr size_t rows = 16 * MT * (SILU ? 2 : 1);
    if (hipError_t x = ensure_lds_limit(fn, rows * krk::adapter_row_bytes(128), done)) return hip_status(x, "adapter_expand_kernel LDS size");
    const hipError_t e = hipLaunchKernel(fn, dim3(plan.col_blocks, (unsigned)cdiv(p.rows, 16 * MT) * p.slots), dim3(krk::kAdapterThreads), kargs,
                                         rows * krk::adapter_row_bytes(p.rank), st);
    return hip_status(e, "adapter_expand_kernel launch");
}

template <bool SILU>
int launch(const krk::AdapterParams& p, const Plan& plan, hipStream_t st) {
    if (int rc = launch_shrink(p, plan, st)) return rc;
    if (!plan.many) return launch_expand<1, SILU, false>(p, plan, st);
    krk::AdapterParams q = p;
    void* kargs[] = {(void*)&q};
    const void* fn = p.splits <= krk::kAdapterFewSplits ? reinterpret_cast<const void*>(&krk::adapter_join_kernel<krk::kAdapterFewSplits>)
                                                        : reinterpret_cast<const void*>(&krk::adapter_join_kernel<krk::kAdapterManySplits>);
    const hipError_t e = hipLaunchKernel(fn, dim3((unsigned)cdiv((int64_t)p.rows * (p.HN / 4), 256)),
                                         dim3(256), kargs, 0, st);
    if (int rc = hip_status(e, "adapter_join_kernel launch")) return rc;
    return launch_expand<kManyTiles<SILU>, SILU, true>(p, plan, st);
}

// A factor of each adapter: [adapters, rows, cols].
int check_factor(const char* name, const void* p, int64_t& adapter, int64_t& row, int64_t adapters, int64_t rows, int64_t cols, Span* out) {
    if (!p) return fail(kErrInvalid, "%s: null pointer", name);
    if (adapters == 1) adapter = 0;
    if (adapter < 0 || adapter > kMaxStride || row < cols || row > kMaxStride)
        return fail(kErrInvalid, "%s: strides %lld and %lld out of range (rows of %lld)", name, (long long)adapter, (long long)row, (long long)cols);
    if (adapter % 8 || row % 8) return fail(kErrAlign, "%s: strides must be multiples of 8 elements", name);
    if (!aligned(p, 16)) return fail(kErrAlign, "%s must be 16-byte aligned", name);
    *out = span(p, (uint64_t)((adapters - 1) * adapter + (rows - 1) * row + cols), 2);
    return 0;
}

}  // namespace

extern "C" {

int krk_adapter_abi_version(void) { return KRK_ADAPTER_ABI_VERSION; }

size_t krk_adapter_struct_size(int which) {
    switch (which) {
        case 0: return sizeof(krk_adapter_shape);
        case 1: return sizeof(krk_adapter_args);
        default: return 0;
    }
}

const char* krk_adapter_last_error(void) { return g_err; }

int krk_adapter_check(const krk_adapter_shape* shape) {
    g_err[0] = '\0';
    if (!shape) return fail(kErrInvalid, "null shape");
    return check_shape(*shape);
}

size_t krk_adapter_workspace_bytes(const krk_adapter_shape* shape) {
    g_err[0] = '\0';
    if (!shape || check_shape(*shape)) return 0;
    return make_plan(*shape).bytes;
}

int krk_adapter_bf16(const krk_adapter_shape* shape, const krk_adapter_args* args, void* workspace, size_t workspace_bytes,
                     void* stream) {
    g_err[0] = '\0';
    if (!shape || !args) return fail(kErrInvalid, "null shape or args");
    const krk_adapter_shape& s = *shape;
    krk_adapter_args a = *args;
    if (int rc = check_shape(s)) return rc;
    if (a.adapters < 1 || a.adapters > kMaxSize) return fail(kErrInvalid, "adapters=%d must be 1 .. %d", a.adapters, kMaxSize);
    const int HN = s.slices * s.rank, out_cols = s.silu ? s.N / 2 : s.N;
    Span in[6] = {}, out, ws;
    if (int rc = check_rows("x", a.x, a.ldx, s.rows, s.K, &in[0])) return rc;
    if (int rc = check_factor("a", a.a, a.a_adapter, a.a_row, a.adapters, HN, s.K, &in[1])) return rc;
    if (int rc = check_factor("b", a.b, a.b_adapter, a.b_row, a.adapters, s.N, s.rank, &in[2])) return rc;
    if (a.scale)
        if (int rc = check_words("scale", a.scale, a.adapters, &in[3])) return rc;
    if (int rc = check_words("index", a.index, s.rows, &in[4])) return rc;
    if (int rc = check_rows("y", a.y, a.ldy, s.rows, s.N, &in[5])) return rc;
    if (int rc = check_rows("out", a.out, a.ldo, s.rows, out_cols, &out)) return rc;
    const Plan plan = make_plan(s);
    if (!workspace || workspace_bytes < plan.bytes)
        return fail(kErrWorkspace, "needs a workspace of %zu bytes, got %zu", plan.bytes, workspace ? workspace_bytes : (size_t)0);
    if (!aligned(workspace, 16)) return fail(kErrAlign, "workspace must be 16-byte aligned");
    ws = span(workspace, plan.bytes, 1);
    const bool same = !s.silu && a.out == a.y && a.ldo == a.ldy;
    for (int i = 0; i < 6; ++i)
        if ((overlaps(out, in[i]) && !(i == 5 && same)) || overlaps(ws, in[i]))
            return fail(kErrAlias, "out (unless it is y, without silu) and the workspace may not share memory with the inputs");
    if (overlaps(out, ws)) return fail(kErrAlias, "out and the workspace may not overlap");
    krk::AdapterParams p{};
    p.x = static_cast<const uint16_t*>(a.x);
    p.ldx = a.ldx;
    p.a = static_cast<const uint16_t*>(a.a);
    p.a_adapter = a.a_adapter;
    p.a_row = a.a_row;
    p.b = static_cast<const uint16_t*>(a.b);
    p.b_adapter = a.b_adapter;
    p.b_row = a.b_row;
    p.scale = a.scale;
    p.index = a.index;
    p.y = static_cast<const uint16_t*>(a.y);
    p.ldy = a.ldy;
    p.out = static_cast<uint16_t*>(a.out);
    p.ldo = a.ldo;
    p.h = static_cast<float*>(workspace);
    p.rows = s.rows;
    p.N = s.N;
    p.K = s.K;
    p.rank = s.rank;
    p.HN = HN;
    p.adapters = a.adapters;
    p.splits = plan.splits;
    p.slices = s.slices;
    p.joined = plan.joined ? reinterpret_cast<uint16_t*>(static_cast<unsigned char*>(workspace) + plan.h) : nullptr;
    p.same = same;
    for (int i = 0; i < s.slices; ++i) {
        p.width[i] = s.widths[i];
        p.first[i] = i ? p.first[i - 1] + s.widths[i - 1] : 0;
        p.block[i + 1] = p.block[i] + (int)cdiv(s.widths[i], krk::kAdapterWaves * krk::kAdapterCols);
    }
    hipStream_t st = static_cast<hipStream_t>(stream);
    return s.silu ? launch<true>(p, plan, st) : launch<false>(p, plan, st);
}

}  // extern "C"
