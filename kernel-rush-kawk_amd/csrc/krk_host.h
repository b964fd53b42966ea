// Host-side pieces that the libraries of several operators share: errors, spans of
// memory, and what a launch needs.
#pragma once

#include <hip/hip_runtime.h>
#include <stdarg.h>
#include <stdint.h>
#include <stdio.h>

#include <atomic>
#include <utility>

namespace {

constexpr int kErrInvalid = -1, kErrAlign = -2, kErrAlias = -3, kErrWorkspace = -4, kErrHip = -5, kErrUnsupported = -6;
constexpr int kCuCount = 256;  // MI355X: 8 XCDs x 32 CUs
constexpr int64_t kMaxStride = (int64_t)1 << 40;

thread_local char g_err[512] = "";

int fail(int code, const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_err, sizeof g_err, fmt, ap);
    va_end(ap);
    return code;
}

inline int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline size_t align_up(size_t v, size_t a) { return (v + a - 1) / a * a; }

int hip_status(hipError_t e, const char* what) {
    return e == hipSuccess ? 0 : fail(kErrHip, "%s: %s", what, hipGetErrorString(e));
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

struct Span {
    uintptr_t a, b;
};
bool overlaps(const Span& x, const Span& y) { return x.a < y.b && y.a < x.b; }
Span span(const void* p, uint64_t elems, size_t size) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(p);
    return p ? Span{a, a + elems * size} : Span{0, 0};
}

bool aligned(const void* p, unsigned bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

// Whether no two elements of a written operand share memory: sorted by stride, each
// is at least the extent of those inside it.  (Strides of extents of one are 0.)
[[maybe_unused]] bool nested(const int64_t (&stride)[3], const int64_t (&n)[3], int64_t inner) {
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

// Whether two written caches of one shape (strides, extents, then `dim` elements)
// share memory.  Views whose spans meet (k and v side by side in one tensor) have to
// have the same strides; they are apart if no step from a row of one to a row of the
// other is shorter than a row.  A step's part along the largest stride is one of the
// two multiples next to it, as what is left has to lie within the extent inside that
// stride.
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
[[maybe_unused]] bool share_memory(const void* x, const Span& xs, const int64_t (&x_stride)[3], const void* y, const Span& ys,
                                   const int64_t (&y_stride)[3], const int64_t (&extent)[3], int dim) {
    if (!overlaps(xs, ys)) return false;
    int64_t stride[3], n[3];
    for (int i = 0; i < 3; ++i) {
        if (x_stride[i] != y_stride[i]) return true;
        stride[i] = x_stride[i];
        n[i] = extent[i];
    }
    const intptr_t bytes = reinterpret_cast<intptr_t>(y) - reinterpret_cast<intptr_t>(x);
    for (int i = 0; i < 3; ++i)
        for (int j = i + 1; j < 3; ++j)
            if (stride[j] > stride[i]) {
                std::swap(stride[i], stride[j]);
                std::swap(n[i], n[j]);
            }
    return !apart(bytes / 2, stride, n, dim);
}

// [rows, cols] bf16 operand; one row's stride is of no matter and set to its
// length.
int check_rows(const char* name, const void* p, int64_t& row, int64_t rows, int64_t cols, Span* out) {
    if (rows == 1) row = cols;
    if (!p) return fail(kErrInvalid, "%s: null pointer", name);
    if (row < cols || row > kMaxStride) return fail(kErrInvalid, "%s: row stride %lld must be >= %lld", name, (long long)row, (long long)cols);
    if (row % 8) return fail(kErrAlign, "%s: the row stride must be a multiple of 8 elements", name);
    if (!aligned(p, 16)) return fail(kErrAlign, "%s must be 16-byte aligned", name);
    *out = span(p, (uint64_t)((rows - 1) * row + cols), 2);
    return 0;
}

// An array of 32-bit values.
[[maybe_unused]] int check_words(const char* name, const void* p, uint64_t n, Span* out) {
    if (!p) return fail(kErrInvalid, "%s: null pointer", name);
    if (!aligned(p, 4)) return fail(kErrAlign, "%s must be 4-byte aligned", name);
    *out = span(p, n, 4);
    return 0;
}

}  // namespace
