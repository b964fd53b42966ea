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
int check_words(const char* name, const void* p, uint64_t n, Span* out) {
    if (!p) return fail(kErrInvalid, "%s: null pointer", name);
    if (!aligned(p, 4)) return fail(kErrAlign, "%s must be 4-byte aligned", name);
    *out = span(p, n, 4);
    return 0;
}

}  // namespace
