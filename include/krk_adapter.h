/*
 * krk_adapter.h — C ABI of low-rank adapters on MI355X (gfx950): rows of many
 * requests, each with its own adapter, beside one projection that they share.
 *
 *   out[row] = y[row] + scale[i] * (x[row] A_i^T) B_i^T,   i = index[row]
 *
 * Stands behind krk_gemm.h's projections, whose output is y; the reference has no
 * adapters.  Operands are bf16 (raw 16-bit patterns) in device memory unless said
 * otherwise.  Nothing here allocates, synchronises or reads device memory on the
 * host: every call enqueues its kernels on `stream` and returns, so it may be
 * recorded into a HIP graph.  Strides are in elements.
 */
#ifndef KRK_ADAPTER_H
#define KRK_ADAPTER_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Return codes: those of krk_gemm.h (0 = success, negative = error). */
enum {
    KRK_ADAPTER_OK = 0,
    KRK_ADAPTER_ERR_INVALID = -1,   /* sizes, null pointers, unknown values */
    KRK_ADAPTER_ERR_ALIGN = -2,     /* a pointer or stride is not aligned */
    KRK_ADAPTER_ERR_ALIAS = -3,     /* an output shares memory with another operand */
    KRK_ADAPTER_ERR_WORKSPACE = -4, /* workspace missing or too small */
    KRK_ADAPTER_ERR_HIP = -5        /* the HIP runtime rejected a launch */
};

#define KRK_ADAPTER_SLICES 4

/* What a call computes, fixed for an object that makes many of them.  The columns of
 * y fall into `slices` slices of widths[s] (multiples of 8) columns, one behind the
 * other, N in all: slice s takes rows s * rank .. (s + 1) * rank - 1 of A_i (the q, k
 * and v parts of a fused projection have first factors of their own).  silu: y is
 * [gate; up] side by side, N / 2 columns each (1 slice, or 2 equal ones), and out is
 * silu(gate) * up, [rows, N / 2]. */
typedef struct krk_adapter_shape {
    int rows;  /* 1 .. 2^18 */
    int N, K;  /* multiples of 8 (silu: N of 16), 8 .. 2^20 */
    int rank;  /* a multiple of 8, 8 .. 128 */
    int silu;  /* 0 or 1 */
    int slices;
    int widths[KRK_ADAPTER_SLICES];
} krk_adapter_shape;

/* An index outside 0 .. adapters - 1 is no adapter: out is y (or silu(gate) * up of
 * it).  Products x A^T are summed in fp32 and enter the second product as two bf16
 * parts (off by 2^-16); the sum with y, and silu, are taken in fp32 with one rounding
 * at the end.  Rows do not reach into each other's results, whatever they hold.
 * An infinite value of B gives NaN (or an infinity, as the two parts have it) to the
 * rows of its adapter. */
typedef struct krk_adapter_args {
    const void* x;            /* [rows, K], row stride ldx (multiple of 8) */
    int64_t ldx;
    const void* a;            /* [adapters, slices * rank, K], strides a_adapter and a_row (multiples of 8) */
    int64_t a_adapter, a_row;
    const void* b;            /* [adapters, N, rank], strides b_adapter and b_row (multiples of 8) */
    int64_t b_adapter, b_row;
    const float* scale;       /* [adapters], or NULL: 1 */
    const int32_t* index;     /* [rows] */
    const void* y;            /* [rows, N], row stride ldy */
    int64_t ldy;
    void* out;                /* [rows, N], or [rows, N / 2] with silu; row stride ldo.  Without silu it may be
                                 y itself (same pointer and stride). */
    int64_t ldo;
    int adapters;             /* 1 .. 2^20 */
} krk_adapter_args;

/* One call.  `workspace`: krk_adapter_workspace_bytes(shape) bytes, 16-byte aligned; what
 * it holds before is of no matter.  Calls that share one must be ordered on one
 * stream.  Results are deterministic. */
int krk_adapter_bf16(const krk_adapter_shape* shape, const krk_adapter_args* args, void* workspace, size_t workspace_bytes,
                     void* stream);

/* 0 for an invalid shape as well; krk_adapter_check and krk_adapter_bf16 then say why. */
size_t krk_adapter_workspace_bytes(const krk_adapter_shape* shape);

/* KRK_ADAPTER_OK, or the error that krk_adapter_bf16 would report for this shape. */
int krk_adapter_check(const krk_adapter_shape* shape);

/* ABI identification: a binding that lays these structs out itself compares the
 * version and the sizes (in the order shape, args) before its first call. */
#define KRK_ADAPTER_ABI_VERSION 1
int krk_adapter_abi_version(void);
size_t krk_adapter_struct_size(int which);

/* Text of the last error raised on the calling thread by a function of this
 * header ("" if none). */
const char* krk_adapter_last_error(void);

#ifdef __cplusplus
}
#endif

#endif /* KRK_ADAPTER_H */
