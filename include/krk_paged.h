/*
 * krk_paged.h — C ABI of the paged key/value cache on MI355X (gfx950): a step
 * over many requests of different lengths, whose keys lie in pages of one pool.
 *
 *   krk_page_step            pages given back and taken for the step's new rows;
 *                            page tables, and each row's slot, position and owner
 *   krk_paged_rope_bf16      per-head RMSNorm of q and k, rotary embedding, and
 *                            the rows' k and v written into their slots
 *   krk_paged_attn_bf16      attention of every request's new rows over its
 *                            pages: single tokens, drafts and chunks of prompts
 *                            in one call
 *
 * Stands beside krk_attn.h, whose caches hold one run of slots per sequence; the
 * reference has no paged cache.
 *
 * A step has B requests; request b brings rows starts[b] .. starts[b + 1] - 1 of
 * the step's `rows` rows (0 of them when it is idle).  Rows behind starts[B] belong
 * to nobody.  Its keys are in pages table[b][0], table[b][1], ... of page_size slots
 * each: position t in slot t % page_size of page table[b][t / page_size].
 *
 * Operands are bf16 (raw 16-bit patterns) in device memory unless said otherwise.
 * Nothing here allocates, synchronises or reads device memory on the host: every
 * call enqueues its kernels on `stream` and returns, so it may be recorded into a
 * HIP graph.  Strides are in elements.
 */
#ifndef KRK_PAGED_H
#define KRK_PAGED_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Return codes: those of krk_gemm.h (0 = success, negative = error). */
enum {
    KRK_PAGED_OK = 0,
    KRK_PAGED_ERR_INVALID = -1,     /* sizes, null pointers, unknown values */
    KRK_PAGED_ERR_ALIGN = -2,       /* a pointer or stride is not aligned */
    KRK_PAGED_ERR_ALIAS = -3,       /* an output shares memory with another operand */
    KRK_PAGED_ERR_WORKSPACE = -4,   /* workspace missing or too small */
    KRK_PAGED_ERR_HIP = -5,         /* the HIP runtime rejected a launch */
    KRK_PAGED_ERR_UNSUPPORTED = -6  /* a head size this build has no kernel for */
};

/* Limits: B <= 4096, rows <= 2^18, page_size a power of two, 8 .. 4096,
 * pages * page_size < 2^31, width * page_size < 2^27. */

/*
 * krk_page_step — for request b, with old = lens[b] taken into 0 .. width * page_size,
 * cut = min(old, max(keep[b], 0)) (keep NULL: old) and n = max(fresh[b], 0):
 *
 *   1. the pages behind ceil(cut / page_size) of its ceil(old / page_size) are pushed on
 *      the stack of free pages, all requests' together so that the first request's
 *      first page ends on top;
 *   2. ceil((cut + n) / page_size) - ceil(cut / page_size) pages are popped, request
 *      after request, each request's first page first, and appended to its table row;
 *   3. lens[b] = cut + n.
 *
 * A request's rows do not fit if they end behind `rows`, cut + n passes the table's
 * width, or the stack does not hold what it and the requests before it need (those
 * that fail the first two tests need nothing).  It then takes no pages, lens[b] = cut,
 * keys[b] = 0 and its rows have no slot.
 *
 *   starts     [B + 1] sums of n, at most `rows`
 *   keys       [B] lens, or 0 where the rows did not fit: what krk_paged_attn takes
 *   slots      [rows] page * page_size + offset; -1 for rows that have none
 *   positions  [rows] cut + i for a request's row i; -1 where slots is
 *   owner      [rows] labels[b], or b where labels is NULL; -1 where slots is
 *
 * free_pages NULL (free_count then too): the caller keeps the tables, and nothing is
 * pushed or popped.  A page number outside 0 .. pages - 1 gives its rows no slot.
 * Table entries behind a request's pages, and the stack behind its count once what
 * was pushed has been popped, are left as they were.
 */
typedef struct krk_page_step_args {
    int32_t* lens;          /* [B] in and out */
    const int32_t* keep;    /* [B] or NULL */
    const int32_t* fresh;   /* [B] new rows */
    const int32_t* labels;  /* [B] or NULL */
    int32_t* table;         /* [B, width], row stride table_row; in and out */
    int64_t table_row;
    int32_t* free_pages;    /* [pages] or NULL; in and out */
    int32_t* free_count;    /* [1] or NULL; in and out */
    int32_t *starts, *keys, *slots, *positions, *owner;
    int B, rows, pages, page_size, width;
} krk_page_step_args;
int krk_page_step(const krk_page_step_args* args, void* stream);

/* A [pages, page_size, heads, head_dim] tensor of keys or values.  Strides in
 * elements, multiples of 8 and not negative (below 2^31, slot below 2^25); base 16-byte aligned;
 * the elements of a head are contiguous.  Rows of a written one may not share memory
 * (sorted by size, each stride is at least the extent of what lies inside it); written
 * k and v may be views of one tensor with the same strides. */
typedef struct krk_pages {
    void* p;
    int64_t page; /* from page to page */
    int64_t slot; /* from key to key */
    int64_t head; /* from head to head */
} krk_pages;

/*
 * krk_paged_rope_bf16 — for each row of qkv = [q heads; k heads; v heads]:
 *
 *   y  = x * rsqrt(mean(x^2) + eps) * gain             per q head and k head
 *   y' = (y_lo cos - y_hi sin, y_hi cos + y_lo sin)    lo, hi: the head's halves
 *
 * q' to q_out, k' and v to the row's slot.  cos and sin are row positions[row] of
 * `table` ([table_rows, head_dim] fp32: cosines, then sines).  All in fp32 with one
 * rounding at the end.  Rows whose slot is outside the pool, or whose position is
 * outside the table, leave q_out and the pages as they were.  Two rows with one
 * slot: either's k and v.
 *
 *   qkv     [rows, (heads + 2 * kv_heads) * head_dim], row stride qkv_row
 *   q_norm, k_norm   [head_dim] gains, 16-byte aligned; NULL both: no norm
 *   q_out   [rows, heads * head_dim], row stride q_row; may be qkv itself
 *           (same pointer and stride: in place)
 */
typedef struct krk_paged_rope_args {
    const void* qkv;
    int64_t qkv_row;
    const void *q_norm, *k_norm;
    float eps;
    const float* table;
    int table_rows;
    const int32_t* slots;     /* [rows] */
    const int32_t* positions; /* [rows] */
    void* q_out;
    int64_t q_row;
    krk_pages k, v;
    int rows, heads, kv_heads, head_dim, pages, page_size;
} krk_paged_rope_args;
int krk_paged_rope_bf16(const krk_paged_rope_args* args, void* stream);

/* What a call of krk_paged_attn_bf16 computes, fixed for an object that makes many of
 * them: it decides the grid and the workspace.  A request's tiles of rows have a
 * workgroup each per key/value head, fewer than 2^24 in all (only shapes of thousands
 * of requests and of key/value heads can have more; krk_paged_check says so). */
typedef struct krk_paged_shape {
    int B, rows;         /* requests; rows of the call (rows * heads < 2^25) */
    int heads, kv_heads; /* heads a multiple of kv_heads */
    int head_dim;        /* 64 or 128 */
    int page_size, width;/* slots of a page; entries of a table row */
    int window;          /* 0: every earlier key; else a row sees the `window` last keys up to itself */
    int sinks;           /* with a window: the first `sinks` positions stay visible */
} krk_paged_shape;

/*
 * Operands of krk_paged_attn_bf16.  With G = heads / kv_heads, query head h reads
 * key/value head h / G.  Row i of request b's n = starts[b + 1] - starts[b] rows has
 * position pos = keys[b] - n + i (keys[b] taken into 0 .. width * page_size, starts into
 * 0 .. rows) and sees position t where t <= pos and (window == 0 or t > pos - window or
 * t < sinks):
 *
 *   out[row, h] = sum_t p_t v_t,   p = softmax over the visible t of scale * (q[row, h] . k_t)
 *
 * Rows of negative position, and rows whose scores are all -infinity, give zeros in
 * out and -infinity in lse.  Rows behind starts[B] are left as they were.  Keys that a
 * row does not see have no part in its result, whatever they hold (NaN and infinities
 * too), and table entries of pages that no row sees are of no matter.  An entry
 * outside 0 .. pages - 1 for a page that is seen reads another page of the pool.
 * starts have to ascend; where they do not, rows may be left as they were.
 *
 * Sums, maxima and weights are held in 32 bits.  The weights enter the products with
 * v as bf16 parts: of a request with up to 16 pairs of a row and a query head per
 * key/value head as three (2^-24), with up to KRK_PAGED_FEW_ROWS as two (2^-16), with
 * more rounded to one: an output is then off by up to 2^-8 of sum p |v| besides its own
 * rounding.
 */
#define KRK_PAGED_FEW_ROWS 64
typedef struct krk_paged_attn_args {
    const void* q;            /* [rows, heads * head_dim], row stride q_row (multiple of 8) */
    int64_t q_row;
    krk_pages k, v;           /* [pages, page_size, kv_heads, head_dim] */
    int pages;
    float scale;              /* > 0, at most 2.3e38 */
    const int32_t* table;     /* [B, width], row stride table_row */
    int64_t table_row;
    const int32_t* starts;    /* [B + 1] */
    const int32_t* keys;      /* [B] */
    void* out;                /* [rows, heads * head_dim], row stride out_row (multiple of 8) */
    int64_t out_row;
    float* lse;               /* [rows, heads] log of the softmax's sum, or NULL */
} krk_paged_attn_args;

/* One call.  `workspace`: krk_paged_workspace_bytes(shape) bytes, 16-byte aligned.  It
 * must be zero-filled once before its first use; every call leaves its counters, at
 * the start, zero again and partial results behind them, so shapes may share one of the
 * largest size.  Calls that share one must be ordered on one stream.  Results are
 * deterministic. */
int krk_paged_attn_bf16(const krk_paged_shape* shape, const krk_paged_attn_args* args, void* workspace,
                        size_t workspace_bytes, void* stream);

/* 0 for an invalid shape as well; krk_paged_check and krk_paged_attn_bf16 then say why. */
size_t krk_paged_workspace_bytes(const krk_paged_shape* shape);

/* KRK_PAGED_OK, or the error that krk_paged_attn_bf16 would report for this shape. */
int krk_paged_check(const krk_paged_shape* shape);

/* ABI identification: a binding that lays these structs out itself compares the
 * version and the sizes (in the order page step, rope, shape, attn) before its first
 * call. */
#define KRK_PAGED_ABI_VERSION 1
int krk_paged_abi_version(void);
size_t krk_paged_struct_size(int which);

/* Text of the last error raised on the calling thread by a function of this
 * header ("" if none). */
const char* krk_paged_last_error(void);

#ifdef __cplusplus
}
#endif

#endif /* KRK_PAGED_H */
