/*
 * krk_attn.h — C ABI of the cache operators of a decode step on MI355X
 * (gfx950): what runs between the qkv projection and the o projection.
 *
 *   krk_qk_norm_rope_bf16   per-head RMSNorm of q and k, rotary embedding, and
 *                           the new rows' k and v written into the cache
 *   krk_attn_bf16           attention of the new rows over the cache: causal,
 *                           with a sliding window and sinks, with the ancestor
 *                           masks of a draft tree, over a prefix shared by the
 *                           whole batch, and with the keys' weights added to
 *                           their scores
 *   krk_cache_evict_bf16    the cache cut down to a budget of slots per head
 *
 * Stands where the reference has engine/kernels/rope.py (qk_norm_rope_cache)
 * and engine/kernels/attention.py (DecodeAttention); the shared prefix, the
 * window, the scores and the eviction have no counterpart there.
 *
 * Operands are bf16 (raw 16-bit patterns) in device memory unless said
 * otherwise.  Nothing here allocates, synchronises or reads device memory on
 * the host: every call enqueues its kernels on `stream` and returns, so it may
 * be recorded into a HIP graph.  Strides are in elements.
 *
 * A batch is B sequences with R new rows each; row b * R + i belongs to
 * sequence b.  Sequence b has lens[b] cached keys (read on the device and
 * taken into 0 .. capacity), the call's own R rows among them and last: row i
 * lies in slot lens[b] - R + i.  Rows whose slot is negative (a sequence shorter
 * than R, an idle one with lens 0) are padding.
 */
#ifndef KRK_ATTN_H
#define KRK_ATTN_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Return codes: those of krk_gemm.h (0 = success, negative = error). */
enum {
    KRK_ATTN_OK = 0,
    KRK_ATTN_ERR_INVALID = -1,     /* sizes, null pointers, unknown values */
    KRK_ATTN_ERR_ALIGN = -2,       /* a pointer or stride is not aligned */
    KRK_ATTN_ERR_ALIAS = -3,       /* an output shares memory with another operand */
    KRK_ATTN_ERR_WORKSPACE = -4,   /* workspace missing or too small */
    KRK_ATTN_ERR_HIP = -5,         /* the HIP runtime rejected a launch */
    KRK_ATTN_ERR_UNSUPPORTED = -6  /* a head size this build has no kernel for */
};

/* A [.., slots, heads, head_dim] tensor of keys or values.  Strides in
 * elements, multiples of 8 and not negative; base 16-byte aligned; the
 * elements of a head are contiguous.  Rows of a written one may not share memory
 * (sorted by size, each stride is at least the extent of what lies inside it);
 * written k and v may be views of one tensor with the same strides. */
typedef struct krk_cache {
    void* p;
    int64_t seq;  /* from sequence to sequence (ignored for a prefix) */
    int64_t slot; /* from key to key */
    int64_t head; /* from head to head */
} krk_cache;

/* What a call of krk_attn_bf16 computes, fixed for an object that makes many
 * of them: it decides how the work is cut and the workspace. */
typedef struct krk_attn_shape {
    int B, R;            /* sequences; new rows of each (R <= 65536, B * R * heads < 2^25, B * kv_heads < 2^23) */
    int heads, kv_heads; /* heads a multiple of kv_heads */
    int head_dim;        /* 64 or 128 */
    int capacity;        /* slots of the cache, >= 1 */
    int window;          /* 0: every earlier key; else a row sees the `window` last keys up to itself */
    int sinks;           /* with a window: the first `sinks` positions stay visible */
    int prefix;          /* keys of the shared prefix, 0 for none; prefix + capacity < 2^27 */
    int scored;          /* 1: scores are updated (no prefix) */
} krk_attn_shape;

/*
 * Operands of krk_attn_bf16.  With G = heads / kv_heads, query head h reads
 * key/value head h / G.  The key in slot s has position prefix + s, prefix key
 * j position j.  Row i at position pos = prefix + lens - R + i sees position t
 * where t <= pos and (window == 0 or t > pos - window or t < sinks), and
 *
 *   out[row, h] = sum_t p_t v_t,   p = softmax over the visible t of scale * (q[row, h] . k_t)
 *
 * With `tree`, bit j of tree[b * R + i] says whether row i sees the call's own
 * row j (its slot lens - R + j), whatever the window; bits R and up, and those of
 * padding rows, are ignored.  The row's position is then that of the sequence's
 * first row that has a slot, plus the bits set, less 1, and it sees the earlier
 * keys by that.  Needs R <= 64 and window 0 or >= R.
 *
 * Padding rows, and rows that see nothing (or whose scores are all -infinity),
 * give zeros in out and -infinity in lse.  Keys that a row does not see have no
 * part in its result, whatever they hold (NaN and infinities too).  Sums, maxima
 * and weights are held in 32 bits.  The weights enter the products with v as two
 * bf16 parts (off by 2^-16), or, where 128 rows share a workgroup (krk_attn_plan
 * tells), rounded to one: an output is then off by up to 2^-8 of sum p |v| besides
 * its own rounding.
 */
typedef struct krk_attn_args {
    const void* q;     /* [B * R, heads * head_dim], row stride q_row (multiple of 8) */
    int64_t q_row;
    krk_cache k, v;    /* [B, capacity, kv_heads, head_dim] */
    krk_cache kp, vp;  /* [prefix, kv_heads, head_dim]; p NULL without a prefix */
    int prefix;        /* its keys in this call, 0 .. shape.prefix */
    float scale;       /* > 0, at most 2.3e38 */
    const int32_t* lens;      /* [B] */
    const int64_t* tree;      /* [B, R] or NULL */
    void* out;                /* [B * R, heads * head_dim], row stride out_row (multiple of 8) */
    int64_t out_row;
    float* lse;               /* [B * R, heads] log of the softmax's sum, or NULL */
    const float* scores;      /* scored: [B, kv_heads, capacity], strides sc_seq, sc_head */
    int64_t sc_seq, sc_head;
    float* scores_out;        /* the scores plus this call's weights, summed over rows and the
                                 G query heads; slots below lens are written.  May be `scores`. */
    int64_t so_seq, so_head;
} krk_attn_args;

/* One call.  `workspace`: krk_attn_workspace_bytes(shape) bytes, 16-byte
 * aligned (may be NULL when that is 0).  It must be zero-filled once before its
 * first use; every call leaves its counters, at the start, zero again and
 * partial results behind them.  Calls that share one workspace must be ordered
 * on one stream.  Shapes of the same B and kv_heads may share one (of the largest
 * one's size); for another B or kv_heads it is zero-filled again first.  Results
 * are deterministic. */
int krk_attn_bf16(const krk_attn_shape* shape, const krk_attn_args* args, void* workspace, size_t workspace_bytes,
                  void* stream);

/* 0 for an invalid shape as well; krk_attn_check and krk_attn_bf16 then say why. */
size_t krk_attn_workspace_bytes(const krk_attn_shape* shape);

/* KRK_ATTN_OK, or the error that krk_attn_bf16 would report for this shape. */
int krk_attn_check(const krk_attn_shape* shape);

/* How the work is cut for this shape.  Rows are pairs of a new row and a query
 * head of one key/value head.  Up to 64 of them (16 or 32 per workgroup) run on
 * a kernel whose waves divide the keys, more (128 per workgroup) on one whose
 * waves divide the rows and which rounds the weights to bf16. */
typedef struct krk_attn_plan_t {
    int rows;           /* of a workgroup: 16, 32 or 128 */
    int splits;         /* key ranges of a sequence's own cache */
    int prefix_rows;    /* the same for the prefix (0 without one) */
    int prefix_splits;
} krk_attn_plan_t;
int krk_attn_plan(const krk_attn_shape* shape, krk_attn_plan_t* out);

/*
 * krk_qk_norm_rope_bf16 — for row b * R + i with qkv = [q heads; k heads; v heads]:
 *
 *   y  = x * rsqrt(mean(x^2) + eps) * gain             per q head and k head
 *   y' = (y_lo cos - y_hi sin, y_hi cos + y_lo sin)    lo, hi: the head's halves
 *
 * q' to q_out, k' and v to slot lens - R + i of the cache.  cos and sin are
 * row `position` of `table` ([table_rows, head_dim] fp32: cosines, then
 * sines), position = positions[row], or the slot where positions is NULL.
 * All in fp32 with one rounding at the end.  Padding rows, and rows whose
 * position is outside the table, leave q_out and the cache as they were.
 *
 *   qkv     [B * R, (heads + 2 * kv_heads) * head_dim], row stride qkv_row
 *   q_norm, k_norm   [head_dim] gains, 16-byte aligned; NULL both: no norm
 *   q_out   [B * R, heads * head_dim], row stride q_row; may be qkv itself
 *           (same pointer and stride: in place)
 */
typedef struct krk_rope_args {
    const void* qkv;
    int64_t qkv_row;
    const void *q_norm, *k_norm;
    float eps;
    const float* table;
    int table_rows;
    const int32_t* positions; /* [B * R] or NULL */
    const int32_t* lens;      /* [B] */
    void* q_out;
    int64_t q_row;
    krk_cache k, v;
    int B, R, heads, kv_heads, head_dim, capacity;
} krk_rope_args;
int krk_qk_norm_rope_bf16(const krk_rope_args* args, void* stream);

/*
 * krk_cache_evict_bf16 — for each sequence b and head: with lens[b] <= budget
 * every slot stays; else the first `sinks` and the last `recent` slots stay,
 * and of the others the budget - sinks - recent with the highest scores (equal
 * scores: the lower slot; NaN above +infinity, -0 equal to +0).  The kept
 * slots, in their order, become slots 0, 1, ... of the k_out, v_out and
 * scores_out; what lies behind them there is left as it was.
 *
 *   keep       [B, kv_heads, budget] int32: the kept slots, ascending, then -1
 *   lens_out   [B] int32: min(lens, budget); may be lens
 *   k_out, v_out   [B, >= budget, kv_heads, head_dim]; may be k and v (in place:
 *              all of the three outputs then), else share no memory with them
 *   scores, scores_out   [B, kv_heads, slots] fp32
 *
 * 0 <= sinks, 0 <= recent, sinks + recent <= budget <= capacity.
 */
typedef struct krk_evict_args {
    krk_cache k, v, k_out, v_out;
    const float* scores;
    int64_t sc_seq, sc_head;
    float* scores_out;
    int64_t so_seq, so_head;
    const int32_t* lens;
    int32_t* lens_out;
    int32_t* keep;
    int B, kv_heads, head_dim, capacity, budget, sinks, recent;
} krk_evict_args;
int krk_cache_evict_bf16(const krk_evict_args* args, void* stream);

/* ABI identification: a binding that lays these structs out itself compares
 * the version and the sizes (in the order shape, args, rope, evict, plan)
 * before its first call. */
#define KRK_ATTN_ABI_VERSION 1
int krk_attn_abi_version(void);
size_t krk_attn_struct_size(int which);

/* Text of the last error raised on the calling thread by a function of this
 * header ("" if none). */
const char* krk_attn_last_error(void);

#ifdef __cplusplus
}
#endif

#endif /* KRK_ATTN_H */
