// Per-head RMSNorm of q and k, rotary embedding and the cache write (gfx950).
//
//   y  = x * rsqrt(mean(x^2) + eps) * gain
//   y' = (y_lo cos - y_hi sin, y_hi cos + y_lo sin)
//
// in fp32, rounded to bf16 once.  Bound by reading and writing qkv once (4 * D
// bytes a head and row).  A head is D / 8 lanes of 8 elements (16-byte loads
// and stores); the sum of squares is a butterfly over those lanes, and the
// other half of the rotation comes from the lane D / 16 away.  Every element
// is read and written by its own lanes' head group alone, so q_out may be qkv.
#pragma once

#include "krk_attn_common.h"

namespace krk {

struct RopeParams {
    const uint16_t* qkv;
    int64_t qkv_row;
    const uint16_t *q_norm, *k_norm;
    float eps;
    const float* table;
    int table_rows;
    const int32_t* positions;
    const int32_t* lens;
    uint16_t* q_out;
    int64_t q_row;
    uint16_t *k, *v;
    int64_t k_seq, k_slot, k_head, v_seq, v_slot, v_head;
    int B, R, heads, kv_heads, capacity;
};

template <int D>
__global__ void __launch_bounds__(256) qk_norm_rope_kernel(RopeParams p) {
    constexpr int L = D / 8;  // lanes of a head
    const int all = p.heads + 2 * p.kv_heads;
    const int64_t unit = ((int64_t)blockIdx.x * 256 + threadIdx.x) / L;  // row * all + head
    const int64_t row = unit / all;
    const bool in = row < (int64_t)p.B * p.R;
    const int64_t at = in ? row : 0;
    const int h = in ? (int)(unit - row * all) : 0;
    const int c = threadIdx.x % L;
    const int b = (int)(at / p.R);
    int len = p.lens[b];
    len = len < 0 ? 0 : len > p.capacity ? p.capacity : len;
    const int slot = len - p.R + (int)(at - (int64_t)b * p.R);
    const int pos = p.positions ? p.positions[at] : slot;
    const bool ok = in && slot >= 0 && pos >= 0 && pos < p.table_rows;
    const u32x4 x = load_stream16(p.qkv + at * p.qkv_row + (int64_t)h * D + 8 * c);
    if (h >= p.heads + p.kv_heads) {  // v: as it is
        if (ok)
            *reinterpret_cast<u32x4*>(p.v + (int64_t)b * p.v_seq + (int64_t)slot * p.v_slot +
                                      (int64_t)(h - p.heads - p.kv_heads) * p.v_head + 8 * c) = x;
        return;  // whole groups of L lanes: no butterfly below reaches them
    }
    float y[8], ss = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t w = x[i];
        y[2 * i] = bf16_to_f32(w & 0xffffu);
        y[2 * i + 1] = __uint_as_float(w & 0xffff0000u);
    }
    const bool is_q = h < p.heads;
    if (p.q_norm) {
#pragma unroll
        for (int i = 0; i < 8; ++i) ss = __builtin_fmaf(y[i], y[i], ss);
#pragma unroll
        for (int s = 1; s < L; s <<= 1) ss += __shfl_xor(ss, s);
        const float rstd = __frsqrt_rn(ss / (float)D + p.eps);
        const u32x4 g = load_cached16((is_q ? p.q_norm : p.k_norm) + 8 * c);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t w = g[i];
            y[2 * i] = y[2 * i] * rstd * bf16_to_f32(w & 0xffffu);
            y[2 * i + 1] = y[2 * i + 1] * rstd * __uint_as_float(w & 0xffff0000u);
        }
    }
    const bool upper = c >= L / 2;
    const float* t = p.table + (int64_t)(ok ? pos : 0) * D + 8 * (upper ? c - L / 2 : c);
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 8; i += 4) {
        const f32x4 cs = *reinterpret_cast<const f32x4*>(t + i);
        const f32x4 sn = *reinterpret_cast<const f32x4*>(t + D / 2 + i);
        float z[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float other = __shfl_xor(y[i + e], L / 2);
            z[e] = __builtin_fmaf(other, upper ? sn[e] : -sn[e], y[i + e] * cs[e]);
        }
        r[i / 2] = pack_bf16(z[0], z[1]);
        r[i / 2 + 1] = pack_bf16(z[2], z[3]);
    }
    if (!ok) return;
    uint16_t* to = is_q ? p.q_out + at * p.q_row + (int64_t)h * D
                        : p.k + (int64_t)b * p.k_seq + (int64_t)slot * p.k_slot + (int64_t)(h - p.heads) * p.k_head;
    *reinterpret_cast<u32x4*>(to + 8 * c) = r;
}

}  // namespace krk
