// gla_rows.h -- addresses of a storage row's elements, and the quantiser of
// Q8_0 storages, shared by the kernels that write and read rows.
//
// Quantize-on-write reproduces KvCacheQ8::quantize_into (src/cache/mod.rs:296-315)
// bit for bit: d = max|x| / 127 (1.0 for an all-zero block), q = clamp(round
// half away from zero(x * (1/d)), -127, 127) computed from the f32 d, NaN -> 0,
// and the stored scale is f16(d) rounded to nearest even.
#pragma once

#include "gla_internal.h"

namespace gla {
namespace {

struct RowOps {
    KvLayout L;
    int64_t n_rows_total;  // valid row ids are [0, n_rows_total)
    int head_dim;
    int head_shift;  // head_dim = 1 << head_shift
    int kv_dim;
    int n_blocks;  // kv_dim / 32
    bool q8;
};

RowOps row_ops(const gla_kv *kv) {
    RowOps o;
    o.L = layout_of(kv);
    o.n_rows_total = kv->n_pages * GLA_PAGE_SIZE;
    o.head_dim = kv->head_dim;
    o.head_shift = __builtin_ctz(kv->head_dim);  // 64, 128 or 256
    o.kv_dim = kv->kv_dim;
    o.n_blocks = kv->kv_dim / 32;
    o.q8 = kv->dtype == GLA_KV_Q8_0;
    return o;
}

// Byte offset of element `gi` (0 .. kv_dim-1) of row `row`, and of its scale.
__device__ __forceinline__ int64_t elem_off(const RowOps &o, int64_t row, int gi, int esize) {
    const int64_t page = row >> 4;
    const int slot = (int)(row & 15);
    const int h = gi >> o.head_shift;
    const int e = gi & (o.head_dim - 1);
    return page * o.L.page_stride + (int64_t)h * o.L.head_stride + (int64_t)slot * o.L.row_stride +
           (int64_t)e * esize;
}
// Byte offset of the Q8_0 scale of (row, element gi) from L.ks (which = 0,
// parity-grouped) or L.vs (which = 1, row-major).
__device__ __forceinline__ int64_t scale_off(const RowOps &o, int64_t row, int gi, int which) {
    const int64_t page = row >> 4;
    const int slot = (int)(row & 15);
    const int h = gi >> o.head_shift;
    const int e = gi & (o.head_dim - 1);
    const int idx = which ? slot * (o.head_dim >> 5) + (e >> 5) : q8ks_off(slot, e >> 5, o.head_dim);
    return page * o.L.page_stride + (int64_t)h * o.L.head_stride + (int64_t)idx * 2;
}

// Byte offset of Q8_0 quant (row, element gi) of K (which = 0) or V (1); the
// quants of a (page, head) are stored in MFMA operand order (q8k_off / q8v_off).
__device__ __forceinline__ int64_t q8_off(const RowOps &o, int64_t row, int gi, int which) {
    const int64_t page = row >> 4;
    const int slot = (int)(row & 15);
    const int h = gi >> o.head_shift;
    const int e = gi & (o.head_dim - 1);
    const int in_head = which ? q8v_off(slot, e, o.head_dim) : q8k_off(slot, e, o.head_dim);
    return page * o.L.page_stride + (int64_t)h * o.L.head_stride + in_head;
}

// max|x| of a block / 127, correctly rounded, or 1 of zeros. The residual of a first
// quotient corrects it (Markstein); that is exact while nothing over- or underflows.
__device__ __forceinline__ float scale_of(float max_abs) {
    if (!__any(max_abs < 0x1p-100f || max_abs > 0x1p100f)) {
        const float q = max_abs * (1.0f / 127.0f);
        return fmaf(fmaf(-127.0f, q, max_abs), 1.0f / 127.0f, q);
    }
    return max_abs > 0.0f ? max_abs / 127.0f : 1.0f;
}

// Half away from zero is truncation of y + copysign(the float below 1/2, y), the sum
// rounded; the conversion truncates, saturates and takes NaN to 0. In few
// instructions: they, not the bytes, bound an append of long prompts.
__device__ __forceinline__ int quantize_one(float x, float inv_d) {
#pragma clang fp contract(off)
    const float y = x * inv_d;
    const float t = y + __builtin_copysignf(0x1.fffffep-2f, y);
    int q;
    asm("v_cvt_i32_f32 %0, %1" : "=v"(q) : "v"(t));
    return min(max(q, -127), 127);
}

// The low bytes of four quants, stored as x + 128.
__device__ __forceinline__ uint32_t quant_bytes(int q0, int q1, int q2, int q3) {
    return (__builtin_amdgcn_perm(q1, q0, 0x0c0c0400u) | __builtin_amdgcn_perm(q3, q2, 0x04000c0cu)) ^ 0x80808080u;
}

// Quantise and store the N (8 or 4) elements gi .. gi + N - 1 of a row's K
// (which = 0) or V (1); the rest of the block of 32 is in the neighbouring lanes
// of an aligned group of 32 / N, which run this together.
template <int N>
__device__ __forceinline__ void store_q8(const RowOps &o, int64_t row, int gi, int which, const float (&x)[N]) {
    static_assert(N == 4 || N == 8, "blocks of 32 in 8 or 4 lanes");
    uint8_t *dst = const_cast<uint8_t *>(which ? o.L.v : o.L.k);
    float max_abs = 0.0f;
#pragma unroll
    for (int j = 0; j < N; j++) max_abs = fmaxf(max_abs, fabsf(x[j]));
    // quad_perm [1 0 3 2], then [2 3 0 1]; of eight lanes then the other quad
    max_abs = fmaxf(max_abs, __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(max_abs), 0xB1, 0xf, 0xf, true)));
    max_abs = fmaxf(max_abs, __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(max_abs), 0x4E, 0xf, 0xf, true)));
    if (N == 4)
        max_abs = fmaxf(max_abs, __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(max_abs), 0x141, 0xf, 0xf, true)));
    const float dsc = scale_of(max_abs);
    const float inv_d = 1.0f / dsc;
    uint32_t w[N / 4];
#pragma unroll
    for (int j = 0; j < N / 4; j++)
        w[j] = quant_bytes(quantize_one(x[4 * j], inv_d), quantize_one(x[4 * j + 1], inv_d), quantize_one(x[4 * j + 2], inv_d),
                           quantize_one(x[4 * j + 3], inv_d));
    if (!which) {  // K: 8 dims of a slot are 8 consecutive bytes
        uint8_t *at = dst + q8_off(o, row, gi, 0);
        if constexpr (N == 8)
            *reinterpret_cast<uint2 *>(at) = make_uint2(w[0], w[1]);
        else
            *reinterpret_cast<uint32_t *>(at) = w[0];
    } else {  // V: one byte per element, 4-position columns
#pragma unroll
        for (int j = 0; j < N; j++) dst[q8_off(o, row, gi + j, 1)] = (uint8_t)(w[j >> 2] >> ((j & 3) * 8));
    }
    if ((gi & 31) == 0) {
        uint8_t *sb = const_cast<uint8_t *>(which ? o.L.vs : o.L.ks);
        *reinterpret_cast<uint16_t *>(sb + scale_off(o, row, gi, which)) = __half_as_ushort(__float2half_rn(dsc));
    }
}

}  // namespace
}  // namespace gla
