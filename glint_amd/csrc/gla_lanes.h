// gla_lanes.h -- what the matrix-core kernels share: exp2, the soft-cap, and maxima and
// sums over lanes by DPP and row swaps.
#pragma once

#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <type_traits>

namespace gla {
namespace lanes {

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// max of two floats as IEEE-754 maximum (a NaN operand gives NaN): gfx950
// has v_maximum3_f32, which needs no NaN-quieting max per operand the way
// fmaxf does after a row swap or a select. Not inline asm: the compiler
// inserts the wait states an MFMA result needs before a VALU read only for
// instructions it emits itself, and these maxima read MFMA results directly.
__device__ __forceinline__ float max2f(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// max / sum over the four 16-lane rows (lane ^ 16, lane ^ 32) with the gfx950
// row swaps: VALU only, no LDS round trip.
__device__ __forceinline__ float max_rows4(float x) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = max2f(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto c = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return max2f(__uint_as_float(c[0]), __uint_as_float(c[1]));
}
__device__ __forceinline__ float sum_rows4(float x) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto c = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(c[0]) + __uint_as_float(c[1]);
}

// sum over the 16 lanes of a row (DPP rotations)
__device__ __forceinline__ float sum_row16(float x) {
    const auto turned = [](float v, auto control) {
        return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), decltype(control)::value, 0xf, 0xf, true));
    };
    x += turned(x, std::integral_constant<int, 0x121>{});  // row_ror 1, 2, 4, 8
    x += turned(x, std::integral_constant<int, 0x122>{});
    x += turned(x, std::integral_constant<int, 0x124>{});
    x += turned(x, std::integral_constant<int, 0x128>{});
    return x;
}

// sum over the wave's lanes up to and with this one: DPP shifts within each 16-lane row, then the
// rows' last lanes into the rows behind them
__device__ __forceinline__ int sum_to_lane(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, true);  // row_shr 1, 2, 4, 8
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // row_bcast 15, into rows 1 and 3
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // row_bcast 31, into rows 2 and 3
    return x;
}

// max / min of unsigned words over the wave, in every lane: DPP rotations within
// each 16-lane row, then the row swaps.
template <bool MAX>
__device__ __forceinline__ uint32_t wave_extreme(uint32_t x) {
    const auto pick = [](uint32_t a, uint32_t b) { return MAX ? max(a, b) : min(a, b); };
    x = pick(x, __builtin_amdgcn_update_dpp(0, x, 0x121, 0xf, 0xf, true));  // row_ror 1, 2, 4, 8
    x = pick(x, __builtin_amdgcn_update_dpp(0, x, 0x122, 0xf, 0xf, true));
    x = pick(x, __builtin_amdgcn_update_dpp(0, x, 0x124, 0xf, 0xf, true));
    x = pick(x, __builtin_amdgcn_update_dpp(0, x, 0x128, 0xf, 0xf, true));
    const auto a = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    x = pick(a[0], a[1]);
    const auto c = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return pick(c[0], c[1]);
}
__device__ __forceinline__ uint32_t umax_rows4(uint32_t x) {
    const auto a = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    x = max(a[0], a[1]);
    const auto c = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return max(c[0], c[1]);
}

// cap * tanh(x / cap) * log2(e), without the long division sequences: x / cap
// by the reciprocal of cap and one correction, 1 / (1 + t) by v_rcp_f32 and one
// Newton step (each then within an ulp).
struct SoftCap {
    float cap, inv, out;
    __device__ __forceinline__ explicit SoftCap(float c) : cap(c), inv(1.0f / c), out(c * kLog2e) {}
    __device__ __forceinline__ float operator()(float x) const {
        const float q = x * inv;
        // past 16 tanh is 1, and an infinite score has no remainder
        const float y = fabsf(q) < 16.0f ? fmaf(fmaf(-cap, q, x), inv, q) : q;
        const float t = fast_exp2(-2.0f * kLog2e * fabsf(y));
        const float d = 1.0f + t;
        float r = __builtin_amdgcn_rcpf(d);
        r = fmaf(fmaf(-d, r, 1.0f), r, r);
        return copysignf((1.0f - t) * r * out, x);
    }
};
__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) x = fmaxf(x, __shfl_xor(x, o));
    return x;
}

}  // namespace lanes
}  // namespace gla
