// What the norm and the gate compute, for the kernels that run them by themselves and in front of a product (gfx950).
#pragma once

#include "m3_common.h"
#include "m3_mfma.h"

namespace m3 {

// Sum over the wave's lanes, in fp64: lane moves within 16 lanes, shuffles across.
__device__ __forceinline__ double wave_sum_f64(double v) {
    auto move = [](double x, auto ctrl) {
        const u32x2 b = __builtin_bit_cast(u32x2, x);
        u32x2 o;
        o[0] = (unsigned)__builtin_amdgcn_update_dpp(0, (int)b[0], decltype(ctrl)::value, 0xF, 0xF, false);
        o[1] = (unsigned)__builtin_amdgcn_update_dpp(0, (int)b[1], decltype(ctrl)::value, 0xF, 0xF, false);
        return __builtin_bit_cast(double, o);
    };
    v += move(v, std::integral_constant<int, 0xB1>{});
    v += move(v, std::integral_constant<int, 0x4E>{});
    v += move(v, std::integral_constant<int, 0x141>{});
    v += move(v, std::integral_constant<int, 0x140>{});
    v += __shfl_xor(v, 16, kWave);
    v += __shfl_xor(v, 32, kWave);
    return v;
}
// 1 / sqrt(m): the hardware's estimate and one step of Newton.
__device__ __forceinline__ float inv_sqrt(float m) {
    const float r = __builtin_amdgcn_rsqf(m);
    const float e = fmaf(-m * r, r, 1.f);
    // m of 0, infinity or NaN: the estimate is the answer
    return fabsf(e) <= 1.f ? fmaf(0.5f * r, e, r) : r;
}

// silu without the overflow of exp(-g): e = exp(-|g|) is at most 1.
__device__ __forceinline__ float silu_any(float g) {
    const float e = expf(-fabsf(g));
    return (g < 0.f ? g * e : g) / (1.f + e);
}

}  // namespace m3
