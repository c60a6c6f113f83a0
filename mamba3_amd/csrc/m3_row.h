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

// For results that are rounded to 8 bits and fewer: 1 / sqrt(m) in two parts, and t r w as fp32 rounded to odd (to the odd one of
// its two neighbours where it is none), so that the next rounding falls as the exact product's would. Rounded to nearest,
// about one e4m3 element in a million would fall on the other side of a tie.
struct RowScale {
    float hi, lo;
};
__device__ __forceinline__ RowScale row_scale(double m) {
    const float r = inv_sqrt((float)m);
    const double e = fma(-m * (double)r, (double)r, 1.0);
    return RowScale{r, fabs(e) < 1e-3 ? (float)(0.5 * (double)r * e) : 0.f};  // (m of 0, infinity or NaN: hi is the answer)
}
__device__ __forceinline__ float norm_odd(float t, float w, RowScale r) {
    const float p = t * r.hi, hi = p * w;  // (t w first could overflow)
    const float rest = fmaf(fmaf(t, r.lo, fmaf(t, r.hi, -p)), w, fmaf(p, w, -hi));
    const unsigned b = __builtin_bit_cast(unsigned, hi), toward = (__builtin_bit_cast(unsigned, rest) ^ b) >> 31;  // 1: toward zero
    constexpr int kNumber = 0x198;  // but for 0, infinity and NaN
    return __builtin_bit_cast(float, __builtin_amdgcn_classf(rest, kNumber) ? (b - toward) | 1u : b);
}
// The sum of eight squares added to s. (Their roundings to fp32 average out over a row: about 2^-28 of its sum.)
__device__ __forceinline__ double add_squares(double s, const float (&t)[8]) {
    float q = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) q = fmaf(t[e], t[e], q);
    return s + (double)q;
}

// v = silu(v) u. With e = exp(-|g|), at most 1: silu = (g < 0 ? g e : g) / (1 + e), which does not overflow. For |g| < 80
// e comes from the hardware's power of two, with the rounding of its argument put right, and 1 / (1 + e) from its reciprocal
// (about 2 units in the last place together); beyond, where e nears the smallest numbers, from the library. With expf and a
// division throughout, gating 8192 x 2112 took 26 us instead of 20 (17.5 with an eight a thread).
__device__ __forceinline__ void silu_mul8(float (&v)[8], const float (&u)[8]) {
    float most = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(v[e]));
    bool near = most < 80.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) near &= v[e] == v[e];
    if (near) {
        constexpr float kHi = 1.44269502f, kLo = 1.92596299e-8f, kLn2 = 0.693147182f;  // log2 e = kHi + kLo
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float g = v[i], a = -fabsf(g), x = a * kHi;
            const float rest = fmaf(a, kLo, fmaf(a, kHi, -x));
            float e = __builtin_amdgcn_exp2f(x);
            e = fmaf(e * kLn2, rest, e);
            v[i] = (g < 0.f ? g * e : g) * __builtin_amdgcn_rcpf(1.f + e) * u[i];
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float g = v[i], e = expf(-fabsf(g));
            v[i] = (g < 0.f ? g * e : g) / (1.f + e) * u[i];
        }
    }
}

}  // namespace m3
