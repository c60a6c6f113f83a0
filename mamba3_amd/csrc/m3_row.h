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

// A 64-bit number as fp32 rounded to odd.
__device__ __forceinline__ float odd_of(double v) {
    const float near = (float)v;
    const double rest = v - (double)near;
    const unsigned b = __builtin_bit_cast(unsigned, near), toward = (unsigned)(__builtin_bit_cast(uint64_t, rest) >> 32 ^ b) >> 31;  // 1: toward zero
    constexpr int kNumber = 0x198;  // but for 0, infinity and NaN
    return __builtin_bit_cast(float, __builtin_amdgcn_class(rest, kNumber) ? (b - toward) | 1u : b);
}
// silu(g) u as fp32 rounded to odd, from 2^-34 of the exact product: e = exp(-|g|) = 2^n 2^f with |f| <= 1/2 and a polynomial for 2^f
// (off by 2^-34.5 of it at most, by Remez's exchange), 1 / (1 + e) from the hardware's estimate and one step of Newton.
__device__ __forceinline__ float silu_mul_odd(float gate, float u) {
    const double g = (double)gate;
    const double x = fmax(fabs(g) * -1.4426950408889634, -1100.0);  // -log2 e; below 2^-1074 e is 0 (NaN comes back in by g)
    const double n = rint(x), f = x - n;
    double p = 1.5201921594169677e-05;
    p = fma(p, f, 0.00015469291141683767);
    p = fma(p, f, 0.001333392256354045);
    p = fma(p, f, 0.00961802725366847);
    p = fma(p, f, 0.05550410353447978);
    p = fma(p, f, 0.24022651198157585);
    p = fma(p, f, 0.693147180728447);
    p = fma(p, f, 0.9999999999616819);
    const double e = ldexp(p, (int)n), d = 1.0 + e;
    const double r = (double)__builtin_amdgcn_rcpf((float)d);
    return odd_of((g < 0.0 ? g * e : g) * fma(r, fma(-d, r, 1.0), r) * (double)u);
}

// v = silu(v) u for results that are rounded to 8 bits and fewer, which fall as the exact product's would (silu_mul_odd). With e = exp(-|g|),
// at most 1: silu = (g < 0 ? g e : g) / (1 + e), which does not overflow. It is computed in 32 bits first: e from the hardware's power of
// two, with the rounding of its argument put right, 1 / (1 + e) from its reciprocal. That is off by at most 4.5 2^-23 of the
// product (e 1.5, the sum 0.5, the reciprocal 1, three products 1.5), nine steps of fp32, which matters next to a tie only. Ties, and
// what the scale turns on, have at most five significant bits whatever the scale: their last 19 bits are zeros. Products within
// kNear steps of such a number (1 in 25000) are computed again. So are those of g < -80, where e nears the smallest numbers, unless the
// lane holds a product that makes zeros of them; and those of |g| > 2^127, whose exponent overflows: they come out as NaN, whose last bits
// are zeros, too. (Products and gates below 2^-126 fp32 itself holds in fewer bits.) Gating 8192 x 2112 in bf16: 18.3 us, 17.5 in 32 bits
// alone, 31 in 64 throughout. In 32 bits alone 83 of 104 million e4m3 elements fell on the other side of a tie, with expf and a division 70.
__device__ __forceinline__ void silu_mul8(float (&v)[8], const float (&u)[8]) {
    constexpr float kHi = 1.44269502f, kLo = 1.92596299e-8f, kLn2 = 0.693147182f;  // log2 e = kHi + kLo
    constexpr unsigned kNear = 10u;
    const auto close = [](float x) __attribute__((always_inline)) { return (__builtin_bit_cast(unsigned, x) + kNear) << 13; };
    float g[8], low = 0.f;
    unsigned nearest = ~0u, any = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        g[i] = v[i];
        const float a = -fabsf(g[i]), x = a * kHi;
        const float rest = fmaf(a, kLo, fmaf(a, kHi, -x));
        float e = __builtin_amdgcn_exp2f(x);
        e = fmaf(e * kLn2, rest, e);
        v[i] = (g[i] < 0.f ? g[i] * e : g[i]) * __builtin_amdgcn_rcpf(1.f + e) * u[i];
        nearest = min(nearest, close(v[i]));
        any |= __builtin_bit_cast(unsigned, v[i]);
        low = fminf(low, g[i]);
    }
    if ((nearest <= 2 * kNear << 13 && any << 1) || low < -80.f) {  // (behind a row's end all are zeros)
        // |g| exp(-|g|) is below 2^-109 for g < -80: times u an element is half its smallest step where it is 2^-19 of the largest
        float top = 0.f, up = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(v[i])), up = fmaxf(up, fabsf(u[i]));
        const bool zeros = top >= 0x1p-50f && up <= 0x1p30f;
        unsigned marks = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) marks |= g[i] < -80.f ? (zeros ? 0u : 1u << i) : close(v[i]) <= 2 * kNear << 13 && v[i] != 0.f ? 1u << i : 0u;
        while (marks) {
            const unsigned at = __builtin_ctz(marks);
            marks &= marks - 1;
            float gate = g[0], up = u[0];
#pragma unroll
            for (int i = 1; i < 8; ++i) gate = at == i ? g[i] : gate, up = at == i ? u[i] : up;
            const float x = silu_mul_odd(gate, up);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = at == i ? x : v[i];
        }
    }
}

}  // namespace m3
