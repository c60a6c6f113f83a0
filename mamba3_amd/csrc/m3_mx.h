// Microscaled values (gfx950): blocks of 32 elements along k share a power of two.
//   value = element * 2^E,  E + 127 in one byte (255: the block held an infinity or NaN, and is NaN)
// Elements are e4m3 (8 bits, largest 448) or e2m1 (4 bits, largest 6). E is the smallest exponent under
// which the block's largest magnitude still rounds to an element: nothing saturates. Elements round
// to nearest, ties to even. A block of zeros has E = 0.
//
// Stored as rows of kp = k rounded up to 128 elements (zeros behind k, E = 0): `data` kp bytes (e4m3) or
// kp / 2 (e2m1, the even k in the low half) a row, `scales` kp / 32 bytes a row. So rows are whole
// 16-byte pieces and whole steps of the matrix instructions, which take 128 k.
#pragma once

#include <atomic>

#include "m3_common.h"
#include "m3_mfma.h"

namespace m3 {

enum MxFormat { kE2m1 = 0, kE4m3 = 1 };
constexpr int kMxStep = 128;  // rows are padded to whole steps
__host__ __device__ constexpr int64_t mx_padded(int64_t k) { return (k + kMxStep - 1) / kMxStep * kMxStep; }
__host__ __device__ constexpr int64_t mx_row_bytes(int64_t kp, int format) { return format == kE4m3 ? kp : kp / 2; }

// Exact n / d for n < 2^31, d >= 2: m = ceil(2^(31 + l) / d) with l = ceil(log2 d); m d - 2^(31 + l) < 2^l keeps
// the error of n m / 2^(31 + l) below 1 / d.
struct FastDiv {
    unsigned m, s, d;
    explicit FastDiv(unsigned d_) : d(d_) {
        unsigned l = 0;
        while ((1ull << l) < d_) ++l;
        m = (unsigned)(((1ull << (31 + l)) + d_ - 1) / d_);
        s = l - 1;
    }
    __device__ __forceinline__ unsigned div(unsigned n) const { return __umulhi(n, m) >> s; }
};

// Allows dynamic LDS past 64 KB, once for each device (a bit of `done`; devices past 63 set it every time).
inline bool allow_lds(const void* kernel, int bytes, std::atomic<uint64_t>& done) {
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess) return false;
    const uint64_t bit = dev < 63 ? (uint64_t)1 << dev : 0;
    if (done.load(std::memory_order_relaxed) & bit) return true;
    if (hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes) != hipSuccess) return false;
    done.fetch_or(bit, std::memory_order_relaxed);
    return true;
}

// Magnitude bits: their order is the magnitudes', an infinity above all numbers and NaN above it.
__device__ __forceinline__ unsigned mag_bits(float v) { return __builtin_bit_cast(unsigned, v) & 0x7fffffffu; }

struct MxScale {
    unsigned byte;
    float inv;  // 2^-E
};
template <int F>
__device__ __forceinline__ MxScale mx_scale(unsigned top) {  // the block's largest magnitude
    const int ex = (int)(top >> 23);
    const unsigned frac = top & 0x7fffffu;
    // the largest element's exponent is 2 or 8; 7 and above round past 6, above 464 past 448
    int s = ex - (F == kE4m3 ? 8 : 2) + (F == kE4m3 ? frac > 0x680000u : frac >= 0x600000u);
    s = s < 0 ? 0 : s;
    s = top == 0 ? 127 : s;
    s = ex == 255 ? 255 : s;
    return MxScale{(unsigned)s, __builtin_bit_cast(float, (unsigned)(254 - s) << 23)};
}
// 2^E of a scale byte: 2^-127 is below the normal numbers, 255 is NaN.
__device__ __forceinline__ float mx_factor(unsigned byte) {
    const unsigned b = byte == 0 ? 0x00400000u : byte == 255 ? 0x7fc00000u : byte << 23;
    return __builtin_bit_cast(float, b);
}

// Largest of aligned groups of four lanes.
__device__ __forceinline__ unsigned quad_max(unsigned v) {
    const unsigned a = (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, false);
    v = a > v ? a : v;
    const unsigned b = (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, false);
    return b > v ? b : v;
}

// Eight elements, scaled: 8 bytes (e4m3) or 4 (e2m1, in x).
template <int F>
__device__ __forceinline__ u32x2 mx_pack8(const float (&v)[8]) {
    u32x2 o{0, 0};
    if constexpr (F == kE4m3) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            int w = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * i], v[4 * i + 1], 0, false);
            w = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * i + 2], v[4 * i + 3], w, true);
            o[i] = (unsigned)w;
        }
    } else {
        unsigned w = 0;
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0], v[1], 1.f, 0);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], 1.f, 1);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4], v[5], 1.f, 2);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6], v[7], 1.f, 3);
        o[0] = w;
    }
    return o;
}

// Quantises the blocks whose 32 elements lie in four consecutive lanes, eight each: this lane's elements go to `data`,
// and in the block's first lane its scale to `scale`.
template <int F>
__device__ __forceinline__ void mx_store8_at(float (&v)[8], uint8_t* data, uint8_t* scale, bool first) {
    unsigned top = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const unsigned b = mag_bits(v[e]);
        top = b > top ? b : top;
    }
    const MxScale s = mx_scale<F>(quad_max(top));
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = s.byte == 255 ? 0.f : v[e] * s.inv;
    const u32x2 o = mx_pack8<F>(v);
    if constexpr (F == kE4m3) *reinterpret_cast<u32x2*>(data) = o;
    else *reinterpret_cast<unsigned*>(data) = o[0];
    if (first) *scale = (uint8_t)s.byte;
}
// The same where they lie in a stored row: `unit` is the index of this lane's eight.
template <int F>
__device__ __forceinline__ void mx_store8(float (&v)[8], uint8_t* data_row, uint8_t* scale_row, int unit) {
    mx_store8_at<F>(v, data_row + unit * (F == kE4m3 ? 8 : 4), scale_row + (unit >> 2), (unit & 3) == 0);
}

// Eight stored elements -> fp32, without their scale.
template <int F>
__device__ __forceinline__ void mx_unpack8(u32x2 w, float (&v)[8]) {
    if constexpr (F == kE4m3) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i], false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i], true);
            v[4 * i] = a[0], v[4 * i + 1] = a[1], v[4 * i + 2] = b[0], v[4 * i + 3] = b[1];
        }
    } else {
        const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[0], 1.f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[0], 1.f, 1);
        const f32x2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[0], 1.f, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[0], 1.f, 3);
        v[0] = a[0], v[1] = a[1], v[2] = b[0], v[3] = b[1], v[4] = c[0], v[5] = c[1], v[6] = d[0], v[7] = d[1];
    }
}

// Eight elements of a row from column c on, those at or past `n` as zero. Whole eights are one or two
// 16-byte reads at the element type's alignment.
template <typename T>
__device__ __forceinline__ void read8(const T* row, int c, int n, T (&t)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) t[e] = (T)0.f;
    if (c + 8 <= n) {
        __builtin_memcpy(t, row + c, 8 * sizeof(T));
    } else if (c < n) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (c + e < n) t[e] = row[c + e];
    }
}
// ... as fp32.
template <typename T>
__device__ __forceinline__ void load8(const T* row, int c, int n, float (&v)[8]) {
    T t[8];
    read8(row, c, n, t);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (float)t[e];
}
// bf16 as it lies in memory, for values that wait in registers.
__device__ __forceinline__ u32x4 raw8(const bf16* row, int c, int n) {
    u32x4 o{0, 0, 0, 0};
    if (c + 8 <= n) {
        __builtin_memcpy(&o, row + c, 16);
    } else if (c < n) {
        const uint16_t* p = reinterpret_cast<const uint16_t*>(row);
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e / 2] |= c + e < n ? (unsigned)p[c + e] << e % 2 * 16 : 0u;
    }
    return o;
}
__device__ __forceinline__ void values8(const u32x4& r, float (&v)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const unsigned w = r[e / 2];
        v[e] = __builtin_bit_cast(float, e % 2 ? w & 0xffff0000u : w << 16);
    }
}
// A row's last columns, where eight do not divide it, are read from late8 columns before and moved by values8_late when they are
// used: a read of single elements is waited for at once (the norm's backward, 16384 x 2050: 99 us, 89 as it is).
__device__ __forceinline__ int late8(int c, int n) { return c < n && c + 8 > n && n >= 8 ? c + 8 - n : 0; }
__device__ __forceinline__ void values8_late(u32x4 r, int late, float (&v)[8]) {
    if (late) {  // down by so many halves
        if (late & 4) r = u32x4{r[2], r[3], 0, 0};
        if (late & 2) r = u32x4{r[1], r[2], r[3], 0};
        if (late & 1) r = u32x4{r[0] >> 16 | r[1] << 16, r[1] >> 16 | r[2] << 16, r[2] >> 16 | r[3] << 16, r[3] >> 16};
    }
    values8(r, v);
}
// Eight elements that stay in registers: bf16 in half as many. kLate: read late8 columns before (the norm, 16384 x 2050: 67 us, 58
// with it; to microscaled values it stays off, whose registers it takes: 4096 x 8192 43 and 51).
template <typename T, bool kLate = false> struct Held8;
template <bool kLate> struct Held8<bf16, kLate> {
    u32x4 raw;
    int late;
    __device__ __forceinline__ void load(const bf16* row, int c, int n) {
        late = kLate ? late8(c, n) : 0;
        raw = raw8(row, c - late, n);
    }
    __device__ __forceinline__ void values(float (&v)[8]) const {
        u32x4 r = raw;
        asm volatile("" : "+v"(r));  // not hoisted out of a loop, where the values would be held after all
        values8_late(r, kLate ? late : 0, v);
    }
};
template <bool kLate> struct Held8<float, kLate> {
    float raw[8];
    __device__ __forceinline__ void load(const float* row, int c, int n) { load8(row, c, n, raw); }
    __device__ __forceinline__ void values(float (&v)[8]) const {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = raw[e];
    }
};
template <typename T>
__device__ __forceinline__ void store8(T* row, int c, int n, const float (&v)[8]) {
    T t[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) t[e] = (T)v[e];
    if (c + 8 <= n) {
        __builtin_memcpy(row + c, t, 8 * sizeof(T));
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (c + e < n) row[c + e] = t[e];
    }
}

}  // namespace m3
