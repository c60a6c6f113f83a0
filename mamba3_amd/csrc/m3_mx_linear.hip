// Products of microscaled activations with 4-bit weights (gfx950):
//   out[m][n] = [res +] scale * sum over k of x(m, k) w(n, k)
// x in e4m3 or e2m1, w in e2m1, both as stored by m3_mx.h, on the matrix instructions that apply the blocks'
// exponents themselves. These add 128 products at a time in fp32 but align e4m3's at about 2^-13 of
// the largest one: up to 3e-4 of that product, 4e-6 of the sum on normal data, far below the operand's own
// rounding (2^-4 of each element) and the bf16 result's (2^-9). e2m1 x e2m1 is exact. An fp32 result takes
// the elements with their scales as bf16 (exact: four significant bits) on the bf16 instructions, whose sums
// are fp32 throughout, at half the rate.
//
// Operand layout of the 16 x 16 x 128 instruction: lane l holds row l % 16; of k, group g = l / 16 holds
// 16 g .. 16 g + 15 and 64 + 16 g .. (e4m3) or 32 g .. 32 g + 31 (e2m1), and the scale of block g. As in
// m3_gemm.h the weights come first, so that a lane gets four consecutive n of one row m.
#include <algorithm>

#include "m3_common.h"
#include "m3_kernels.h"
#include "m3_mx.h"
#include "mamba3_amd.h"

namespace m3 {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

struct MxLinearArgs {
    const uint8_t *x, *xs, *w, *ws;
    const void* res;
    void* out;
    float scale;
    int M, N, steps;  // steps of 128 k
};

__device__ __forceinline__ i32x8 wide(i32x4 lo, i32x4 hi) {
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}

// One operand's 16 rows of 128 k as a lane holds them.
template <int F>
struct MxFrag {
    i32x4 p[F == kE4m3 ? 2 : 1];
    int s;
    // k in the order of the scaled instructions, or (kLinear) lane group g its block's 32 in order
    template <bool kLinear>
    __device__ __forceinline__ void load(const uint8_t* row, const uint8_t* srow, int step, int g) {
        if constexpr (F == kE4m3) {
            const uint8_t* at = row + (int64_t)step * 128;
            p[0] = *reinterpret_cast<const i32x4*>(at + (kLinear ? 32 * g : 16 * g));
            p[1] = *reinterpret_cast<const i32x4*>(at + (kLinear ? 32 * g + 16 : 64 + 16 * g));
        } else {
            p[0] = *reinterpret_cast<const i32x4*>(row + (int64_t)step * 64 + 16 * g);
        }
        s = srow[(int64_t)step * 4 + g];
    }
    __device__ __forceinline__ i32x8 all() const {
        if constexpr (F == kE4m3) return wide(p[0], p[1]);
        else return wide(p[0], i32x4{0, 0, 0, 0});
    }
    // elements 8 j .. 8 j + 7 of the lane's block with their scale, in bf16
    __device__ __forceinline__ bf16x8 part(int j, float f) const {
        float v[8];
        if constexpr (F == kE4m3) mx_unpack8<F>(u32x2{(unsigned)p[j / 2][j % 2 * 2], (unsigned)p[j / 2][j % 2 * 2 + 1]}, v);
        else mx_unpack8<F>(u32x2{(unsigned)p[0][j], 0}, v);
        bf16x8 o;
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = (bf16)(v[e] * f);
        return o;
    }
};

template <int FA>
__device__ __forceinline__ f32x4 mx_mma(const MxFrag<kE2m1>& w, const MxFrag<FA>& x, f32x4 c) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w.all(), x.all(), c, 4, FA == kE4m3 ? 0 : 4, 0, w.s, 0, x.s);
}

// out[m][n .. n + 3] from four sums; `whole`: rows of out are 16-byte (fp32) or 8-byte (bf16) pieces.
template <typename TO>
__device__ __forceinline__ void mx_out4(const MxLinearArgs& a, int m, int n, f32x4 v, bool whole) {
    typedef TO T4 __attribute__((ext_vector_type(4)));
    if (m >= a.M || n >= a.N) return;
    const int64_t at = (int64_t)m * a.N + n;
    TO* out = reinterpret_cast<TO*>(a.out) + at;
    const TO* res = reinterpret_cast<const TO*>(a.res) + at;
    if (whole) {
        T4 o, r{};
        if (a.res) r = *reinterpret_cast<const T4*>(res);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = (TO)(a.res ? fmaf(a.scale, v[e], (float)r[e]) : a.scale * v[e]);
        *reinterpret_cast<T4*>(out) = o;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (n + e < a.N) out[e] = (TO)(a.res ? fmaf(a.scale, v[e], (float)res[e]) : a.scale * v[e]);
    }
}

// Few rows: a block takes 16 FM rows and 16 FN columns, its four waves every fourth step of k, straight from
// memory to registers; their sums meet in LDS. Bound by the weights' read.
constexpr int kMlWaves = 4;
template <int FA, int FM, int FN, typename TO>
__global__ __launch_bounds__(kMlWaves * 64) void mx_linear_few_kernel(MxLinearArgs a, int tiles_n, bool whole) {
    constexpr bool kExact = sizeof(TO) == 4;
    __shared__ f32x4 part[kMlWaves][FM * FN][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
    const int tm = (int)blockIdx.x / tiles_n, tn = (int)blockIdx.x - tm * tiles_n;
    const int m0 = tm * 16 * FM, n0 = tn * 16 * FN;
    const int64_t xb = (int64_t)a.steps * (FA == kE4m3 ? 128 : 64), wb = (int64_t)a.steps * 64, sb = (int64_t)a.steps * 4;
    const uint8_t *xp[FM], *xsp[FM], *wp[FN], *wsp[FN];
#pragma unroll
    for (int i = 0; i < FM; ++i) {
        const int m = m0 + i * 16 + r < a.M ? m0 + i * 16 + r : a.M - 1;  // rows past the last are not stored
        xp[i] = a.x + m * xb, xsp[i] = a.xs + m * sb;
    }
#pragma unroll
    for (int j = 0; j < FN; ++j) {
        const int n = n0 + j * 16 + r < a.N ? n0 + j * 16 + r : a.N - 1;
        wp[j] = a.w + n * wb, wsp[j] = a.ws + n * sb;
    }
    f32x4 acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int step = wave; step < a.steps; step += kMlWaves) {
        MxFrag<FA> x[FM];
        MxFrag<kE2m1> w[FN];
#pragma unroll
        for (int j = 0; j < FN; ++j) w[j].template load<kExact>(wp[j], wsp[j], step, g);
#pragma unroll
        for (int i = 0; i < FM; ++i) x[i].template load<kExact>(xp[i], xsp[i], step, g);
        if constexpr (kExact) {
            float fx[FM], fw[FN];
#pragma unroll
            for (int i = 0; i < FM; ++i) fx[i] = mx_factor((unsigned)x[i].s);
#pragma unroll
            for (int j = 0; j < FN; ++j) fw[j] = mx_factor((unsigned)w[j].s);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                bf16x8 xq[FM];
#pragma unroll
                for (int i = 0; i < FM; ++i) xq[i] = x[i].part(q, fx[i]);
#pragma unroll
                for (int j = 0; j < FN; ++j) {
                    const bf16x8 wq = w[j].part(q, fw[j]);
#pragma unroll
                    for (int i = 0; i < FM; ++i) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wq, xq[i], acc[i][j], 0, 0, 0);
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < FN; ++j)
#pragma unroll
                for (int i = 0; i < FM; ++i) acc[i][j] = mx_mma<FA>(w[j], x[i], acc[i][j]);
        }
    }
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) part[wave][i * FN + j][lane] = acc[i][j];
    __syncthreads();
    for (int f = wave; f < FM * FN; f += kMlWaves) {
        f32x4 v = part[0][f][lane];
#pragma unroll
        for (int q = 1; q < kMlWaves; ++q) v += part[q][f][lane];
        mx_out4<TO>(a, m0 + f / FN * 16 + r, n0 + f % FN * 16 + g * 4, v, whole);
    }
}

template <int FA, int FM, int FN, typename TO>
static int few_t(const MxLinearArgs& a, hipStream_t stream) {
    const int64_t tn = (a.N + 16 * FN - 1) / (16 * FN), tm = (a.M + 16 * FM - 1) / (16 * FM);
    if (tn * tm > 0x7fffffff) return M3_ERR_UNSUPPORTED;
    const size_t piece = 4 * sizeof(TO);
    const bool whole = a.N % 4 == 0 && reinterpret_cast<uintptr_t>(a.out) % piece == 0 && (!a.res || reinterpret_cast<uintptr_t>(a.res) % piece == 0);
    hipLaunchKernelGGL((mx_linear_few_kernel<FA, FM, FN, TO>), dim3((unsigned)(tn * tm)), dim3(kMlWaves * 64), 0, stream, a, (int)tn, whole);
    return hipGetLastError() == hipSuccess ? M3_OK : M3_ERR_LAUNCH;
}
template <int FA, typename TO>
static int linear_t(const MxLinearArgs& a, hipStream_t stream) {
    if (a.M <= 16) return few_t<FA, 1, 1, TO>(a, stream);
    if (a.M <= 32) return few_t<FA, 2, 2, TO>(a, stream);
    return few_t<FA, 4, 4, TO>(a, stream);
}

int launch_mx_linear(const void* x, const void* xs, int x_format, const void* w, const void* ws, const void* res, float scale,
                     void* out, int out_dtype, int m, int n, int k, hipStream_t stream) {
    const auto b = [](const void* p) { return reinterpret_cast<const uint8_t*>(p); };
    const MxLinearArgs a{b(x), b(xs), b(w), b(ws), res, out, scale, m, n, (int)(mx_padded(k) / kMxStep)};
    if (out_dtype == M3_DTYPE_BF16) return x_format == kE4m3 ? linear_t<kE4m3, bf16>(a, stream) : linear_t<kE2m1, bf16>(a, stream);
    return x_format == kE4m3 ? linear_t<kE4m3, float>(a, stream) : linear_t<kE2m1, float>(a, stream);
}

}  // namespace m3
