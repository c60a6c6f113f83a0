// Microscaled quantisation (m3_mx.h), with silu(gate) * up in front of it, and its inverse.
// Bound by HBM: one read and one write; gated by the gate's arithmetic as well. 32000 x 768 in bf16 to e2m1 13.4 us (4.6 TB/s), gated
// 8192 x 2112 to e4m3 18.7 us (4.7 TB/s), its values 10.2 (5.1 TB/s). A lane takes eight elements (one 16-byte read of bf16), four
// lanes a block of 32, whose largest magnitude they find with two lane moves.
#include <algorithm>

#include "m3_common.h"
#include "m3_kernels.h"
#include "m3_mx.h"
#include "m3_row.h"
#include "mamba3_amd.h"

namespace m3 {

constexpr int kMxThreads = 256;

// A thread an eight: two or four a thread, asked for at once, took longer (gated 8192 x 2112, the gate in 32 bits alone, 17.5 us, 19.7 and 25).
template <typename T, int F, bool kGated>
__global__ __launch_bounds__(kMxThreads) void mx_quantize_kernel(const T* __restrict__ x, uint8_t* __restrict__ data,
                                                                 uint8_t* __restrict__ scales, unsigned units, int k,
                                                                 int kp, FastDiv per_row) {
    const unsigned id = blockIdx.x * kMxThreads + threadIdx.x;
    if (id >= units) return;  // whole blocks of 32: units of a row come in sixteens
    const unsigned row = per_row.div(id);
    const int unit = (int)(id - row * per_row.d);
    const T* r = x + (int64_t)row * (kGated ? 2 * (int64_t)k : k);
    Held8<T> x8, u8;
    x8.load(r, unit * 8, k);
    if constexpr (kGated) u8.load(r + k, unit * 8, k);
    float v[8];
    x8.values(v);
    if constexpr (kGated) {
        float u[8];
        u8.values(u);
        silu_mul8(v, u);
    }
    mx_store8<F>(v, data + (int64_t)row * (F == kE4m3 ? kp : kp / 2), scales + (int64_t)row * (kp / 32), unit);
}

template <typename T, int F>
__global__ __launch_bounds__(kMxThreads) void mx_dequantize_kernel(const uint8_t* __restrict__ data, const uint8_t* __restrict__ scales,
                                                                   T* __restrict__ out, unsigned units, int k, int kp, FastDiv per_row) {
    const unsigned id = blockIdx.x * kMxThreads + threadIdx.x;
    if (id >= units) return;
    const unsigned row = per_row.div(id);
    const int unit = (int)(id - row * per_row.d);
    const uint8_t* p = data + (int64_t)row * (F == kE4m3 ? kp : kp / 2);
    u32x2 w;
    if constexpr (F == kE4m3) w = *reinterpret_cast<const u32x2*>(p + unit * 8);
    else w = u32x2{*reinterpret_cast<const unsigned*>(p + unit * 4), 0};
    const float f = mx_factor(scales[(int64_t)row * (kp / 32) + (unit >> 2)]);
    float v[8];
    mx_unpack8<F>(w, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] *= f;
    store8(out + (int64_t)row * k, unit * 8, k, v);
}

// Launches of fewer than 2^31 units.
template <typename Launch>
static int mx_rows(int64_t rows, int64_t per_row, Launch launch) {
    const int64_t most = (((int64_t)1 << 31) - 1) / per_row;
    for (int64_t r = 0; r < rows; r += most) {
        const unsigned units = (unsigned)(std::min(most, rows - r) * per_row);
        launch(r, units, dim3((units + kMxThreads - 1) / kMxThreads));
        if (hipGetLastError() != hipSuccess) return M3_ERR_LAUNCH;
    }
    return M3_OK;
}

template <typename T, int F, bool kGated>
static int quantize_t(const void* x, void* data, void* scales, int64_t rows, int k, hipStream_t stream) {
    const int kp = (int)mx_padded(k);
    return mx_rows(rows, kp / 8, [&](int64_t r, unsigned units, dim3 grid) {
        hipLaunchKernelGGL((mx_quantize_kernel<T, F, kGated>), grid, dim3(kMxThreads), 0, stream,
                           reinterpret_cast<const T*>(x) + r * k * (kGated ? 2 : 1),
                           reinterpret_cast<uint8_t*>(data) + r * mx_row_bytes(kp, F), reinterpret_cast<uint8_t*>(scales) + r * (kp / 32),
                           units, k, kp, FastDiv(kp / 8));
    });
}
template <typename T>
static int quantize_f(const void* x, bool gated, int format, void* data, void* scales, int64_t rows, int k, hipStream_t stream) {
    if (format == kE4m3)
        return gated ? quantize_t<T, kE4m3, true>(x, data, scales, rows, k, stream) : quantize_t<T, kE4m3, false>(x, data, scales, rows, k, stream);
    return gated ? quantize_t<T, kE2m1, true>(x, data, scales, rows, k, stream) : quantize_t<T, kE2m1, false>(x, data, scales, rows, k, stream);
}
int launch_mx_quantize(const void* x, int dtype, bool gated, int format, void* data, void* scales, int64_t rows, int k, hipStream_t stream) {
    return dtype == M3_DTYPE_BF16 ? quantize_f<bf16>(x, gated, format, data, scales, rows, k, stream)
                                  : quantize_f<float>(x, gated, format, data, scales, rows, k, stream);
}

template <typename T, int F>
static int dequantize_t(const void* data, const void* scales, void* out, int64_t rows, int k, hipStream_t stream) {
    const int kp = (int)mx_padded(k);
    return mx_rows(rows, kp / 8, [&](int64_t r, unsigned units, dim3 grid) {
        hipLaunchKernelGGL((mx_dequantize_kernel<T, F>), grid, dim3(kMxThreads), 0, stream,
                           reinterpret_cast<const uint8_t*>(data) + r * mx_row_bytes(kp, F),
                           reinterpret_cast<const uint8_t*>(scales) + r * (kp / 32), reinterpret_cast<T*>(out) + r * k, units, k, kp, FastDiv(kp / 8));
    });
}
int launch_mx_dequantize(const void* data, const void* scales, int format, void* out, int dtype, int64_t rows, int k, hipStream_t stream) {
    if (dtype == M3_DTYPE_BF16)
        return format == kE4m3 ? dequantize_t<bf16, kE4m3>(data, scales, out, rows, k, stream) : dequantize_t<bf16, kE2m1>(data, scales, out, rows, k, stream);
    return format == kE4m3 ? dequantize_t<float, kE4m3>(data, scales, out, rows, k, stream) : dequantize_t<float, kE2m1>(data, scales, out, rows, k, stream);
}

}  // namespace m3
