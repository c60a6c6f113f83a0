// The residual's addition with the norm behind it, forward and backward (gfx950):
//   t = T(residual + s x)   (or t = x),   r = 1 / sqrt(mean t^2 + eps),   y = t r w
// in one pass: a row stays in registers between its sum of squares and its result. y is rounded once, to
// the inputs' type or to microscaled elements (m3_mx.h). The squares are of t as it is stored, since
// that is what the next block adds to. Backward, with g = w dy and a = sum g t:
//   dt = dtotal + r g - t r^3 a / d,   dresidual = dt,   dx = s dt,   dw = sum over rows of dy t r
// Bound by HBM: x, residual, t and y once each; backward t, dtotal, dy, dx and dresidual once each. bf16, 16384 x 2048: forward
// 43 us (6.2 TB/s, partly from the last-level cache), to e4m3 40 (5.9), backward 64 and 5 for dw (5.2 TB/s); fp32 107, 85 and 138. bf16 rows and
// weights wait as they lie in memory and are taken apart where they are used: at half the registers, four to six waves a SIMD
// instead of three or four (51 us and 58 as fp32).
//
// One wave a row where it holds it: no barriers, and the rows of a block's four waves hide one another's latency.
// A row is taken by one wave (to 2048 columns) or by a block's four (to 8192), eight consecutive
// columns a lane and piece, so that four lanes hold a block of 32; wider rows are read a second time.
// Squares are added in fp32 within a lane (at most 32 of them) and in fp64 across lanes; for microscaled results in fp64
// from eight on, and the product is rounded once (m3_row.h).
#include <algorithm>

#include "m3_common.h"
#include "m3_kernels.h"
#include "m3_mx.h"
#include "m3_row.h"
#include "mamba3_amd.h"

namespace m3 {

constexpr int kAnThreads = 256;
constexpr int kAnWaves = kAnThreads / 64;
constexpr int kSame = -1;  // y in the inputs' type

// The same over the waves of a row: `red` has kAnWaves places, one set for each call in turn.
template <int kWpr>
__device__ __forceinline__ double row_sum(double v, double* red) {
    v = wave_sum_f64(v);
    if constexpr (kWpr > 1) {
        __syncthreads();  // what the places held has been read
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
        __syncthreads();
        v = red[0];
#pragma unroll
        for (int i = 1; i < kWpr; ++i) v += red[i];
    }
    return v;
}
struct AddNormArgs {
    const void *x, *res, *w;
    void *total, *y;
    uint8_t *data, *scales;
    float* rstd;
    int64_t rows;
    int d, kp;
    float scale, eps;
};

// kNp pieces of eight a lane, kWpr waves a row. kF: kSame or a microscaled format.
template <typename T, int kF, bool kRes, int kWpr, int kNp>
__global__ __launch_bounds__(kAnThreads) void add_norm_kernel(AddNormArgs a) {
    constexpr int kLanes = kWpr * 64, kRpb = kAnWaves / kWpr;  // lanes a row, rows a block
    __shared__ double red[kAnWaves];
    const int lane = threadIdx.x % kLanes;
    const int d = a.d, units = (kF == kSame ? d + 7 : a.kp) / 8;
    const double share = 1.0 / d;
    Held8<T> w[kNp];
#pragma unroll
    for (int p = 0; p < kNp; ++p) w[p].load(reinterpret_cast<const T*>(a.w), (lane + p * kLanes) * 8, d);
    for (int64_t row = (int64_t)blockIdx.x * kRpb + threadIdx.x / kLanes; row < a.rows; row += (int64_t)gridDim.x * kRpb) {
        const int64_t base = row * d;
        float t[kNp][8];
        Held8<T, kF == kSame> x[kNp], r[kRes ? kNp : 1];
#pragma unroll
        for (int p = 0; p < kNp; ++p) {
            const int c = (lane + p * kLanes) * 8;
            x[p].load(reinterpret_cast<const T*>(a.x) + base, c, d);
            if constexpr (kRes) r[p].load(reinterpret_cast<const T*>(a.res) + base, c, d);
        }
        float ss = 0.f;
        double squares = 0.0;
#pragma unroll
        for (int p = 0; p < kNp; ++p) {
            x[p].values(t[p]);
            if constexpr (kRes) {
                float v[8];
                r[p].values(v);
#pragma unroll
                for (int e = 0; e < 8; ++e) t[p][e] = (float)(T)fmaf(a.scale, t[p][e], v[e]);
                const int c = (lane + p * kLanes) * 8;
                if (c < d) store8(reinterpret_cast<T*>(a.total) + base, c, d, t[p]);
            }
            if constexpr (kF != kSame) {
                squares = add_squares(squares, t[p]);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) ss = fmaf(t[p][e], t[p][e], ss);
            }
        }
        const double mean = row_sum<kWpr>(kF != kSame ? squares : (double)ss, red) * share + (double)a.eps;
        const RowScale r2 = row_scale(mean);
        const float rs = r2.hi;
        if (a.rstd && lane == 0) a.rstd[row] = rs;
#pragma unroll
        for (int p = 0; p < kNp; ++p) {
            const int unit = lane + p * kLanes;
            if (unit >= units) continue;
            float v[8];
            w[p].values(v);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = kF != kSame ? norm_odd(t[p][e], v[e], r2) : t[p][e] * rs * v[e];
            if constexpr (kF == kSame) store8(reinterpret_cast<T*>(a.y) + base, unit * 8, d, v);
            else mx_store8<kF>(v, a.data + row * (kF == kE4m3 ? a.kp : a.kp / 2), a.scales + row * (a.kp / 32), unit);
        }
    }
}

// Rows of any width, one block each: t is read a second time.
template <typename T, int kF, bool kRes>
__global__ __launch_bounds__(kAnThreads) void add_norm_wide_kernel(AddNormArgs a) {
    __shared__ double red[kAnWaves];
    const int d = a.d, units = (kF == kSame ? d + 7 : a.kp) / 8;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const int64_t base = row * d;
        double sum = 0.0;
        for (int unit = threadIdx.x; unit < units; unit += kAnThreads) {
            float t[8], r[8], ss = 0.f;
            load8(reinterpret_cast<const T*>(a.x) + base, unit * 8, d, t);
            if constexpr (kRes) {
                load8(reinterpret_cast<const T*>(a.res) + base, unit * 8, d, r);
#pragma unroll
                for (int e = 0; e < 8; ++e) t[e] = (float)(T)fmaf(a.scale, t[e], r[e]);
                store8(reinterpret_cast<T*>(a.total) + base, unit * 8, d, t);
            }
            if constexpr (kF != kSame) {
                sum = add_squares(sum, t);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) ss = fmaf(t[e], t[e], ss);
                sum += (double)ss;
            }
        }
        const RowScale r2 = row_scale(row_sum<kAnWaves>(sum, red) * (1.0 / d) + (double)a.eps);
        const float rs = r2.hi;
        if (a.rstd && threadIdx.x == 0) a.rstd[row] = rs;
        for (int unit = threadIdx.x; unit < units; unit += kAnThreads) {
            float t[8], w[8];  // t: what this thread wrote above
            load8(reinterpret_cast<const T*>(kRes ? a.total : a.x) + base, unit * 8, d, t);
            load8(reinterpret_cast<const T*>(a.w), unit * 8, d, w);
#pragma unroll
            for (int e = 0; e < 8; ++e) t[e] = kF != kSame ? norm_odd(t[e], w[e], r2) : t[e] * rs * w[e];
            if constexpr (kF == kSame) store8(reinterpret_cast<T*>(a.y) + base, unit * 8, d, t);
            else mx_store8<kF>(t, a.data + row * (kF == kE4m3 ? a.kp : a.kp / 2), a.scales + row * (a.kp / 32), unit);
        }
    }
}

constexpr int64_t kAnMaxBlocks = 2048;  // eight a CU: each keeps its columns of w in registers over its rows

template <typename T, int kF, bool kRes>
static int add_norm_t(const AddNormArgs& a, hipStream_t stream) {
    const int units = (kF == kSame ? a.d + 7 : a.kp) / 8;
    auto grid = [&](int64_t rows_a_block) {
        return dim3((unsigned)std::min((a.rows + rows_a_block - 1) / rows_a_block, kAnMaxBlocks));
    };
    const dim3 block(kAnThreads);
    if (units <= 64) hipLaunchKernelGGL((add_norm_kernel<T, kF, kRes, 1, 1>), grid(4), block, 0, stream, a);
    else if (units <= 128) hipLaunchKernelGGL((add_norm_kernel<T, kF, kRes, 1, 2>), grid(4), block, 0, stream, a);
    else if (units <= 256) hipLaunchKernelGGL((add_norm_kernel<T, kF, kRes, 1, 4>), grid(4), block, 0, stream, a);
    else if (units <= 512) hipLaunchKernelGGL((add_norm_kernel<T, kF, kRes, 4, 2>), grid(1), block, 0, stream, a);
    else if (units <= 1024) hipLaunchKernelGGL((add_norm_kernel<T, kF, kRes, 4, 4>), grid(1), block, 0, stream, a);
    else hipLaunchKernelGGL((add_norm_wide_kernel<T, kF, kRes>), grid(1), block, 0, stream, a);
    return hipGetLastError() == hipSuccess ? M3_OK : M3_ERR_LAUNCH;
}
template <typename T>
static int add_norm_f(const AddNormArgs& a, int format, hipStream_t stream) {
    if (format == kSame) return add_norm_t<T, kSame, true>(a, stream);
    if (format == kE4m3) return a.res ? add_norm_t<T, kE4m3, true>(a, stream) : add_norm_t<T, kE4m3, false>(a, stream);
    return a.res ? add_norm_t<T, kE2m1, true>(a, stream) : add_norm_t<T, kE2m1, false>(a, stream);
}

int launch_add_norm(const void* x, const void* res, const void* w, int dtype, float scale, float eps, void* total, void* y,
                    float* rstd, int64_t rows, int d, hipStream_t stream) {
    const AddNormArgs a{x, res, w, total, y, nullptr, nullptr, rstd, rows, d, 0, scale, eps};
    return dtype == M3_DTYPE_BF16 ? add_norm_f<bf16>(a, kSame, stream) : add_norm_f<float>(a, kSame, stream);
}
int launch_add_norm_mx(const void* x, const void* res, const void* w, int dtype, float scale, float eps, void* total, int format,
                       void* data, void* scales, int64_t rows, int d, hipStream_t stream) {
    const AddNormArgs a{x, res, w, total, nullptr, reinterpret_cast<uint8_t*>(data), reinterpret_cast<uint8_t*>(scales), nullptr,
                        rows, d, (int)mx_padded(d), scale, eps};
    return dtype == M3_DTYPE_BF16 ? add_norm_f<bf16>(a, format, stream) : add_norm_f<float>(a, format, stream);
}

// ---- backward
struct AddNormBwdArgs {
    const void *t, *w, *dtotal, *dy;
    const float* rstd;
    void *dx, *dres;
    float* part;  // [blocks][d]: each block's rows of dw
    int64_t rows;
    int d;
    float scale;
};

template <typename T>
__device__ __forceinline__ void store_grads(const AddNormBwdArgs& a, int64_t base, int c, const float (&dt)[8]) {
    if (a.dres) store8(reinterpret_cast<T*>(a.dres) + base, c, a.d, dt);
    if (a.dx) {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = a.scale * dt[e];
        store8(reinterpret_cast<T*>(a.dx) + base, c, a.d, v);
    }
}

// A block's waves walk rows; each lane adds up dw of its columns, and the waves' sums meet in LDS. bf16 rows
// wait as they lie in memory, the next one's while this one's are used, and so do the weights (16384 x 2048 62 us and 5 for dw; 86
// without; fp32, at twice the bytes, 137).
template <typename T, int kWaves, int kWpr, int kNp>
__global__ __launch_bounds__(kWaves * 64) void add_norm_bwd_kernel(AddNormBwdArgs a) {
    constexpr int kLanes = kWpr * 64, kRpb = kWaves / kWpr;
    __shared__ double red[kWaves];
    __shared__ float sum[kWpr == 1 ? kWaves * 64 * 8 : 1];
    const int lane = threadIdx.x % kLanes, d = a.d;
    Held8<T> w[kNp];
    float dw[kNp][8];
#pragma unroll
    for (int p = 0; p < kNp; ++p) {
        w[p].load(reinterpret_cast<const T*>(a.w), (lane + p * kLanes) * 8, d);
#pragma unroll
        for (int e = 0; e < 8; ++e) dw[p][e] = 0.f;
    }
    constexpr bool kHalf = sizeof(T) == 2, kAhead = kHalf && kWpr * kNp < 16;  // (more would take more than half the registers)
    u32x4 tr[kNp], gr[kNp], dr[kNp];
    float rr;
    auto read = [&](int64_t row) __attribute__((always_inline)) {
        const int64_t base = row * d;
#pragma unroll
        for (int p = 0; p < kNp; ++p) {
            const int c0 = (lane + p * kLanes) * 8, c = c0 - late8(c0, d);
            tr[p] = raw8(reinterpret_cast<const bf16*>(a.t) + base, c, d);
            gr[p] = raw8(reinterpret_cast<const bf16*>(a.dy) + base, c, d);
            dr[p] = a.dtotal ? raw8(reinterpret_cast<const bf16*>(a.dtotal) + base, c, d) : u32x4{0, 0, 0, 0};
        }
        rr = a.rstd[row];
    };
    const int64_t step = (int64_t)gridDim.x * kRpb;
    int64_t row = (int64_t)blockIdx.x * kRpb + threadIdx.x / kLanes;
    if (kAhead && row < a.rows) read(row);
    for (; row < a.rows; row += step) {
        const int64_t base = row * d;
        float t[kNp][8], g[kNp][8], dt[kNp][8];
        if constexpr (kHalf) {
            if constexpr (!kAhead) read(row);
#pragma unroll
            for (int p = 0; p < kNp; ++p) {
                const int late = late8((lane + p * kLanes) * 8, d);
                values8_late(tr[p], late, t[p]), values8_late(gr[p], late, g[p]), values8_late(dr[p], late, dt[p]);
            }
        } else {
#pragma unroll
            for (int p = 0; p < kNp; ++p) {
                const int c = (lane + p * kLanes) * 8;
                load8(reinterpret_cast<const T*>(a.t) + base, c, d, t[p]);
                load8(reinterpret_cast<const T*>(a.dy) + base, c, d, g[p]);
                if (a.dtotal) {
                    load8(reinterpret_cast<const T*>(a.dtotal) + base, c, d, dt[p]);
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) dt[p][e] = 0.f;
                }
            }
            rr = a.rstd[row];
        }
        const float rs = rr;
        if (kAhead && row + step < a.rows) read(row + step);
        float dot = 0.f;
#pragma unroll
        for (int p = 0; p < kNp; ++p) {
            float w8[8];
            w[p].values(w8);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                dw[p][e] = fmaf(g[p][e], t[p][e] * rs, dw[p][e]);
                g[p][e] *= w8[e];
                dot = fmaf(g[p][e], t[p][e], dot);
            }
        }
        const float mean = (float)(row_sum<kWpr>((double)dot, red) / d * (double)rs * (double)rs);
#pragma unroll
        for (int p = 0; p < kNp; ++p) {
            const int c = (lane + p * kLanes) * 8;
            if (c >= d) continue;
#pragma unroll
            for (int e = 0; e < 8; ++e) dt[p][e] = fmaf(rs, fmaf(-t[p][e], mean, g[p][e]), dt[p][e]);
            store_grads<T>(a, base, c, dt[p]);
        }
    }
    if (!a.part) return;
    float* out = a.part + (int64_t)blockIdx.x * d;
#pragma unroll
    for (int p = 0; p < kNp; ++p) {
        if constexpr (kWpr == 1) {
            __syncthreads();
            store8(sum + (threadIdx.x >> 6) * 512, lane * 8, 512, dw[p]);
            __syncthreads();
            for (int c = threadIdx.x; c < 512; c += kWaves * 64) {
                float v = sum[c];
#pragma unroll
                for (int i = 1; i < kWaves; ++i) v += sum[i * 512 + c];
                if (p * 512 + c < d) out[p * 512 + c] = v;
            }
        } else {
            const int c = (lane + p * kLanes) * 8;
            if (c < d) store8(out, c, d, dw[p]);
        }
    }
}

// Rows of any width, one block each, read twice; dw has a kernel of its own.
template <typename T>
__global__ __launch_bounds__(kAnThreads) void add_norm_bwd_wide_kernel(AddNormBwdArgs a) {
    __shared__ double red[kAnWaves];
    const int d = a.d, units = (d + 7) / 8;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const int64_t base = row * d;
        double sum = 0.0;
        float t[8], g[8], w[8], dt[8];
        for (int unit = threadIdx.x; unit < units; unit += kAnThreads) {
            load8(reinterpret_cast<const T*>(a.t) + base, unit * 8, d, t);
            load8(reinterpret_cast<const T*>(a.dy) + base, unit * 8, d, g);
            load8(reinterpret_cast<const T*>(a.w), unit * 8, d, w);
            float dot = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) dot = fmaf(g[e] * w[e], t[e], dot);
            sum += (double)dot;
        }
        const float rs = a.rstd[row];
        const float mean = (float)(row_sum<kAnWaves>(sum, red) / d * (double)rs * (double)rs);
        for (int unit = threadIdx.x; unit < units; unit += kAnThreads) {
            load8(reinterpret_cast<const T*>(a.t) + base, unit * 8, d, t);
            load8(reinterpret_cast<const T*>(a.dy) + base, unit * 8, d, g);
            load8(reinterpret_cast<const T*>(a.w), unit * 8, d, w);
#pragma unroll
            for (int e = 0; e < 8; ++e) dt[e] = 0.f;
            if (a.dtotal) load8(reinterpret_cast<const T*>(a.dtotal) + base, unit * 8, d, dt);
#pragma unroll
            for (int e = 0; e < 8; ++e) dt[e] = fmaf(rs, fmaf(-t[e], mean, g[e] * w[e]), dt[e]);
            store_grads<T>(a, base, unit * 8, dt);
        }
    }
}
// dw of wide rows: block (x, y) adds part y of the rows up over 512 columns.
template <typename T>
__global__ __launch_bounds__(64) void add_norm_dw_wide_kernel(AddNormBwdArgs a, int64_t rows_a_part) {
    const int c = ((int)blockIdx.x * 64 + (int)threadIdx.x) * 8;
    if (c >= a.d) return;
    const int64_t r0 = (int64_t)blockIdx.y * rows_a_part, r1 = r0 + rows_a_part < a.rows ? r0 + rows_a_part : a.rows;
    float dw[8] = {}, t[8], g[8];
    for (int64_t row = r0; row < r1; ++row) {
        load8(reinterpret_cast<const T*>(a.t) + row * a.d, c, a.d, t);
        load8(reinterpret_cast<const T*>(a.dy) + row * a.d, c, a.d, g);
        const float rs = a.rstd[row];
#pragma unroll
        for (int e = 0; e < 8; ++e) dw[e] = fmaf(g[e], t[e] * rs, dw[e]);
    }
    store8(a.part + (int64_t)blockIdx.y * a.d, c, a.d, dw);
}

// dw = the blocks' sums in order: 64 columns a block, whose 16 waves take every 16th.
template <typename T>
__global__ __launch_bounds__(1024) void add_norm_dw_kernel(const float* __restrict__ part, T* __restrict__ dw, int parts, int d) {
    __shared__ float sum[16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int c = (int)blockIdx.x * 64 + lane, cc = c < d ? c : d - 1;
    float v = 0.f;
#pragma unroll 8
    for (int i = wave; i < parts; i += 16) v += part[(int64_t)i * d + cc];
    sum[wave][lane] = v;
    __syncthreads();
    if (wave == 0 && c < d) {
#pragma unroll
        for (int i = 1; i < 16; ++i) v += sum[i][lane];
        dw[c] = (T)v;
    }
}

constexpr int kAnNarrow = 8192;  // columns that stay in registers
// Blocks of the backward: as many waves as run at once by the registers that a row's pieces take (65536 x 768: eight waves a CU
// 122 us, twelve 106), in few blocks, since each has its line in dw's sum (32768 x 512: four waves a block 34.4, eight 32.4).
static int add_norm_bwd_waves(int d) { return d <= 512 ? 8 : d <= 1024 ? 12 : 4; }
static int64_t add_norm_parts(int64_t rows, int d) {
    const int waves = add_norm_bwd_waves(d);
    if (d <= 1024) return std::min<int64_t>(d <= 512 ? 512 : 256, (rows + waves - 1) / waves);
    return d <= 2048 ? std::min<int64_t>(512, (rows + waves - 1) / waves) : std::min<int64_t>(d <= 4096 ? 768 : 512, rows);
}
size_t add_norm_bwd_workspace(int64_t rows, int d) { return (size_t)add_norm_parts(rows, d) * d * sizeof(float); }

template <typename T>
static int add_norm_bwd_t(AddNormBwdArgs a, void* dw, hipStream_t stream) {
    const int64_t parts = add_norm_parts(a.rows, a.d);
    const dim3 grid((unsigned)parts), block(64 * add_norm_bwd_waves(a.d));
    if (a.d <= 512) hipLaunchKernelGGL((add_norm_bwd_kernel<T, 8, 1, 1>), grid, block, 0, stream, a);
    else if (a.d <= 1024) hipLaunchKernelGGL((add_norm_bwd_kernel<T, 12, 1, 2>), grid, block, 0, stream, a);
    else if (a.d <= 2048) hipLaunchKernelGGL((add_norm_bwd_kernel<T, 4, 1, 4>), grid, block, 0, stream, a);
    else if (a.d <= 4096) hipLaunchKernelGGL((add_norm_bwd_kernel<T, 4, 4, 2>), grid, block, 0, stream, a);
    else if (a.d <= kAnNarrow) hipLaunchKernelGGL((add_norm_bwd_kernel<T, 4, 4, 4>), grid, block, 0, stream, a);
    else {
        if (a.dx || a.dres)
            hipLaunchKernelGGL((add_norm_bwd_wide_kernel<T>), dim3((unsigned)std::min(a.rows, kAnMaxBlocks)), dim3(kAnThreads), 0, stream, a);
        if (dw) {
            const int64_t each = (a.rows + parts - 1) / parts;
            hipLaunchKernelGGL((add_norm_dw_wide_kernel<T>), dim3((unsigned)((a.d + 511) / 512), (unsigned)parts), dim3(64), 0, stream, a, each);
        }
    }
    if (hipGetLastError() != hipSuccess) return M3_ERR_LAUNCH;
    if (!dw) return M3_OK;
    hipLaunchKernelGGL((add_norm_dw_kernel<T>), dim3((unsigned)((a.d + 63) / 64)), dim3(1024), 0, stream, a.part,
                       reinterpret_cast<T*>(dw), (int)parts, a.d);
    return hipGetLastError() == hipSuccess ? M3_OK : M3_ERR_LAUNCH;
}
int launch_add_norm_bwd(const void* total, const void* w, const float* rstd, const void* dtotal, const void* dy, int dtype,
                        float scale, void* dx, void* dres, void* dw, void* ws, int64_t rows, int d, hipStream_t stream) {
    const AddNormBwdArgs a{total, w, dtotal, dy, rstd, dx, dres, dw ? reinterpret_cast<float*>(ws) : nullptr, rows, d, scale};
    return dtype == M3_DTYPE_BF16 ? add_norm_bwd_t<bf16>(a, dw, stream) : add_norm_bwd_t<float>(a, dw, stream);
}

}  // namespace m3
