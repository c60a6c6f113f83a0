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
#include <atomic>
#include <utility>

#include "m3_common.h"
#include "m3_kernels.h"
#include "m3_mx.h"
#include "m3_row.h"
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
    int ld;           // columns of a row of out and res
};
struct MxBefore {  // of a tensor: its norm's weight
    const void* norm;
    float eps;
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
    const int64_t at = (int64_t)m * a.ld + n;
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

// Few rows: a block takes 16 FM rows and 16 FN columns, its kW waves every kW-th step of k, straight from memory to
// registers; their sums meet in LDS. Bound by the latency of its few reads, and by the weights' read. Eight waves where FM FN is at
// most eight, or 16 where k is above 3968 and the block takes 16 columns (few_waves): weights that come from
// HBM, as a model's do, are then on their way at once (1 x 768 x 3696 2.8 us in a graph, 3.2 with four waves; 1 x 5504 x 2048 5.0, 5.7
// with eight, 8.2 with four; 1 x 2048 x 8800 7.8, 6.9 with four). Blocks of 64 x 64 hold more sums: four waves.

// Adds w x^T of one step of k.
template <int FA, int FM, int FN, bool kExact>
__device__ __forceinline__ void few_step(const MxFrag<kE2m1> (&w)[FN], const MxFrag<FA> (&x)[FM], f32x4 (&acc)[FM][FN]) {
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
// The waves' sums and their store.
template <int kW, int FM, int FN, typename TO>
__device__ __forceinline__ void few_store(const MxLinearArgs& a, f32x4* part, const f32x4 (&acc)[FM][FN], int m0, int n0, bool whole) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) part[(wave * FM * FN + i * FN + j) * 64 + lane] = acc[i][j];
    __syncthreads();
    for (int f = wave; f < FM * FN; f += kW) {
        f32x4 v = part[f * 64 + lane];
#pragma unroll
        for (int q = 1; q < kW; ++q) v += part[(q * FM * FN + f) * 64 + lane];
        mx_out4<TO>(a, m0 + f / FN * 16 + (lane & 15), n0 + f % FN * 16 + (lane >> 4) * 4, v, whole);
    }
}

template <int kW, int FA, int FM, int FN, typename TO>
__global__ __launch_bounds__(kW * 64) void mx_linear_few_kernel(MxLinearArgs a, int tiles_n, bool whole) {
    constexpr bool kExact = sizeof(TO) == 4;
    extern __shared__ __align__(16) char mx_smem[];
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
    for (int step = wave; step < a.steps; step += kW) {
        MxFrag<FA> x[FM];
        MxFrag<kE2m1> w[FN];
#pragma unroll
        for (int j = 0; j < FN; ++j) w[j].template load<kExact>(wp[j], wsp[j], step, g);
#pragma unroll
        for (int i = 0; i < FM; ++i) x[i].template load<kExact>(xp[i], xsp[i], step, g);
        few_step<FA, FM, FN, kExact>(w, x, acc);
    }
    few_store<kW, FM, FN, TO>(a, reinterpret_cast<f32x4*>(mx_smem), acc, m0, n0, whole);
}

// The same for at most 16 rows of a tensor, which each block quantises to e4m3 into LDS first: one launch less, and the
// weights' first reads are on their way meanwhile. Rows of LDS are XOR-swizzled in 16-byte pieces. The sums are those of
// the kernel above on the quantised rows, bit for bit. In front of the rounding may stand the norm (a wave takes a row as
// m3_add_norm.hip's does: the same sums) or silu(gate) * up.
constexpr int kMlRawRows = 16;
// The work that is worth a launch less when every block does it (bf16, us in a graph, one launch against two): quantising
// 4 x 5504 elements 5.7 against 6.9, 16 x 1536 5.5 against 5.8, 16 x 2048 6.8 against 6.5; gating 2 x 5504 6.6 against 7.0, 8 x 1536 5.8
// against 5.7, 8 x 2112 (the gate in 32 bits alone) 7.1 against 5.6; a norm
// of 8 rows, one a wave, of 768 4.9 against 5.6, of 2048 7.4 against 8.5, of 16 rows of 768 7.1 against 5.8.
constexpr int kMlRawElements = 24576, kMlGatedElements = 12288, kMlNormRows = 8;
constexpr int kMlNormPieces = 4;    // of 512 columns: a wave's row
enum { kAsIs, kNormed, kGated };
template <int kW, typename T, int kPre, int FN, typename TO>
__global__ __launch_bounds__(kW * 64) void mx_linear_raw_kernel(MxLinearArgs a, MxBefore before, int k, bool whole) {
    constexpr bool kExact = sizeof(TO) == 4;
    extern __shared__ __align__(16) char mx_smem[];  // [M][kp] elements, [M][kp / 32] scales; then the waves' sums
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
    const int n0 = (int)blockIdx.x * 16 * FN, kp = a.steps * kMxStep;
    const int64_t wb = (int64_t)a.steps * 64, sb = (int64_t)a.steps * 4;
    const uint8_t *wp[FN], *wsp[FN];
    MxFrag<kE2m1> w[FN];
    uint8_t* xs = reinterpret_cast<uint8_t*>(mx_smem) + a.M * kp;
    const int units = kp / 8;
    auto put = [&](float (&v)[8], int row, int unit) __attribute__((always_inline)) {
        const int at = (unit >> 1 ^ (row & 7)) * 2 + (unit & 1);  // its 16-byte piece
        mx_store8_at<kE4m3>(v, reinterpret_cast<uint8_t*>(mx_smem) + row * kp + at * 8, xs + row * (kp / 32) + (unit >> 2), (unit & 3) == 0);
    };
    // the weights' first step, asked for behind x's first elements: memory answers in order, and these are nearer
    auto ask = [&]() __attribute__((always_inline)) {
        M3_FENCE();
#pragma unroll
        for (int j = 0; j < FN; ++j) {
            const int n = n0 + j * 16 + r < a.N ? n0 + j * 16 + r : a.N - 1;
            wp[j] = a.w + n * wb, wsp[j] = a.ws + n * sb;
            w[j].template load<kExact>(wp[j], wsp[j], wave < a.steps ? wave : a.steps - 1, g);
        }
        M3_FENCE();
    };
    if constexpr (kPre == kNormed) {
        Held8<T> nw[kMlNormPieces], tt[kMlNormPieces];
#pragma unroll
        for (int p = 0; p < kMlNormPieces; ++p) {
            tt[p].load(reinterpret_cast<const T*>(a.x) + (int64_t)(wave < a.M ? wave : 0) * k, (lane + p * 64) * 8, k);
            nw[p].load(reinterpret_cast<const T*>(before.norm), (lane + p * 64) * 8, k);
        }
        ask();
        const double share = 1.0 / k;  // while they are on their way
        if (const int row = wave; row < a.M) {
            float t[kMlNormPieces][8];
            double squares = 0.0;
#pragma unroll
            for (int p = 0; p < kMlNormPieces; ++p) {
                tt[p].values(t[p]);
                squares = add_squares(squares, t[p]);
            }
            const RowScale rs = row_scale(wave_sum_f64(squares) * share + (double)before.eps);
#pragma unroll
            for (int p = 0; p < kMlNormPieces; ++p) {
                if (lane + p * 64 >= units) continue;
                float w8[8];
                nw[p].values(w8);
#pragma unroll
                for (int e = 0; e < 8; ++e) t[p][e] = norm_odd(t[p][e], w8[e], rs);
                put(t[p], row, lane + p * 64);
            }
        }
    } else {
        // whole groups of four: units come in sixteens
        constexpr int kHalves = kPre == kGated ? 2 : 1;
        const int all = a.M * units;
        Held8<T> v, u;
        auto read = [&](int i) __attribute__((always_inline)) {
            const int row = i / units, unit = i - row * units;
            const T* x = reinterpret_cast<const T*>(a.x) + (int64_t)row * k * kHalves;
            v.load(x, unit * 8, k);
            if constexpr (kPre == kGated) u.load(x + k, unit * 8, k);
        };
        if ((int)threadIdx.x < all) read(threadIdx.x);
        ask();
        for (int i = threadIdx.x; i < all; i += kW * 64) {
            const int row = i / units, unit = i - row * units;
            float f[8], h[8];
            v.values(f);
            if constexpr (kPre == kGated) u.values(h);
            if (i + kW * 64 < all) read(i + kW * 64);
            if constexpr (kPre == kGated) silu_mul8(f, h);
            put(f, row, unit);
        }
    }
    __syncthreads();
    f32x4 acc[1][FN];
#pragma unroll
    for (int j = 0; j < FN; ++j) acc[0][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int m = r < a.M ? r : a.M - 1;
    const char* xr = mx_smem + m * kp;
    const uint8_t* xsr = xs + m * (kp / 32);
    for (int step = wave; step < a.steps; step += kW) {
        if (step != wave) {
#pragma unroll
            for (int j = 0; j < FN; ++j) w[j].template load<kExact>(wp[j], wsp[j], step, g);
        }
        MxFrag<kE4m3> x[1];
        const int p0 = step * 8 + (kExact ? 2 * g : g), p1 = step * 8 + (kExact ? 2 * g + 1 : 4 + g);
        x[0].p[0] = *reinterpret_cast<const i32x4*>(xr + (p0 ^ (m & 7)) * 16);
        x[0].p[1] = *reinterpret_cast<const i32x4*>(xr + (p1 ^ (m & 7)) * 16);
        x[0].s = xsr[step * 4 + g];
        few_step<kE4m3, 1, FN, kExact>(w, x, acc);
    }
    __syncthreads();  // the rows have been read
    few_store<kW, 1, FN, TO>(a, reinterpret_cast<f32x4*>(mx_smem), acc, 0, n0, whole);
}

// Rows of the result are whole pieces of four.
template <typename TO>
static bool out4(const MxLinearArgs& a) {
    const size_t piece = 4 * sizeof(TO);
    return a.ld % 4 == 0 && reinterpret_cast<uintptr_t>(a.out) % piece == 0 && (!a.res || reinterpret_cast<uintptr_t>(a.res) % piece == 0);
}
// Waves of a block (the measurements: above).
template <int FM, int FN, typename F>
static void few_waves(const MxLinearArgs& a, F launch) {
    // at most 64 KB of sums
    if constexpr (FM * FN <= 4) {
        if (FN == 1 && a.steps >= 32) return launch(std::integral_constant<int, 16>{});
    }
    launch(std::integral_constant<int, FM * FN <= 8 ? 8 : 4>{});
}
template <int FA, int FM, int FN, typename TO>
static int few_t(const MxLinearArgs& a, hipStream_t stream) {
    const int64_t tn = (a.N + 16 * FN - 1) / (16 * FN), tm = (a.M + 16 * FM - 1) / (16 * FM);
    if (tn * tm >= (1 << 24)) return M3_ERR_UNSUPPORTED;  // a grid holds less than 2^32 threads, and 256 a block where there are so many
    few_waves<FM, FN>(a, [&](auto w) {
        constexpr int kW = decltype(w)::value;
        hipLaunchKernelGGL((mx_linear_few_kernel<kW, FA, FM, FN, TO>), dim3((unsigned)(tn * tm)), dim3(kW * 64), kW * FM * FN * 1024, stream, a, (int)tn,
                           out4<TO>(a));
    });
    return hipGetLastError() == hipSuccess ? M3_OK : M3_ERR_LAUNCH;
}
// Columns of a block: the fewest with which at most 256 blocks (one a CU) cover the result, since every block reads its rows
// of x anew (M = 64, K = 768: N = 3696 takes 4.4, 5.0 and 6.2 us with 16, 32 and 64 columns, N = 32000 17, 11 and 9.3).
static int few_columns(const MxLinearArgs& a, int rows) {
    const int64_t tm = (a.M + rows - 1) / rows;
    return tm * ((a.N + 15) / 16) <= 256 ? 1 : tm * ((a.N + 31) / 32) <= 256 ? 2 : 4;
}
template <int FA, int FM, typename TO>
static int few_m(const MxLinearArgs& a, hipStream_t stream) {
    const int fn = few_columns(a, 16 * FM);
    if (fn == 1) return few_t<FA, FM, 1, TO>(a, stream);
    if (fn == 2) return few_t<FA, FM, 2, TO>(a, stream);
    return few_t<FA, FM, 4, TO>(a, stream);
}
template <typename T, int kPre, int FN, typename TO>
static int raw_t(const MxLinearArgs& a, const MxBefore& before, int k, hipStream_t stream) {
    few_waves<1, FN>(a, [&](auto w) {
        constexpr int kW = decltype(w)::value;
        const int lds = std::max(a.M * a.steps * (kMxStep + 4), kW * FN * 1024);
        hipLaunchKernelGGL((mx_linear_raw_kernel<kW, T, kPre, FN, TO>), dim3((unsigned)((a.N + 16 * FN - 1) / (16 * FN))), dim3(kW * 64), lds, stream, a, before,
                           k, out4<TO>(a));
    });
    return hipGetLastError() == hipSuccess ? M3_OK : M3_ERR_LAUNCH;
}
template <typename T, int kPre, typename TO>
static int raw_n(const MxLinearArgs& a, const MxBefore& before, int k, hipStream_t stream) {
    const int fn = few_columns(a, 16);
    if (fn == 1) return raw_t<T, kPre, 1, TO>(a, before, k, stream);
    if (fn == 2) return raw_t<T, kPre, 2, TO>(a, before, k, stream);
    return raw_t<T, kPre, 4, TO>(a, before, k, stream);
}
template <typename T>
static int raw_pre(const MxLinearArgs& a, int pre, const MxBefore& before, int k, hipStream_t stream) {
    if (pre == kNormed) return raw_n<T, kNormed, T>(a, before, k, stream);
    if (pre == kGated) return raw_n<T, kGated, T>(a, before, k, stream);
    return raw_n<T, kAsIs, T>(a, before, k, stream);
}

// Many rows: tiles through LDS, as in m3_gemm.h. A block of WGM x WGN waves owns a BM x BN tile (a wave 32 FM x 64)
// and walks k in steps of 128, fetched straight to LDS as many steps ahead as it has stages (two or four); operand rows past the end come as zeros by
// the descriptors' bounds. The 32 x 32 x 64 instruction takes a step in two halves; half s of a step takes the step's blocks
// of 32 s and 2 + s, so that a lane's two scales of an operand row are one 16-bit read: group g = lane / 32 holds
// block 2 g + s (e2m1) or 16 elements of either block (e4m3), and the scale of block 2 g + s.
//
// LDS of a step: x rows of 128 (e4m3) or 64 bytes, w rows of 64, then a word of scales for each row of x and of w.
// 16-byte pieces lie XOR-swizzled, by which piece a lane fetches: piece c of row r at c ^ (r & 7), in rows of 64 bytes at
// c ^ (r >> 1 & 3), so that eight consecutive rows of a read fall on eight places.
//
// A step is 2 FM groups of two instructions, each with a fragment of x; fragments are read two groups ahead, into a ring of
// four. The barrier lies before the last two groups: by then all waves have read the step, whose place is refilled with
// the one so many stages further on, and the next step has landed. (With a whole half's fragments ahead the 256 x 256 tile spilled 94
// registers.) Blocks stay for further tiles, whose first steps are fetched by the last steps of the tile before; the
// epilogue turns the results into whole rows in a part of LDS of each wave's own.
template <int FA_, int BM_, int BN_, int WGM_, int WGN_, int STAGES_, int ER_>
struct MxTile {
    static constexpr int FA = FA_, BM = BM_, BN = BN_, WGM = WGM_, WGN = WGN_, STAGES = STAGES_;
    static constexpr int ER = ER_;  // rows of results a wave turns at once
    static constexpr int NW = WGM * WGN, NT = NW * 64;
    static constexpr int FM = BM / WGM / 32, FN = 2;
    static constexpr int XROW = FA == kE4m3 ? 128 : 64;  // bytes of x a row and step
    // copies a wave and step: of 1 KB of x and of w, of 64 rows' scales (those past the last row's fetch nothing)
    static constexpr int NX = BM * XROW / 1024 / NW, NWL = BN * 64 / 1024 / NW, NS = ((BM + BN) / 64 + NW - 1) / NW, NLD = NX + NWL + NS;
    static constexpr int kX = BM * XROW, kW = BN * 64, kS = NS * NW * 256;
    static constexpr int kStage = kX + kW + kS;
    static constexpr int kLds = STAGES * kStage + NW * ER * 128;
    static constexpr int kStores = FM * 4;  // of an epilogue, a wave
    static_assert(BN / WGN == 64 && NX * NW * 1024 == kX && NWL * NW * 1024 == kW && (ER == 16 || ER == 32), "whole copies");
};

template <int... I, typename F>
__device__ __forceinline__ void mx_each(std::integer_sequence<int, I...>, F f) {
    (f(std::integral_constant<int, I>{}), ...);
}

template <typename Tile>
__global__ __launch_bounds__(Tile::NT, 2) void mx_linear_tile_kernel(MxLinearArgs a, int tiles_m, int tiles_n) {
    constexpr int FA = Tile::FA, FM = Tile::FM, FN = Tile::FN, ST = Tile::STAGES, XROW = Tile::XROW, NLD = Tile::NLD;
    constexpr int XP = FA == kE4m3 ? 2 : 1;  // 16-byte pieces of an x fragment
    extern __shared__ __align__(16) char mx_smem[];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / Tile::WGN, wn = wave % Tile::WGN;
    const int total = tiles_m * tiles_n, grid = (int)gridDim.x;
    const int xld = a.steps * XROW, wld = a.steps * 64, sld = a.steps * 4;

    // ids -> tiles: those of one XCD (every eighth id) are a contiguous run, in groups of 8 row tiles walked column by
    // column, so that an XCD's L2 serves both operands
    auto tile_of = [&](int id, int& m0, int& n0) __attribute__((always_inline)) {
        constexpr int G = 8;
        const int x = id & 7, per = total >> 3, rest = total & 7;
        const int at = x * per + (x < rest ? x : rest) + (id >> 3);
        const int group = __builtin_amdgcn_readfirstlane(at / (G * tiles_n)), first = group * G;
        const int rows = tiles_m - first < G ? tiles_m - first : G;
        const int in = at - group * (G * tiles_n);
        const int tn = __builtin_amdgcn_readfirstlane(in / rows);
        m0 = (first + in - tn * rows) * Tile::BM, n0 = tn * Tile::BN;
    };

    // ---- copies: this wave's NX of x, NWL of w and one of the scales (64 rows of x or of w)
    unsigned xoff[Tile::NX], woff[Tile::NWL];
#pragma unroll
    for (int i = 0; i < Tile::NX; ++i) {
        constexpr int CPR = XROW / 16, RPI = 64 / CPR;
        const int r = (wave * Tile::NX + i) * RPI + lane / CPR, c = lane % CPR;
        xoff[i] = (unsigned)(r * xld + ((FA == kE4m3 ? c ^ (r & 7) : c ^ (r >> 1 & 3)) * 16));
    }
#pragma unroll
    for (int i = 0; i < Tile::NWL; ++i) {
        const int r = (wave * Tile::NWL + i) * 16 + lane / 4, c = lane % 4;
        woff[i] = (unsigned)(r * wld + ((c ^ (r >> 1 & 3)) * 16));
    }
    const unsigned soff = (unsigned)(lane * sld);
    const char *px, *pw, *ps[Tile::NS];
    int bx, bw, bs[Tile::NS], f_id, fs;
    auto enter = [&](int id) __attribute__((always_inline)) {
        f_id = id, fs = 0;
        int m0 = 0, n0 = 0;
        const bool there = id < total;
        if (there) tile_of(id, m0, n0);
        const int xr = a.M - m0 < Tile::BM ? a.M - m0 : Tile::BM, wr = a.N - n0 < Tile::BN ? a.N - n0 : Tile::BN;
        px = reinterpret_cast<const char*>(a.x) + (int64_t)m0 * xld;
        pw = reinterpret_cast<const char*>(a.w) + (int64_t)n0 * wld;
        bx = there ? (xr - 1) * xld + XROW : 0;
        bw = there ? (wr - 1) * wld + 64 : 0;
#pragma unroll
        for (int i = 0; i < Tile::NS; ++i) {
            const int c = wave * Tile::NS + i;  // of BM / 64 copies of x's scales, then BN / 64 of w's
            const bool sx = c < Tile::BM / 64;
            const int row = (sx ? c : c - Tile::BM / 64) * 64, left = (sx ? xr : wr) - row;
            ps[i] = (sx ? reinterpret_cast<const char*>(a.xs) + (int64_t)(m0 + row) * sld : reinterpret_cast<const char*>(a.ws) + (int64_t)(n0 + row) * sld);
            bs[i] = there && c < (Tile::BM + Tile::BN) / 64 && left > 0 ? ((left < 64 ? left : 64) - 1) * sld + 4 : 0;
        }
    };
    auto advance = [&]() __attribute__((always_inline)) {
        if (++fs == a.steps) enter(f_id + grid);
        else {
            px += XROW, pw += 64;
#pragma unroll
            for (int i = 0; i < Tile::NS; ++i) ps[i] += 4;
        }
    };
    const unsigned lds0 = (unsigned)reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)mx_smem);
    auto rsrc = [](const char* base, int bytes) __attribute__((always_inline)) {
        return u32x4{(unsigned)reinterpret_cast<uintptr_t>(base), (unsigned)(reinterpret_cast<uintptr_t>(base) >> 32), (unsigned)bytes,
                     (unsigned)kRsrcFlags};
    };
    // In assembly for the reason that m3_gemm.h gives: the kernel waits for its copies itself.
    auto copy16 = [](u32x4 rs, unsigned off, unsigned at) __attribute__((always_inline)) {
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" : : "s"(at), "v"(off), "s"(rs) : "memory");
    };
    auto copy4 = [](u32x4 rs, unsigned off, unsigned at) __attribute__((always_inline)) {
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds" : : "s"(at), "v"(off), "s"(rs) : "memory");
    };
    auto fetch = [&](int i, int slot) __attribute__((always_inline)) {
        const unsigned at = lds0 + slot * Tile::kStage;
        if (i < Tile::NX) copy16(rsrc(px, bx), xoff[i], at + (wave * Tile::NX + i) * 1024);
        else if (i < Tile::NX + Tile::NWL) copy16(rsrc(pw, bw), woff[i - Tile::NX], at + Tile::kX + (wave * Tile::NWL + i - Tile::NX) * 1024);
        else copy4(rsrc(ps[i - Tile::NX - Tile::NWL], bs[i - Tile::NX - Tile::NWL]), soff, at + Tile::kX + Tile::kW + (wave * Tile::NS + i - Tile::NX - Tile::NWL) * 256);
    };

    // ---- fragments
    const int r = lane & 31, g = lane >> 5;
    int xat[2][XP], wat[2];  // of the two halves, within 32 rows
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        if constexpr (FA == kE4m3) {
            xat[h][0] = r * 128 + (((2 * h + g) ^ (r & 7)) * 16);
            xat[h][XP - 1] = r * 128 + (((4 + 2 * h + g) ^ (r & 7)) * 16);
        } else {
            xat[h][0] = r * 64 + (((2 * g + h) ^ (r >> 1 & 3)) * 16);
        }
        wat[h] = r * 64 + (((2 * g + h) ^ (r >> 1 & 3)) * 16);
    }
    const int sat = r * 4 + 2 * g;
    constexpr int G = 2 * FM;  // groups of a step
    i32x4 fx[4][XP], fw[2][FN];
    int sxr[FM], swr[FN], sxn[FM], swn[FN];  // scales of this step and of the next
    typedef float f32x16 __attribute__((ext_vector_type(16)));
    f32x16 acc[FM][FN];
    auto read_x = [&](int gi, int slot) __attribute__((always_inline)) {  // group gi's
        const char* p = mx_smem + slot * Tile::kStage + (wm * FM + gi % FM) * 32 * XROW;
#pragma unroll
        for (int q = 0; q < XP; ++q) fx[gi % 4][q] = *reinterpret_cast<const i32x4*>(p + xat[gi / FM][q]);
    };
    auto read_w = [&](int h, int slot) __attribute__((always_inline)) {
        const char* p = mx_smem + slot * Tile::kStage + Tile::kX + wn * FN * 2048 + wat[h];
#pragma unroll
        for (int i = 0; i < FN; ++i) fw[h][i] = *reinterpret_cast<const i32x4*>(p + i * 2048);
    };
    auto read_scales = [&](int slot) __attribute__((always_inline)) {
        const char* p = mx_smem + slot * Tile::kStage + Tile::kX + Tile::kW + sat;
#pragma unroll
        for (int i = 0; i < FN; ++i) swn[i] = *reinterpret_cast<const unsigned short*>(p + Tile::BM * 4 + (wn * FN + i) * 128);
#pragma unroll
        for (int i = 0; i < FM; ++i) sxn[i] = *reinterpret_cast<const unsigned short*>(p + (wm * FM + i) * 128);
    };
    auto take_scales = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < FN; ++i) swr[i] = swn[i];
#pragma unroll
        for (int i = 0; i < FM; ++i) sxr[i] = sxn[i];
    };
    auto group = [&](auto gc) __attribute__((always_inline)) {
        constexpr int gi = decltype(gc)::value, h = gi / FM, i = gi % FM;
        i32x8 x;
        if constexpr (XP == 2) x = wide(fx[gi % 4][0], fx[gi % 4][XP - 1]);
        else x = wide(fx[gi % 4][0], i32x4{0, 0, 0, 0});
#pragma unroll
        for (int j = 0; j < FN; ++j)
            acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wide(fw[h][j], i32x4{0, 0, 0, 0}), x, acc[i][j], 4,
                                                                       FA == kE4m3 ? 0 : 4, h, swr[j], h, sxr[i]);
    };

    // ---- epilogue: ER rows of 64 columns at a time. Stores go out unconditionally, those past the end to an offset
    // that the descriptor drops, so that their number is known to the next wait.
    const bool whole = a.N % 8 == 0 && a.ld % 8 == 0 && reinterpret_cast<uintptr_t>(a.out) % 16 == 0 && reinterpret_cast<uintptr_t>(a.res) % 16 == 0;
    auto epilogue = [&](int id, auto with_res) __attribute__((always_inline)) {
        constexpr bool kRes = decltype(with_res)::value;
        constexpr int ER = Tile::ER, T = ER / 8;
        int m0, n0;
        tile_of(id, m0, n0);
        m0 += wm * FM * 32, n0 += wn * 64;
        const int lane = opaque((int)threadIdx.x) & 63, r = lane & 31, g = lane >> 5;  // not held across the steps
        char* mine = mx_smem + ST * Tile::kStage + wave * (ER * 128);
        const bf16* res = reinterpret_cast<const bf16*>(a.res);
        bf16* out = reinterpret_cast<bf16*>(a.out);
        // scale times the sums of a round's rows, plus what lies in their place
        auto combine = [&](int round) __attribute__((always_inline)) {
            const int i = round * ER / 32;
            if (ER == 32 || (r >> 4) == round % 2) {
#pragma unroll
                for (int j = 0; j < FN; ++j)
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        bf16x4* at = reinterpret_cast<bf16x4*>(mine + (r & (ER - 1)) * 128 + (((j * 4 + q) ^ (r & 7)) * 16) + g * 8);
                        bf16x4 o{};
                        if constexpr (kRes) o = *at;
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[e] = (bf16)fmaf(a.scale, acc[i][j][q * 4 + e], kRes ? (float)o[e] : 0.f);
                        *at = o;
                    }
            }
            M3_LDS_FENCE();  // the fours and the rows' pieces are other types to the compiler
        };
        if (whole) {
            const int rr = lane >> 3, n = n0 + (lane & 7) * 8;
            // the residual's rows as they lie, a round ahead; past the end a neighbour's, which are not stored
            bf16x8 rv[kRes ? 2 : 1][T];
            auto read_res = [&](int round, int to) __attribute__((always_inline)) {
#pragma unroll
                for (int t = 0; t < T; ++t) {
                    const int m = m0 + round * ER + t * 8 + rr;
                    rv[kRes ? to : 0][t] = *reinterpret_cast<const bf16x8*>(res + (int64_t)(m < a.M ? m : a.M - 1) * a.ld + (n < a.N ? n : a.N - 8));
                }
            };
            if constexpr (kRes) read_res(0, 0);
#pragma unroll
            for (int round = 0; round < FM * 32 / ER; ++round) {
                if constexpr (kRes) {
                    if (round + 1 < FM * 32 / ER) read_res(round + 1, (round + 1) % 2);
#pragma unroll
                    for (int t = 0; t < T; ++t)
                        *reinterpret_cast<bf16x8*>(mine + (t * 8 + rr) * 128 + (((lane & 7) ^ rr) * 16)) = rv[round % 2][t];
                    M3_LDS_FENCE();
                }
                combine(round);
                const int m1 = m0 + round * ER, rows = a.M - m1 < ER ? a.M - m1 : ER;
                const __amdgpu_buffer_rsrc_t to = make_rsrc(out + (int64_t)m1 * a.ld, rows > 0 ? (int64_t)rows * a.ld * 2 : 0);
#pragma unroll
                for (int t = 0; t < T; ++t) {
                    const u32x4 v = *reinterpret_cast<const u32x4*>(mine + (t * 8 + rr) * 128 + (((lane & 7) ^ rr) * 16));
                    __builtin_amdgcn_raw_buffer_store_b128(v, to, n < a.N ? ((t * 8 + rr) * a.ld + n) * 2 : (int)0x80000000u, 0, 0);
                }
                M3_LDS_FENCE();
            }
        } else {
            // rows of any alignment: a column a lane
            const int n = n0 + lane, nc = n < a.N ? n : a.N - 1;
            bf16* cell = reinterpret_cast<bf16*>(mine) + (lane & 7);
            auto at = [&](int row) __attribute__((always_inline)) { return cell + row * 64 + (((lane >> 3) ^ (row & 7)) * 8); };
#pragma unroll
            for (int round = 0; round < FM * 32 / ER; ++round) {
                const int m1 = m0 + round * ER;
                if constexpr (kRes) {
                    bf16 v[ER];
#pragma unroll
                    for (int e = 0; e < ER; ++e) v[e] = res[(int64_t)(m1 + e < a.M ? m1 + e : a.M - 1) * a.ld + nc];
#pragma unroll
                    for (int e = 0; e < ER; ++e) *at(e) = v[e];
                    M3_LDS_FENCE();
                }
                combine(round);
#pragma unroll
                for (int e = 0; e < ER; ++e) {
                    const bf16 v = *at(e);
                    if (m1 + e < a.M && n < a.N) out[(int64_t)(m1 + e) * a.ld + n] = v;
                }
                M3_LDS_FENCE();
            }
            asm volatile("s_waitcnt vmcnt(0)" : : : "memory");  // the stores' number is not known
        }
    };

    if ((int)blockIdx.x >= total) return;
    enter((int)blockIdx.x);
#pragma unroll
    for (int s = 0; s < ST; ++s) {
        if (s) advance();
#pragma unroll
        for (int i = 0; i < NLD; ++i) fetch(i, s);
    }
    auto wait = [](auto n) __attribute__((always_inline)) {
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" : : "n"(decltype(n)::value) : "memory");
    };
    wait(std::integral_constant<int, NLD*(ST - 1)>{});
    M3_LDS_FENCE();
    __builtin_amdgcn_s_barrier();
    M3_LDS_FENCE();
    int slot = 0;
    read_scales(0);
    read_w(0, 0);
    read_x(0, 0);
    read_x(1, 0);
    take_scales();
    constexpr int kPerLd = (NLD + 1) / 2;
    // kStored: the epilogue before has just sent its stores, behind the copies that this step waits for
    auto step = [&](auto stored) __attribute__((always_inline)) {
        constexpr int kYounger = NLD * (ST - 2) + (decltype(stored)::value ? Tile::kStores : 0);
        const int next = slot + 1 == ST ? 0 : slot + 1;
        auto at = [&](auto gc) __attribute__((always_inline)) {
            constexpr int gi = decltype(gc)::value;
            if constexpr (gi == G - 2) {
                // the next step has landed (memory operations end in order: what may be on its way is what was sent
                // after its copies), and all waves have read this one
                wait(std::integral_constant<int, kYounger>{});
                M3_LDS_FENCE();
                __builtin_amdgcn_s_barrier();
                M3_LDS_FENCE();
                read_scales(next);
                read_w(0, next);
            }
            if constexpr (gi >= G - 2) {
#pragma unroll
                for (int t = (gi - G + 2) * kPerLd; t < (gi - G + 3) * kPerLd && t < NLD; ++t) fetch(t, slot);
                read_x(gi + 2 - G, next);
            } else {
                if constexpr (gi == FM - 2) read_w(1, slot);
                read_x(gi + 2, slot);
            }
            M3_FENCE();
            group(gc);
            M3_FENCE();
        };
        advance();
        M3_FENCE();
        mx_each(std::make_integer_sequence<int, G>{}, at);  // (no branch: the compiler would move products behind it)
        take_scales();
        slot = next;
    };
    for (int id = (int)blockIdx.x; id < total; id += grid) {
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j) acc[i][j] = f32x16{};
        if (id == (int)blockIdx.x) step(std::false_type{});
        else step(std::true_type{});
        for (int n = a.steps; n > 1; --n) step(std::false_type{});
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j) asm volatile("" : "+v"(acc[i][j]));  // the last products before the epilogue's branches
        if (a.res) epilogue(id, std::true_type{});
        else epilogue(id, std::false_type{});
    }
    // no copy outlives its block
    wait(std::integral_constant<int, 0>{});
}

constexpr int kMlTileLd = 1 << 25;  // 32 rows of fewer columns are below 2^31 bytes, the end of a descriptor

template <typename Tile>
static int tile_t(const MxLinearArgs& a, hipStream_t stream) {
    const int64_t tm = (a.M + Tile::BM - 1) / Tile::BM, tn = (a.N + Tile::BN - 1) / Tile::BN;
    if (tm * tn > (1 << 30) || a.ld >= kMlTileLd) return M3_ERR_UNSUPPORTED;
    static std::atomic<uint64_t> done{0};
    if (!allow_lds(reinterpret_cast<const void*>(&mx_linear_tile_kernel<Tile>), Tile::kLds, done)) return M3_ERR_LAUNCH;
    const int64_t most = 256 * std::min(2, (160 << 10) / Tile::kLds);  // blocks at once
    hipLaunchKernelGGL((mx_linear_tile_kernel<Tile>), dim3((unsigned)std::min(tm * tn, most)), dim3(Tile::NT), Tile::kLds, stream, a,
                       (int)tm, (int)tn);
    return hipGetLastError() == hipSuccess ? M3_OK : M3_ERR_LAUNCH;
}
// Which kernel, by the number of tiles of 128 columns and the steps of k (us in a graph of weights from HBM, e4m3, few
// rows' kernel and tiles of 64 x 128, which have four steps on their way):
//   8 rows: 2048 x 128000 41.9 and 38.8, 2048 x 25600 11.8 and 11.5, 1024 x 128000 21.7 and 21.9
//   16 rows: 2048 x 128000 46.1 and 39.4, 2048 x 25600 12.8 and 11.6, 1536 x 32000 9.9 and 10.1, 768 x 128000 16.6 and 18.3, 2048 x 16000 8.8 and 10.7
//   32 rows: 2048 x 25600 16.2 and 12.0, 1024 x 32000 9.8 and 8.2, 768 x 32000 7.1 and 7.4, 768 x 128000 22 and 18, 2048 x 16000 9.7 and 10.8
//   64 rows: 2048 x 11000 14.3 and 11.4, 768 x 11000 7.9 and 6.9, 768 x 7168 5.4 and 6.7
// and with tiles of 128 x 128 (weights from the caches) 256 x 768 x 3696 6.5 and 5.9, 1000 x 768 x 4224 19 and 9.1. Tiles of 128 x 128 for
// 64 rows: 2048 x 11000 14.3, 2048 x 128000 45 (42.6). 128 x 128 and 256 x 256 tiles: 8192 x 768 x 4224 32 and 37,
// 8192 x 2112 x 768 19 and 27, 8192 x 5504 x 2048 105 and 76.
static bool takes_tiles(const MxLinearArgs& a) {
    if (a.ld >= kMlTileLd) return false;
    const int64_t tiles = (int64_t)((a.M + 127) / 128) * ((a.N + 127) / 128);
    if (a.M > 64) return tiles >= 56;
    if (a.M > 32) return tiles >= 72;
    if (a.M > 16) return tiles >= (a.steps >= 8 ? 200 : 512);
    if (a.M > 8) return tiles >= (a.steps >= 12 ? 200 : 512) && a.steps >= 8;
    return tiles >= 512 && a.steps >= 16;
}
template <int FA, typename TO>
static int linear_t(const MxLinearArgs& a, hipStream_t stream) {
    if constexpr (sizeof(TO) == 2) {
        if (takes_tiles(a)) {
            typedef MxTile<FA, 256, 256, 2, 4, 2, 32> Large;
            typedef MxTile<FA, 128, 128, 2, 2, 2, 32> Middle;
            if (a.M <= 64) return tile_t<MxTile<FA, 64, 128, 1, 2, 4, 32>>(a, stream);
            const int64_t tm = (a.M + 255) / 256, large = tm * ((a.N + 255) / 256);
            if (large < 192 || a.steps < 12 || a.M <= 128) return tile_t<Middle>(a, stream);
            // Whole rounds of large tiles, one a CU, and for the columns that are left one round of the others, two a CU, if they
            // fit it (us, all in large tiles and so: 1.2 rounds, 300 x 1700 x 40008, 43 and 38; 1.3, 2100 x 1600 x 9000, 45 and 42; 4.4, 8192 x 2048 x
            // 8800, 138 and 134). After five rounds the power that idle CUs leave to the others is worth as much (5.4, 8192 x 2048 x 11008,
            // 177 and 177, with a residual 210 and 218).
            const int64_t cols = large / 256 * 256 / tm * 256, left = a.N - cols;
            if (large >= 1280 || large % 256 == 0 || cols == 0 || (int64_t)((a.M + 127) / 128) * ((left + 127) / 128) > 512) return tile_t<Large>(a, stream);
            MxLinearArgs rest = a, most = a;
            most.N = (int)cols, rest.N = (int)left;
            rest.w += cols * a.steps * 64, rest.ws += cols * a.steps * 4;
            rest.out = reinterpret_cast<bf16*>(a.out) + cols;
            if (a.res) rest.res = reinterpret_cast<const bf16*>(a.res) + cols;
            const int st = tile_t<Large>(most, stream);
            return st == M3_OK ? tile_t<Middle>(rest, stream) : st;
        }
    }
    // rows of a block: the fewest with which 256 blocks of 16 columns do (64 x 2112 x 768 3.6, 4.7 and 7.1 us with 16, 32 and 64,
    // 32 x 5504 x 2048 6.1 and 8.6 with 16 and 32), and not 64 for 32
    const int64_t tn = (a.N + 15) / 16;
    if (a.M <= 16 || (a.M + 15) / 16 * tn <= 256) return few_m<FA, 1, TO>(a, stream);
    if (a.M <= 32 || (a.M + 31) / 32 * tn <= 256) return few_m<FA, 2, TO>(a, stream);
    return few_m<FA, 4, TO>(a, stream);
}

static MxLinearArgs linear_args(const void* x, const void* xs, const void* w, const void* ws, const void* res, float scale, void* out,
                                int m, int n, int k) {
    const auto b = [](const void* p) { return reinterpret_cast<const uint8_t*>(p); };
    return MxLinearArgs{b(x), b(xs), b(w), b(ws), res, out, scale, m, n, (int)(mx_padded(k) / kMxStep), n};
}
bool mx_linear_takes_tensor(int64_t m, int64_t n, int64_t k, int x_dtype, int out_dtype, int before) {
    if (m > kMlRawRows || m * mx_padded(k) > (before == kGated ? kMlGatedElements : kMlRawElements)) return false;
    if (before != kAsIs && x_dtype != out_dtype) return false;
    if (before == kNormed && (m > kMlNormRows || k > kMlNormPieces * 512)) return false;
    const MxLinearArgs a = linear_args(nullptr, nullptr, nullptr, nullptr, nullptr, 1.f, nullptr, (int)m, (int)n, (int)k);
    return out_dtype != M3_DTYPE_BF16 || !takes_tiles(a);
}
int launch_mx_linear_tensor(const void* x, int x_dtype, int before, const void* norm, float eps, const void* w, const void* ws, const void* res,
                            float scale, void* out, int out_dtype, int m, int n, int k, hipStream_t stream) {
    const MxLinearArgs a = linear_args(x, nullptr, w, ws, res, scale, out, m, n, k);
    const MxBefore b{norm, eps};
    if (x_dtype == out_dtype) return x_dtype == M3_DTYPE_BF16 ? raw_pre<bf16>(a, before, b, k, stream) : raw_pre<float>(a, before, b, k, stream);
    return x_dtype == M3_DTYPE_BF16 ? raw_n<bf16, kAsIs, float>(a, b, k, stream) : raw_n<float, kAsIs, bf16>(a, b, k, stream);
}
int launch_mx_linear(const void* x, const void* xs, int x_format, const void* w, const void* ws, const void* res, float scale,
                     void* out, int out_dtype, int m, int n, int k, hipStream_t stream) {
    const MxLinearArgs a = linear_args(x, xs, w, ws, res, scale, out, m, n, k);
    if (out_dtype == M3_DTYPE_BF16) return x_format == kE4m3 ? linear_t<kE4m3, bf16>(a, stream) : linear_t<kE2m1, bf16>(a, stream);
    return x_format == kE4m3 ? linear_t<kE4m3, float>(a, stream) : linear_t<kE2m1, float>(a, stream);
}

}  // namespace m3
