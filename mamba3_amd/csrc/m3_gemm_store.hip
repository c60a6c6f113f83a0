// Products whose result is stored as it is (m3_gemm.h): the MLP's down projection with its
// residual, the input and weight gradients, and the joining of partial sums.
#include "m3_gemm_host.h"
#include "m3_kernels.h"

namespace m3 {

template <typename T>
__device__ __forceinline__ void store4(T* p, f32x4 v) {
    if constexpr (sizeof(T) == 2) {
        bf16x4 o;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = (bf16)v[e];
        *reinterpret_cast<bf16x4*>(p) = o;
    } else {
        *reinterpret_cast<f32x4*>(p) = v;
    }
}

// alpha with the factor that lies on the device
__device__ __forceinline__ float store_scale(const GemmStore& s) {
    float f = s.alpha;
    if (s.num) f *= s.num[0];
    if (s.den) f = s.den[0] == 0.f ? 0.f : f / s.den[0];
    return f;
}

struct EpiStore {
    GemmStore s;
    bool vec;  // whole 16-byte pieces

    template <typename T, typename Tile, int kMode>
    __device__ __forceinline__ void run(const GemmArgs& a, const GemmPlace<Tile, kMode>& at,
                                        typename Tile::Acc (&acc)[Tile::FM][Tile::FN], char* smem, const GemmItem& it) const {
        const int z = it.batch;
        T* out = reinterpret_cast<T*>(s.out[z]);
        const T* res = reinterpret_cast<const T*>(s.res);
        const float alpha = s.part ? 1.f : store_scale(s);
        if (s.part) {
            float* part = s.part + ((int64_t)it.split * a.batch + z) * s.rows * s.cols;
            each(at, acc, [&](int m, int n, f32x4 v) {
                float* p = part + (int64_t)m * s.cols + n;
                if (vec) {
                    if (s.add) v += *reinterpret_cast<const f32x4*>(p);
                    *reinterpret_cast<f32x4*>(p) = v;
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (n + e < s.cols) p[e] = s.add ? p[e] + v[e] : v[e];
                }
            });
        } else if (vec) {
            const GemmRows<T, Tile, Tile::FN * Tile::MF> rows(smem, at.wave(), at.lane);
#pragma unroll
            for (int i = 0; i < Tile::FM; ++i) {
                const int m = at.m(i), r0 = at.row0(i), c0 = at.col0();
#pragma unroll
                for (int j = 0; j < Tile::FN; ++j)
#pragma unroll
                    for (int q = 0; q < Tile::Q; ++q) {
                        f32x4 v = four(acc[i][j], q) * alpha;
                        const int n = at.n(j, q);
                        if (res && m < s.rows && n < s.cols) {
                            typedef T T4 __attribute__((ext_vector_type(4)));
                            const T4 r = *reinterpret_cast<const T4*>(res + (int64_t)m * s.ldo + n);
#pragma unroll
                            for (int e = 0; e < 4; ++e) v[e] += (float)r[e];
                        }
                        rows.put(j, q, v);
                    }
                rows.store(out + (int64_t)r0 * s.ldo + c0, s.ldo, s.rows - r0, s.cols - c0);
            }
        } else {
            each(at, acc, [&](int m, int n, f32x4 v) {
                const int64_t o = (int64_t)m * s.ldo + n;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (n + e < s.cols) out[o + e] = (T)(v[e] * alpha + (res ? (float)res[o + e] : 0.f));
            });
        }
    }

    // f(m, n, four) for the fours that begin inside the result
    template <typename Place, typename Acc, int FM, int FN, typename F>
    __device__ __forceinline__ void each(const Place& at, Acc (&acc)[FM][FN], F f) const {
        constexpr int Q = sizeof(Acc) / 16;
#pragma unroll
        for (int i = 0; i < FM; ++i) {
            const int m = at.m(i);
            if (m >= s.rows) continue;
#pragma unroll
            for (int j = 0; j < FN * Q; ++j) {
                const int n = at.n(j / Q, j % Q);
                if (n < s.cols) f(m, n, four(acc[i][j / Q], j % Q));
            }
        }
    }
};

static bool whole_pieces(int dtype, const GemmStore& s) {
    const int e = dtype == M3_DTYPE_BF16 ? 8 : 4;
    auto al = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
    return s.cols % e == 0 && s.ldo % e == 0 && al(s.out[0]) && al(s.out[1]) && al(s.res);
}

int gemm_store(GemmForm form, int dtype, const GemmPlan& p, GemmArgs a, const GemmStore& st, int batch,
               hipStream_t stream) {
    a.splits = p.splits;
    EpiStore e{st, whole_pieces(dtype, st)};
    if (p.splits == 1 && !st.add && st.out[0]) e.s.part = nullptr;
    int r;
    if (form == kFormNT) r = gemm_dispatch<true, true, kPlain>(dtype, p, a, e, st.rows, st.cols, 1, stream);
    else if (form == kFormNN) r = gemm_dispatch<true, false, kSeg2>(dtype, p, a, e, st.rows, st.cols, 1, stream);
    else r = gemm_dispatch<false, false, kBatch2>(dtype, p, a, e, st.rows, st.cols, batch, stream);
    if (r != M3_OK || !e.s.part || !st.out[0]) return r;
    return gemm_reduce(dtype, st, p.splits, batch, stream);
}

// One thread joins four columns of a row; parts are added in order.
template <typename T, bool kVec>
__global__ __launch_bounds__(256) void gemm_reduce_kernel(GemmStore s, int splits) {
    const int z = blockIdx.y;
    const int64_t each = (int64_t)s.rows * s.cols, stride = each * gridDim.y;
    const float* part = s.part + z * each;
    T* out = reinterpret_cast<T*>(s.out[z]);
    const T* res = reinterpret_cast<const T*>(s.res);
    const float alpha = store_scale(s);
    const int64_t pieces = kVec ? each / 4 : each;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < pieces; i += (int64_t)gridDim.x * 256) {
        const int64_t at = kVec ? i * 4 : i;
        const int64_t m = at / s.cols, o = m * s.ldo + (at - m * s.cols);
        if constexpr (kVec) {
            f32x4 v{0.f, 0.f, 0.f, 0.f};
            for (int k = 0; k < splits; ++k) v += *reinterpret_cast<const f32x4*>(part + k * stride + at);
            v *= alpha;
            if (res)
                for (int e = 0; e < 4; ++e) v[e] += (float)res[o + e];
            store4(out + o, v);
        } else {
            float v = 0.f;
            for (int k = 0; k < splits; ++k) v += part[k * stride + at];
            out[o] = (T)(v * alpha + (res ? (float)res[o] : 0.f));
        }
    }
}

int gemm_reduce(int dtype, const GemmStore& st, int splits, int batch, hipStream_t stream) {
    const bool vec = whole_pieces(dtype, st);
    const int64_t pieces = (int64_t)st.rows * st.cols / (vec ? 4 : 1);
    const dim3 grid((unsigned)std::min<int64_t>((pieces + 255) / 256, 8192), (unsigned)batch);
    if (dtype == M3_DTYPE_BF16) {
        if (vec) hipLaunchKernelGGL((gemm_reduce_kernel<bf16, true>), grid, dim3(256), 0, stream, st, splits);
        else hipLaunchKernelGGL((gemm_reduce_kernel<bf16, false>), grid, dim3(256), 0, stream, st, splits);
    } else {
        if (vec) hipLaunchKernelGGL((gemm_reduce_kernel<float, true>), grid, dim3(256), 0, stream, st, splits);
        else hipLaunchKernelGGL((gemm_reduce_kernel<float, false>), grid, dim3(256), 0, stream, st, splits);
    }
    return hipGetLastError() == hipSuccess ? M3_OK : M3_ERR_LAUNCH;
}

// One thread writes 16 bytes of a row; src rows of whole, aligned pieces are read the same way.
template <typename T>
__global__ __launch_bounds__(256) void gemm_pad_kernel(GemmPads pads, const int64_t* __restrict__ target, int64_t ignore) {
    constexpr int E = 16 / sizeof(T);
    typedef T Piece __attribute__((ext_vector_type(E)));
    const int64_t all = pads.first[pads.n];
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (int64_t)gridDim.x * 256) {
        GemmPad p = pads.p[0];
        int64_t at = i;
#pragma unroll
        for (int k = 1; k < kPadCopies; ++k)
            if (k < pads.n && i >= pads.first[k]) p = pads.p[k], at = i - pads.first[k];
        const int per = p.ldd / E;
        const int64_t r = at / per;
        const int c = (int)(at - r * per) * E;
        const T* src = reinterpret_cast<const T*>(p.src) + r * p.cols + c;
        Piece v;
        if (target && target[r] == ignore) {
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] = (T)0.f;
        } else if (p.cols % E == 0) {
            v = *reinterpret_cast<const Piece*>(src);
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] = c + e < p.cols ? src[e] : (T)0.f;
        }
        *reinterpret_cast<Piece*>(reinterpret_cast<T*>(p.dst) + r * p.ldd + c) = v;
    }
}

int gemm_pad_copy(int dtype, const GemmPads& pads, const int64_t* target, int64_t ignore, hipStream_t stream) {
    if (pads.n == 0) return M3_OK;
    const dim3 grid((unsigned)std::min<int64_t>((pads.first[pads.n] + 255) / 256, 16384));
    if (dtype == M3_DTYPE_BF16)
        hipLaunchKernelGGL(gemm_pad_kernel<bf16>, grid, dim3(256), 0, stream, pads, target, ignore);
    else
        hipLaunchKernelGGL(gemm_pad_kernel<float>, grid, dim3(256), 0, stream, pads, target, ignore);
    return hipGetLastError() == hipSuccess ? M3_OK : M3_ERR_LAUNCH;
}

// Estimated us of each choice, from launches of 256, 512 and 1024 tiles of 8 and 64 k steps (torch on the
// same card: 8192^3 bf16 668 us): a step of a 256 x 256 tile takes 1.45 us, of a 128 x 128 tile 0.62 us
// alone on its CU and 0.90 us next to another, of a 64 x 64 tile 0.20 and 0.37 us; to that come a
// tile's start and epilogue. Parts of k cost the fp32 partial sums' write and read and a launch.
// What it decides, both sides measured: the gated product of 8192 x 11008 x 2048 takes 80 us less on 256 x 256
// tiles than on 128 x 128, that of 8192 x 4224 x 768 8 us more; the 8192 x 768 product over 16128 takes
// 70 us less in two parts on 256 x 256 tiles than in two on 128 x 128.
GemmPlan gemm_plan(int dtype, int64_t rows, int64_t cols, int64_t steps, int batch, int max_splits) {
    struct Cost { int size, at_once; double alone, all, fixed; };
    static const Cost bf[3] = {{256, 1, 1.45, 1.45, 8.0}, {128, 2, 0.62, 0.90, 4.5}, {64, 2, 0.20, 0.37, 3.5}};
    static const Cost fp[3] = {{0, 0, 0, 0, 0}, {128, 2, 1.90, 3.60, 5.0}, {64, 2, 0.65, 1.07, 4.0}};
    const Cost* c = dtype == M3_DTYPE_BF16 ? bf : fp;
    GemmPlan best{kTileS, 1, 64, 64};
    double least = 1e30;
    for (int t = dtype == M3_DTYPE_BF16 ? kTileL : kTileM; t <= kTileS; ++t) {
        const int64_t tiles = ((rows + c[t].size - 1) / c[t].size) * ((cols + c[t].size - 1) / c[t].size) * batch;
        for (int s = 1; s <= max_splits && s <= steps; ++s) {
            const int64_t items = tiles * s, slots = (int64_t)256 * c[t].at_once;
            const double per = (double)((steps + s - 1) / s);
            const int64_t rest = items % slots;
            double us = items / slots * (per * c[t].all + c[t].fixed);
            if (rest) us += per * (rest > 256 ? c[t].all : c[t].alone) + c[t].fixed;
            if (s > 1) us += 4.0 + (double)rows * cols * batch * 8.0 * s / 5.0e6;
            if (us < least) {
                least = us;
                best = GemmPlan{t, s, c[t].size, c[t].size};
            }
        }
    }
    return best;
}

}  // namespace m3
