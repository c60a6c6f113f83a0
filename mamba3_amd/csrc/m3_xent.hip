// Softmax cross entropy of a vocabulary projection without its logits (gfx950): for rows h_m and a
// weight W of V rows,
//   z = h W^T, lse_m = log sum over v of exp z_mv, loss_m = lse_m - z_m,target,
//   dz_mv = (exp(z_mv - lse_m) - [v = target]) gl_m, dh = dz W, dW = dz^T h.
// Forward: the product's epilogue (m3_gemm.h) reduces each tile's columns to a maximum and a sum
// of exponentials per row, so one pair per row and tile of the vocabulary leaves the kernel
// instead of the logits; a second kernel joins a row's pairs, a third the rows. Backward, in
// pieces of the vocabulary: the same product again, whose epilogue writes dz of the piece, and
// the two gradient products on it: dW's rows of the piece are final, dh is summed over the
// pieces in fp32. Recomputing z costs 2 M V d operations (a quarter of the pass) and keeps the memory at one piece.
//
// Rows whose target is ignored count nowhere: their loss and dz are zero by selection, and
// products over rows read them as zeros, whatever the row holds. A target outside [0, V) that is
// not the ignored value makes its row's loss, and the gradients it enters, NaN.
#include "m3_gemm_host.h"
#include "m3_kernels.h"

namespace m3 {

constexpr int kXentSplits = 16;
constexpr int64_t kXentPieceBytes = (int64_t)256 << 20;
constexpr int64_t kXentPieceMost = (int64_t)1 << 20;  // columns: a tile's rows stay within 32-bit offsets

template <typename T> __device__ __forceinline__ float exp_of(float x);
template <> __device__ __forceinline__ float exp_of<bf16>(float x) { return fast_exp(x); }
template <> __device__ __forceinline__ float exp_of<float>(float x) { return expf(x); }

// (max, sum of exp(z - max)) of two disjoint sets. An empty set is (-inf, 0).
__device__ __forceinline__ void join(float& m, float& s, float m2, float s2) {
    const float top = fmaxf(m, m2);
    const float a = m == top ? s : s * expf(m - top), b = m2 == top ? s2 : s2 * expf(m2 - top);
    m = top;
    s = a + b;
}

struct EpiXentFwd {
    float2* part;           // [tiles_n][rows]
    float* zt;              // [rows]: the target's logit
    const int64_t* target;  // [rows]
    int rows, vocab;

    template <typename T, typename Tile, int kMode>
    __device__ __forceinline__ void run(const GemmArgs&, const GemmPlace<Tile, kMode>& at,
                                        typename Tile::Acc (&acc)[Tile::FM][Tile::FN], char* smem, int tm, int tn, int) const {
        float2* red = reinterpret_cast<float2*>(smem);  // [WGN][BM]
#pragma unroll
        for (int i = 0; i < Tile::FM; ++i) {
            const int m = at.m(i);
            const int64_t t = m < rows ? target[m] : -1;
            float top = -INFINITY;
#pragma unroll
            for (int j = 0; j < Tile::FN * Tile::Q; ++j) {
                const int n = at.n(j / Tile::Q, j % Tile::Q);
                const f32x4 v = four(acc[i][j / Tile::Q], j % Tile::Q);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (n + e < vocab) {
                        top = fmaxf(top, v[e]);
                        if (t == n + e) zt[m] = v[e];
                    }
                }
            }
#pragma unroll
            for (int off = Tile::MF; off < 64; off *= 2) top = fmaxf(top, __shfl_xor(top, off, kWave));
            float sum = 0.f;
            const float ref = top == -INFINITY ? 0.f : top;  // a row without finite logits
#pragma unroll
            for (int j = 0; j < Tile::FN * Tile::Q; ++j) {
                const int n = at.n(j / Tile::Q, j % Tile::Q);
                const f32x4 v = four(acc[i][j / Tile::Q], j % Tile::Q);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (n + e < vocab) sum += exp_of<T>(v[e] - ref);
            }
#pragma unroll
            for (int off = Tile::MF; off < 64; off *= 2) sum += __shfl_xor(sum, off, kWave);
            if (at.lane < Tile::MF) red[at.wn * Tile::BM + at.local_m(i)] = make_float2(top, sum);
        }
        __syncthreads();
        for (int r = threadIdx.x; r < Tile::BM; r += Tile::NT) {
            const int m = tm * Tile::BM + r;
            if (m >= rows) break;
            float2 v = red[r];
#pragma unroll
            for (int w = 1; w < Tile::WGN; ++w) join(v.x, v.y, red[w * Tile::BM + r].x, red[w * Tile::BM + r].y);
            part[(int64_t)tn * rows + m] = v;
        }
    }
};

struct EpiXentBwd {
    void* dz;  // rows x ld: the piece's columns, zero past the vocabulary
    int ld;
    const float* lse;
    const float* count;      // [1]: rows that count
    const float* gl;         // dL/dloss: [1], or [rows] for no reduction
    const int64_t* target;
    int64_t ignore;
    int reduction;
    int v0, vocab, rows;     // first column of the piece

    template <typename T, typename Tile, int kMode>
    __device__ __forceinline__ void run(const GemmArgs&, const GemmPlace<Tile, kMode>& at,
                                        typename Tile::Acc (&acc)[Tile::FM][Tile::FN], char*, int, int, int) const {
        typedef T T4 __attribute__((ext_vector_type(4)));
        const float all = reduction == M3_REDUCTION_NONE ? 0.f : gl[0];
        const float each = reduction == M3_REDUCTION_MEAN ? all / count[0] : all;
#pragma unroll
        for (int i = 0; i < Tile::FM; ++i) {
            const int m = at.m(i);
            if (m >= rows) continue;
            const int64_t t = target[m];
            const bool live = t != ignore;
            float g = reduction == M3_REDUCTION_NONE ? gl[m] : each;
            if (t < 0 || t >= vocab) g = NAN;
            const float l = lse[m];
#pragma unroll
            for (int j = 0; j < Tile::FN * Tile::Q; ++j) {
                const int n = at.n(j / Tile::Q, j % Tile::Q);
                if (n >= ld) continue;
                const f32x4 v = four(acc[i][j / Tile::Q], j % Tile::Q);
                T4 o;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float p = exp_of<T>(v[e] - l);
                    if (t == v0 + n + e) p -= 1.f;
                    o[e] = (T)(live && v0 + n + e < vocab ? p * g : 0.f);
                }
                *reinterpret_cast<T4*>(reinterpret_cast<T*>(dz) + (int64_t)m * ld + n) = o;
            }
        }
    }
};

constexpr int kXentRows = 64;  // rows a block of xent_rows_kernel

// lse and loss of 64 rows: 4 threads a row take every 4th pair, then meet in LDS.
__global__ __launch_bounds__(256) void xent_rows_kernel(const float2* __restrict__ part, const float* __restrict__ zt,
                                                        const int64_t* __restrict__ target, int64_t ignore, int tiles,
                                                        int rows, int vocab, float* __restrict__ loss,
                                                        float* __restrict__ lse, double* __restrict__ sums) {
    __shared__ float2 red[4][kXentRows];
    __shared__ double s_sum[kXentRows];
    const int r = threadIdx.x & 63, q = threadIdx.x >> 6;
    const int m = blockIdx.x * kXentRows + r;
    float top = -INFINITY, sum = 0.f;
    if (m < rows)
        for (int t = q; t < tiles; t += 4) {
            const float2 v = part[(int64_t)t * rows + m];
            join(top, sum, v.x, v.y);
        }
    red[q][r] = make_float2(top, sum);
    __syncthreads();
    if (q == 0) {
        double mine = 0.0, counts = 0.0;
        if (m < rows) {
#pragma unroll
            for (int k = 1; k < 4; ++k) join(top, sum, red[k][r].x, red[k][r].y);
            const float l = top + logf(sum);
            const int64_t t = target[m];
            float v = 0.f;
            if (t != ignore) {
                v = t >= 0 && t < vocab ? l - zt[m] : NAN;
                counts = 1.0;
            }
            lse[m] = l;
            if (loss) loss[m] = v;
            mine = (double)v;
        }
        if (sums) {
            // lanes in a fixed order
#pragma unroll
            for (int off = 32; off > 0; off >>= 1) {
                mine += __shfl_xor(mine, off, kWave);
                counts += __shfl_xor(counts, off, kWave);
            }
            if (r == 0) {
                sums[2 * blockIdx.x] = mine;
                sums[2 * blockIdx.x + 1] = counts;
            }
        }
    }
}

// The blocks' sums in a fixed order: the loss and the number of rows that count.
__global__ __launch_bounds__(256) void xent_total_kernel(const double* __restrict__ sums, int n, int reduction,
                                                         float* __restrict__ loss, float* __restrict__ count) {
    __shared__ double red[2][256];
    double a = 0.0, b = 0.0;
    for (int i = threadIdx.x; i < n; i += 256) {
        a += sums[2 * i];
        b += sums[2 * i + 1];
    }
    red[0][threadIdx.x] = a;
    red[1][threadIdx.x] = b;
    __syncthreads();
    for (int off = 128; off > 0; off >>= 1) {
        if (threadIdx.x < off) {
            red[0][threadIdx.x] += red[0][threadIdx.x + off];
            red[1][threadIdx.x] += red[1][threadIdx.x + off];
        }
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        // no row counts: the mean of nothing is NaN
        if (reduction != M3_REDUCTION_NONE)
            loss[0] = (float)(reduction == M3_REDUCTION_MEAN ? red[0][0] / red[1][0] : red[0][0]);
        count[0] = (float)red[1][0];
    }
}

namespace {

struct Bump {
    char* p;
    size_t used = 0;
    void* take(int64_t bytes) {
        void* r = p ? p + used : nullptr;
        used += (size_t)up256(bytes);
        return r;
    }
};

struct XentFwd {
    GemmPlan z;
    int tiles;
    void *h, *w;
    float2* part;
    float* zt;
    double* sums;
    size_t bytes;
};
XentFwd xent_fwd_layout(int64_t rows, int64_t d, int64_t vocab, int dtype, void* ws) {
    XentFwd f;
    Bump b{reinterpret_cast<char*>(ws)};
    const int64_t dp = gemm_pad(d, dtype), size = dtype == M3_DTYPE_BF16 ? 2 : 4;
    f.z = gemm_plan(dtype, rows, vocab, gemm_steps(d, dtype), 1, 1);
    f.tiles = (int)((vocab + f.z.bn - 1) / f.z.bn);
    f.h = dp != d ? b.take(rows * dp * size) : nullptr;
    f.w = dp != d ? b.take(vocab * dp * size) : nullptr;
    f.part = reinterpret_cast<float2*>(b.take((int64_t)f.tiles * rows * 8));
    f.zt = reinterpret_cast<float*>(b.take(rows * 4));
    f.sums = reinterpret_cast<double*>(b.take((rows + kXentRows - 1) / kXentRows * 16));
    f.bytes = b.used;
    return f;
}

struct XentBwd {
    int64_t piece;  // columns of a piece (its row stride)
    GemmPlan z, dh, dw;
    void *h, *w, *dz;
    float* part;      // dh's sums
    float* part_dw;
    size_t bytes;
};
XentBwd xent_bwd_layout(int64_t rows, int64_t d, int64_t vocab, int dtype, bool want_dh, bool want_dw, void* ws) {
    XentBwd f;
    Bump b{reinterpret_cast<char*>(ws)};
    const int64_t dp = gemm_pad(d, dtype), size = dtype == M3_DTYPE_BF16 ? 2 : 4;
    // pieces of equal width within the bound, whole 256-column tiles
    const int64_t most = std::min<int64_t>(std::max<int64_t>(kXentPieceBytes / (rows * size) / 256 * 256, 256), kXentPieceMost);
    const int64_t pieces = (vocab + most - 1) / most;
    f.piece = pieces == 1 ? gemm_pad(vocab, dtype) : ((vocab + pieces - 1) / pieces + 255) / 256 * 256;
    f.z = gemm_plan(dtype, rows, f.piece, gemm_steps(d, dtype), 1, 1);
    f.dh = gemm_plan(dtype, rows, d, gemm_steps(f.piece, dtype), 1, kXentSplits);
    f.dw = gemm_plan(dtype, f.piece, d, gemm_steps(rows, dtype), 1, kXentSplits);
    f.h = b.take(rows * dp * size);
    f.w = dp != d ? b.take(vocab * dp * size) : nullptr;
    f.dz = b.take(rows * f.piece * size);
    f.part = want_dh ? reinterpret_cast<float*>(b.take((int64_t)f.dh.splits * rows * d * 4)) : nullptr;
    f.part_dw = want_dw ? reinterpret_cast<float*>(b.take((int64_t)gemm_part_bytes(f.dw, 1, f.piece, d))) : nullptr;
    f.bytes = b.used;
    return f;
}

}  // namespace

#define M3_TRY(e)                       \
    do {                                \
        const int st_ = (e);            \
        if (st_ != M3_OK) return st_;   \
    } while (0)

size_t xent_fwd_workspace(int64_t rows, int64_t d, int64_t vocab, int dtype) {
    return xent_fwd_layout(rows, d, vocab, dtype, nullptr).bytes;
}
size_t xent_bwd_workspace(int64_t rows, int64_t d, int64_t vocab, int dtype, bool want_dh, bool want_dw) {
    return xent_bwd_layout(rows, d, vocab, dtype, want_dh, want_dw, nullptr).bytes;
}

int launch_xent_fwd(int64_t rows, int64_t d, int64_t vocab, int dtype, int reduction, const void* hidden,
                    const void* weight, const int64_t* target, int64_t ignore, float* loss, float* lse, float* count,
                    void* ws, hipStream_t stream) {
    const XentFwd f = xent_fwd_layout(rows, d, vocab, dtype, ws);
    const int64_t dp = gemm_pad(d, dtype);
    if (f.h) {
        M3_TRY(gemm_pad_copy(dtype, hidden, f.h, rows, d, dp, nullptr, 0, stream));
        M3_TRY(gemm_pad_copy(dtype, weight, f.w, vocab, d, dp, nullptr, 0, stream));
        hidden = f.h, weight = f.w;
    }
    M3_TRY((gemm_dispatch<true, true, kPlain>(dtype, f.z, gemm_args({hidden, dp}, {weight, dp}, rows, vocab, dp, 1),
                                              EpiXentFwd{f.part, f.zt, target, (int)rows, (int)vocab}, rows, vocab, 1, stream)));
    const bool none = reduction == M3_REDUCTION_NONE;
    const int blocks = (int)((rows + kXentRows - 1) / kXentRows);
    hipLaunchKernelGGL(xent_rows_kernel, dim3(blocks), dim3(256), 0, stream, f.part, f.zt, target, ignore, f.tiles,
                       (int)rows, (int)vocab, none ? loss : nullptr, lse, none ? nullptr : f.sums);
    if (!none) hipLaunchKernelGGL(xent_total_kernel, dim3(1), dim3(256), 0, stream, f.sums, blocks, reduction, loss, count);
    return hipGetLastError() == hipSuccess ? M3_OK : M3_ERR_LAUNCH;
}

int launch_xent_bwd(int64_t rows, int64_t d, int64_t vocab, int dtype, int reduction, const void* hidden,
                    const void* weight, const int64_t* target, int64_t ignore, const float* lse, const float* count,
                    const float* grad_loss, void* dhidden, void* dweight, void* ws, hipStream_t stream) {
    const XentBwd f = xent_bwd_layout(rows, d, vocab, dtype, dhidden != nullptr, dweight != nullptr, ws);
    const int64_t dp = gemm_pad(d, dtype), size = dtype == M3_DTYPE_BF16 ? 2 : 4;
    M3_TRY(gemm_pad_copy(dtype, hidden, f.h, rows, d, dp, target, ignore, stream));
    if (f.w) {
        M3_TRY(gemm_pad_copy(dtype, weight, f.w, vocab, d, dp, nullptr, 0, stream));
        weight = f.w;
    }
    const int r = (int)rows;
    GemmStore dh{{nullptr, nullptr}, d, nullptr, 1.f, f.part, 0, r, (int)d};
    for (int64_t v0 = 0; v0 < vocab; v0 += f.piece) {
        const int64_t have = std::min(f.piece, vocab - v0);
        const char* w = reinterpret_cast<const char*>(weight) + v0 * dp * size;
        // dz of the piece; columns past the vocabulary, up to the row stride, are written as zeros
        M3_TRY((gemm_dispatch<true, true, kPlain>(
            dtype, f.z, gemm_args({f.h, dp}, {w, dp}, rows, have, dp, 1),
            EpiXentBwd{f.dz, (int)f.piece, lse, count, grad_loss, target, ignore, reduction, (int)v0, (int)vocab, r},
            rows, f.piece, 1, stream)));
        if (dhidden) {
            GemmArgs a = gemm_args({f.dz, f.piece}, {w, dp}, rows, dp, f.piece, 1);
            a.KB[0] = (int)have;
            M3_TRY(gemm_store(kFormNN, dtype, f.dh, a, dh, 1, stream));
            dh.add = 1;
        }
        if (dweight) {
            void* out = reinterpret_cast<char*>(dweight) + v0 * d * size;
            const GemmStore dw{{out, nullptr}, d, nullptr, 1.f, f.part_dw, 0, (int)have, (int)d};
            M3_TRY(gemm_store(kFormTN, dtype, f.dw, gemm_args({f.dz, f.piece}, {f.h, dp}, f.piece, dp, rows, 1), dw, 1, stream));
        }
    }
    if (dhidden) {
        dh.out[0] = dhidden;
        M3_TRY(gemm_reduce(dtype, dh, f.dh.splits, 1, stream));
    }
    return M3_OK;
}

}  // namespace m3
