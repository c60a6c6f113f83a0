// Softmax cross entropy of a vocabulary projection without its logits (gfx950): for rows h_m and a
// weight W of V rows,
//   z = h W^T, lse_m = log sum over v of exp z_mv, loss_m = lse_m - z_m,target,
//   dz_mv = (exp(z_mv - lse_m) - [v = target]) gl_m, dh = dz W, dW = dz^T h,
// where one gl for all rows (a mean or a sum) is left to the products' results: dz then holds
// softmax - 1 in the target's place, not rounded multiples of 1 / rows.
// Forward: the product's epilogue (m3_gemm.h) reduces each tile's columns to a maximum and a sum
// of exponentials per row, so one pair per row and tile of the vocabulary leaves the kernel
// instead of the logits; a second kernel joins a row's pairs, a third the rows. Backward, in
// pieces of the vocabulary: the same product again, whose epilogue writes dz of the piece, and
// the two gradient products on it: dW's rows of the piece are final, dh is summed over the
// pieces in fp32. Recomputing z costs 2 M V d operations (a quarter of the pass) and keeps the memory at one piece.
//
// Measured, bf16, forward + backward: 8192 rows, d 768, 32000 tokens 1.48 - 1.57 ms (z 381 - 398 us, dz in two pieces
// 234 us each, gradients 360 us each and 18 for dh's parts: 1,050 TF/s); 4096 rows, d 2048, 128000 tokens
// 6.6 - 6.9 ms (1,701, 4 x 454, 4 x 811: 1,260 TF/s). Bound by the MFMAs, and over short k by the epilogues,
// which a CU's one block of 256 x 256 does not overlap with products: at d 768 an exponential for each
// 768 multiply-adds. Two blocks of 128 x 128 overlap them and are slower: z 446 - 464 us, dz 309 - 316.
// Pieces of 256 MiB: two of 16128 columns at the first size. 16 rows, d 2048, 128000 tokens, fp32: 1.2 ms (z 335 and
// 311 us, dh 318, dW 354: 64-row tiles a quarter full, and 1 GB written).
//
// Rows whose target is ignored count nowhere: their loss and dz are zero by selection, and
// products over rows read them as zeros, whatever the row holds. A target outside [0, V) that is
// not the ignored value makes its row's loss, and the gradients it enters, NaN.
#include <type_traits>

#include "m3_gemm_host.h"
#include "m3_kernels.h"

namespace m3 {

constexpr int64_t kXentPieceBytes = (int64_t)256 << 20;
constexpr int64_t kXentPieceMost = (int64_t)1 << 20;  // columns: a tile's rows stay within 32-bit offsets

template <typename T> __device__ __forceinline__ float exp_of(float x);
template <> __device__ __forceinline__ float exp_of<bf16>(float x) { return fast_exp(x); }
template <> __device__ __forceinline__ float exp_of<float>(float x) { return expf(x); }

// (max, sum of exp(z - max)) of two disjoint sets. An empty set is (-inf, 0). S: the sum's type; a row's pairs come one
// after another, hundreds of them for a large vocabulary, and are summed in fp64.
template <typename S>
__device__ __forceinline__ void join(float& m, S& s, float m2, S s2) {
    const float top = fmaxf(m, m2);
    const S a = m == top ? s : s * (S)expf(m - top), b = m2 == top ? s2 : s2 * (S)expf(m2 - top);
    m = top;
    s = a + b;
}

struct EpiXentFwd {
    float2* part;           // [tiles_n][rows]
    float* zt;              // [rows]: the target's logit
    const int64_t* target;  // [rows]
    int rows, vocab;

    template <typename T, typename Tile, int kMode>
    __device__ __forceinline__ void run(const GemmPlace<Tile, kMode>& at,
                                        typename Tile::Acc (&acc)[Tile::FM][Tile::FN], char* smem, const GemmItem& it) const {
        float2* red = reinterpret_cast<float2*>(smem);  // [WGN][BM]
        if (at.n0 + Tile::BN <= vocab) rows_of<T, Tile, kMode, true>(at, acc, red);
        else rows_of<T, Tile, kMode, false>(at, acc, red);
        __syncthreads();
        for (int r = threadIdx.x; r < Tile::BM; r += Tile::NT) {
            const int m = it.tm * Tile::BM + r;
            if (m >= rows) break;
            float2 v = red[r];
#pragma unroll
            for (int w = 1; w < Tile::WGN; ++w) join(v.x, v.y, red[w * Tile::BM + r].x, red[w * Tile::BM + r].y);
            part[(int64_t)it.tn * rows + m] = v;
        }
    }

    // The lanes of a row hold 4 columns of each piece; kAll: every column of the tile exists.
    template <typename T, typename Tile, int kMode, bool kAll>
    __device__ __forceinline__ void rows_of(const GemmPlace<Tile, kMode>& at, typename Tile::Acc (&acc)[Tile::FM][Tile::FN],
                                            float2* red) const {
        constexpr int J = Tile::FN * Tile::Q;
        const int first = at.n(0, 0);
        // the target's place among this wave's columns, of all pieces' rows
        int rel[Tile::FM];
#pragma unroll
        for (int i = 0; i < Tile::FM; ++i) {
            const int m = at.m(i);
            const int64_t t = m < rows ? target[m] : -1;
            rel[i] = t >= 0 && t < vocab ? (int)t - first : -1;
        }
        auto logit = [&](int i, int j, int e) __attribute__((always_inline)) {
            const float v = four(acc[i][j / Tile::Q], j % Tile::Q)[e];
            return kAll || at.n(j / Tile::Q, j % Tile::Q) + e < vocab ? v : -INFINITY;
        };
        float top[Tile::FM];
#pragma unroll
        for (int i = 0; i < Tile::FM; ++i) {
            top[i] = -INFINITY;
#pragma unroll
            for (int j = 0; j < J; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) top[i] = fmaxf(top[i], logit(i, j, e));
            // few waves hold the target of one of their rows
            if (__any(rel[i] >= 0 && rel[i] < Tile::FN * Tile::MF)) {
#pragma unroll
                for (int j = 0; j < J; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (rel[i] == at.n(j / Tile::Q, j % Tile::Q) - first + e) zt[at.m(i)] = logit(i, j, e);
            }
        }
        bool any_far = false;
#pragma unroll
        for (int i = 0; i < Tile::FM; ++i) {
#pragma unroll
            for (int off = Tile::MF; off < 64; off *= 2) top[i] = fmaxf(top[i], __shfl_xor(top[i], off, kWave));
            any_far = any_far || far(top[i]);
        }
        // The sums of exp(z - top). bf16: as one fma before the instruction, but for far rows; `some`: there are such
        // rows in this wave (the others' sums do not change by it).
        auto sums = [&](auto some) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < Tile::FM; ++i) {
                const float ref = top[i] == -INFINITY ? 0.f : top[i];  // a row without finite logits
                const float low = -ref * kLog2e;
                float sum = 0.f, apart = 0.f;
#pragma unroll
                for (int j = 0; j < J; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float z = logit(i, j, e);
                        if constexpr (sizeof(T) == 2) sum += __builtin_amdgcn_exp2f(__builtin_fmaf(z, kLog2e, low));
                        if constexpr (decltype(some)::value) apart += exp_of<T>(z - ref);
                    }
                // every term is off by low's rounding, which the fma sees
                if constexpr (sizeof(T) == 2) sum *= __builtin_amdgcn_exp2f(-__builtin_fmaf(ref, kLog2e, low));
                if constexpr (decltype(some)::value) sum = sizeof(T) == 4 || far(ref) ? apart : sum;
#pragma unroll
                for (int off = Tile::MF; off < 64; off *= 2) sum += __shfl_xor(sum, off, kWave);
                if (at.lane < Tile::MF) red[at.wn * Tile::BM + at.local_m(i)] = make_float2(top[i], sum);
            }
        };
        if (sizeof(T) == 4 || __any(any_far)) sums(std::true_type{});
        else sums(std::false_type{});
    }
    // logits at the type's ends: their product with log2(e) overflows
    static __device__ __forceinline__ bool far(float top) { return fabsf(top) > 1e38f && top != -INFINITY; }
};

struct EpiXentBwd {
    void* dz;  // rows x ld: the piece's columns, zero past the vocabulary
    int ld;
    const float* lse;
    const float* gl;         // dL/dloss [rows] without a reduction, else nullptr
    const int64_t* target;
    int64_t ignore;
    int v0, have, vocab, rows;  // first column of the piece, its columns that exist

    template <typename T, typename Tile, int kMode>
    __device__ __forceinline__ void run(const GemmPlace<Tile, kMode>& at,
                                        typename Tile::Acc (&acc)[Tile::FM][Tile::FN], char* smem, const GemmItem&) const {
        constexpr int J = Tile::FN * Tile::Q;
        GemmRows<T, Tile, Tile::FN * Tile::MF> out(smem, at.wave(), at.lane);
        const int first = at.n(0, 0);
        const bool all = at.n0 + Tile::BN <= have;  // every column of the tile exists
        float low[Tile::FM], g[Tile::FM];
        int rel[Tile::FM];  // the target's place among this wave's columns
#pragma unroll
        for (int i = 0; i < Tile::FM; ++i) {
            const int m = at.m(i) < rows ? at.m(i) : rows - 1;
            const int64_t t = target[m];
            const bool live = t != ignore;
            // a target outside the vocabulary makes its row NaN
            low[i] = !live ? INFINITY : t < 0 || t >= vocab ? NAN : lse[m];
            g[i] = gl && live ? gl[m] : 1.f;
            rel[i] = live && t >= v0 && t < v0 + have ? (int)(t - v0) - first : -1;
        }
#pragma unroll
        for (int i = 0; i < Tile::FM; ++i) {
            const bool hit = __any(rel[i] >= 0 && rel[i] < Tile::FN * Tile::MF);
            const int r0 = at.row0(i), c0 = at.col0();
            out.begin(reinterpret_cast<T*>(dz) + (int64_t)r0 * ld + c0, ld, rows - r0, ld - c0);
#pragma unroll
            for (int j = 0; j < J; ++j) {
                const int n = at.n(j / Tile::Q, j % Tile::Q);
                const f32x4 z = four(acc[i][j / Tile::Q], j % Tile::Q);
                f32x4 p;
#pragma unroll
                for (int e = 0; e < 4; ++e) p[e] = exp_of<T>(z[e] - low[i]);
                if (hit)
#pragma unroll
                    for (int e = 0; e < 4; ++e) p[e] -= rel[i] == n - first + e ? 1.f : 0.f;
                if (gl) p *= g[i];
                // ignored: zero whatever the weight holds (hidden reads as zero there, and 0 * inf is NaN)
#pragma unroll
                for (int e = 0; e < 4; ++e) p[e] = low[i] == INFINITY ? 0.f : p[e];
                if (!all)
#pragma unroll
                    for (int e = 0; e < 4; ++e) p[e] = n + e < have ? p[e] : 0.f;
                out.put(j / Tile::Q, j % Tile::Q, p);
            }
            out.store();
        }
    }
};

constexpr int kXentRows = 16;  // rows a block of xent_rows_kernel

// lse and loss of 16 rows: 16 threads a row take every 16th pair (a read of the block takes 128 bytes
// of each of 16 tiles' pairs), then meet in LDS. 4096 rows of 500 pairs: 64 rows a block, 4
// threads each, took 62 us.
__global__ __launch_bounds__(256) void xent_rows_kernel(const float2* __restrict__ part, const float* __restrict__ zt,
                                                        const int64_t* __restrict__ target, int64_t ignore, int tiles,
                                                        int rows, int vocab, float* __restrict__ loss,
                                                        float* __restrict__ lse, double* __restrict__ sums) {
    constexpr int Q = 256 / kXentRows;
    __shared__ float red_top[Q][kXentRows];
    __shared__ double red_sum[Q][kXentRows];
    const int r = threadIdx.x % kXentRows, q = threadIdx.x / kXentRows;
    const int m = blockIdx.x * kXentRows + r;
    float top = -INFINITY;
    double sum = 0.0;
    if (m < rows) {
#pragma unroll 4
        for (int t = q; t < tiles; t += Q) {
            const float2 v = part[(int64_t)t * rows + m];
            join(top, sum, v.x, (double)v.y);
        }
    }
    red_top[q][r] = top;
    red_sum[q][r] = sum;
    __syncthreads();
    if (threadIdx.x >= 64) return;
    double mine = 0.0, counts = 0.0;
    if (q == 0 && m < rows) {
#pragma unroll
        for (int k = 1; k < Q; ++k) join(top, sum, red_top[k][r], red_sum[k][r]);
        // the loss from the difference of the logits, not of numbers as large as they are
        const float log_sum = logf((float)sum);
        const int64_t t = target[m];
        float v = 0.f;
        if (t != ignore) {
            v = t >= 0 && t < vocab ? (top - zt[m]) + log_sum : NAN;
            counts = 1.0;
        }
        lse[m] = top + log_sum;
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
        if (threadIdx.x == 0) {
            sums[2 * blockIdx.x] = mine;
            sums[2 * blockIdx.x + 1] = counts;
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
    f.z = gemm_plan(dtype, rows, vocab, gemm_steps(d, dtype), 1);
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
    GemmPlan z;
    GemmPairPlan grads;  // dh, dW
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
    f.z = gemm_plan(dtype, rows, f.piece, gemm_steps(d, dtype), 1);
    const GemmTask tasks[2] = {{want_dh ? rows : 0, d, gemm_steps(f.piece, dtype), kMostSplits, false},
                               {want_dw ? f.piece : 0, d, gemm_steps(rows, dtype), kMaxSplits, true}};
    f.grads = gemm_pair_plan(dtype, tasks);
    const int dh_splits = f.grads.p[0].splits[0];
    f.h = b.take(rows * dp * size);
    f.w = dp != d ? b.take(vocab * dp * size) : nullptr;
    f.dz = b.take(rows * f.piece * size);
    f.part = want_dh && (pieces > 1 || dh_splits > 1) ? reinterpret_cast<float*>(b.take((int64_t)dh_splits * rows * d * 4)) : nullptr;
    f.part_dw = want_dw ? reinterpret_cast<float*>(b.take((int64_t)gemm_part_bytes(f.grads.p[1].splits[1], f.piece, d))) : nullptr;
    f.bytes = b.used;
    return f;
}

}  // namespace

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
        GemmPads pads;
        pads.add(dtype, hidden, f.h, rows, d, dp);
        pads.add(dtype, weight, f.w, vocab, d, dp);
        M3_TRY(gemm_pad_copy(dtype, pads, nullptr, 0, stream));
        hidden = f.h, weight = f.w;
    }
    M3_TRY((gemm_dispatch<true, true, kPlain>(dtype, f.z, gemm_args({hidden, dp}, {weight, dp}, rows, vocab, dp, 1),
                                              EpiXentFwd{f.part, f.zt, target, (int)rows, (int)vocab}, rows, vocab, stream)));
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
    GemmPads live, pads;
    live.add(dtype, hidden, f.h, rows, d, dp);
    M3_TRY(gemm_pad_copy(dtype, live, target, ignore, stream));
    if (f.w) {
        pads.add(dtype, weight, f.w, vocab, d, dp);
        M3_TRY(gemm_pad_copy(dtype, pads, nullptr, 0, stream));
        weight = f.w;
    }
    const int r = (int)rows;
    const bool none = reduction == M3_REDUCTION_NONE;
    GemmGrads g;
    GemmStore& dh = g.st[0];
    if (dhidden) dh = GemmStore{nullptr, d, nullptr, 1.f, f.part, 0, r, (int)d};
    if (!none) dh.num = grad_loss;
    if (reduction == M3_REDUCTION_MEAN) dh.den = count;
    for (int64_t v0 = 0; v0 < vocab; v0 += f.piece) {
        const int64_t have = std::min(f.piece, vocab - v0);
        const char* w = reinterpret_cast<const char*>(weight) + v0 * dp * size;
        // dz of the piece; columns past the vocabulary, up to the row stride, are written as zeros
        M3_TRY((gemm_dispatch<true, true, kPlain>(
            dtype, f.z, gemm_args({f.h, dp}, {w, dp}, rows, have, dp, 1),
            EpiXentBwd{f.dz, (int)f.piece, lse, none ? grad_loss : nullptr, target, ignore, (int)v0, (int)have, (int)vocab, r},
            rows, f.piece, stream)));
        if (dhidden) {
            g.a[0] = gemm_args({f.dz, f.piece}, {w, dp}, rows, dp, f.piece, 1);
            g.a[0].KB[0] = (int)have;
            if (f.piece >= vocab) dh.out = dhidden;  // one piece: no sum over calls
        }
        if (dweight) {
            g.a[1] = gemm_args({f.dz, f.piece}, {f.h, dp}, f.piece, dp, rows, 1);
            g.st[1] = GemmStore{reinterpret_cast<char*>(dweight) + v0 * d * size, d, nullptr, 1.f, f.part_dw, 0, (int)have, (int)d};
            g.st[1].num = dh.num, g.st[1].den = dh.den;
        }
        if (f.grads.apart) {
            GemmGrads one;
            one.a[0] = g.a[0], one.st[0] = g.st[0];
            M3_TRY(gemm_grads(dtype, f.grads.p[0], one, stream));
            one = GemmGrads{};
            one.a[1] = g.a[1], one.st[1] = g.st[1];
            M3_TRY(gemm_grads(dtype, f.grads.p[1], one, stream));
        } else {
            M3_TRY(gemm_grads(dtype, f.grads.p[0], g, stream));
        }
        dh.add = 1;
    }
    if (dhidden && f.piece < vocab) {
        dh.out = dhidden;
        dh.splits = f.grads.p[0].splits[0];
        M3_TRY(gemm_reduce(dtype, &dh, 1, stream));
    }
    return M3_OK;
}

}  // namespace m3
