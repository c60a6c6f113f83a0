// fp32 products of many rows of microscaled values with e2m1 weights (gfx950): both are written out in bf16, which holds them
// exactly, and go through the tiled bf16 product with fp32 sums (m3_gemm.h). The few-row kernel (m3_mx_linear.hip) takes the
// values apart again in every block, at 460 TFLOP/s; here the product makes 1,200, behind two launches that write the copies.
#include "m3_gemm_host.h"
#include "m3_kernels.h"
#include "m3_mx.h"

namespace m3 {

// [res +] scale * sums, a four of columns a lane.
struct EpiFloat {
    float* out;
    const float* res;
    float scale;
    int rows, cols;
    bool whole;  // rows are whole, aligned fours

    template <typename T, typename Tile, int kMode>
    __device__ __forceinline__ void run(const GemmPlace<Tile, kMode>& at, typename Tile::Acc (&acc)[Tile::FM][Tile::FN], char*, const GemmItem&) const {
#pragma unroll
        for (int i = 0; i < Tile::FM; ++i) {
            const int m = at.m(i);
            if (m >= rows) continue;
#pragma unroll
            for (int j = 0; j < Tile::FN * Tile::Q; ++j) {
                const int n = at.n(j / Tile::Q, j % Tile::Q);
                if (n >= cols) continue;
                const int64_t o = (int64_t)m * cols + n;
                f32x4 v = four(acc[i][j / Tile::Q], j % Tile::Q) * scale;
                if (whole) {
                    if (res) v += *reinterpret_cast<const f32x4*>(res + o);
                    *reinterpret_cast<f32x4*>(out + o) = v;
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (n + e < cols) out[o + e] = v[e] + (res ? res[o + e] : 0.f);
                }
            }
        }
    }
};

// From 256 rows and 10^10 products on (us, few-row kernel and this: 8192 x 2048 x 11008 811 and 341, 8192 x 768 x 3696 116 and 70,
// 8192 x 2112 x 768 57 and 47, 256 x 2048 x 32000 87 and 80, 256 x 2048 x 11008 37 and 43, 1000 x 768 x 4224 25 and 27).
size_t mx_linear_exact_workspace(int64_t m, int64_t n, int64_t k) {
    if (m < 256 || (double)m * (double)n * (double)k < 1e10) return 0;
    return (size_t)(up256(m * mx_padded(k) * 2) + up256(n * mx_padded(k) * 2));
}
int launch_mx_linear_exact(const void* x, const void* xs, int x_format, const void* w, const void* ws, const float* res, float scale,
                           float* out, int m, int n, int k, void* workspace, hipStream_t stream) {
    const int kp = (int)mx_padded(k);
    Bump room{reinterpret_cast<char*>(workspace)};
    void* xb = room.take((int64_t)m * kp * 2);
    void* wb = room.take((int64_t)n * kp * 2);
    M3_TRY(launch_mx_dequantize(x, xs, x_format, xb, M3_DTYPE_BF16, m, kp, stream));
    M3_TRY(launch_mx_dequantize(w, ws, kE2m1, wb, M3_DTYPE_BF16, n, kp, stream));
    const auto fours = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
    const EpiFloat epi{out, res, scale, m, n, n % 4 == 0 && fours(out) && fours(res)};
    const GemmPlan plan = gemm_plan(M3_DTYPE_BF16, m, n, gemm_steps(kp, M3_DTYPE_BF16), 1);
    return gemm_dispatch<true, true, kPlain>(M3_DTYPE_BF16, plan, gemm_args({xb, kp}, {wb, kp}, m, n, kp, 1), epi, m, n, stream);
}

}  // namespace m3
