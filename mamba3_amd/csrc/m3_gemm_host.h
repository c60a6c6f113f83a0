// Host side of the tiled products: tile and split choice, launches (m3_gemm.h).
#pragma once

#include <algorithm>
#include <atomic>

#include "m3_gemm.h"
#include "m3_gemm_plan.h"

namespace m3 {

// Tiles: 256 x 256 by 8 waves (bf16 only; one block a CU), 128 x 128 by 4 waves (two blocks a
// CU), 64 x 64 by 4 waves, four steps deep (two blocks a CU).
typedef GemmTile<256, 256, 2, 4, 2, 16> TileL;
template <typename T> using TileM = GemmTile<128, 128, 2, 2, 2, sizeof(T) == 2 ? 16 : 32>;
typedef GemmTile<64, 64, 2, 2, 4, 16> TileS;

struct GemmPlan {
    int tile;
    int splits;
    int bm, bn;
};

// search_plan and pair_plan (m3_gemm_plan.h), kept for the next calls of the same sizes.
GemmGroupPlan gemm_group_plan(int dtype, const GemmTask* tasks, int n);
GemmPairPlan gemm_pair_plan(int dtype, const GemmTask (&tasks)[2]);
GemmPlan gemm_plan(int dtype, int64_t rows, int64_t cols, int64_t steps, int max_splits);

inline int64_t gemm_steps(int64_t k, int dtype) {
    const int bk = dtype == M3_DTYPE_BF16 ? 64 : 32;
    return (k + bk - 1) / bk;
}
inline int64_t gemm_pad(int64_t n, int dtype) {  // to 16 bytes
    const int e = dtype == M3_DTYPE_BF16 ? 8 : 4;
    return (n + e - 1) / e * e;
}
inline int64_t up256(int64_t n) { return (n + 255) / 256 * 256; }

// A running pointer through the workspace.
struct Bump {
    char* p;
    size_t used = 0;
    void* take(int64_t bytes) {
        void* r = p ? p + used : nullptr;
        used += (size_t)up256(bytes);
        return r;
    }
};

#define M3_TRY(e)                       \
    do {                                \
        const int st_ = (e);            \
        if (st_ != M3_OK) return st_;   \
    } while (0)

// Launches k over the items of a group: as many blocks as run at once, each takes every grid-th item.
template <typename Tile, int kN, typename... Rest>
int gemm_launch_group(void (*k)(GemmGroup<kN>, Rest...), GemmGroup<kN> g, const int64_t (&rows)[kN], const int64_t (&cols)[kN],
                      std::atomic<uint64_t>& done, hipStream_t stream, const Rest&... rest) {
    int64_t items = 0;
    for (int p = 0; p < kN; ++p) {
        g.first[p] = (int)items;
        g.a[p].tiles_m = (int)((rows[p] + Tile::BM - 1) / Tile::BM);
        g.a[p].tiles_n = (int)((cols[p] + Tile::BN - 1) / Tile::BN);
        items += (int64_t)g.a[p].tiles_m * g.a[p].tiles_n * g.a[p].splits;
        if (items > 0x3fffffff) return M3_ERR_UNSUPPORTED;
    }
    g.first[kN] = (int)items;
    // once for each device (a bit of `done`; devices past 63 set it every time)
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess) return M3_ERR_DEVICE;
    const uint64_t bit = dev < 63 ? (uint64_t)1 << dev : 0;
    if (!(done.load(std::memory_order_relaxed) & bit)) {
        if (hipFuncSetAttribute(reinterpret_cast<const void*>(k), hipFuncAttributeMaxDynamicSharedMemorySize, Tile::kLds) != hipSuccess)
            return M3_ERR_LAUNCH;
        done.fetch_or(bit, std::memory_order_relaxed);
    }
    constexpr int64_t kAtOnce = 256 * (Tile::NT >= 512 ? 1 : 2);
    hipLaunchKernelGGL(k, dim3((unsigned)std::min(items, kAtOnce)), dim3(Tile::NT), Tile::kLds, stream, g, rest...);
    return hipGetLastError() == hipSuccess ? M3_OK : M3_ERR_LAUNCH;
}

template <typename T, typename Tile, bool kAKc, bool kBKc, int kMode, typename Epi>
int gemm_launch(const GemmArgs& a, const Epi& epi, int64_t rows, int64_t cols, hipStream_t stream) {
    static std::atomic<uint64_t> done{0};
    GemmGroup<1> g;
    g.a[0] = a;
    return gemm_launch_group<Tile, 1, Epi>(gemm_kernel<T, Tile, kAKc, kBKc, kMode, Epi>, g, {rows}, {cols}, done, stream, epi);
}

template <bool kAKc, bool kBKc, int kMode, typename Epi>
int gemm_dispatch(int dtype, const GemmPlan& p, const GemmArgs& a, const Epi& epi, int64_t rows, int64_t cols,
                  hipStream_t stream) {
    if (dtype == M3_DTYPE_BF16) {
        if (p.tile == kTileL) return gemm_launch<bf16, TileL, kAKc, kBKc, kMode>(a, epi, rows, cols, stream);
        if (p.tile == kTileM) return gemm_launch<bf16, TileM<bf16>, kAKc, kBKc, kMode>(a, epi, rows, cols, stream);
        return gemm_launch<bf16, TileS, kAKc, kBKc, kMode>(a, epi, rows, cols, stream);
    }
    if (p.tile == kTileM) return gemm_launch<float, TileM<float>, kAKc, kBKc, kMode>(a, epi, rows, cols, stream);
    return gemm_launch<float, TileS, kAKc, kBKc, kMode>(a, epi, rows, cols, stream);
}

// Stores a product (m3_gemm_store.hip): out (rows x cols, row stride ldo) = alpha * num / den * (A B)
// [+ res], or, split or accumulated over calls, fp32 partial sums in `part` that gemm_reduce joins.
struct GemmStore {
    void* out;
    int64_t ldo;
    const void* res;  // rows x cols, row stride ldo, or nullptr
    float alpha;
    float* part;      // [splits][rows][cols]
    int add;          // the partial sums of an earlier call stay in `part`
    int rows, cols;
    const float *num = nullptr, *den = nullptr;  // on the device: a factor num / den (0 where den is 0)
    int splits = 1;
};
// x W^T: A and B rows of k
int gemm_store(int dtype, const GemmPlan& p, GemmArgs a, GemmStore st, hipStream_t stream);
// Gradient products of one launch: the first (which may be left out, rows 0) dy W, A rows of k and B
// [k][n], of one or two terms; up to three dy^T x, A [k][m] and B [k][n]. A product whose `out` is nullptr
// leaves its partial sums; the others' are joined here.
struct GemmGrads {
    GemmArgs a[kGroupMax];
    GemmStore st[kGroupMax];
    int n = 1;  // entry 0 is dy W's
    GemmGrads() {
        for (int p = 0; p < kGroupMax; ++p) {
            a[p] = GemmArgs{};
            st[p] = GemmStore{};
        }
    }
};
int gemm_grads(int dtype, const GemmGroupPlan& plan, GemmGrads g, hipStream_t stream);
// out = alpha * num / den * sum over s of part[s] [+ res], for each entry with an `out` and parts
int gemm_reduce(int dtype, const GemmStore* st, int n, hipStream_t stream);
inline size_t gemm_part_bytes(int splits, int64_t rows, int64_t cols) {
    return splits > 1 ? (size_t)up256((int64_t)splits * rows * cols * 4) : 0;
}
// dst [rows][ldd] = src [rows][cols] with zeros in the columns past cols, for up to kPadCopies arrays in
// one launch; rows whose target is `ignore` are zero where a target is given. ldd * size is a
// multiple of 16.
constexpr int kPadCopies = 5;
struct GemmPad {
    const void* src;
    void* dst;
    int64_t rows;
    int cols, ldd;
};
struct GemmPads {
    GemmPad p[kPadCopies];
    int64_t first[kPadCopies + 1];  // first 16-byte piece of each in a row of all pieces
    int n = 0;
    void add(int dtype, const void* src, void* dst, int64_t rows, int64_t cols, int64_t ldd) {
        p[n] = GemmPad{src, dst, rows, (int)cols, (int)ldd};
        first[0] = 0;
        first[n + 1] = first[n] + rows * (ldd / (dtype == M3_DTYPE_BF16 ? 8 : 4));
        ++n;
    }
};
int gemm_pad_copy(int dtype, const GemmPads& pads, const int64_t* target, int64_t ignore, hipStream_t stream);

inline GemmArgs gemm_args(GemmOp a, GemmOp b, int64_t m, int64_t n, int64_t k, int splits) {
    GemmArgs g;
    g.a[0] = g.a[1] = a;
    g.b[0] = g.b[1] = b;
    g.M = (int)m, g.N = (int)n;
    g.K[0] = g.KB[0] = (int)k;
    g.K[1] = g.KB[1] = 0;
    g.splits = splits;
    g.tiles_m = g.tiles_n = 0;
    return g;
}

}  // namespace m3
