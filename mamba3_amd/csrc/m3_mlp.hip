// The gated MLP of a residual block and its backward (gfx950):
//   g = x Wg^T, u = x Wu^T, h = silu(g) * u, y = [res +] s (h Wd^T)
//   dh = s dy Wd, du = dh silu(g), dg = dh u silu'(g), silu'(g) = sig(g) (1 + g (1 - sig(g)))
//   dx = dg Wg + du Wu, dWg = dg^T x, dWu = du^T x, dWd = s dy^T h
// on the tiled products of m3_gemm.h. Both projections, the activation and the product are one
// kernel: a tile holds the gate and the up columns of the same hidden units, so g and u meet in
// a lane's registers in fp32 and only h is stored. The backward's dh is never stored either: its
// epilogue reads g and u and writes dg and du, the operands of the four gradient products, which
// are one launch (dx is one product of two terms).
//
// Measured, bf16, 8192 rows, d 768, ff 2112 (forward + backward 347 - 362 us, 239 GFLOP): gated product 75 us,
// down 48, dh 67, gradients 149 and their sums 12; d 2048, ff 5504 (1.47 - 1.53 ms, 1,110 TF/s): 333, 167, 229, 757
// and 27. Bound by the MFMAs; the small size by 4.1 and 2.1 rounds of tiles that take 5 and 3, and by the kept
// values' bytes next to twelve k steps a tile.
//
// For the backward the forward keeps g and u. bf16: rounded to 24 bits (the upper 16 of each, and the
// next 8 of both in another 16), a relative 2^-16: a bf16 copy alone would put a rounding
// of g and one of u (2^-8 each) into dg and du next to their own; 24 bits cost 2 more
// bytes an element. fp32: as they are.
#include "m3_gemm_host.h"
#include "m3_kernels.h"

namespace m3 {

typedef unsigned short u16x4 __attribute__((ext_vector_type(4)));
typedef unsigned short u16x8 __attribute__((ext_vector_type(8)));

template <typename T> __device__ __forceinline__ float sigmoid_of(float g);
template <> __device__ __forceinline__ float sigmoid_of<bf16>(float g) { return __builtin_amdgcn_rcpf(1.f + fast_exp(-g)); }
template <> __device__ __forceinline__ float sigmoid_of<float>(float g) { return sigmoid_f(g); }

// Where g and u of four columns n .. n + 3 of row m are kept: blocks of 16 x 16 elements in a row of
// blocks, in a block the fours of 16 rows side by side for each four columns. The 16 lanes that
// hold the same columns of a piece (m3_gemm.h) then write and read a contiguous run, where rows
// would take 8 bytes of each of 16 rows.
struct KeptGu {
    void* p;
    int64_t elements;  // rows and columns rounded up to 16
    int blocks;        // a row of blocks
    __device__ __forceinline__ int64_t at(int m, int n) const {
        return ((int64_t)(m >> 4) * blocks + (n >> 4)) * 256 + ((n & 15) >> 2) * 64 + (m & 15) * 4;
    }
};

// A float's bits, to be cut to the upper 24: rounded to the nearest (ties away from zero; past the largest, to
// infinity). Infinities stay, and NaNs: of bf16 operands they have zeros in their low bits.
__device__ __forceinline__ unsigned round24(float v) { return __builtin_bit_cast(unsigned, v) + 0x80; }

// bf16: [element fours][g upper 16 x 4, u upper 16 x 4], then [element fours][the next 8 of both x 4].
// fp32: g, then u.
template <typename T>
__device__ __forceinline__ void keep_gu(const KeptGu& k, int64_t at, f32x4 g, f32x4 u) {
    if constexpr (sizeof(T) == 2) {
        u16x8 hi;
        u16x4 lo;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            // (__builtin_bit_cast of a vector's component takes component 0 on this compiler)
            const float ge = g[e], ue = u[e];
            const unsigned gb = round24(ge), ub = round24(ue);
            hi[e] = (unsigned short)(gb >> 16);
            hi[4 + e] = (unsigned short)(ub >> 16);
            lo[e] = (unsigned short)((gb >> 8 & 0xff) | (ub & 0xff00));
        }
        unsigned short* p = reinterpret_cast<unsigned short*>(k.p);
        *reinterpret_cast<u16x8*>(p + 2 * at) = hi;
        *reinterpret_cast<u16x4*>(p + 2 * k.elements + at) = lo;
    } else {
        float* p = reinterpret_cast<float*>(k.p) + at;
        *reinterpret_cast<f32x4*>(p) = g;
        *reinterpret_cast<f32x4*>(p + k.elements) = u;
    }
}

template <typename T>
struct KeptFour {
    u16x8 hi;
    u16x4 lo;
    f32x4 g, u;
    __device__ __forceinline__ void load(const KeptGu& k, int64_t at) {
        if constexpr (sizeof(T) == 2) {
            const unsigned short* p = reinterpret_cast<const unsigned short*>(k.p);
            hi = *reinterpret_cast<const u16x8*>(p + 2 * at);
            lo = *reinterpret_cast<const u16x4*>(p + 2 * k.elements + at);
        } else {
            const float* p = reinterpret_cast<const float*>(k.p) + at;
            g = *reinterpret_cast<const f32x4*>(p);
            u = *reinterpret_cast<const f32x4*>(p + k.elements);
        }
    }
    __device__ __forceinline__ void get(int e, float& ge, float& ue) const {
        if constexpr (sizeof(T) == 2) {
            ge = __builtin_bit_cast(float, (unsigned)hi[e] << 16 | (lo[e] & 0xffu) << 8);
            ue = __builtin_bit_cast(float, (unsigned)hi[4 + e] << 16 | (lo[e] & 0xff00u));
        } else {
            ge = g[e];
            ue = u[e];
        }
    }
};

// Columns come in whole 16-byte pieces: the hidden width is padded to 16 bytes, its pad columns are
// zero (their weight rows read as zero) and are stored as zeros.
struct EpiGated {
    void* h;      // rows x ldh
    KeptGu kept;  // p nullptr: no backward
    int rows, ldh;

    template <typename T, typename Tile, int kMode>
    __device__ __forceinline__ void run(const GemmPlace<Tile, kMode>& at,
                                        typename Tile::Acc (&acc)[Tile::FM][Tile::FN], char* smem, const GemmItem&) const {
        GemmRows<T, Tile, Tile::FN / 2 * Tile::MF> out(smem, at.wave(), at.lane);
#pragma unroll
        for (int i = 0; i < Tile::FM; ++i) {
            const int m = at.m(i), r0 = at.row0(i), c0 = at.col0();
            out.begin(reinterpret_cast<T*>(h) + (int64_t)r0 * ldh + c0, ldh, rows - r0, ldh - c0);
#pragma unroll
            for (int jq = 0; jq < Tile::FN / 2 * Tile::Q; ++jq) {
                const int j = jq / Tile::Q, q = jq % Tile::Q;
                const int n = at.n(j, q);
                const f32x4 g = four(acc[i][j], q), u = four(acc[i][j + Tile::FN / 2], q);
                f32x4 v;
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = g[e] * sigmoid_of<T>(g[e]) * u[e];
                out.put(j, q, v);
                if (kept.p && m < rows && n < ldh) keep_gu<T>(kept, kept.at(m, n), g, u);
            }
            out.store();
        }
    }
};

struct EpiGateBwd {
    void *dg, *du;
    KeptGu kept;
    float alpha;
    int rows, ldh;

    template <typename T, typename Tile, int kMode>
    __device__ __forceinline__ void run(const GemmPlace<Tile, kMode>& at,
                                        typename Tile::Acc (&acc)[Tile::FM][Tile::FN], char* smem, const GemmItem&) const {
        constexpr int J = Tile::FN * Tile::Q;
        GemmRows<T, Tile, Tile::FN * Tile::MF> out(smem, at.wave(), at.lane);
        // the kept values of a piece's row are fetched while the one before is worked on
        KeptFour<T> k[2][J];
        auto fetch = [&](int i) {
            const int m = at.m(i) < rows ? at.m(i) : rows - 1;
#pragma unroll
            for (int jq = 0; jq < J; ++jq) {
                const int n = at.n(jq / Tile::Q, jq % Tile::Q);
                k[i & 1][jq].load(kept, kept.at(m, n < ldh ? n : 0));
            }
        };
        fetch(0);
#pragma unroll
        for (int i = 0; i < Tile::FM; ++i) {
            const int r0 = at.row0(i), c0 = at.col0();
            const int64_t o = (int64_t)r0 * ldh + c0;
            if (i + 1 < Tile::FM) fetch(i + 1);
            out.begin(reinterpret_cast<T*>(dg) + o, ldh, rows - r0, ldh - c0);
            f32x4 b[J];
#pragma unroll
            for (int jq = 0; jq < J; ++jq) {
                const f32x4 v = four(acc[i][jq / Tile::Q], jq % Tile::Q);
                f32x4 a;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float g, u;
                    k[i & 1][jq].get(e, g, u);
                    const float s = sigmoid_of<T>(g), dh = v[e] * alpha;
                    // s, which is 0 for far gates, meets each large factor before they meet one another
                    a[e] = dh * (u * (s * (1.f + g * (1.f - s))));
                    b[jq][e] = dh * (g * s);
                }
                out.put(jq / Tile::Q, jq % Tile::Q, a);
            }
            out.store();
            out.begin(reinterpret_cast<T*>(du) + o, ldh, rows - r0, ldh - c0);
#pragma unroll
            for (int jq = 0; jq < J; ++jq) out.put(jq / Tile::Q, jq % Tile::Q, b[jq]);
            out.store();
        }
    }
};

namespace {

struct MlpShape {
    int64_t rows, d, ff, dp, fp;
    int dtype;
    int64_t size;
    bool pad_d, pad_f;  // rows of d (ff) are not whole 16-byte pieces
};
MlpShape mlp_shape(int64_t rows, int64_t d, int64_t ff, int dtype) {
    MlpShape s{rows, d, ff, gemm_pad(d, dtype), gemm_pad(ff, dtype), dtype, dtype == M3_DTYPE_BF16 ? 2 : 4, false, false};
    s.pad_d = s.dp != d, s.pad_f = s.fp != ff;
    return s;
}

struct MlpFwd {
    GemmPlan up, down;
    void *x, *wg, *wu, *wd, *h;
    float* part;
    size_t bytes;
};
MlpFwd mlp_fwd_layout(const MlpShape& s, bool keeps_h, void* ws) {
    MlpFwd f;
    Bump b{reinterpret_cast<char*>(ws)};
    f.up = gemm_plan(s.dtype, s.rows, 2 * s.ff, gemm_steps(s.d, s.dtype), 1);
    f.down = gemm_plan(s.dtype, s.rows, s.d, gemm_steps(s.ff, s.dtype), kMaxSplits);
    f.x = s.pad_d ? b.take(s.rows * s.dp * s.size) : nullptr;
    f.wg = s.pad_d ? b.take(s.ff * s.dp * s.size) : nullptr;
    f.wu = s.pad_d ? b.take(s.ff * s.dp * s.size) : nullptr;
    f.wd = s.pad_f ? b.take(s.d * s.fp * s.size) : nullptr;
    f.h = keeps_h ? nullptr : b.take(s.rows * s.fp * s.size);
    f.part = reinterpret_cast<float*>(b.take((int64_t)gemm_part_bytes(f.down.splits, s.rows, s.d)));
    f.bytes = b.used;
    return f;
}

// What the backward computes, in the order of the grouped launch.
enum { kDx, kDwGate, kDwUp, kDwDown };
struct MlpBwd {
    GemmPlan dh;
    GemmGroupPlan grads;
    void *x, *dy, *wg, *wu, *wd, *dg, *du;
    float* part[kGroupMax];
    size_t bytes;
};
MlpBwd mlp_bwd_layout(const MlpShape& s, void* ws) {
    MlpBwd f;
    Bump b{reinterpret_cast<char*>(ws)};
    f.dh = gemm_plan(s.dtype, s.rows, s.ff, gemm_steps(s.d, s.dtype), 1);
    const int64_t over_rows = gemm_steps(s.rows, s.dtype);
    const GemmTask tasks[kGroupMax] = {{s.rows, s.d, 2 * gemm_steps(s.fp, s.dtype), kMaxSplits, false},
                                       {s.ff, s.d, over_rows, kMaxSplits, true},
                                       {s.ff, s.d, over_rows, kMaxSplits, true},
                                       {s.d, s.ff, over_rows, kMaxSplits, true}};
    f.grads = gemm_group_plan(s.dtype, tasks, kGroupMax);
    f.x = s.pad_d ? b.take(s.rows * s.dp * s.size) : nullptr;
    f.dy = s.pad_d ? b.take(s.rows * s.dp * s.size) : nullptr;
    f.wg = s.pad_d ? b.take(s.ff * s.dp * s.size) : nullptr;
    f.wu = s.pad_d ? b.take(s.ff * s.dp * s.size) : nullptr;
    f.wd = s.pad_f ? b.take(s.d * s.fp * s.size) : nullptr;
    f.dg = b.take(s.rows * s.fp * s.size);
    f.du = b.take(s.rows * s.fp * s.size);
    for (int p = 0; p < kGroupMax; ++p)
        f.part[p] = reinterpret_cast<float*>(b.take((int64_t)gemm_part_bytes(f.grads.splits[p], tasks[p].rows, tasks[p].cols)));
    f.bytes = b.used;
    return f;
}

// h behind what is kept of g and u
KeptGu kept_gu(const MlpShape& s, const void* saved) {
    const int64_t blocks = (s.fp + 15) / 16, rows = (s.rows + 15) / 16 * 16;
    return KeptGu{const_cast<void*>(saved), rows * blocks * 16, (int)blocks};
}
int64_t gu_bytes(const MlpShape& s) { return up256(kept_gu(s, nullptr).elements * (s.dtype == M3_DTYPE_BF16 ? 6 : 8)); }

// src as it is, or its padded copy, which `pads` will make
const void* padded(const MlpShape& s, GemmPads& pads, const void* src, void* dst, int64_t rows, int64_t cols, int64_t ldd) {
    if (!dst) return src;
    pads.add(s.dtype, src, dst, rows, cols, ldd);
    return dst;
}

}  // namespace

size_t swiglu_saved(int64_t rows, int64_t d, int64_t ff, int dtype) {
    const MlpShape s = mlp_shape(rows, d, ff, dtype);
    return (size_t)(gu_bytes(s) + up256(rows * s.fp * s.size));
}
size_t swiglu_fwd_workspace(int64_t rows, int64_t d, int64_t ff, int dtype, bool keeps) {
    return mlp_fwd_layout(mlp_shape(rows, d, ff, dtype), keeps, nullptr).bytes;
}
size_t swiglu_bwd_workspace(int64_t rows, int64_t d, int64_t ff, int dtype) {
    return mlp_bwd_layout(mlp_shape(rows, d, ff, dtype), nullptr).bytes;
}

int launch_swiglu_fwd(int64_t rows, int64_t d, int64_t ff, int dtype, const void* x, const void* wg, const void* wu,
                      const void* wd, const void* res, float scale, void* y, void* saved, void* ws,
                      hipStream_t stream) {
    const MlpShape s = mlp_shape(rows, d, ff, dtype);
    const MlpFwd f = mlp_fwd_layout(s, saved != nullptr, ws);
    GemmPads pads;
    x = padded(s, pads, x, f.x, rows, d, s.dp);
    wg = padded(s, pads, wg, f.wg, ff, d, s.dp);
    wu = padded(s, pads, wu, f.wu, ff, d, s.dp);
    wd = padded(s, pads, wd, f.wd, d, ff, s.fp);
    M3_TRY(gemm_pad_copy(dtype, pads, nullptr, 0, stream));
    void* h = saved ? reinterpret_cast<char*>(saved) + gu_bytes(s) : f.h;
    GemmArgs a = gemm_args({x, s.dp}, {wg, s.dp}, rows, ff, s.dp, 1);
    a.b[1] = {wu, s.dp};
    M3_TRY((gemm_dispatch<true, true, kGated>(dtype, f.up, a, EpiGated{h, kept_gu(s, saved), (int)rows, (int)s.fp}, rows, 2 * s.fp, stream)));
    const GemmStore st{y, d, res, scale, f.part, 0, (int)rows, (int)d};
    return gemm_store(dtype, f.down, gemm_args({h, s.fp}, {wd, s.fp}, rows, d, s.fp, 1), st, stream);
}

int launch_swiglu_bwd(int64_t rows, int64_t d, int64_t ff, int dtype, const void* x, const void* wg, const void* wu,
                      const void* wd, float scale, const void* saved, const void* dy, void* dx, void* dwg, void* dwu,
                      void* dwd, void* ws, hipStream_t stream) {
    const MlpShape s = mlp_shape(rows, d, ff, dtype);
    const MlpBwd f = mlp_bwd_layout(s, ws);
    const void* h = reinterpret_cast<const char*>(saved) + gu_bytes(s);
    const bool gates = dx || dwg || dwu;
    GemmPads pads;
    dy = padded(s, pads, dy, f.dy, rows, d, s.dp);
    if (gates) wd = padded(s, pads, wd, f.wd, d, ff, s.fp);
    if (dx) {
        wg = padded(s, pads, wg, f.wg, ff, d, s.dp);
        wu = padded(s, pads, wu, f.wu, ff, d, s.dp);
    }
    if (dwg || dwu) x = padded(s, pads, x, f.x, rows, d, s.dp);
    M3_TRY(gemm_pad_copy(dtype, pads, nullptr, 0, stream));
    if (gates) {
        // rows of Wd past d do not exist: A's pad columns meet zeros
        GemmArgs a = gemm_args({dy, s.dp}, {wd, s.fp}, rows, s.fp, s.dp, 1);
        a.KB[0] = (int)d;
        M3_TRY((gemm_dispatch<true, false, kPlain>(dtype, f.dh, a, EpiGateBwd{f.dg, f.du, kept_gu(s, saved), scale, (int)rows, (int)s.fp}, rows, s.fp, stream)));
    }
    // a gradient that is not wanted has no rows, and no items
    GemmGrads g;
    if (dx) {
        g.a[kDx] = gemm_args({f.dg, s.fp}, {wg, s.dp}, rows, s.dp, s.fp, 1);
        g.a[kDx].a[1] = {f.du, s.fp}, g.a[kDx].b[1] = {wu, s.dp};
        g.a[kDx].K[1] = (int)s.fp;
        g.a[kDx].KB[0] = g.a[kDx].KB[1] = (int)ff;
        g.st[kDx] = GemmStore{dx, d, nullptr, 1.f, f.part[kDx], 0, (int)rows, (int)d};
    }
    if (dwg) {
        g.a[kDwGate] = gemm_args({f.dg, s.fp}, {x, s.dp}, s.fp, s.dp, rows, 1);
        g.st[kDwGate] = GemmStore{dwg, d, nullptr, 1.f, f.part[kDwGate], 0, (int)ff, (int)d};
    }
    if (dwu) {
        g.a[kDwUp] = gemm_args({f.du, s.fp}, {x, s.dp}, s.fp, s.dp, rows, 1);
        g.st[kDwUp] = GemmStore{dwu, d, nullptr, 1.f, f.part[kDwUp], 0, (int)ff, (int)d};
    }
    if (dwd) {
        g.a[kDwDown] = gemm_args({dy, s.dp}, {h, s.fp}, s.dp, s.fp, rows, 1);
        g.st[kDwDown] = GemmStore{dwd, ff, nullptr, scale, f.part[kDwDown], 0, (int)d, (int)ff};
    }
    return gates || dwd ? gemm_grads(dtype, f.grads, g, stream) : M3_OK;
}

}  // namespace m3
