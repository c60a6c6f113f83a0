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

template <int kN>
__device__ __forceinline__ GemmStore pick_store(const GemmStore (&v)[kN], int p) {
    if constexpr (kN == 1) {
        return v[0];
    } else {
        GemmStore r;
        M3_PICK(r, v, p, out);
        M3_PICK(r, v, p, ldo);
        M3_PICK(r, v, p, res);
        M3_PICK(r, v, p, alpha);
        M3_PICK(r, v, p, part);
        M3_PICK(r, v, p, add);
        M3_PICK(r, v, p, rows);
        M3_PICK(r, v, p, cols);
        M3_PICK(r, v, p, num);
        M3_PICK(r, v, p, den);
        M3_PICK(r, v, p, splits);
        return r;
    }
}

// alpha with the factor that lies on the device
__device__ __forceinline__ float store_scale(const GemmStore& s) {
    float f = s.alpha;
    if (s.num) f *= s.num[0];
    if (s.den) f = s.den[0] == 0.f ? 0.f : f / s.den[0];
    return f;
}

template <int kN>
struct EpiStore {
    GemmStore st[kN];
    bool whole[kN];  // results come in whole, aligned 16-byte pieces

    template <typename T, typename Tile, int kMode>
    __device__ __forceinline__ void run(const GemmPlace<Tile, kMode>& at, typename Tile::Acc (&acc)[Tile::FM][Tile::FN],
                                        char* smem, const GemmItem& it) const {
        const GemmStore s = pick_store(st, it.prob);
        bool vec;
        if constexpr (kN == 1) vec = whole[0];
        else vec = pick4(it.prob, whole[0], whole[1], whole[2], whole[3]);
        T* out = reinterpret_cast<T*>(s.out);
        const T* res = reinterpret_cast<const T*>(s.res);
        const float alpha = s.part ? 1.f : store_scale(s);
        if (s.part) {
            float* part = s.part + (int64_t)it.split * s.rows * s.cols;
            each(s, at, acc, [&](int m, int n, f32x4 v) {
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
            GemmRows<T, Tile, Tile::FN * Tile::MF> rows(smem, at.wave(), at.lane);
#pragma unroll
            for (int i = 0; i < Tile::FM; ++i) {
                const int m = at.m(i), r0 = at.row0(i), c0 = at.col0();
                rows.begin(out + (int64_t)r0 * s.ldo + c0, s.ldo, s.rows - r0, s.cols - c0);
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
                rows.store();
            }
        } else {
            each(s, at, acc, [&](int m, int n, f32x4 v) {
                const int64_t o = (int64_t)m * s.ldo + n;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (n + e < s.cols) out[o + e] = (T)(v[e] * alpha + (res ? (float)res[o + e] : 0.f));
            });
        }
    }

    // f(m, n, four) for the fours that begin inside the result
    template <typename Place, typename Acc, int FM, int FN, typename F>
    static __device__ __forceinline__ void each(const GemmStore& s, const Place& at, Acc (&acc)[FM][FN], F f) {
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
    return s.cols % e == 0 && s.ldo % e == 0 && al(s.out) && al(s.res);
}

// Where one part of a whole result goes: straight to `out`, unless sums are kept or joined.
static void direct(GemmStore& st) {
    if (st.splits == 1 && !st.add && st.out) st.part = nullptr;
}

int gemm_store(int dtype, const GemmPlan& p, GemmArgs a, GemmStore st, hipStream_t stream) {
    a.splits = st.splits = p.splits;
    EpiStore<1> e{{st}, {whole_pieces(dtype, st)}};
    direct(e.st[0]);
    const int r = gemm_dispatch<true, true, kPlain>(dtype, p, a, e, st.rows, st.cols, stream);
    if (r != M3_OK || !e.st[0].part) return r;
    return gemm_reduce(dtype, &st, 1, stream);
}

template <typename T, typename Tile>
__global__ __launch_bounds__(Tile::NT, 2) void gemm_grads_kernel(GemmGroup<kGroupMax> grp, EpiStore<kGroupMax> epi) {
    gemm_run<T, Tile, true, false, kSeg2, 0, 1>(grp, epi);
    gemm_run<T, Tile, false, false, kPlain, 1, kGroupMax>(grp, epi);
}

template <typename T, typename Tile>
static int launch_grads(const GemmGroup<kGroupMax>& grp, const EpiStore<kGroupMax>& e, hipStream_t stream) {
    static std::atomic<uint64_t> done{0};
    int64_t rows[kGroupMax], cols[kGroupMax];
    for (int p = 0; p < kGroupMax; ++p) rows[p] = e.st[p].rows, cols[p] = e.st[p].cols;
    return gemm_launch_group<Tile, kGroupMax, EpiStore<kGroupMax>>(gemm_grads_kernel<T, Tile>, grp, rows, cols, done, stream, e);
}

// The products share one launch: what one of them leaves of the last round of tiles the next one takes,
// and there is one reduction. The four products of 8192 x 768 x 2112 take 192 us apart and 161 together,
// with their reductions (12 us): 133 GFLOP at 890 TF/s in the products' launch; of 8192 x 2048 x 5504
// 757 us, 1,220 TF/s. Bound by the MFMAs, and at the smaller size by the parts of k, whose fp32 sums are
// written and read.
int gemm_grads(int dtype, const GemmGroupPlan& plan, GemmGrads g, hipStream_t stream) {
    GemmGroup<kGroupMax> grp;
    EpiStore<kGroupMax> e;
    bool join = false;
    for (int p = 0; p < kGroupMax; ++p) {
        g.st[p].splits = plan.splits[p];
        grp.a[p] = g.a[p];
        grp.a[p].splits = plan.splits[p];
        e.st[p] = g.st[p];
        e.whole[p] = whole_pieces(dtype, g.st[p]);
        direct(e.st[p]);
        join = join || (e.st[p].part && e.st[p].out && e.st[p].rows);
        if (!e.st[p].part) g.st[p].part = nullptr;
    }
    int r;
    if (dtype == M3_DTYPE_BF16) {
        r = plan.tile == kTileL   ? launch_grads<bf16, TileL>(grp, e, stream)
            : plan.tile == kTileM ? launch_grads<bf16, TileM<bf16>>(grp, e, stream)
                                  : launch_grads<bf16, TileS>(grp, e, stream);
    } else {
        r = plan.tile == kTileM ? launch_grads<float, TileM<float>>(grp, e, stream) : launch_grads<float, TileS>(grp, e, stream);
    }
    return r != M3_OK || !join ? r : gemm_reduce(dtype, g.st, kGroupMax, stream);
}

struct GemmReduce {
    GemmStore st[kGroupMax];
    bool whole[kGroupMax];
};

// One thread joins four columns of a row (or one element); parts are added in order. A grid row for each
// result. Bound by the parts' read: 27 us for two parts of 16128 x 768 sums (99 MB, 25 MB written: 4.6 TB/s).
template <typename T>
__global__ __launch_bounds__(256) void gemm_reduce_kernel(GemmReduce r) {
    const GemmStore s = pick_store(r.st, (int)blockIdx.y);
    if (!s.part || !s.out) return;
    const bool vec = pick4((int)blockIdx.y, r.whole[0], r.whole[1], r.whole[2], r.whole[3]);
    const int64_t each = (int64_t)s.rows * s.cols;
    T* out = reinterpret_cast<T*>(s.out);
    const T* res = reinterpret_cast<const T*>(s.res);
    const float alpha = store_scale(s);
    const int64_t pieces = vec ? each / 4 : each;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < pieces; i += (int64_t)gridDim.x * 256) {
        const int64_t at = vec ? i * 4 : i;
        const int64_t m = at / s.cols, o = m * s.ldo + (at - m * s.cols);
        if (vec) {
            f32x4 v{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
            for (int k = 0; k < s.splits; ++k) v += *reinterpret_cast<const f32x4*>(s.part + k * each + at);
            v *= alpha;
            if (res)
                for (int e = 0; e < 4; ++e) v[e] += (float)res[o + e];
            store4(out + o, v);
        } else {
            float v = 0.f;
            for (int k = 0; k < s.splits; ++k) v += s.part[k * each + at];
            out[o] = (T)(v * alpha + (res ? (float)res[o] : 0.f));
        }
    }
}

int gemm_reduce(int dtype, const GemmStore* st, int n, hipStream_t stream) {
    GemmReduce r;
    int64_t most = 0;
    for (int p = 0; p < kGroupMax; ++p) {
        r.st[p] = p < n ? st[p] : GemmStore{};
        r.whole[p] = whole_pieces(dtype, r.st[p]);
        if (r.st[p].part && r.st[p].out)
            most = std::max(most, (int64_t)r.st[p].rows * r.st[p].cols / (r.whole[p] ? 4 : 1));
    }
    if (most == 0) return M3_OK;
    const dim3 grid((unsigned)std::min<int64_t>((most + 255) / 256, 8192), (unsigned)n);
    if (dtype == M3_DTYPE_BF16) hipLaunchKernelGGL(gemm_reduce_kernel<bf16>, grid, dim3(256), 0, stream, r);
    else hipLaunchKernelGGL(gemm_reduce_kernel<float>, grid, dim3(256), 0, stream, r);
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

// A search takes 20 us of host time or more, and a call asks three times (the workspace's size, its check, the
// launch): each thread keeps its last plans, in any of four places that follow a hash of their tasks.
template <typename Plan, typename F>
static const Plan& kept_plan(int dtype, const GemmTask* tasks, int n, F search) {
    struct Kept {
        int dtype = -1, n = 0;
        GemmTask t[kGroupMax];
        Plan plan;
    };
    static thread_local Kept kept[64];
    static thread_local unsigned turn = 0;
    uint64_t h = (uint64_t)dtype * 31 + (uint64_t)n;
    for (int p = 0; p < n; ++p)
        h = (h * 0x9e3779b97f4a7c15ull + (uint64_t)tasks[p].rows * 3 + (uint64_t)tasks[p].cols * 5 + (uint64_t)tasks[p].steps * 7) ^ (h >> 29);
    auto same = [](const GemmTask& a, const GemmTask& b) {
        return a.rows == b.rows && a.cols == b.cols && a.steps == b.steps && a.max_splits == b.max_splits && a.tn == b.tn;
    };
    Kept* at = nullptr;
    for (unsigned i = 0; i < 4; ++i) {
        Kept& k = kept[((h >> 58) + i) & 63];
        bool hit = k.dtype == dtype && k.n == n;
        for (int p = 0; hit && p < n; ++p) hit = same(k.t[p], tasks[p]);
        if (hit) return k.plan;
        if (!at && k.n == 0) at = &k;
    }
    if (!at) at = &kept[((h >> 58) + turn++ % 4) & 63];
    at->plan = search();
    at->dtype = dtype, at->n = n;
    for (int p = 0; p < n; ++p) at->t[p] = tasks[p];
    return at->plan;
}

GemmGroupPlan gemm_group_plan(int dtype, const GemmTask* tasks, int n) {
    return kept_plan<GemmGroupPlan>(dtype, tasks, n, [&] { return search_plan(dtype == M3_DTYPE_BF16, tasks, n); });
}

GemmPairPlan gemm_pair_plan(int dtype, const GemmTask (&tasks)[2]) {
    return kept_plan<GemmPairPlan>(dtype, tasks, 2, [&] {
        return pair_plan(tasks, [&](const GemmTask (&t)[2]) { return search_plan(dtype == M3_DTYPE_BF16, t, 2); });
    });
}

GemmPlan gemm_plan(int dtype, int64_t rows, int64_t cols, int64_t steps, int max_splits) {
    const GemmTask t{rows, cols, steps, max_splits, false};
    const GemmGroupPlan g = gemm_group_plan(dtype, &t, 1);
    const int size = g.tile == kTileL ? 256 : g.tile == kTileM ? 128 : 64;
    return GemmPlan{g.tile, g.splits[0], size, size};
}

}  // namespace m3
