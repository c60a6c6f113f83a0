// The next token of each row of logits, from a given random number (gfx950):
//   mass(v) = exp((z_v - max z) / T);  tokens in the order of z, ties from the lowest index;
//   kept: the first k of them, of these the shortest run whose mass reaches p of the k's, and of these the
//   ones with mass >= m; token = the first whose running mass passes u times the kept mass.
// Every bound cuts the same order, so what is kept is a prefix, and each step is the question which
// token of the order a count or a mass falls on. It is answered without sorting the row. One block takes a row and holds
// its first 112 KB in LDS (the rest is read anew in each pass: 256 rows of 128000 fp32 logits come from the last-level
// cache). It finds the largest logit; adds up masses (and where top_k asks, counts) by distance from it, in 2048 bins
// of T / 64; narrows every answer to a few bins, since what lies before and in a bin bounds the mass that the next question takes
// its share of; gathers the tokens of all these bins in one pass, up to 1024, sorts them and reads the answers off. With
// more (equal logits, low temperatures), each question gathers the one bin that it falls in, which is split by its keys' bits
// until it fits.
// With q = 64 (max z - z) / T in 64 bits, a token's mass is exp(-b / 64) exp(-r / 64), b the bin and r < 1: the bins add up
// exp(-r / 64), five terms of its series to 2e-14, as whole numbers of 2^-45 (131072 tokens; 2^-51 to 2048, 2^-40 for 2^22), so that sums do not depend
// on their order; exp(-b / 64), of two table values, comes in once a bin. (An exponential for each token took three times as long.) What
// lies past the last bin but one, below exp(-32) of the likeliest, is counted but has no mass. A running mass of n tokens is off by
// about 2e-14 of itself and a quarter of sqrt(n) of these units (3e-12 of the likeliest's mass at 131072 tokens, to 2048 below 2e-14), where sums of
// 64-bit floating numbers would be off by about 1e-14 and depend on their order. That is how probable it is for a border that u falls
// on its other side.
// Bound by the reads and the bins' atomics for large batches (256 rows of 128000 fp32 logits, a setting for each row: 80 us, where one
// read of them takes 22; a row alone on its CU takes 50-60), by the chain of passes, barriers and first fetches of code for few
// (4 rows of 32000: 20-21 us, of which greedy choice and launch take 6). After the bins one wave does what is left but
// gathering and sorting: with all 16 and their barriers, and the library's exponential at each place that needs one, 23-26 us. 16 waves a
// block: with 8, which leaves the compiler more registers, the large case took 97 us for 78 (with four terms of the series).
#include <algorithm>
#include <atomic>

#include "m3_common.h"
#include "m3_kernels.h"
#include "m3_mx.h"
#include "mamba3_amd.h"

namespace m3 {

typedef unsigned long long u64;
constexpr int kSpThreads = 1024;
constexpr int kSpWaves = kSpThreads / 64;
constexpr int kSpBins = 2048;
constexpr double kSpPerT = 64.0;  // bins of T / 64
constexpr int kSpList = 1024;
constexpr int kSpShare = kSpBins / kSpWaves;  // a wave's bins
constexpr int kSpParts = 1024;  // of a bin's keys
constexpr int kSpHeld = 112 << 10;  // bytes of a row in LDS

struct SampleArgs {
    const void* z;
    const float* u;
    // a setting for each row, or one for all
    const float *temperature, *top_p, *min_p;
    const int32_t* top_k;
    double temperature1, top_p1, min_p1;
    int64_t top_k1;
    int64_t* token;
    float* logprob;
    int64_t rows;
    int vocab;
    int shift;  // masses are whole numbers of 2^-shift
};

// Logits as whole numbers that keep their order, -0 as 0.
__device__ __forceinline__ unsigned sp_key(float z) {
    const unsigned b = __builtin_bit_cast(unsigned, z + 0.f);
    return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float sp_logit(unsigned key) {
    return __builtin_bit_cast(float, key ^ ((key >> 31) ? 0x80000000u : 0xffffffffu));
}
constexpr unsigned kSpNone = 0x007fffffu;  // the key of -infinity

// Distances from the largest logit in bins, as 64-bit numbers (NaN for NaN).
struct SampleScale {
    double top, per;  // per = kSpPerT / T
    int shift;        // masses are whole numbers of 2^-shift
    __device__ __forceinline__ double far(float z) const { return (top - (double)z) * per; }
    // a logit at least as near as q, with room for rounding: what is below it is further
    __device__ __forceinline__ float near(double q) const {
        const double z = top - (q + 1e-6) / per;
        return (float)(z - fabs(z) * 1e-6);
    }
    // a logit at least as far as q: what is above it is nearer
    __device__ __forceinline__ float beyond(double q) const {
        const double z = top - (q - 1e-6) / per;
        return (float)(z + fabs(z) * 1e-6);
    }
};
__device__ __forceinline__ int sp_bin(double q) { return q < (double)(kSpBins - 1) ? (int)q : kSpBins - 1; }
__device__ __forceinline__ bool sp_in(double q, int bin) { return q >= (double)bin && (q < (double)(bin + 1) || bin == kSpBins - 1); }
constexpr double kSpWhole = 4503599627370496.0;  // 2^52: what is added to it is rounded to a whole number, in its low bits
__device__ __forceinline__ u64 sp_whole(double v) {  // of 0 <= v < 2^52
    return __builtin_bit_cast(u64, v + kSpWhole) & 0x000fffffffffffffull;
}
// exp(-i) and exp(-i / 64): a bin's mass is a product of two, and a token's that times five terms of exp(-d / 64)'s series for
// what it lies behind its bin's start (to 2e-14).
struct SampleTables {
    double whole[kSpBins / 64], part[64];
};
constexpr double sp_exp_of(double x) {  // Taylor's series for |x| <= 1
    double term = 1.0, sum = 1.0;
    for (int i = 1; i < 24; ++i) term *= x / i, sum += term;
    return sum;
}
constexpr SampleTables sp_tables() {
    SampleTables t{};
    for (int i = 0; i < kSpBins / 64; ++i) t.whole[i] = i == 0 ? 1.0 : t.whole[i - 1] * sp_exp_of(-1.0);
    for (int i = 0; i < 64; ++i) t.part[i] = sp_exp_of(-i / 64.0);
    return t;
}
__constant__ const SampleTables kSpTables = sp_tables();
__device__ __forceinline__ double sp_series(double d) {
    constexpr double c1 = -1.0 / kSpPerT, c2 = c1 * c1 / 2, c3 = c2 * c1 / 3, c4 = c3 * c1 / 4, c5 = c4 * c1 / 5;
    return fma(fma(fma(fma(fma(c5, d, c4), d, c3), d, c2), d, c1), d, 1.0);
}
__device__ __forceinline__ double sp_bin_mass(const SampleTables& t, int b) { return t.whole[b >> 6] * t.part[b & 63]; }
// A token's mass times 2^shift as a whole number (shift <= 51), none past the last bin but one.
__device__ __forceinline__ u64 sp_mass(const SampleTables& t, const SampleScale& s, float z) {
    const double q = s.far(z);
    if (!(q < (double)(kSpBins - 1))) return 0;
    const int b = (int)q;
    return sp_whole(ldexp(sp_bin_mass(t, b) * sp_series(q - (double)b), s.shift));
}

struct SampleRow {
    double t, p, m;
    int64_t k;
};
__device__ __forceinline__ SampleRow sp_row(const SampleArgs& a, int64_t row) {
    SampleRow r;
    r.t = a.temperature ? (double)a.temperature[row] : a.temperature1;
    r.p = a.top_p ? (double)a.top_p[row] : a.top_p1;
    r.m = a.min_p ? (double)a.min_p[row] : a.min_p1;
    r.k = a.top_k ? (int64_t)a.top_k[row] : a.top_k1;
    if (r.k <= 0 || r.k > a.vocab) r.k = a.vocab;
    return r;
}

// A row's logits, in pieces of 16 bytes: the first `held` in LDS, the others in memory.
template <typename T>
struct SampleLogits {
    static constexpr int E = 16 / sizeof(T);
    u32x4* lds;
    const T* z;
    int vocab, held;

    static __device__ __forceinline__ float get(const u32x4& w, int e) {
        // (a bit cast of the vector's component itself takes the first one with this compiler)
        const unsigned u = w[sizeof(T) == 4 ? e : e / 2];
        return __builtin_bit_cast(float, sizeof(T) == 4 ? u : e & 1 ? u & 0xffff0000u : u << 16);
    }
    // element e, known at run time only
    static __device__ __forceinline__ float pick(const u32x4& w, int e) {
        const int d = sizeof(T) == 4 ? e : e >> 1;
        const unsigned a = w[0], b = w[1], c = w[2], g = w[3];
        const unsigned u = d < 2 ? (d == 0 ? a : b) : (d == 2 ? c : g);
        return __builtin_bit_cast(float, sizeof(T) == 4 ? u : e & 1 ? u & 0xffff0000u : u << 16);
    }
    // piece p; past the row's end -infinity
    __device__ __forceinline__ u32x4 read(int p) const {
        const int v = p * E;
        T t[E];
        if (v + E <= vocab) {
            __builtin_memcpy(t, z + v, 16);
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) t[e] = v + e < vocab ? z[v + e] : (T)-INFINITY;
        }
        return __builtin_bit_cast(u32x4, t);
    }
    template <typename F>
    __device__ __forceinline__ void pieces_from(int p0, int p1, F f) const {  // f(piece, its index), three more in flight
        const int p = p0 + (int)threadIdx.x;
        if (p0 >= p1) return;
        u32x4 w0 = read(p), w1 = read(p + kSpThreads), w2 = read(p + 2 * kSpThreads), w3 = read(p + 3 * kSpThreads);
#pragma unroll 1
        for (int i = p; i < p1; i += kSpThreads) {
            f(w0, i);
            w0 = w1, w1 = w2, w2 = w3, w3 = read(i + 4 * kSpThreads);
        }
    }
    // f(logit, index) for all of them, by the whole block; what is past the end comes as -infinity.
    // kFirst: the pass that fills LDS.
    template <bool kFirst, typename F>
    __device__ __forceinline__ void each(F f) const {
        auto one = [&](const u32x4& w, int p) __attribute__((always_inline)) {
#pragma unroll
            for (int e = 0; e < E; ++e) f(get(w, e), p * E + e);
        };
        if constexpr (kFirst) {
            pieces_from(0, held, [&](const u32x4& w, int p) __attribute__((always_inline)) {
                lds[p] = w;
                one(w, p);
            });
        } else {
#pragma unroll 2
            for (int p = threadIdx.x; p < held; p += kSpThreads) one(lds[p], p);
        }
        pieces_from(held, (vocab + E - 1) / E, one);
    }
    // The same for the logits in one of kSpans spans [lo, hi]: a piece's are marked first, without a branch, and then taken
    // one by one.
    template <int kSpans, typename F>
    __device__ __forceinline__ void each_in(const float (&lo)[kSpans], const float (&hi)[kSpans], F f) const {
        auto one = [&](const u32x4& w, int p) __attribute__((always_inline)) {
            unsigned marks = 0;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float x = get(w, e);
                bool in = false;
#pragma unroll
                for (int i = 0; i < kSpans; ++i) in |= (x >= lo[i]) & (x <= hi[i]);
                marks |= in ? 1u << e : 0u;
            }
            while (marks) {
                const int e = __builtin_ctz(marks);
                marks &= marks - 1;
                f(pick(w, e), p * E + e);
            }
        };
#pragma unroll 2
        for (int p = threadIdx.x; p < held; p += kSpThreads) one(lds[p], p);
        pieces_from(held, (vocab + E - 1) / E, one);
    }
};

// A place in the row's order: everything before it has `count` tokens and `mass`; it is the tie-th token (from 0)
// of those with this key.
struct SamplePlace {
    unsigned key;
    int64_t tie;
    u64 count, mass;  // before it
    u64 own;          // its mass
    int index;        // -1: not known yet
};

// What the first wave finds out from the bins.
struct SamplePlan {
    static constexpr int kSpans = 3;  // k's; p's and min_p's; the token's
    int from[kSpans], to[kSpans];     // of bins
    int skipped[kSpans];              // bins before a span that are in none
    float lo[kSpans], hi[kSpans];
    double parts;                     // of the sort, a bin
    bool by_k, by_p, by_m;
    int k_bin, m_from, m_to;
    unsigned some;                    // tokens of the spans (without counts, at least)
    u64 total, kept, before_m;
};

// The block's working memory.
struct SampleShared {
    SampleTables tables;
    SamplePlan plan;
    u64 begin_mass[kSpWaves];  // of all bins before a wave's share of them
    unsigned begin_count[kSpWaves];
    unsigned tail;
    // of the row's bins, and a place for each lane's tokens without mass; then of a wave's share of bins up to each
    u64 mass[kSpBins + 64];
    unsigned count[kSpBins + 64];
    union {
        struct {
            u64 list[kSpList];    // key, complement of the index: as gathered, then from the largest down
            u64 parted[kSpList];  // by parts of the keys' span
        };
        struct {            // of a split bin's parts
            u64 smass[kSpParts];
            unsigned scount[kSpParts];
        };
    };
    unsigned parts[kSpList];
    u64 wmass[kSpWaves];
    unsigned wcount[kSpWaves];
    unsigned n;
    int at;
    SamplePlace place;
};

// Sums over a wave's lanes, by lane moves.
template <int kCtrl, int kRows>
__device__ __forceinline__ unsigned sp_move(unsigned v) { return (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, kCtrl, kRows, 0xf, true); }
template <int kCtrl, int kRows = 0xf>
__device__ __forceinline__ void sp_add(unsigned& c, u64& m) {
    c += sp_move<kCtrl, kRows>(c);
    m += (u64)sp_move<kCtrl, kRows>((unsigned)(m >> 32)) << 32 | sp_move<kCtrl, kRows>((unsigned)m);
}
// The largest over a wave's lanes.
__device__ __forceinline__ unsigned sp_max(unsigned v) {
    auto with = [&](auto ctrl) __attribute__((always_inline)) {
        const unsigned o = (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, decltype(ctrl)::value, 0xF, 0xF, false);
        v = o > v ? o : v;
    };
    with(std::integral_constant<int, 0xB1>{});
    with(std::integral_constant<int, 0x4E>{});
    with(std::integral_constant<int, 0x141>{});
    with(std::integral_constant<int, 0x140>{});
#pragma unroll
    for (int off = 16; off < 64; off <<= 1) {
        const unsigned o = __shfl_xor(v, off, kWave);
        v = o > v ? o : v;
    }
    return v;
}
// Inclusive sums over rows of 16 lanes, and over a wave.
__device__ __forceinline__ void sp_row_scan(unsigned& c, u64& m) {
    sp_add<kRowShr + 1>(c, m);
    sp_add<kRowShr + 2>(c, m);
    sp_add<kRowShr + 4>(c, m);
    sp_add<kRowShr + 8>(c, m);
}
__device__ __forceinline__ void sp_wave_scan(unsigned& c, u64& m) {
    sp_row_scan(c, m);
    sp_add<kRowBcast15, 0xa>(c, m);
    sp_add<kRowBcast31, 0xc>(c, m);
}
// Exclusive sums of c and m over the block's threads, in their order, and all of them.
__device__ __forceinline__ void sp_scan(SampleShared& s, unsigned& c, u64& m, unsigned& all_c, u64& all_m) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    unsigned ic = c;
    u64 im = m;
    sp_wave_scan(ic, im);
    __syncthreads();
    if (lane == 63) s.wcount[wave] = ic, s.wmass[wave] = im;
    __syncthreads();
    unsigned bc = 0;
    u64 bm = 0;
    all_c = 0, all_m = 0;
#pragma unroll
    for (int w = 0; w < kSpWaves; ++w) {
        if (w == wave) bc = all_c, bm = all_m;
        all_c += s.wcount[w], all_m += s.wmass[w];
    }
    c = bc + ic - c, m = bm + im - m;
}

// What is looked for: the `count`-th token (kCount), or the first whose running mass is at least (kReach), or above
// (kPass), `mass`.
enum { kCount, kReach, kPass };
struct SampleGoal {
    int kind;
    u64 count;
    double mass;
    __device__ __forceinline__ bool reached(u64 c, u64 m) const {
        return kind == kCount ? c >= count : kind == kReach ? (double)m >= mass : (double)m > mass;
    }
};

// The bins' running sums in place of the bins' own; all of them.
template <int kBins>
__device__ __forceinline__ void sp_run(SampleShared& s, u64* mass, unsigned* count, unsigned& all_c, u64& all_m) {
    constexpr int kPer = kBins / kSpThreads;
    static_assert(kPer * kSpThreads == kBins && kSpList % kSpThreads == 0, "whole shares");
    unsigned c[kPer], tc = 0;
    u64 m[kPer], tm = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        c[i] = tc += count[threadIdx.x * kPer + i];
        m[i] = tm += mass[threadIdx.x * kPer + i];
    }
    sp_scan(s, tc, tm, all_c, all_m);
#pragma unroll
    for (int i = 0; i < kPer; ++i) count[threadIdx.x * kPer + i] = tc + c[i], mass[threadIdx.x * kPer + i] = tm + m[i];
    __syncthreads();
}
// The bin s.at whose end reaches the goal and whose start does not, or where none does `otherwise` (-1: none).
template <int kBins>
__device__ __forceinline__ void sp_find_bin(SampleShared& s, const u64* mass, const unsigned* count, u64 base_c, u64 base_m, const SampleGoal& goal,
                                            int otherwise) {
    constexpr int kPer = kBins / kSpThreads;
    if (threadIdx.x == 0) s.at = otherwise;
    const int first = (int)threadIdx.x * kPer;
    bool before = goal.reached(base_c + (first ? count[first - 1] : 0), base_m + (first ? mass[first - 1] : 0));
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const bool now = goal.reached(base_c + count[first + i], base_m + mass[first + i]);
        if (now & !before) s.at = first + i;
        before = now;
    }
    __syncthreads();
}

// The smallest lo and the largest hi of the block's threads.
__device__ __forceinline__ void sp_span(SampleShared& s, unsigned& lo, unsigned& hi) {
    const unsigned a = ~sp_max(~lo), b = sp_max(hi);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s.wmass[threadIdx.x >> 6] = (u64)a << 32 | b;
    __syncthreads();
    lo = 0xffffffffu, hi = 0;
#pragma unroll
    for (int w = 0; w < kSpWaves; ++w) {
        const unsigned x = (unsigned)(s.wmass[w] >> 32), y = (unsigned)s.wmass[w];
        lo = x < lo ? x : lo;
        hi = y > hi ? y : hi;
    }
}
// Sorts the first n of the list from the largest key (and the lowest index) down: by 1024 parts, and within
// a part by counting the larger ones; where a part has more than 48 (equal logits), all by exchanges of pairs.
// place(key): its part, below 1024, not falling as keys fall; with kByKeys parts of the keys' span.
// (Counting alone, without parts: sp_count_sort.)
template <bool kByKeys, typename F>
__device__ __forceinline__ void sp_sort(SampleShared& s, unsigned n, F place) {
    constexpr int kPer = kSpList / kSpThreads;
    u64 mine[kPer];
    unsigned klo = 0xffffffffu, khi = 0, part[kPer], nth[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const unsigned j = threadIdx.x + i * kSpThreads;
        s.parts[j] = 0;
        mine[i] = j < n ? s.list[j] : 0;
        const unsigned key = (unsigned)(mine[i] >> 32);
        if (j < n) klo = key < klo ? key : klo, khi = key > khi ? key : khi;
    }
    int shift = 0;
    if constexpr (kByKeys) {
        sp_span(s, klo, khi);
        while ((khi - klo) >> shift >= (unsigned)kSpList) ++shift;
    } else {
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const unsigned key = (unsigned)(mine[i] >> 32);
        part[i] = kByKeys ? (khi - key) >> shift : place(key);
        nth[i] = threadIdx.x + i * kSpThreads < n ? atomicAdd(&s.parts[part[i]], 1u) : 0;
    }
    __syncthreads();
    // the parts' first places: a thread's are consecutive
    unsigned c[kPer], first = 0, all_c;
    u64 none = 0, all_m;
#pragma unroll
    for (int i = 0; i < kPer; ++i) c[i] = s.parts[threadIdx.x * kPer + i], first += c[i];
    unsigned most = 0, unused = 0xffffffffu;
#pragma unroll
    for (int i = 0; i < kPer; ++i) most = c[i] > most ? c[i] : most;
    sp_span(s, unused, most);
    if (most > 48) {
        unsigned size = 128;
        while (size < n) size <<= 1;
        for (unsigned i = n + threadIdx.x; i < size; i += kSpThreads) s.list[i] = 0;
        static_assert(kSpList <= 2 * kSpThreads, "a pair a thread");
        const unsigned i = threadIdx.x;
        // pairs up to 64 apart lie with one wave, whose LDS operations run in order: barriers stand only between the others
        bool apart = true;
        for (unsigned w = 2; w <= size; w <<= 1)
            for (unsigned d = w >> 1; d > 0; d >>= 1) {
                if (apart || d > 64) __syncthreads();
                apart = d > 64;
                if (i < size / 2) {
                    const unsigned x = 2 * i - (i & (d - 1)), y = x + d;
                    volatile u64* list = s.list;
                    const u64 p = list[x], q = list[y];
                    if ((p < q) == ((x & w) == 0)) list[x] = q, list[y] = p;
                }
            }
        __syncthreads();
        return;
    }
    sp_scan(s, first, none, all_c, all_m);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        s.parts[threadIdx.x * kPer + i] = first;
        first += c[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kPer; ++i)
        if (threadIdx.x + i * kSpThreads < n) s.parted[s.parts[part[i]] + nth[i]] = mine[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        if (threadIdx.x + i * kSpThreads >= n) continue;
        const unsigned from = s.parts[part[i]], to = part[i] + 1 < (unsigned)kSpList ? s.parts[part[i] + 1] : n;
        unsigned above = 0;
        for (unsigned j = from; j < to; ++j) above += s.parted[j] > mine[i];
        s.list[from + above] = mine[i];
    }
    __syncthreads();
}
constexpr unsigned kSpCounted = 256;
__device__ __forceinline__ void sp_count_sort(SampleShared& s, unsigned n) {  // of at most so many, into s.parted
    if (threadIdx.x < n) {
        const u64 mine = s.list[threadIdx.x];
        unsigned above = 0;
#pragma unroll 4
        for (unsigned j = 0; j < n; ++j) above += s.list[j] > mine;
        s.parted[above] = mine;
    }
    __syncthreads();
}
// A thread's part of the sorted list: each token's count and mass before it, and the mass up to it.
struct SampleWalk {
    static constexpr int kPer = kSpList / kSpThreads;
    unsigned n;
    u64 count[kPer], before[kPer], after[kPer];
    // of tokens that follow each other in the row's order, behind base_c and base_m
    __device__ __forceinline__ void start(SampleShared& s, unsigned n_, const SampleScale& scale, u64 base_c, u64 base_m) {
        n = n_;
        u64 m[kPer], all_m, at = 0;
        unsigned tc = 0, all_c;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const unsigned j = threadIdx.x * kPer + i;
            m[i] = j < n ? sp_mass(s.tables, scale, sp_logit((unsigned)(s.list[j] >> 32))) : 0;
            at += m[i];
        }
        sp_scan(s, tc, at, all_c, all_m);
        at += base_m;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            count[i] = base_c + threadIdx.x * kPer + i;
            before[i] = at;
            after[i] = at += m[i];
        }
    }
    // the token that the goal falls on, in s.place, or the last where none reaches it: the masses of a bin, added up at once,
    // may differ from its tokens' in the last bits (the caller waits)
    __device__ __forceinline__ void find(SampleShared& s, const SampleGoal& goal) const {
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const unsigned j = threadIdx.x * kPer + i;
            if (j < n && !goal.reached(count[i], before[i]) && (j + 1 == n || goal.reached(count[i] + 1, after[i]))) {
                const unsigned key = (unsigned)(s.list[j] >> 32);
                unsigned less = 0, more = j;  // the first of its ties
                while (less < more) {
                    const unsigned mid = (less + more) / 2;
                    if ((unsigned)(s.list[mid] >> 32) > key) less = mid + 1;
                    else more = mid;
                }
                s.place = SamplePlace{key, (int64_t)(j - less), count[i], before[i], after[i] - before[i], (int)~(unsigned)s.list[j]};
            }
        }
    }
};

// The token of the row's order that the goal falls on, in s.place; goals lie within the row. (Counts are those of the tokens
// before it only if the row's bins have counts.)
template <typename L>
__device__ __forceinline__ void sp_locate(SampleShared& s, const L& z, const SampleScale& scale, const SampleGoal& goal) {
    __syncthreads();
    sp_find_bin<kSpBins>(s, s.mass, s.count, 0, 0, goal, -1);
    const int bin = s.at;
    u64 base_c = bin > 0 ? s.count[bin - 1] : 0, base_m = bin > 0 ? s.mass[bin - 1] : 0;
    // first what may lie in the bin, by one comparison each way
    float lo[1] = {bin < kSpBins - 1 ? scale.near((double)(bin + 1)) : -INFINITY}, hi[1] = {bin > 0 ? scale.beyond((double)bin) : INFINITY};
    bool few = bin >= 0;
    if (!few && threadIdx.x == 0) s.place = SamplePlace{kSpNone, 0, 0, 0, 0, 0};  // not within the row: the caller's goals rule it out
    while (few) {
        // gather the bin's tokens in [lo, hi]
        __syncthreads();
        if (threadIdx.x == 0) s.n = 0;
        __syncthreads();
        z.template each_in<1>(lo, hi, [&](float x, int v) __attribute__((always_inline)) {
            if (x > -INFINITY && sp_in(scale.far(x), bin)) {
                const unsigned i = atomicAdd(&s.n, 1u);
                if (i < (unsigned)kSpList) s.list[i] = (u64)sp_key(x) << 32 | (unsigned)~v;
            }
        });
        __syncthreads();
        const unsigned n = s.n;
        if (n <= (unsigned)kSpList) {
            sp_sort<true>(s, n, [](unsigned) { return 0u; });
            SampleWalk walk;
            walk.start(s, n, scale, base_c, base_m);
            walk.find(s, goal);
            few = false;
            continue;
        }
        // too many to sort: split the keys' span in 1024, or find one key
        unsigned klo = 0xffffffffu, khi = 0;
        for (int b = threadIdx.x; b < kSpParts; b += kSpThreads) s.smass[b] = 0, s.scount[b] = 0;  // seen by all behind sp_span's barriers
        z.template each_in<1>(lo, hi, [&](float x, int) __attribute__((always_inline)) {
            if (x > -INFINITY && sp_in(scale.far(x), bin)) {
                const unsigned key = sp_key(x);
                klo = key < klo ? key : klo;
                khi = key > khi ? key : khi;
            }
        });
        sp_span(s, klo, khi);
        if (klo == khi) {
            // equal logits: which of them, by division
            if (threadIdx.x == 0) {
                const u64 own = sp_mass(s.tables, scale, sp_logit(khi));
                int64_t before = 0, with = n;  // not reached with `before` of them, reached with `with`
                while (with - before > 1) {
                    const int64_t mid = (before + with) / 2;
                    if (goal.reached(base_c + (u64)mid, base_m + (u64)mid * own)) with = mid;
                    else before = mid;
                }
                s.place = SamplePlace{khi, before, base_c + (u64)before, base_m + (u64)before * own, own, -1};
            }
            few = false;
            continue;
        }
        int parts = 0;
        while ((khi - klo) >> parts >= (unsigned)kSpParts) ++parts;
        // from the largest key down
        z.template each_in<1>(lo, hi, [&](float x, int) __attribute__((always_inline)) {
            if (x > -INFINITY && sp_in(scale.far(x), bin)) {
                const int b = (int)((khi - sp_key(x)) >> parts);
                atomicAdd(&s.scount[b], 1u);
                atomicAdd(&s.smass[b], sp_mass(s.tables, scale, x));
            }
        });
        __syncthreads();
        unsigned all_c;
        u64 all_m;
        sp_run<kSpParts>(s, s.smass, s.scount, all_c, all_m);
        sp_find_bin<kSpParts>(s, s.smass, s.scount, base_c, base_m, goal, (int)((khi - klo) >> parts));
        const unsigned b = (unsigned)s.at;
        if (b) base_c += s.scount[b - 1], base_m += s.smass[b - 1];
        const unsigned new_hi = khi - (b << parts), span = (1u << parts) - 1u;
        lo[0] = sp_logit(new_hi - klo > span ? new_hi - span : klo);
        hi[0] = sp_logit(new_hi);
    }
    __syncthreads();
}

// The index of the tie-th token with this logit.
template <typename T>
__device__ __forceinline__ int sp_index(SampleShared& s, const T* z, int vocab, float logit, int64_t tie) {
    __syncthreads();
    if (threadIdx.x == 0) s.at = 0;
    int64_t before = 0;
    for (int v0 = 0; v0 < vocab; v0 += kSpThreads * 8) {
        const int v = v0 + (int)threadIdx.x * 8;
        float x[8];
        unsigned mine = 0, c, all_c;
        u64 none = 0, all_m;
        if (v < vocab) {
            load8(z, v, vocab, x);
#pragma unroll
            for (int e = 0; e < 8; ++e) mine += v + e < vocab && x[e] == logit;
        }
        c = mine;
        sp_scan(s, c, none, all_c, all_m);
        int64_t at = before + c;
        if (mine && at <= tie && at + mine > tie) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (v + e < vocab && x[e] == logit && at++ == tie) s.at = v + e;
        }
        before += all_c;
        if (before > tie) break;
    }
    __syncthreads();
    return s.at;
}

template <typename T>
__global__ __launch_bounds__(kSpThreads) void sample_kernel(SampleArgs a, int held) {
    extern __shared__ __align__(16) char sp_smem[];
    __shared__ SampleShared s;
    const int64_t row = blockIdx.x;
    const SampleLogits<T> z{reinterpret_cast<u32x4*>(sp_smem), reinterpret_cast<const T*>(a.z) + row * a.vocab, a.vocab, held};
    const SampleRow r = sp_row(a, row);
    for (int b = threadIdx.x; b < kSpBins + 64; b += kSpThreads) s.mass[b] = 0, s.count[b] = 0;
    if (threadIdx.x < sizeof(SampleTables) / 8) reinterpret_cast<double*>(&s.tables)[threadIdx.x] = reinterpret_cast<const double*>(&kSpTables)[threadIdx.x];
    if (threadIdx.x == 0) s.tail = s.n = 0;

    // the largest logit (NaN is none), for a greedy choice its lowest index
    float top = -INFINITY;
    unsigned first = 0xffffffffu;
    const bool greedy = !(r.t > 0.0);
    if (greedy)
        z.template each<true>([&](float x, int v) __attribute__((always_inline)) {
            if (x > top) top = x, first = (unsigned)v;  // a thread's indexes rise
        });
    else z.template each<true>([&](float x, int) __attribute__((always_inline)) { top = x > top ? x : top; });
    u64 best = (u64)sp_key(top) << 32 | (unsigned)~first;
    if (greedy) {
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) {
            const u64 o = __shfl_xor(best, off, kWave);
            best = o > best ? o : best;
        }
    } else {
        best = (u64)sp_max((unsigned)(best >> 32)) << 32;
    }
    if ((threadIdx.x & 63) == 0) s.wmass[threadIdx.x >> 6] = best;
    __syncthreads();
    static_assert(kSpWaves == 16, "a value for each lane of a row of 16");
    best = s.wmass[threadIdx.x & 15];
    if (greedy) {
#pragma unroll
        for (int off = 8; off > 0; off >>= 1) {
            const u64 o = __shfl_xor(best, off, kWave);
            best = o > best ? o : best;
        }
    } else {
        best = (u64)sp_max((unsigned)(best >> 32)) << 32;
    }
    top = sp_logit((unsigned)(best >> 32));
    if (greedy || top == -INFINITY) {
        if (threadIdx.x == 0) {
            a.token[row] = top == -INFINITY ? -1 : (int64_t)(int)~(unsigned)best;
            if (a.logprob) a.logprob[row] = top == -INFINITY ? __builtin_nanf("") : 0.f;
        }
        return;
    }
    const double u = (double)a.u[row];
    if (top == INFINITY) {
        // infinite logits: all have the same mass, the others none
        unsigned c = 0, all_c;
        u64 none = 0, all_m;
        z.template each<false>([&](float x, int) { c += x == top; });
        sp_scan(s, c, none, all_c, all_m);
        double n = r.k < (int64_t)all_c ? (double)r.k : (double)all_c;
        if (r.p < 1.0) n = fmax(ceil(r.p * n), 1.0);
        const double at = floor(fmax(u, 0.0) * n);
        const int index = sp_index(s, z.z, a.vocab, top, (int64_t)(at < n ? at : n - 1.0));
        if (threadIdx.x == 0) {
            a.token[row] = index;
            if (a.logprob) a.logprob[row] = (float)-log(n);
        }
        return;
    }
    const SampleScale scale{(double)top, fmin(kSpPerT / r.t, 1e300), a.shift};  // finite: the first lies at 0 times it

    // masses, and counts where a count is asked for
    const bool counts = r.k < (int64_t)a.vocab;
    unsigned tail = 0;  // tokens of the last bin, which have no mass
    {
        const double unit = ldexp(1.0, a.shift), c1 = unit * (-1.0 / kSpPerT), c2 = c1 * (-1.0 / (2 * kSpPerT)), c3 = c2 * (-1.0 / (3 * kSpPerT)),
                     c4 = c3 * (-1.0 / (4 * kSpPerT)), c5 = c4 * (-1.0 / (5 * kSpPerT));  // sp_series, times 2^shift
        const int aside = kSpBins + ((int)threadIdx.x & 63);
        auto add = [&](float x, auto counted) __attribute__((always_inline)) {
            // without a branch: what has no mass (NaN, too) goes where nobody looks
            const double q = scale.far(x);
            const bool in = q < (double)(kSpBins - 1);
            const int b = (int)q, at = in ? b : aside;
            const double d = q - (double)b;
            atomicAdd(&s.mass[at], sp_whole(fma(fma(fma(fma(fma(c5, d, c4), d, c3), d, c2), d, c1), d, unit)));
            if constexpr (decltype(counted)::value) {
                atomicAdd(&s.count[at], 1u);
                tail += !in & (x > -INFINITY);
            }
        };
        if (counts) {
            z.template each<false>([&](float x, int) __attribute__((always_inline)) { add(x, std::true_type{}); });
            if (tail) atomicAdd(&s.tail, tail);
        } else z.template each<false>([&](float x, int) __attribute__((always_inline)) { add(x, std::false_type{}); });
    }
    __syncthreads();
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    SamplePlan& plan = s.plan;
    {
        // running sums of each wave's share of bins
        constexpr int kPer = kSpBins / kSpThreads;
        unsigned c[kPer], ic = 0;
        u64 m[kPer], im = 0;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int b = (int)threadIdx.x * kPer + i;
            const u64 raw = s.mass[b];
            // without counts, at least so many tokens are in a bin
            c[i] = ic += !counts ? (unsigned)((raw + ((u64)1 << a.shift) - 1) >> a.shift) : b == kSpBins - 1 ? s.tail : s.count[b];
            m[i] = im += (u64)((double)raw * sp_bin_mass(s.tables, b) + 0.5);
        }
        const unsigned own_c = ic;
        const u64 own_m = im;
        sp_wave_scan(ic, im);
        if (lane == 63) s.wcount[wave] = ic, s.wmass[wave] = im;
#pragma unroll
        for (int i = 0; i < kPer; ++i) s.count[threadIdx.x * kPer + i] = ic - own_c + c[i], s.mass[threadIdx.x * kPer + i] = im - own_m + m[i];
    }
    __syncthreads();
    const auto share = [&](u64 of) __attribute__((always_inline)) {  // the token that reaches p is the last; the first stays whatever p is
        const double m = r.p > 0.0 ? r.p * (double)of : 0.0;
        return SampleGoal{kReach, 0, m > 1.0 ? m : 1.0};
    };
    const auto draw = [&](u64 of) __attribute__((always_inline)) {  // u below 1 falls within the kept mass; others are taken to its ends
        const double m = u > 0.0 ? u * (double)of : 0.0, most = (double)of * (1.0 - 0x1p-30);
        return SampleGoal{kPass, 0, m < most ? m : most};
    };
    // min_p keeps what is nearer than this; rounding of the logarithm matters to tokens that are as near as makes no
    // difference to a bin, and these are asked for their mass itself
    const double min_p = r.m < 1.0 ? r.m : 1.0;
    const double far_m = r.m > 0.0 ? log(min_p) * -kSpPerT : (double)kSpBins;
    auto kept_by_m = [&](float x) __attribute__((always_inline)) {
        const double q = scale.far(x);
        return q < far_m - 1e-6 || (q < far_m + 1e-6 && exp(q * (-1.0 / kSpPerT)) >= min_p);
    };
    auto mass_to = [&](int bin) __attribute__((always_inline)) { return bin < 0 ? (u64)0 : s.begin_mass[bin / kSpShare] + s.mass[bin]; };
    auto count_to = [&](int bin) __attribute__((always_inline)) { return bin < 0 ? 0u : s.begin_count[bin / kSpShare] + s.count[bin]; };
    if (wave == 0) {
        // The bins in which the answers lie: the k-th token's, that in which p of the k's mass is reached, the bound of min_p and
        // the token's. What is known of a mass is that it lies between those of all before its bin and of all up to its end.
        unsigned ic = s.wcount[lane & 15];
        u64 im = s.wmass[lane & 15];
        const unsigned own_c = ic;
        const u64 own_m = im;
        sp_row_scan(ic, im);
        if (lane < kSpWaves) s.begin_mass[lane] = im - own_m, s.begin_count[lane] = ic - own_c;
        const u64 total = __shfl(im, 15, kWave);
        __builtin_amdgcn_wave_barrier();
        // the bin whose end reaches the goal and whose start does not
        auto find = [&](const SampleGoal& goal, int otherwise) __attribute__((always_inline)) {
            const u64 shares = __ballot(goal.reached(ic, im)) & 0xffffu;
            if (!shares) return otherwise;
            const int first = __builtin_ctzll(shares), at = first * kSpShare + 2 * lane;
            const u64 bm = s.begin_mass[first];
            const unsigned bc = s.begin_count[first];
            const bool r0 = goal.reached((u64)bc + s.count[at], bm + s.mass[at]), r1 = goal.reached((u64)bc + s.count[at + 1], bm + s.mass[at + 1]);
            const u64 m0 = __ballot(r0), m1 = __ballot(r1);
            if (!m1) return otherwise;
            const int l = __builtin_ctzll(m1);
            return first * kSpShare + 2 * l + ((m0 >> l & 1) ? 0 : 1);
        };
        static_assert(kSpShare == 128, "two bins a lane");
        constexpr int kSpans = SamplePlan::kSpans;
        int from[kSpans] = {0, 0, 0}, to[kSpans] = {-1, -1, -1};
        u64 low = total, high = total, kept = total, before_m = 0;
        int k_bin = 0;
        bool by_k = counts, by_p = r.p < 1.0, by_m = far_m < (double)(kSpBins - 2);  // what is beyond has no mass
        if (by_k) {
            const int at = find(SampleGoal{kCount, (u64)r.k, 0.0}, -1);
            by_k = at >= 0;  // the row has so many tokens
            if (by_k) {
                from[0] = to[0] = k_bin = at;
                low = mass_to(at - 1), high = mass_to(at);
                if (low == high) by_k = false, to[0] = -1, kept = low;  // whichever it is
            }
        }
        if (by_p) {
            from[1] = find(share(low), kSpBins - 1), to[1] = find(share(high), kSpBins - 1);
            low = mass_to(from[1] - 1), high = mass_to(to[1]);
        }
        const int m_from = by_m ? (int)fmax(far_m - 1e-6, 0.0) : 0, m_to = by_m ? (int)(far_m + 1e-6) : -1;
        if (by_m) {
            before_m = mass_to(m_from - 1);
            const u64 up_to_m = mass_to(m_to);
            if (before_m >= high) {  // the others leave less
                by_m = false;
            } else if (up_to_m <= low) {  // more, of which min_p leaves a part
                by_k = by_p = false;
                from[0] = 0, to[0] = -1, from[1] = m_from, to[1] = m_to;
                kept = total, low = before_m, high = up_to_m;
            } else {
                // side by side with p's, a span holds both
                from[1] = to[1] < 0 ? m_from : min(from[1], m_from), to[1] = max(to[1], m_to);
                low = min(low, before_m), high = min(high, up_to_m);
            }
        }
        from[2] = find(draw(low), kSpBins - 1), to[2] = find(draw(high), kSpBins - 1);
        // the spans one after the other: the token's, p's and min_p's, k's
        int bins = 0;
        unsigned some = 0;
#pragma unroll
        for (int i = kSpans - 1, done = 0; i >= 0; --i) {
            from[i] = max(from[i], done);
            const bool is = to[i] >= from[i];
            if (lane == 0) {
                plan.from[i] = from[i], plan.to[i] = to[i], plan.skipped[i] = from[i] - bins;
                plan.lo[i] = !is ? INFINITY : to[i] < kSpBins - 1 ? scale.near((double)(to[i] + 1)) : -INFINITY;
                plan.hi[i] = !is ? -INFINITY : from[i] > 0 ? scale.beyond((double)from[i]) : INFINITY;
            }
            if (is) {
                bins += to[i] - from[i] + 1, done = to[i] + 1;
                some += count_to(to[i]) - count_to(from[i] - 1);
            }
        }
        if (lane == 0) {
            plan.parts = (double)kSpList / (double)bins;
            plan.k_bin = k_bin;
            plan.by_k = by_k, plan.by_p = by_p, plan.by_m = by_m, plan.m_from = m_from, plan.m_to = m_to;
            plan.some = some, plan.total = total, plan.kept = kept, plan.before_m = before_m;
        }
    }
    __syncthreads();
    unsigned n = kSpList + 1;
    if (plan.some <= (unsigned)kSpList) {
        constexpr int kSpans = SamplePlan::kSpans;
        float lo[kSpans], hi[kSpans];
        int from[kSpans], to[kSpans];
#pragma unroll
        for (int i = 0; i < kSpans; ++i) lo[i] = plan.lo[i], hi[i] = plan.hi[i], from[i] = plan.from[i], to[i] = plan.to[i];
        z.template each_in<kSpans>(lo, hi, [&](float x, int v) __attribute__((always_inline)) {
            const int b = sp_bin(scale.far(x));
            bool in = false;
#pragma unroll
            for (int i = 0; i < kSpans; ++i) in |= (b >= from[i]) & (b <= to[i]);
            if (in && x > -INFINITY) {
                const unsigned i = atomicAdd(&s.n, 1u);
                if (i < (unsigned)kSpList) s.list[i] = (u64)sp_key(x) << 32 | (unsigned)~v;
            }
        });
        __syncthreads();
        n = s.n;
    }

    u64 kept = plan.kept;
    float logit;
    int index;
    if (n <= (unsigned)kSpList) {
        const u64* list = s.list;
        u64* after = s.parted;  // the mass up to each token of the list
        if (n <= kSpCounted) {
            sp_count_sort(s, n);
            list = s.parted, after = s.list;
        } else {
            // its parts: the spans' bins one after the other, without those between
            sp_sort<false>(s, n, [&](unsigned key) __attribute__((always_inline)) {
                const double q = scale.far(sp_logit(key));
                const int b = sp_bin(q);
                const int less = b <= plan.to[2] ? plan.skipped[2] : b <= plan.to[1] ? plan.skipped[1] : plan.skipped[0];
                return (unsigned)fmin(fmax((q - (double)less) * plan.parts, 0.0), (double)(kSpList - 1));
            });
        }
        if (wave != 0) return;
        // The first wave reads the answers off. A bin's first token starts where the bin does, its last ends where the bin does
        // (the masses of a bin, added up at once, may differ from its tokens' in the last bits); a lane takes `per`
        // tokens in a row.
        const unsigned per = (n + 63) / 64, j0 = lane * per, j1 = min(j0 + per, n);
        auto far_of = [&](unsigned j) __attribute__((always_inline)) { return scale.far(sp_logit((unsigned)(list[j] >> 32))); };
        u64 v = 0;
        bool known = false;  // v is the mass of all before, not only of this lane's
        int b_before = j0 > 0 && j0 < n ? sp_bin(far_of(j0 - 1)) : -1;
        {
            int pb = b_before;
#pragma unroll 1
            for (unsigned j = j0; j < j1; ++j) {
                const int b = sp_bin(far_of(j));
                const u64 m = sp_mass(s.tables, scale, sp_logit((unsigned)(list[j] >> 32)));
                if (b != pb) v = mass_to(b - 1), known = true;
                v += m, pb = b;
                after[j] = m;
            }
        }
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const u64 ov = __shfl_up(v, off, kWave);
            const bool ok = __shfl_up((int)known, off, kWave);
            if (lane >= off && !known) v += ov, known = ok;
        }
        v = __shfl_up(v, 1, kWave);  // up to this lane's first
        {
            int pb = b_before, b = j0 < n ? sp_bin(far_of(j0)) : -1;
#pragma unroll 1
            for (unsigned j = j0; j < j1; ++j) {
                const int next = j + 1 < n ? sp_bin(far_of(j + 1)) : -1;
                if (b != pb) v = mass_to(b - 1);
                v += after[j];
                const u64 end = mass_to(b);
                after[j] = next != b || v > end ? end : v;
                pb = b, b = next;
            }
        }
        __builtin_amdgcn_wave_barrier();
        // the first token that reaches a goal (not a count)
        auto find = [&](const SampleGoal& goal) __attribute__((always_inline)) {
            const u64 lanes = __ballot(j0 < n && goal.reached(0, after[j1 - 1]));
            if (!lanes) return n - 1;
            const unsigned at = __builtin_ctzll(lanes) * per + lane;
            const u64 places = __ballot(lane < per && at < n && goal.reached(0, after[at < n ? at : n - 1]));
            return (unsigned)(at - lane) + (unsigned)__builtin_ctzll(places);
        };
        if (plan.by_k) {
            // it is so many behind its bin's start; the list may lack tokens before that
            const int bin = plan.k_bin;
            unsigned nearer = 0;
#pragma unroll 1
            for (unsigned j = j0; j < j1; ++j) nearer += sp_bin(far_of(j)) < bin;
            u64 none = 0;
            sp_wave_scan(nearer, none);
            kept = after[min(__shfl(nearer, 63, kWave) + (unsigned)(r.k - 1 - count_to(bin - 1)), n - 1)];
        }
        if (plan.by_p) kept = after[find(share(kept))];
        if (plan.by_m) {
            int last = -1;
#pragma unroll 1
            for (unsigned j = j0; j < j1; ++j) {
                const float x = sp_logit((unsigned)(list[j] >> 32));
                const int b = sp_bin(scale.far(x));
                if (b >= plan.m_from && b <= plan.m_to && kept_by_m(x)) last = (int)j;
            }
            last = (int)sp_max((unsigned)(last + 1)) - 1;
            kept = min(kept, last < 0 ? plan.before_m : after[last]);
        }
        const unsigned at = find(draw(kept));
        logit = sp_logit((unsigned)(list[at] >> 32)), index = (int)~(unsigned)list[at];
    } else {
        // the running sums of all bins
        constexpr int kPer = kSpBins / kSpThreads;
#pragma unroll
        for (int i = 0; i < kPer; ++i) s.count[threadIdx.x * kPer + i] += s.begin_count[wave], s.mass[threadIdx.x * kPer + i] += s.begin_mass[wave];
        const bool by_k = plan.by_k, by_p = plan.by_p;
        SamplePlace q;
        for (int step = by_k ? 0 : by_p ? 1 : 2; step < 3; step = step == 0 && !by_p ? 2 : step + 1) {
            if (step == 2 && plan.by_m) {
                u64 mine = 0, all_m;
                unsigned none = 0, all_c;
                const int m_from = plan.m_from, m_to = plan.m_to;
                const float least[1] = {scale.near((double)(m_to + 1))}, most[1] = {m_from > 0 ? scale.beyond((double)m_from) : INFINITY};
                z.template each_in<1>(least, most, [&](float x, int) __attribute__((always_inline)) {
                    const int b = sp_bin(scale.far(x));
                    if (b >= m_from && b <= m_to && kept_by_m(x)) mine += sp_mass(s.tables, scale, x);
                });
                sp_scan(s, none, mine, all_c, all_m);
                kept = min(kept, plan.before_m + all_m);
            }
            sp_locate(s, z, scale, step == 0 ? SampleGoal{kCount, (u64)r.k, 0.0} : step == 1 ? share(kept) : draw(kept));
            q = s.place;
            if (step < 2) kept = q.mass + q.own;
        }
        logit = sp_logit(q.key);
        index = q.index >= 0 ? q.index : sp_index(s, z.z, a.vocab, logit, q.tie);
    }
    if (threadIdx.x == 0) {
        a.token[row] = index;
        // the likeliest token's mass is 1: what the others add may be far below it
        if (a.logprob) a.logprob[row] = (float)(scale.far(logit) * (-1.0 / kSpPerT) - log1p(ldexp((double)(int64_t)(kept - ((u64)1 << a.shift)), -a.shift)));
    }
}

template <typename T>
static int sample_t(const SampleArgs& a, hipStream_t stream) {
    const int pieces = (int)(((int64_t)a.vocab * (int)sizeof(T) + 15) / 16), held = std::min(pieces, kSpHeld / 16);
    static std::atomic<uint64_t> done{0};
    if (!allow_lds(reinterpret_cast<const void*>(&sample_kernel<T>), kSpHeld, done)) return M3_ERR_LAUNCH;
    // a grid holds less than 2^32 threads
    constexpr int64_t kRows = ((int64_t)1 << 32) / kSpThreads / 2;
    for (int64_t r = 0; r < a.rows; r += kRows) {
        SampleArgs b = a;
        const auto from = [&](auto* p) { return p ? p + r : p; };
        b.z = reinterpret_cast<const T*>(a.z) + r * a.vocab;
        b.u = from(a.u), b.temperature = from(a.temperature), b.top_p = from(a.top_p), b.min_p = from(a.min_p), b.top_k = from(a.top_k);
        b.token = from(a.token), b.logprob = from(a.logprob);
        hipLaunchKernelGGL((sample_kernel<T>), dim3((unsigned)std::min(kRows, a.rows - r)), dim3(kSpThreads), held * 16, stream, b, held);
        if (hipGetLastError() != hipSuccess) return M3_ERR_LAUNCH;
    }
    return M3_OK;
}

int launch_sample(const void* logits, int dtype, int64_t rows, int vocab, const float* u, const float* temperature,
                  double temperature1, const int32_t* top_k, int64_t top_k1, const float* top_p, double top_p1,
                  const float* min_p, double min_p1, int64_t* token, float* logprob, hipStream_t stream) {
    int bits = 0;
    while (((int64_t)1 << bits) < vocab) ++bits;
    // a row's mass stays below 2^62, a token's within the 52 bits that sp_mass has
    const SampleArgs a{logits, u, temperature, top_p, min_p, top_k, temperature1, top_p1, min_p1, top_k1, token, logprob, rows, vocab,
                       std::min(62 - bits, 51)};
    return dtype == M3_DTYPE_BF16 ? sample_t<bf16>(a, stream) : sample_t<float>(a, stream);
}

}  // namespace m3
