// The next token of each row of logits, from a given random number (gfx950):
//   mass(v) = exp((z_v - max z) / T);  tokens in the order of z, ties from the lowest index;
//   kept: the first k of them, of these the shortest run whose mass reaches p of the k's, and of these the
//   ones with mass >= m; token = the first whose running mass passes u times the kept mass.
// Every bound cuts the same order, so what is kept is a prefix, and each step is the question which
// token of the order a count or a mass falls on. It is answered without sorting the row:
//   sample_top:   each row's largest logit (its lowest index), in slices over many blocks;
//   sample_bins:  counts and masses by distance from it, 1024 bins of 1/32;
//   sample_pick:  one block a row finds the bin, gathers its tokens (the row is read once more), sorts them
//                 and walks on; a bin with more than 2048 tokens is split by its keys' bits first.
// Masses are added as whole numbers of 2^-45 or so, so that sums do not depend on their order, and come
// from an exponential in 64 bits (a Taylor series of 2^f, |f| <= 1/2, to 1e-13 of its value): a border is
// missed with a probability of about 1e-9 a row, as with 64-bit sums over sorted probabilities.
// Bound by the row's three reads.
#include <algorithm>

#include "m3_common.h"
#include "m3_kernels.h"
#include "m3_mx.h"
#include "mamba3_amd.h"

namespace m3 {

typedef unsigned long long u64;
constexpr int kSpThreads = 256;
constexpr int kSpBins = 1024;
constexpr int kSpList = 2048;
constexpr int kSpSlices = 64;  // most of a row
constexpr int kSpPick = 1024;  // threads of sample_pick

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
    int rows, vocab, slices, slice;  // slice: logits of each
    u64* top;       // [rows][slices]
    u64* mass;      // [rows][kSpBins]
    unsigned* count;
    int shift;      // masses are whole numbers of 2^-shift
};

// Order of logits as whole numbers; -0 as 0, NaN as -infinity, which is no token.
__device__ __forceinline__ unsigned sp_key(float z) {
    z = z != z ? -INFINITY : z + 0.f;
    const unsigned b = __builtin_bit_cast(unsigned, z);
    return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float sp_logit(unsigned key) {
    return __builtin_bit_cast(float, key ^ ((key >> 31) ? 0x80000000u : 0xffffffffu));
}
constexpr unsigned kSpNone = 0x007fffffu;  // the key of -infinity

__device__ __forceinline__ int sp_bin(float top, float z) {
    const float far = (top - z) * 32.f;  // NaN for two infinities, which are the same logit
    return z == top ? 0 : far < (float)(kSpBins - 1) ? (int)far : kSpBins - 1;
}
// 2^shift mass of a logit, rounded: c = log2(e) / T.
__device__ __forceinline__ u64 sp_mass(float top, float z, double c, int shift) {
    const double x = z == top ? 0.0 : ((double)z - (double)top) * c;
    if (!(x > -64.0)) return 0;  // below half of 2^-62; NaN, an infinity times 0, too
    const double n = rint(x), f = (x - n) * 0.69314718055994530942;
    double e = 1.0 / 6227020800.0;
    e = fma(e, f, 1.0 / 479001600.0);
    e = fma(e, f, 1.0 / 39916800.0);
    e = fma(e, f, 1.0 / 3628800.0);
    e = fma(e, f, 1.0 / 362880.0);
    e = fma(e, f, 1.0 / 40320.0);
    e = fma(e, f, 1.0 / 5040.0);
    e = fma(e, f, 1.0 / 720.0);
    e = fma(e, f, 1.0 / 120.0);
    e = fma(e, f, 1.0 / 24.0);
    e = fma(e, f, 1.0 / 6.0);
    e = fma(e, f, 0.5);
    e = fma(e, f, 1.0);
    e = fma(e, f, 1.0);
    return (u64)(ldexp(e, (int)n + shift) + 0.5);
}

struct SampleRow {
    double t, p, m;
    int64_t k;
};
__device__ __forceinline__ SampleRow sp_row(const SampleArgs& a, int row) {
    SampleRow r;
    r.t = a.temperature ? (double)a.temperature[row] : a.temperature1;
    r.p = a.top_p ? (double)a.top_p[row] : a.top_p1;
    r.m = a.min_p ? (double)a.min_p[row] : a.min_p1;
    r.k = a.top_k ? (int64_t)a.top_k[row] : a.top_k1;
    if (r.k <= 0 || r.k > a.vocab) r.k = a.vocab;
    return r;
}

template <typename T>
__global__ __launch_bounds__(kSpThreads) void sample_top_kernel(SampleArgs a) {
    const int row = blockIdx.y, s = blockIdx.x;
    const T* z = reinterpret_cast<const T*>(a.z) + (int64_t)row * a.vocab;
    const int v0 = s * a.slice, v1 = v0 + a.slice < a.vocab ? v0 + a.slice : a.vocab;
    u64 best = 0;  // key, then the complement of the index
    for (int v = v0 + (int)threadIdx.x * 8; v < v1; v += kSpThreads * 8) {
        float f[8];
        load8(z, v, v1, f);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const u64 k = (u64)sp_key(f[e]) << 32 | (unsigned)~(v + e);
            if (v + e < v1 && k > best) best = k;
        }
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        const u64 o = __shfl_xor(best, off, kWave);
        best = o > best ? o : best;
    }
    __shared__ u64 red[kSpThreads / 64];
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = best;
    __syncthreads();
    if (threadIdx.x == 0) {
#pragma unroll
        for (int i = 1; i < kSpThreads / 64; ++i) best = red[i] > best ? red[i] : best;
        a.top[(int64_t)row * a.slices + s] = best;
    }
    // this slice's share of the row's bins, for the next kernel to add to
    for (int b = s * kSpThreads + (int)threadIdx.x; b < kSpBins; b += a.slices * kSpThreads) {
        a.mass[(int64_t)row * kSpBins + b] = 0;
        a.count[(int64_t)row * kSpBins + b] = 0;
    }
}

// The row's largest logit and its index's complement, by one wave.
__device__ __forceinline__ u64 sp_top(const SampleArgs& a, int row) {
    const int lane = threadIdx.x & 63;
    u64 v = lane < a.slices ? a.top[(int64_t)row * a.slices + lane] : 0;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        const u64 o = __shfl_xor(v, off, kWave);
        v = o > v ? o : v;
    }
    return v;
}

template <typename T>
__global__ __launch_bounds__(kSpThreads) void sample_bins_kernel(SampleArgs a) {
    __shared__ u64 mass[kSpBins];
    __shared__ unsigned count[kSpBins];
    const int row = blockIdx.y;
    const SampleRow r = sp_row(a, row);
    const unsigned key = (unsigned)(sp_top(a, row) >> 32);
    if (!(r.t > 0.0) || key <= kSpNone) return;  // greedy, or no token
    const float top = sp_logit(key);
    const double c = 1.4426950408889634074 / r.t;
    for (int b = threadIdx.x; b < kSpBins; b += kSpThreads) mass[b] = 0, count[b] = 0;
    __syncthreads();
    const T* z = reinterpret_cast<const T*>(a.z) + (int64_t)row * a.vocab;
    const int v0 = (int)blockIdx.x * a.slice, v1 = v0 + a.slice < a.vocab ? v0 + a.slice : a.vocab;
    for (int v = v0 + (int)threadIdx.x * 8; v < v1; v += kSpThreads * 8) {
        float f[8];
        load8(z, v, v1, f);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if (v + e >= v1 || !(f[e] > -INFINITY)) continue;
            const int b = sp_bin(top, f[e]);
            atomicAdd(&count[b], 1u);
            const u64 m = sp_mass(top, f[e], c, a.shift);
            if (m) atomicAdd(&mass[b], m);
        }
    }
    __syncthreads();
    for (int b = threadIdx.x; b < kSpBins; b += kSpThreads) {
        if (count[b]) {
            atomicAdd(&a.count[(int64_t)row * kSpBins + b], count[b]);
            atomicAdd(&a.mass[(int64_t)row * kSpBins + b], mass[b]);
        }
    }
}

// A place in the row's order: everything before it has `count` tokens and `mass`; it is the tie-th token (from 0)
// of those with this key.
struct SamplePlace {
    unsigned key;
    int64_t tie;
    u64 count, mass;  // before it
    u64 own;          // its mass
    int index;        // -1: not known yet
};

// One block's working memory.
struct SampleShared {
    u64 mass[kSpBins];
    unsigned count[kSpBins];
    u64 list[kSpList];      // key, complement of the index
    u64 wmass[kSpPick / 64];
    unsigned wcount[kSpPick / 64];
    unsigned n, lo, hi;
    int at;
    u64 before_mass, found;
    unsigned before_count;
    SamplePlace place;
};

// Exclusive sums of c and m over the block's threads, in their order.
__device__ __forceinline__ void sp_scan(SampleShared& s, unsigned& c, u64& m, unsigned& all_c, u64& all_m) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    unsigned ic = c;
    u64 im = m;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const unsigned oc = __shfl_up(ic, off, kWave);
        const u64 om = __shfl_up(im, off, kWave);
        if (lane >= off) ic += oc, im += om;
    }
    __syncthreads();
    if (lane == 63) s.wcount[wave] = ic, s.wmass[wave] = im;
    __syncthreads();
    unsigned bc = 0;
    u64 bm = 0;
    all_c = 0, all_m = 0;
#pragma unroll
    for (int w = 0; w < kSpPick / 64; ++w) {
        if (w == wave) bc = all_c, bm = all_m;
        all_c += s.wcount[w], all_m += s.wmass[w];
    }
    c = bc + ic - c, m = bm + im - m;
}

// Which bin of s.mass / s.count is the first whose end reaches the goal: `goal_c` tokens, or with kByMass a mass
// of at least (kPast: above) `goal_m`. s.at: the bin (-1: none), s.before_*: what lies before it, base included.
template <bool kByMass, bool kPast>
__device__ __forceinline__ void sp_find_bin(SampleShared& s, u64 base_c, u64 base_m, u64 goal_c, double goal_m) {
    constexpr int kPer = kSpBins / kSpPick;
    static_assert(kPer * kSpPick == kSpBins && kSpList % kSpPick == 0, "whole shares");
    unsigned c[kPer], tc = 0, all_c;
    u64 m[kPer], tm = 0, all_m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        c[i] = s.count[threadIdx.x * kPer + i], m[i] = s.mass[threadIdx.x * kPer + i];
        tc += c[i], tm += m[i];
    }
    if (threadIdx.x == 0) s.at = -1;
    unsigned pc = tc;
    u64 pm = tm;
    sp_scan(s, pc, pm, all_c, all_m);
    __syncthreads();
    auto reached = [&](u64 cc, u64 mm) { return kByMass ? (kPast ? (double)mm > goal_m : (double)mm >= goal_m) : cc >= goal_c; };
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        // the one bin that is reached and whose start is not
        if (c[i] && reached(base_c + pc + c[i], base_m + pm + m[i]) && !reached(base_c + pc, base_m + pm)) {
            s.at = (int)threadIdx.x * kPer + i;
            s.before_count = pc, s.before_mass = pm;
        }
        pc += c[i], pm += m[i];
    }
    __syncthreads();
}

// Calls f(key, index, logit) for the row's tokens, by the whole block: 32 logits a thread are read at once.
template <typename T, typename F>
__device__ __forceinline__ void sp_all(const T* z, int vocab, F f) {
    constexpr int kU = 4;
    for (int v0 = (int)threadIdx.x * 8; v0 < vocab; v0 += kSpPick * 8 * kU) {
        float x[kU][8];
#pragma unroll
        for (int i = 0; i < kU; ++i) load8(z, v0 + i * kSpPick * 8, vocab, x[i]);
#pragma unroll
        for (int i = 0; i < kU; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int v = v0 + i * kSpPick * 8 + e;
                const unsigned key = sp_key(x[i][e]);
                if (v < vocab && key > kSpNone) f(key, v, x[i][e]);
            }
    }
}
// For those of bin `bin` with keys in [lo, hi].
template <typename T, typename F>
__device__ __forceinline__ void sp_each(const T* z, int vocab, float top, int bin, unsigned lo, unsigned hi, F f) {
    sp_all(z, vocab, [&](unsigned key, int v, float x) {
        if (key >= lo && key <= hi && sp_bin(top, x) == bin) f(key, v, x);
    });
}

// The token of the row's order on which a count (`goal_c`: the goal_c-th token is the answer) or a mass falls
// (kByMass: the first whose running mass is at least, or with kPast above, goal_m). mass0 / count0: the row's bins
// in global memory. The answer is in s.place; goals lie within the row.
template <typename T, bool kByMass, bool kPast>
__device__ void sp_locate(const SampleArgs& a, SampleShared& s, const T* z, int row, float top, double c, u64 goal_c, double goal_m) {
    __syncthreads();
    for (int b = threadIdx.x; b < kSpBins; b += kSpPick) {
        s.mass[b] = a.mass[(int64_t)row * kSpBins + b];
        s.count[b] = a.count[(int64_t)row * kSpBins + b];
    }
    sp_find_bin<kByMass, kPast>(s, 0, 0, goal_c, goal_m);
    const int bin = s.at;
    if (bin < 0) {  // not within the row: the caller's goals rule it out
        if (threadIdx.x == 0) s.place = SamplePlace{kSpNone, 0, 0, 0, 0, 0};
        __syncthreads();
        return;
    }
    u64 base_c = s.before_count, base_m = s.before_mass;
    unsigned lo = 0, hi = 0xffffffffu, n = s.count[bin];
    // too many to sort: split the keys' span in 1024 until few are left, or one key
    while (n > kSpList) {
        __syncthreads();
        if (threadIdx.x == 0) s.lo = 0xffffffffu, s.hi = 0;
        for (int b = threadIdx.x; b < kSpBins; b += kSpPick) s.mass[b] = 0, s.count[b] = 0;
        __syncthreads();
        unsigned klo = 0xffffffffu, khi = 0;
        sp_each(z, a.vocab, top, bin, lo, hi, [&](unsigned key, int, float) {
            klo = key < klo ? key : klo;
            khi = key > khi ? key : khi;
        });
        atomicMin(&s.lo, klo);
        atomicMax(&s.hi, khi);
        __syncthreads();
        lo = s.lo, hi = s.hi;
        if (lo == hi) break;
        int shift = 0;
        while ((hi - lo) >> shift >= (unsigned)kSpBins) ++shift;
        // from the largest key down
        sp_each(z, a.vocab, top, bin, lo, hi, [&](unsigned key, int, float x) {
            const int b = (int)((hi - key) >> shift);
            atomicAdd(&s.count[b], 1u);
            atomicAdd(&s.mass[b], sp_mass(top, x, c, a.shift));
        });
        sp_find_bin<kByMass, kPast>(s, base_c, base_m, goal_c, goal_m);
        const unsigned b = s.at < 0 ? 0u : (unsigned)s.at;
        base_c += s.before_count, base_m += s.before_mass;
        n = s.count[b];
        const unsigned new_hi = hi - (b << shift);
        const unsigned span = (1u << shift) - 1u;
        lo = new_hi - lo > span ? new_hi - span : lo;
        hi = new_hi;
    }
    __syncthreads();
    if (n > kSpList) {  // equal logits: which of them, by division
        if (threadIdx.x == 0) {
            const u64 own = sp_mass(top, sp_logit(hi), c, a.shift);
            int64_t tie;
            if constexpr (!kByMass) {
                tie = (int64_t)(goal_c - base_c) - 1;
            } else {
                auto reached = [&](int64_t t) {  // with t of them
                    const double m = (double)(base_m + (u64)t * own);
                    return kPast ? m > goal_m : m >= goal_m;
                };
                int64_t few = 0, many = n;  // not reached with few, reached with many
                while (many - few > 1) {
                    const int64_t mid = (few + many) / 2;
                    if (reached(mid)) many = mid;
                    else few = mid;
                }
                tie = many - 1;
            }
            s.place = SamplePlace{hi, tie, base_c + (u64)tie, base_m + (u64)tie * own, own, -1};
        }
        __syncthreads();
        return;
    }
    // few: gather, sort from the largest key (and the lowest index) down, add up
    if (threadIdx.x == 0) s.n = 0;
    unsigned size = 64;
    while (size < n) size <<= 1;
    __syncthreads();
    sp_each(z, a.vocab, top, bin, lo, hi, [&](unsigned key, int v, float) {
        const unsigned i = atomicAdd(&s.n, 1u);
        if (i < (unsigned)kSpList) s.list[i] = (u64)key << 32 | (unsigned)~v;
    });
    __syncthreads();
    for (unsigned i = threadIdx.x; i < size; i += kSpPick)
        if (i >= n) s.list[i] = 0;
    for (unsigned w = 2; w <= size; w <<= 1)
        for (unsigned d = w >> 1; d > 0; d >>= 1) {
            __syncthreads();
            for (unsigned i = threadIdx.x; i < size / 2; i += kSpPick) {
                const unsigned x = 2 * i - (i & (d - 1)), y = x + d;
                const u64 p = s.list[x], q = s.list[y];
                if ((p < q) == ((x & w) == 0)) s.list[x] = q, s.list[y] = p;
            }
        }
    __syncthreads();
    constexpr int kPer = kSpList / kSpPick;
    u64 m[kPer], tm = 0, all_m;
    unsigned tc = 0, all_c;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const unsigned j = threadIdx.x * kPer + i;
        m[i] = j < n ? sp_mass(top, sp_logit((unsigned)(s.list[j] >> 32)), c, a.shift) : 0;
        tm += m[i];
    }
    u64 pm = tm;
    sp_scan(s, tc, pm, all_c, all_m);
    auto reached = [&](u64 cc, u64 mm) { return kByMass ? (kPast ? (double)mm > goal_m : (double)mm >= goal_m) : cc >= goal_c; };
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const unsigned j = threadIdx.x * kPer + i;
        const u64 bm = base_m + pm, bc = base_c + j;
        if (j < n && reached(bc + 1, bm + m[i]) && !reached(bc, bm)) {
            const unsigned key = (unsigned)(s.list[j] >> 32);
            unsigned less = 0, more = j;  // the first of its ties
            while (less < more) {
                const unsigned mid = (less + more) / 2;
                if ((unsigned)(s.list[mid] >> 32) > key) less = mid + 1;
                else more = mid;
            }
            s.place = SamplePlace{key, (int64_t)(j - less), bc, bm, m[i], (int)~(unsigned)s.list[j]};
        }
        pm += m[i];
    }
    __syncthreads();
}

// The index of the tie-th token with this key.
template <typename T>
__device__ __forceinline__ int sp_index(SampleShared& s, const T* z, int vocab, unsigned key, int64_t tie) {
    __syncthreads();
    if (threadIdx.x == 0) s.at = 0;
    int64_t before = 0;
    for (int v0 = 0; v0 < vocab; v0 += kSpPick * 8) {
        const int v = v0 + (int)threadIdx.x * 8;
        float x[8];
        unsigned mine = 0, c, all_c;
        u64 none = 0, all_m;
        if (v < vocab) {
            load8(z, v, vocab, x);
#pragma unroll
            for (int e = 0; e < 8; ++e) mine += v + e < vocab && sp_key(x[e]) == key;
        }
        c = mine;
        sp_scan(s, c, none, all_c, all_m);
        int64_t at = before + c;
        if (mine && at <= tie && at + mine > tie) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (v + e < vocab && sp_key(x[e]) == key && at++ == tie) s.at = v + e;
        }
        before += all_c;
        if (before > tie) break;
    }
    __syncthreads();
    return s.at;
}

template <typename T>
__global__ __launch_bounds__(kSpPick) void sample_pick_kernel(SampleArgs a) {
    __shared__ SampleShared s;
    const int row = blockIdx.x;
    const T* z = reinterpret_cast<const T*>(a.z) + (int64_t)row * a.vocab;
    const SampleRow r = sp_row(a, row);
    const u64 first = sp_top(a, row);
    const unsigned key = (unsigned)(first >> 32);
    if (!(r.t > 0.0) || key <= kSpNone) {
        if (threadIdx.x == 0) {
            a.token[row] = key <= kSpNone ? -1 : (int64_t)(int)~(unsigned)first;
            if (a.logprob) a.logprob[row] = key <= kSpNone ? __builtin_nanf("") : 0.f;
        }
        return;
    }
    const float top = sp_logit(key);
    const double c = 1.4426950408889634074 / r.t;
    // all tokens and their mass
    unsigned tc = 0, tokens;
    u64 tm = 0, total;
    for (int b = threadIdx.x; b < kSpBins; b += kSpPick) {
        tc += a.count[(int64_t)row * kSpBins + b];
        tm += a.mass[(int64_t)row * kSpBins + b];
    }
    sp_scan(s, tc, tm, tokens, total);
    // the kept prefix ends behind (end_key, end_tie) and has `kept` of mass
    unsigned end_key = 0;
    int64_t end_tie = a.vocab;
    u64 kept = total;
    if (r.k < (int64_t)tokens) {
        sp_locate<T, false, false>(a, s, z, row, top, c, (u64)r.k, 0.0);
        end_key = s.place.key, end_tie = s.place.tie, kept = s.place.mass + s.place.own;
    }
    if (r.p < 1.0) {
        // the token that reaches p of the k's mass is the last; the first stays whatever p is
        const double goal = r.p > 0.0 ? r.p * (double)kept : 0.0;
        sp_locate<T, true, false>(a, s, z, row, top, c, 0, goal > 0.0 ? goal : 1.0);
        const SamplePlace q = s.place;
        if (q.key > end_key || (q.key == end_key && q.tie < end_tie)) end_key = q.key, end_tie = q.tie, kept = q.mass + q.own;
    }
    if (r.m > 0.0) {
        const double m = r.m < 1.0 ? r.m : 1.0;
        // mass falls with the key: the lowest key with mass >= m, found in 64 steps a time
        unsigned lo = kSpNone + 1, hi = key;  // hi has it
        while (lo < hi) {
            const unsigned span = hi - lo, step = span / 64 + 1, lane = threadIdx.x & 63;
            const u64 probe = (u64)lo + (u64)step * lane;  // 64 places from lo up
            const bool in = probe < hi;
            const double x = in ? ((double)sp_logit((unsigned)probe) - (double)top) / r.t : 0.0;
            const bool has = !in || exp(x) >= m;
            const u64 votes = __ballot(has);  // from some lane on; lanes past hi have it
            if (votes == 0) {
                const u64 next = (u64)lo + (u64)step * 63 + 1;
                lo = next < hi ? (unsigned)next : hi;
                continue;
            }
            const unsigned firsthas = (unsigned)__ffsll((unsigned long long)votes) - 1;
            const u64 nh = (u64)lo + (u64)step * firsthas;
            const unsigned new_hi = nh < hi ? (unsigned)nh : hi;
            const unsigned new_lo = firsthas ? (unsigned)((u64)lo + (u64)step * (firsthas - 1) + 1) : new_hi;
            hi = new_hi, lo = new_lo < new_hi ? new_lo : new_hi;
        }
        if (hi > end_key) {
            // the mass down to that key
            u64 mine = 0;
            sp_all(z, a.vocab, [&](unsigned k, int, float x) {
                if (k >= hi) mine += sp_mass(top, x, c, a.shift);
            });
            unsigned none = 0, all_c;
            u64 all;
            sp_scan(s, none, mine, all_c, all);
            end_key = hi, end_tie = a.vocab, kept = all;
        }
    }
    const double u = (double)a.u[row];
    // u below 1 falls within the kept mass; others are taken to its ends
    double goal = u > 0.0 ? u * (double)kept : 0.0;
    const double most = (double)kept * (1.0 - 0x1p-50);
    goal = goal < most ? goal : most;
    sp_locate<T, true, true>(a, s, z, row, top, c, 0, goal);
    const SamplePlace q = s.place;
    const int index = q.index >= 0 ? q.index : sp_index(s, z, a.vocab, q.key, q.tie);
    if (threadIdx.x == 0) {
        a.token[row] = index;
        if (a.logprob) {
            const float x = sp_logit(q.key);
            a.logprob[row] = (float)((x == top ? 0.0 : ((double)x - (double)top) / r.t) - log(ldexp((double)kept, -a.shift)));
        }
    }
}

// Slices of a row: enough blocks to fill the card (four a CU), none below 2048 logits.
static int sample_slices(int64_t rows, int64_t vocab) {
    const int64_t most = std::max<int64_t>(1, std::min<int64_t>(kSpSlices, vocab / 2048));
    return (int)std::max<int64_t>(1, std::min(most, (1024 + rows - 1) / rows));
}
constexpr int64_t kSpRows = 32768;  // of a launch (grids hold 65535)
size_t sample_workspace(int64_t rows, int64_t vocab) {
    rows = std::min(rows, kSpRows);
    return (size_t)rows * ((size_t)sample_slices(rows, vocab) * 8 + kSpBins * 12);
}

template <typename T>
static int sample_t(const SampleArgs& a, hipStream_t stream) {
    const dim3 grid((unsigned)a.slices, (unsigned)a.rows);
    hipLaunchKernelGGL((sample_top_kernel<T>), grid, dim3(kSpThreads), 0, stream, a);
    hipLaunchKernelGGL((sample_bins_kernel<T>), grid, dim3(kSpThreads), 0, stream, a);
    hipLaunchKernelGGL((sample_pick_kernel<T>), dim3((unsigned)a.rows), dim3(kSpPick), 0, stream, a);
    return hipGetLastError() == hipSuccess ? M3_OK : M3_ERR_LAUNCH;
}

int launch_sample(const void* logits, int dtype, int64_t rows, int vocab, const float* u, const float* temperature,
                  double temperature1, const int32_t* top_k, int64_t top_k1, const float* top_p, double top_p1,
                  const float* min_p, double min_p1, int64_t* token, float* logprob, void* ws, hipStream_t stream) {
    SampleArgs a;
    a.temperature1 = temperature1, a.top_p1 = top_p1, a.min_p1 = min_p1, a.top_k1 = top_k1;
    a.vocab = vocab;
    a.slices = sample_slices(std::min(rows, kSpRows), vocab);
    a.slice = (vocab + a.slices - 1) / a.slices;
    a.mass = reinterpret_cast<u64*>(ws);
    a.top = a.mass + std::min(rows, kSpRows) * kSpBins;
    a.count = reinterpret_cast<unsigned*>(a.top + std::min(rows, kSpRows) * a.slices);
    int bits = 0;
    while (((int64_t)1 << bits) < vocab) ++bits;
    a.shift = 62 - bits;  // a whole row's mass stays below 2^62
    const int size = dtype == M3_DTYPE_BF16 ? 2 : 4;
    for (int64_t r = 0; r < rows; r += kSpRows) {
        a.rows = (int)std::min(rows - r, kSpRows);
        a.z = reinterpret_cast<const char*>(logits) + r * vocab * size;
        a.u = u + r;
        a.temperature = temperature ? temperature + r : nullptr;
        a.top_k = top_k ? top_k + r : nullptr;
        a.top_p = top_p ? top_p + r : nullptr;
        a.min_p = min_p ? min_p + r : nullptr;
        a.token = token + r;
        a.logprob = logprob ? logprob + r : nullptr;
        const int st = dtype == M3_DTYPE_BF16 ? sample_t<bf16>(a, stream) : sample_t<float>(a, stream);
        if (st != M3_OK) return st;
    }
    return M3_OK;
}

}  // namespace m3
