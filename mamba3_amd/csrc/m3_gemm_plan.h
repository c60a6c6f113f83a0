// Tile and split choice of the tiled products (m3_gemm.h): plain C++ on the host, without HIP.
#pragma once

#include <algorithm>
#include <cstdint>

namespace m3 {

enum { kTileL = 0, kTileM = 1, kTileS = 2 };

// One product to be planned: rows x cols results (for a gated product, cols counts both halves) over
// k steps of 128 bytes; max_splits 1 where the epilogue needs the whole sum; tn: both operands in rows of
// m and n.
struct GemmTask {
    int64_t rows, cols, steps;
    int max_splits;
    bool tn;
};
constexpr int kGroupMax = 4;
constexpr int kMaxSplits = 16;
// Of a product whose inner length is the vocabulary: a few rows' tiles are few, and each is one chain of
// additions over thousands of steps (rows 16 x 64 over 128000 tokens in fp32: 291 us in 16 parts, 95 in 64
// by the estimate below).
constexpr int kMostSplits = 64;
struct GemmGroupPlan {
    int tile;
    int splits[kGroupMax];
    double us = 0;  // estimated
};

// Estimated us of each choice, from launches of 256, 512 and 1024 tiles of 8 and 64 k steps (torch on the
// same card: 8192^3 bf16 668 us): a step of a 256 x 256 tile takes 1.45 us (1.38 where both operands
// are rows of m and n), of a 128 x 128 tile 0.62 us alone on its CU and 0.90 us (1.05) next to another, of a
// 64 x 64 tile 0.20 and 0.37 us; to that come a tile's start and epilogue. Parts of k cost the
// fp32 partial sums' write and read and a launch.
// What it decides, both sides measured: the gated product of 8192 x 11008 x 2048 takes 80 us less on 256 x 256
// tiles than on 128 x 128, that of 8192 x 4224 x 768 8 us more; the 8192 x 768 product over 16128 takes
// 33 us less in two parts on 256 x 256 tiles than whole on 128 x 128.
struct TileCost { int size, at_once; double alone, all, tn, fixed; };
inline const TileCost* tile_costs(bool bf16) {
    static const TileCost b[3] = {{256, 1, 1.45, 1.45, 1.38, 8.0}, {128, 2, 0.62, 0.90, 1.05, 4.5}, {64, 2, 0.20, 0.37, 0.38, 3.5}};
    static const TileCost f[3] = {{0, 0, 0, 0, 0, 0}, {128, 2, 1.90, 3.60, 3.60, 5.0}, {64, 2, 0.65, 1.07, 1.07, 4.0}};
    return bf16 ? b : f;
}

inline int64_t group_items(const TileCost& c, const GemmTask& t, int splits) {
    return ((t.rows + c.size - 1) / c.size) * ((t.cols + c.size - 1) / c.size) * splits;
}

// Rounds of as many items as run at once, each as long as its longest item.
inline double group_us(const TileCost& c, const GemmTask* t, const int* splits, int n) {
    const int64_t slots = (int64_t)256 * c.at_once;
    double us = 0, longest = 0, alone = 0;  // of the current round's items, and with a CU to themselves
    int64_t room = slots;                   // left in the current round
    bool joined = false;
    for (int p = 0; p < n; ++p) {
        int64_t items = group_items(c, t[p], splits[p]);
        if (items == 0) continue;
        const double steps = (double)((t[p].steps + splits[p] - 1) / splits[p]);
        const double one = steps * (t[p].tn ? c.tn : c.all) + c.fixed, own = std::min(one, steps * c.alone + c.fixed);
        if (splits[p] > 1) {
            us += (double)t[p].rows * t[p].cols * 8.0 * splits[p] / 5.0e6;
            joined = true;
        }
        const int64_t in = std::min(items, room);
        longest = std::max(longest, one), alone = std::max(alone, own);
        room -= in, items -= in;
        if (room == 0) us += longest, longest = alone = 0, room = slots;
        us += items / slots * one;
        items %= slots;
        if (items) longest = one, alone = own, room = slots - items;
    }
    // the last round may leave each item a CU to itself
    return us + (slots - room <= 256 ? alone : longest) + (joined ? 4.0 : 0.0);
}

// The numbers of parts of one tile size with the least estimate; s comes in as ones. A product of many
// rounds of tiles gains nothing from parts of its own, whatever else its launch holds: next to it a few tiles
// over a long k (dh of few rows over a vocabulary, beside dW's many short tiles) gain most.
inline double search_splits(const TileCost& c, const GemmTask* tasks, int n, int* s) {
    double us = group_us(c, tasks, s, n);
    auto fits = [&](int p, int k) {
        return k == 1 || (k <= tasks[p].max_splits && k <= tasks[p].steps && group_items(c, tasks[p], 1) <= (int64_t)256 * c.at_once * 6);
    };
    if (n == 2) {
        // both at once: where each product's uncut tiles take as long, neither gains alone
        static const int kTry[] = {1, 2, 3, 4, 5, 6, 7, 8, 10, 12, 14, 16, 20, 24, 28, 32, 40, 48, 56, 64};
        int v[kGroupMax] = {1, 1, 1, 1};
        for (int i : kTry) {
            if (!fits(0, i)) break;
            v[0] = i;
            for (int j : kTry) {
                if (!fits(1, j)) break;
                v[1] = j;
                const double u = group_us(c, tasks, v, n);
                if (u < us) us = u, s[0] = i, s[1] = j;
            }
        }
        return us;
    }
    // all dy^T x alike first, then one product after the other
    static const int kTry[] = {1, 2, 3, 4, 5, 6, 8, 10, 12, 16};
    int alike = 1;
    for (int k : kTry) {
        int v[kGroupMax] = {1, 1, 1, 1};
        for (int p = 0; p < n; ++p)
            if (tasks[p].tn && fits(p, k)) v[p] = k;
        const double u = group_us(c, tasks, v, n);
        if (u < us) us = u, alike = k;
    }
    for (int p = 0; p < n; ++p)
        if (tasks[p].tn && fits(p, alike)) s[p] = alike;
    for (int pass = 0; pass < 2; ++pass)
        for (int p = 0; p < n; ++p) {
            int keep = s[p];
            for (int k : kTry) {
                if (!fits(p, k)) break;
                s[p] = k;
                const double u = group_us(c, tasks, s, n);
                if (u < us) us = u, keep = k;
            }
            s[p] = keep;
        }
    return us;
}

// The tile for products of one launch and the number of k parts of each with the least estimated time.
inline GemmGroupPlan search_plan(bool bf16, const GemmTask* tasks, int n) {
    const TileCost* c = tile_costs(bf16);
    GemmGroupPlan best{kTileS, {1, 1, 1, 1}, 1e30};
    for (int t = bf16 ? kTileL : kTileM; t <= kTileS; ++t) {
        int s[kGroupMax] = {1, 1, 1, 1};
        const double us = search_splits(c[t], tasks, n, s);
        if (us < best.us) {
            best.us = us;
            best.tile = t;
            for (int p = 0; p < kGroupMax; ++p) best.splits[p] = s[p];
        }
    }
    return best;
}

// Two products, planned by `plan` (search_plan), in one launch or each in its own. Together, one fills the last round of
// the other; a few tiles over a long k and many tiles of a step or two want other tile sizes. Estimates within
// a tenth are taken for equal, and a second launch costs 5 us. (dh and dW of 16 rows x 2048 over 128000 tokens in
// fp32: 908 us together, 366 and 328 apart.)
struct GemmPairPlan {
    GemmGroupPlan p[2];  // of each product, or twice that of both
    bool apart;
};
template <typename F>
GemmPairPlan pair_plan(const GemmTask (&t)[2], F plan) {
    const GemmGroupPlan both = plan(t);
    GemmPairPlan r{{both, both}, false};
    if (t[0].rows == 0 || t[1].rows == 0) return r;
    GemmTask first[2] = {t[0], t[1]}, second[2] = {t[0], t[1]};
    first[1].rows = second[0].rows = 0;
    const GemmGroupPlan a = plan(first), b = plan(second);
    if (a.us + b.us + 5.0 < 0.9 * both.us) r = GemmPairPlan{{a, b}, true};
    return r;
}

}  // namespace m3
