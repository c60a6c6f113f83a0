// Tiled matrix products for the training operators (gfx950, wave64), bf16 or fp32 operands
// with fp32 accumulation:
//   C[m][n] = sum over k of A(m, k) B(n, k),
// each operand stored either with k contiguous (rows of k) or with its own index contiguous
// (rows of m or n), so that x W^T, dy W and dy^T x all run on one kernel without a transposed
// copy. Epilogues get the fp32 accumulators (m3_mlp.hip, m3_xent.hip).
//
// A block of WGM x WGN waves owns a BM x BN tile and walks k in steps of 128 bytes per row
// (64 bf16 or 32 fp32). Tiles go from HBM straight to LDS (16 bytes a lane, no registers in
// between), STAGES deep; operand reads past the end of a row or of the array return zero by
// the buffer descriptor's bound, so ragged edges cost no branch. LDS rows are XOR-swizzled by
// choosing which 16 bytes each lane fetches:
//   k-contiguous tiles: [row][8 pieces], piece c of row r at c ^ (r & 7);
//   others: [k][row of m or n], 32-byte units (bf16) or 64-byte units (fp32) at u ^ key(k),
// which leaves the ds_read_b128 / ds_read_b64_tr_b16 / ds_read_b32 operand reads without
// bank conflicts beyond the two cycles that 512 bytes need.
//
// The MFMA takes B as its first operand: a lane then holds four consecutive n of one row m,
// and epilogues load and store 8 or 16 bytes a lane.
#pragma once

#include "m3_common.h"
#include "m3_mfma.h"

namespace m3 {

constexpr unsigned kOob = 0x80000000u;  // a byte offset past every descriptor's bound

template <typename T> struct GemmType;
template <> struct GemmType<bf16> {
    typedef bf16x8 Frag;  // 8 consecutive k of one row
    static __device__ __forceinline__ f32x4 mma(Frag b, Frag a, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(b, a, c, 0, 0, 0);
    }
};
template <> struct GemmType<float> {
    typedef f32x4 Frag;  // 4 consecutive k of one row: MFMA j takes element j of every lane
    static __device__ __forceinline__ f32x4 mma(Frag b, Frag a, f32x4 c) {
#pragma unroll
        for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(b[j], a[j], c, 0, 0, 0);
        return c;
    }
};

// One operand of a product. kc: rows of k (p[row * ld + k]); else rows of m or n
// (p[k * ld + row]). 16-byte aligned, ld * sizeof(T) a multiple of 16.
struct GemmOp {
    const void* p;
    int64_t ld;
};

// Two terms (kSeg2: C = A0 B0 + A1 B1), two problems (kBatch2: blockIdx.y) or two B halves
// of a tile (kGated: columns [0, BN/2) from B0 and [BN/2, BN) from B1).
enum GemmMode { kPlain, kSeg2, kBatch2, kGated };

struct GemmArgs {
    GemmOp a[2], b[2];
    int M, N;    // rows of A and of B (kGated: of one half): what the tiles may read
    int K[2];    // inner lengths of the terms; multiples of 16 bytes for k-contiguous operands
    int KB[2];   // rows of B that exist where B is not k-contiguous (<= K: the rest reads as zero)
    int splits;  // k is cut into so many parts (blockIdx.z)
    int tiles_m, tiles_n;
};

// Global -> LDS copies of one operand's tile by the whole block.
template <typename T, bool kKc, int BX, int NW>
struct GemmLoader {
    static constexpr int kInstr = BX * 128 / 1024;  // wave instructions a tile
    static constexpr int NI = kInstr / NW;          // of which each wave issues NI
    static constexpr int SZ = sizeof(T);
    static constexpr int CPR = kKc ? 8 : BX * SZ / 16;  // 16-byte pieces a row
    static constexpr int RPI = 64 / CPR;                // rows an instruction
    static_assert(kInstr % NW == 0 && NI >= 1, "tile too small for the block");
    unsigned voff[NI];
    int piece;  // kKc: the lane's 16-byte piece of the row

    // row0: first row of this wave's part when it differs from its place in the tile (kGated)
    __device__ __forceinline__ void init(int wave, int lane, int64_t ld, int row_shift) {
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int r = (wave * NI + i) * RPI + lane / CPR, c = lane % CPR;
            if constexpr (kKc) {
                piece = c ^ (r & 7);
                voff[i] = (unsigned)((r - row_shift) * (int)ld * SZ + piece * 16);
            } else if constexpr (SZ == 2) {
                const int key = ((r & 3) | ((r >> 3) & 3) << 2) & (BX / 16 - 1);
                voff[i] = (unsigned)(r * (int)ld * SZ + (((c >> 1) ^ key) << 1 | (c & 1)) * 16);
            } else {
                const int key = (r >> 2) & 3;
                voff[i] = (unsigned)(r * (int)ld * SZ + (((c >> 2) ^ key) << 2 | (c & 3)) * 16);
            }
        }
    }
    // bytes: what the descriptor spans; pieces: valid 16-byte pieces of the rows (kKc)
    __device__ __forceinline__ void issue(const char* base, int64_t bytes, int pieces, char* lds, int wave) const {
        const __amdgpu_buffer_rsrc_t rs = make_rsrc(base, bytes < 0 ? 0 : bytes);
        const bool live = !kKc || piece < pieces;
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const unsigned v = live ? voff[i] : kOob;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(
                rs, (__attribute__((address_space(3))) void*)(lds + (wave * NI + i) * 1024), 16, (int)v, 0, 0, 0);
        }
    }
};

// LDS -> MFMA operand: 16 rows (unit u of the tile), k step ks (of two).
template <typename T, bool kKc, int BX>
struct GemmReader {
    typedef typename GemmType<T>::Frag Frag;
    int off[2];
    int key;
    __device__ __forceinline__ void init(int lane) {
        const int r = lane & 15, g = lane >> 4;
        if constexpr (kKc) {
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) off[ks] = r * 128 + (((ks * 4 + g) ^ (r & 7)) * 16);
        } else if constexpr (sizeof(T) == 2) {
            key = (r >> 2 | g << 2) & (BX / 16 - 1);
            off[0] = (g * 8 + (r >> 2)) * (BX * 2) + (r & 3) * 8;
        } else {
            key = g;
            off[0] = g * 4 * (BX * 4) + r * 4;
        }
    }
    __device__ __forceinline__ Frag read(const char* tile, int u, int ks) const {
        if constexpr (kKc) {
            return *reinterpret_cast<const Frag*>(tile + u * 2048 + off[ks]);
        } else if constexpr (sizeof(T) == 2) {
            const char* p = tile + off[0] + ((u ^ key) << 5) + ks * 32 * (BX * 2);
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p);
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (__attribute__((address_space(3))) s16x4*)(p + 4 * (BX * 2)));
            const bf16x4 l4 = __builtin_bit_cast(bf16x4, lo), h4 = __builtin_bit_cast(bf16x4, hi);
            return __builtin_shufflevector(l4, h4, 0, 1, 2, 3, 4, 5, 6, 7);
        } else {
            const char* p = tile + off[0] + ((u ^ key) << 6) + ks * 16 * (BX * 4);
            Frag f;
#pragma unroll
            for (int j = 0; j < 4; ++j) f[j] = *reinterpret_cast<const float*>(p + j * (BX * 4));
            return f;
        }
    }
};

template <int kN>
__device__ __forceinline__ void wait_vm_lds() {  // at most kN loads in flight, no LDS read
    __builtin_amdgcn_s_waitcnt((kN & 15) | (7 << 4) | ((kN >> 4) << 14));
}

template <int BM_, int BN_, int WGM_, int WGN_, int STAGES_>
struct GemmTile {
    static constexpr int BM = BM_, BN = BN_, WGM = WGM_, WGN = WGN_, STAGES = STAGES_;
    static constexpr int NW = WGM * WGN, NT = NW * 64;
    static constexpr int FM = BM / WGM / 16, FN = BN / WGN / 16;  // 16 x 16 pieces of a wave
    static constexpr int kStageBytes = (BM + BN) * 128;
    static constexpr int kLds = STAGES * kStageBytes;
};

// Where a wave's accumulators lie: piece (fm, fn), lane: row m(fm), columns n(fn) .. n(fn) + 3.
template <typename Tile, int kMode>
struct GemmPlace {
    int m0, n0, wm, wn, lane;
    __device__ __forceinline__ int local_m(int fm) const { return (wm * Tile::FM + fm) * 16 + (lane & 15); }
    __device__ __forceinline__ int m(int fm) const { return m0 + local_m(fm); }
    // kGated: fn < FN / 2 of the gate; the up piece of the same columns is fn + FN / 2
    __device__ __forceinline__ int n(int fn) const {
        constexpr int F = kMode == kGated ? Tile::FN / 2 : Tile::FN;
        return n0 + (wn * F + fn) * 16 + (lane >> 4) * 4;
    }
};

// Block -> tile: the blocks of one XCD (dispatch is round robin over 8) take a contiguous run of
// tiles, and runs walk groups of 8 row tiles column by column, so that an XCD's L2 serves
// both operands.
__device__ __forceinline__ void gemm_tile_of(int tiles_m, int tiles_n, int& tm, int& tn) {
    const int total = tiles_m * tiles_n, b = (int)blockIdx.x;
    const int x = b & 7, per = total >> 3, rest = total & 7;
    const int id = x * per + (x < rest ? x : rest) + (b >> 3);
    constexpr int G = 8;
    const int group = id / (G * tiles_n), first = group * G;
    const int rows = tiles_m - first < G ? tiles_m - first : G;
    const int in = id - group * (G * tiles_n);
    tm = first + in % rows;
    tn = in / rows;
}

template <typename T, typename Tile, bool kAKc, bool kBKc, int kMode, typename Epi>
__global__ __launch_bounds__(Tile::NT, Tile::NT >= 512 ? 2 : 1) void gemm_kernel(GemmArgs a, Epi epi) {
    constexpr int BM = Tile::BM, BN = Tile::BN, FM = Tile::FM, FN = Tile::FN, ST = Tile::STAGES;
    constexpr int BK = 128 / sizeof(T), SZ = sizeof(T);
    typedef GemmLoader<T, kAKc, BM, Tile::NW> LA;
    typedef GemmLoader<T, kBKc, BN, Tile::NW> LB;
    constexpr int NLD = LA::NI + LB::NI;
    extern __shared__ __align__(16) char gemm_smem[];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int tm, tn;
    gemm_tile_of(a.tiles_m, a.tiles_n, tm, tn);
    const int m0 = tm * BM, n0 = tn * (kMode == kGated ? BN / 2 : BN);
    const int z = kMode == kBatch2 ? (int)blockIdx.y : 0;

    // the k steps of this block: steps [s0, s1) of the terms' steps in a row
    const int st0 = (a.K[0] + BK - 1) / BK;
    const int steps = st0 + (kMode == kSeg2 ? (a.K[1] + BK - 1) / BK : 0);
    const int s0 = (int)((int64_t)steps * blockIdx.z / a.splits), s1 = (int)((int64_t)steps * (blockIdx.z + 1) / a.splits);

    const bool second = kMode == kGated && wave * LB::NI >= LB::kInstr / 2;
    static_assert(kMode != kGated || (LB::kInstr / 2) % LB::NI == 0, "a wave fetches from one half");
    LA la;
    LB lb;
    la.init(wave, lane, a.a[z].ld, 0);
    lb.init(wave, lane, a.b[z].ld, second ? BN / 2 : 0);

    auto issue = [&](int s, int slot) {
        const int seg = kMode == kSeg2 && s >= st0 ? 1 : 0;
        const int k0 = (seg ? s - st0 : s) * BK;
        const int krem = s < s1 ? a.K[seg] - k0 : 0;
        const int ia = kMode == kSeg2 ? seg : z, ib = kMode == kGated ? (second ? 1 : 0) : ia;
        char* sl = gemm_smem + slot * Tile::kStageBytes;
        const int64_t lda = a.a[ia].ld, ldb = a.b[ib].ld;
        const char* pa = reinterpret_cast<const char*>(a.a[ia].p);
        const char* pb = reinterpret_cast<const char*>(a.b[ib].p);
        // spans end with the last valid row's last valid element
        if constexpr (kAKc) pa += (m0 * lda + k0) * SZ;
        else pa += (k0 * lda + m0) * SZ;
        if constexpr (kBKc) pb += (n0 * ldb + k0) * SZ;
        else pb += (k0 * ldb + n0) * SZ;
        const int64_t ba = krem <= 0 ? 0 : kAKc ? ((int64_t)(a.M - m0 - 1) * lda + krem) * SZ : ((int64_t)(krem - 1) * lda + (a.M - m0)) * SZ;
        const int kb = kBKc || krem <= 0 ? krem : a.KB[seg] - k0;
        const int64_t bb = kb <= 0 ? 0 : kBKc ? ((int64_t)(a.N - n0 - 1) * ldb + kb) * SZ : ((int64_t)(kb - 1) * ldb + (a.N - n0)) * SZ;
        const int pieces = krem <= 0 ? 0 : (krem * SZ) >> 4;
        la.issue(pa, ba, pieces, sl, wave);
        lb.issue(pb, bb, pieces, sl + BM * 128, wave);
    };

    GemmReader<T, kAKc, BM> ra;
    GemmReader<T, kBKc, BN> rb;
    ra.init(lane);
    rb.init(lane);
    const int wm = wave / Tile::WGN, wn = wave % Tile::WGN;
    auto unit_b = [&](int fn) {
        if constexpr (kMode == kGated)
            return fn < FN / 2 ? wn * (FN / 2) + fn : BN / 32 + wn * (FN / 2) + fn - FN / 2;
        else
            return wn * FN + fn;
    };

    f32x4 acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

#pragma unroll
    for (int s = 0; s < ST - 1; ++s) issue(s0 + s, s);
    int slot = 0;
    for (int s = s0; s < s1; ++s) {
        // step s has landed, and every wave has read step s - 1 out of the slot to be refilled
        wait_vm_lds<NLD * (ST - 2)>();
        M3_LDS_FENCE();
        __builtin_amdgcn_s_barrier();
        M3_LDS_FENCE();
        {
            int next = slot + ST - 1;
            next = next >= ST ? next - ST : next;
            issue(s + ST - 1, next);
        }
        const char* ta = gemm_smem + slot * Tile::kStageBytes;
        const char* tb = ta + BM * 128;
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            typename GemmType<T>::Frag fa[FM], fb[FN];
#pragma unroll
            for (int j = 0; j < FN; ++j) fb[j] = rb.read(tb, unit_b(j), ks);
#pragma unroll
            for (int i = 0; i < FM; ++i) fa[i] = ra.read(ta, wm * FM + i, ks);
#pragma unroll
            for (int i = 0; i < FM; ++i)
#pragma unroll
                for (int j = 0; j < FN; ++j) acc[i][j] = GemmType<T>::mma(fb[j], fa[i], acc[i][j]);
        }
        slot = slot + 1 == ST ? 0 : slot + 1;
    }
    wait_vm_lds<0>();  // nothing writes LDS once the epilogue uses it
    M3_LDS_FENCE();
    __builtin_amdgcn_s_barrier();
    M3_LDS_FENCE();
    const GemmPlace<Tile, kMode> at{m0, n0, wm, wn, lane};
    epi.template run<T, Tile, kMode>(a, at, acc, gemm_smem, tm, tn, z);
}

}  // namespace m3
