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

typedef float f32x16 __attribute__((ext_vector_type(16)));

// The MFMA of a type: bf16 16 x 16 results of 32 k; fp32 MF x MF (16 or 32) of four times 4 or 2 k.
template <typename T, int MF> struct GemmType;
template <> struct GemmType<bf16, 16> {
    typedef bf16x8 Frag;  // 8 consecutive k of one row
    typedef f32x4 Acc;
    static __device__ __forceinline__ Acc mma(Frag b, Frag a, Acc c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(b, a, c, 0, 0, 0);
    }
};
template <> struct GemmType<float, 16> {
    typedef f32x4 Frag;
    typedef f32x4 Acc;
    static __device__ __forceinline__ Acc mma(Frag b, Frag a, Acc c) {
#pragma unroll
        for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(b[j], a[j], c, 0, 0, 0);
        return c;
    }
};
template <> struct GemmType<float, 32> {
    typedef f32x4 Frag;  // 4 consecutive k of one row: MFMA j takes element j of every lane
    typedef f32x16 Acc;
    static __device__ __forceinline__ Acc mma(Frag b, Frag a, Acc c) {
#pragma unroll
        for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(b[j], a[j], c, 0, 0, 0);
        return c;
    }
};

// One operand of a product. kc: rows of k (p[row * ld + k]); else rows of m or n
// (p[k * ld + row]). 16-byte aligned, ld * sizeof(T) a multiple of 16.
struct GemmOp {
    const void* p;
    int64_t ld;
};

// Two terms (kSeg2: C = A0 B0 + A1 B1) or two B halves of a tile (kGated: columns [0, BN/2) from B0
// and [BN/2, BN) from B1).
enum GemmMode { kPlain, kSeg2, kGated };

struct GemmArgs {
    GemmOp a[2], b[2];
    int M, N;    // rows of A and of B (kGated: of one half): what the tiles may read
    int K[2];    // inner lengths of the terms; multiples of 16 bytes for k-contiguous operands
    int KB[2];   // rows of B that exist where B is not k-contiguous (<= K: the rest reads as zero)
    int splits;  // k is cut into so many parts
    int tiles_m, tiles_n;
};

// Products of one launch: product p has the work ids [first[p], first[p + 1]).
template <int kN>
struct GemmGroup {
    GemmArgs a[kN];
    int first[kN + 1];
};
// One of four scalars, field by field: an index known at run time only, a loop over the products or a
// struct chosen as a whole would put the kernel argument into scratch memory.
template <typename V>
__device__ __forceinline__ V pick4(int p, V a, V b, V c, V d) {
    const V lo = p == 1 ? b : a, hi = p == 3 ? d : c;
    return p < 2 ? lo : hi;
}
#define M3_PICK(r, v, p, f) (r).f = pick4(p, (v)[0].f, (v)[1].f, (v)[2].f, (v)[3].f)

template <int kN>
__device__ __forceinline__ GemmArgs pick_args(const GemmArgs (&v)[kN], int p) {
    if constexpr (kN == 1) {
        return v[0];
    } else {
        static_assert(kN == 4, "one product or four");
        GemmArgs r;
        M3_PICK(r, v, p, a[0].p);
        M3_PICK(r, v, p, a[0].ld);
        M3_PICK(r, v, p, a[1].p);
        M3_PICK(r, v, p, a[1].ld);
        M3_PICK(r, v, p, b[0].p);
        M3_PICK(r, v, p, b[0].ld);
        M3_PICK(r, v, p, b[1].p);
        M3_PICK(r, v, p, b[1].ld);
        M3_PICK(r, v, p, K[0]);
        M3_PICK(r, v, p, K[1]);
        M3_PICK(r, v, p, KB[0]);
        M3_PICK(r, v, p, KB[1]);
        M3_PICK(r, v, p, M);
        M3_PICK(r, v, p, N);
        M3_PICK(r, v, p, splits);
        M3_PICK(r, v, p, tiles_m);
        M3_PICK(r, v, p, tiles_n);
        return r;
    }
}

// Global -> LDS copies of one operand's tile by the whole block.
template <typename T, bool kKc, int BX, int NW, int MF>
struct GemmLoader {
    static constexpr int kInstr = BX * 128 / 1024;  // wave instructions a tile
    static constexpr int NI = kInstr / NW;          // of which each wave issues NI
    static constexpr int SZ = sizeof(T);
    static constexpr int CPR = kKc ? 8 : BX * SZ / 16;  // 16-byte pieces a row
    static constexpr int RPI = 64 / CPR;                // rows an instruction
    static_assert(kInstr % NW == 0 && NI >= 1, "tile too small for the block");
    unsigned voff[NI];

    // Which of the tile's instructions is a wave's i-th: with rows of m or n the first half of them
    // fetches the first half of the step's k.
    static __device__ __forceinline__ int instr(int wave, int i) {
        if constexpr (kKc || NI == 1) return wave * NI + i;
        else return i / (NI / 2) * (kInstr / 2) + wave * (NI / 2) + i % (NI / 2);
    }
    // ld: row stride in elements; row_shift: rows before this wave's in the tile (kGated); pieces: valid
    // 16-byte pieces of the rows (kKc), the others are read out of bounds, as zeros
    __device__ __forceinline__ void init(int wave, int lane, int ld, int row_shift, int pieces) {
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int r = instr(wave, i) * RPI + lane / CPR, c = lane % CPR;
            if constexpr (kKc) {
                const int piece = c ^ (r & 7);
                voff[i] = piece < pieces ? (unsigned)((r - row_shift) * ld * SZ + piece * 16) : kOob;
            } else if constexpr (SZ == 2) {
                const int key = (r & 3) | ((r >> 3) & 3) << 2;
                voff[i] = (unsigned)(r * ld * SZ + (((c >> 1) ^ (key & (BX / 16 - 1))) << 1 | (c & 1)) * 16);
            } else {
                constexpr int U = MF / 4;  // pieces of a unit
                const int key = (r >> 2) & (64 / MF - 1);
                voff[i] = (unsigned)(r * ld * SZ + ((c / U ^ key) * U + c % U) * 16);
            }
        }
    }
    // Instruction i of this wave; bytes is what lies behind base. In assembly because the compiler takes
    // every later ds_read_b64_tr_b16 for a reader of what the builtin copies and waits for all copies
    // before it; the kernel waits itself (wait_vm_lds). m0 holds no value of the compiler between
    // instructions (a reserved register). No vector register is written, so none is
    // live while the copy runs.
    __device__ __forceinline__ void issue(int i, const char* base, int bytes, unsigned lds, int wave) const {
        const u32x4 rs{(unsigned)reinterpret_cast<uintptr_t>(base), (unsigned)(reinterpret_cast<uintptr_t>(base) >> 32),
                       (unsigned)bytes, (unsigned)kRsrcFlags};
        const unsigned at = lds + instr(wave, i) * 1024;
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                     :
                     : "s"(at), "v"(voff[i]), "s"(rs)
                     : "memory");
    }
};

// LDS -> MFMA operand: MF rows (unit u of the tile), k step ks (of 2 for MF 16, of 4 for MF 32).
template <typename T, bool kKc, int BX, int MF>
struct GemmReader {
    typedef typename GemmType<T, MF>::Frag Frag;
    static constexpr int KS = MF == 16 ? 2 : 4, G = 64 / MF;  // lane groups along k
    int off[KS];
    int key;
    __device__ __forceinline__ void init(int lane) {
        const int r = lane % MF, g = lane / MF;
        if constexpr (kKc) {
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) off[ks] = r * 128 + (((ks * G + g) ^ (r & 7)) * 16);
        } else if constexpr (sizeof(T) == 2) {
            // 16 lanes read a 4 x 16 block and get its columns
            const int j = lane & 15;
            key = ((j >> 2) | g << 2) & (BX / 16 - 1);
            off[0] = (g * 8 + (j >> 2)) * (BX * 2) + (j & 3) * 8;
        } else {
            key = g;
            off[0] = g * 4 * (BX * 4) + r * 4;
        }
    }
    __device__ __forceinline__ Frag read(const char* tile, int u, int ks) const {
        if constexpr (kKc) {
            return *reinterpret_cast<const Frag*>(tile + u * (MF * 128) + off[ks]);
        } else if constexpr (sizeof(T) == 2) {
            const char* p = tile + off[0] + ((u ^ key) << 5) + ks * (8 * G) * (BX * 2);
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p);
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (__attribute__((address_space(3))) s16x4*)(p + 4 * (BX * 2)));
            const bf16x4 l4 = __builtin_bit_cast(bf16x4, lo), h4 = __builtin_bit_cast(bf16x4, hi);
            return __builtin_shufflevector(l4, h4, 0, 1, 2, 3, 4, 5, 6, 7);
        } else {
            const char* p = tile + off[0] + (u ^ key) * (MF * 4) + ks * (4 * G) * (BX * 4);
            Frag f;
#pragma unroll
            for (int j = 0; j < 4; ++j) f[j] = *reinterpret_cast<const float*>(p + j * (BX * 4));
            return f;
        }
    }
};

template <int kN>
__device__ __forceinline__ void wait_vm_lds() {  // at most kN copies in flight, no LDS read
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" : : "n"(kN) : "memory");
}

template <int BM_, int BN_, int WGM_, int WGN_, int STAGES_, int MF_>
struct GemmTile {
    static constexpr int BM = BM_, BN = BN_, WGM = WGM_, WGN = WGN_, STAGES = STAGES_, MF = MF_;
    static constexpr int NW = WGM * WGN, NT = NW * 64;
    static constexpr int FM = BM / WGM / MF, FN = BN / WGN / MF;  // MF x MF pieces of a wave
    static constexpr int Q = MF * MF / 256;                       // fours of columns a lane holds of a piece
    static constexpr int kStageBytes = (BM + BN) * 128;
    // behind the stages: an epilogue's bf16 rows, or a pair of floats for each row and column of waves
    static constexpr int kStages = STAGES * kStageBytes;
    static constexpr int kEpi = MF == 32 ? WGN * BM * 8 : NW * MF * (FN * MF * 2 + 16);
    static constexpr int kLds = kStages + kEpi;
    typedef typename GemmType<float, MF>::Acc Acc;
};

// Where a wave's accumulators lie: piece (fm, fn), four q, lane: row m(fm), columns n(fn, q) ..
// n(fn, q) + 3.
template <typename Tile, int kMode>
struct GemmPlace {
    static constexpr int MF = Tile::MF;
    int m0, n0, wm, wn, lane;
    __device__ __forceinline__ int local_m(int fm) const { return (wm * Tile::FM + fm) * MF + lane % MF; }
    __device__ __forceinline__ int m(int fm) const { return m0 + local_m(fm); }
    __device__ __forceinline__ int wave() const { return wm * Tile::WGN + wn; }
    __device__ __forceinline__ int row0(int fm) const { return m0 + (wm * Tile::FM + fm) * MF; }  // of the piece
    __device__ __forceinline__ int col0() const {  // of the wave
        constexpr int F = kMode == kGated ? Tile::FN / 2 : Tile::FN;
        return n0 + wn * F * MF;
    }
    // kGated: fn < FN / 2 of the gate; the up piece of the same columns is fn + FN / 2
    __device__ __forceinline__ int n(int fn, int q) const {
        constexpr int F = kMode == kGated ? Tile::FN / 2 : Tile::FN;
        return n0 + (wn * F + fn) * MF + q * 8 + lane / MF * 4;
    }
};
template <typename Acc>
__device__ __forceinline__ f32x4 four(const Acc& v, int q) {
    return f32x4{v[q * 4], v[q * 4 + 1], v[q * 4 + 2], v[q * 4 + 3]};
}

// Stores MF rows of a wave's results. bf16: as whole rows, fours go into a wave-private part of LDS and
// leave it as 16 bytes a lane, kCols columns of a row side by side (64 or 128 bytes), where storing
// them as the MFMA leaves them would write 8 bytes to each of 16 rows; LDS operations of one wave run
// in order, so no barrier is needed. fp32: 16 bytes a lane at once (the LDS would cost the second block on
// a CU).
template <typename T, typename Tile, int kCols>
struct GemmRows {
    static constexpr int MF = Tile::MF, E = 16 / sizeof(T);
    static constexpr int kPitch = kCols * (int)sizeof(T) + 16;
    static constexpr int LPR = kCols / E, RPI = 64 / LPR;  // lanes a row, rows an instruction
    static_assert(sizeof(T) == 4 || Tile::NW * MF * kPitch <= Tile::kEpi, "rows fit LDS");
    typedef T T4 __attribute__((ext_vector_type(4)));
    typedef T Piece __attribute__((ext_vector_type(E)));
    char* mine;
    int lane;
    T* out;
    int64_t ld;
    int rows, cols;
    __device__ __forceinline__ GemmRows(char* smem, int wave, int lane_) : mine(smem + wave * (MF * kPitch)), lane(lane_) {}
    // the next MF rows go to out_ + r * ld_ for r < rows_; columns come in whole 16-byte pieces, cols_ of them exist
    __device__ __forceinline__ void begin(T* out_, int64_t ld_, int rows_, int cols_) {
        out = out_, ld = ld_, rows = rows_, cols = cols_;
    }
    // columns fn * MF + q * 8 + ... of row lane % MF
    __device__ __forceinline__ void put(int fn, int q, f32x4 v) const {
        const int r = lane % MF, c = fn * MF + q * 8 + lane / MF * 4;
        T4 o;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = (T)v[e];
        if constexpr (sizeof(T) == 4) {
            if (r < rows && c < cols) *reinterpret_cast<T4*>(out + r * ld + c) = o;
        } else {
            *reinterpret_cast<T4*>(mine + r * kPitch + c * (int)sizeof(T)) = o;
        }
    }
    __device__ __forceinline__ void store() const {
        if constexpr (sizeof(T) == 2) {
            const int r0 = lane / LPR, c = lane % LPR * E;
            M3_LDS_FENCE();  // the fours and the pieces are other types to the compiler
#pragma unroll
            for (int i = 0; i < (MF + RPI - 1) / RPI; ++i) {
                const int r = i * RPI + r0;
                if (r < MF && r < rows && c < cols)
                    *reinterpret_cast<Piece*>(out + r * ld + c) = *reinterpret_cast<const Piece*>(mine + r * kPitch + c * (int)sizeof(T));
            }
            M3_LDS_FENCE();
        }
    }
};

// A block's piece of work: one tile of one product, one part of its k.
struct GemmItem {
    int prob, tm, tn, split;
};
// Work id (counted from the product's first) -> item. Ids go to the XCDs round robin (blocks are
// dispatched so, and a block's later ids are a multiple of 8 further on): those of one XCD take a
// contiguous run of tiles, and runs walk groups of 8 row tiles column by column, so that an
// XCD's L2 serves both operands.
// (Quotients come from the vector unit: readfirstlane brings these back to scalar registers, which the
// copies' operands have to be in.)
__device__ __forceinline__ int scalar(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ GemmItem gemm_item(const GemmArgs& a, int prob, int id) {
    const int total = a.tiles_m * a.tiles_n;
    const int split = scalar(id / total), b = id - split * total;
    const int x = b & 7, per = total >> 3, rest = total & 7;
    const int at = x * per + (x < rest ? x : rest) + (b >> 3);
    constexpr int G = 8;
    const int group = scalar(at / (G * a.tiles_n)), first = group * G;
    const int rows = a.tiles_m - first < G ? a.tiles_m - first : G;
    const int in = at - group * (G * a.tiles_n);
    const int tn = scalar(in / rows);
    return GemmItem{prob, first + in - tn * rows, tn, split};
}
// The k steps of a product, and where part `split` of them begins (steps < 2^26, splits <= 64).
template <int kMode, int BK>
__device__ __forceinline__ int gemm_steps_of(const GemmArgs& a) {
    return (a.K[0] + BK - 1) / BK + (kMode == kSeg2 ? (a.K[1] + BK - 1) / BK : 0);
}
__device__ __forceinline__ int gemm_first_step(int steps, int splits, int split) {
    return scalar((int)((unsigned)steps * (unsigned)split / (unsigned)splits));
}

// The items of products [kP0, kP1) of a group that fall to this block: ids congruent to its own.
template <typename T, typename Tile, bool kAKc, bool kBKc, int kMode, int kP0, int kP1, int kN, typename Epi>
__device__ __forceinline__ void gemm_run(const GemmGroup<kN>& grp, const Epi& epi) {
    constexpr int BM = Tile::BM, BN = Tile::BN, FM = Tile::FM, FN = Tile::FN, ST = Tile::STAGES, MF = Tile::MF;
    constexpr int BK = 128 / sizeof(T), SZ = sizeof(T);
    typedef GemmLoader<T, kAKc, BM, Tile::NW, MF> LA;
    typedef GemmLoader<T, kBKc, BN, Tile::NW, MF> LB;
    typedef GemmType<T, MF> Type;
    constexpr int NLD = LA::NI + LB::NI;
    extern __shared__ __align__(16) char gemm_smem[];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int grid = (int)gridDim.x, id_end = grp.first[kP1];
    int id0 = grp.first[kP0];
    if constexpr (kP0 > 0) {
        const int r = id0 - scalar(id0 / grid) * grid;  // whose turn it is
        id0 += ((int)blockIdx.x >= r ? 0 : grid) + (int)blockIdx.x - r;
    } else {
        id0 = (int)blockIdx.x;
    }
    if (id0 >= id_end) return;
    auto args_of = [&](int p) __attribute__((always_inline)) {
        if constexpr (kP1 - kP0 == 1) return grp.a[kP0];
        else return pick_args(grp.a, p);
    };
    static_assert(kP1 - kP0 <= 1 || (kP0 == 1 && kP1 == 4), "one product, or the last three of four");
    auto item_of = [&](int id) __attribute__((always_inline)) {
        int p = kP0, first = grp.first[kP0];
        if constexpr (kP1 - kP0 == 3) {
            const int f2 = grp.first[2], f3 = grp.first[3];
            p = id >= f3 ? 3 : id >= f2 ? 2 : 1;
            first = id >= f3 ? f3 : id >= f2 ? f2 : first;
        }
        return gemm_item(args_of(p), p, id - first);
    };

    const bool second = kMode == kGated && wave * LB::NI >= LB::kInstr / 2;
    static_assert(kMode != kGated || (LB::kInstr / 2) % LB::NI == 0, "a wave fetches from one half");
    LA la;
    LB lb;
    // What is fetched next: step fs of item f_id, which ends before step f_end. From step to step
    // the pointers advance by pa_step and pb_step; at step `turn` (the end, a term's last, partial step
    // or the second term's first) everything is set up anew. Behind the last item nothing is read.
    const char *pa, *pb;
    int64_t pa_step, pb_step;
    int ba, bb, turn, fs, f_id, f_end;
    auto set_up = [&]() __attribute__((always_inline)) {
        const GemmItem it = item_of(f_id);
        const GemmArgs a = args_of(it.prob);
        const int st0 = (a.K[0] + BK - 1) / BK, steps = gemm_steps_of<kMode, BK>(a);
        const int m0 = it.tm * BM, n0 = it.tn * (kMode == kGated ? BN / 2 : BN);
        // rows that exist in this tile: spans end with the last one's last valid element (< 2^31 bytes)
        const int ra_rows = a.M - m0 < BM ? a.M - m0 : BM, rb_rows = a.N - n0 < BN ? a.N - n0 : BN;
        const int seg = kMode == kSeg2 && fs >= st0 ? 1 : 0;
        const int k0 = (seg ? fs - st0 : fs) * BK;
        const int K = seg ? a.K[1] : a.K[0], KB = seg ? a.KB[1] : a.KB[0];
        const int left = K - k0, krem = left < BK ? left : BK;
        const GemmOp oa = seg ? a.a[1] : a.a[0], ob = seg || second ? a.b[1] : a.b[0];
        const int bleft = KB - k0;
        const int brem = kBKc || krem < bleft ? krem : bleft;  // may be negative
        const int lda = (int)oa.ld, ldb = (int)ob.ld;
        pa = reinterpret_cast<const char*>(oa.p) + (kAKc ? (int64_t)m0 * lda + k0 : (int64_t)k0 * lda + m0) * SZ;
        pb = reinterpret_cast<const char*>(ob.p) + (kBKc ? (int64_t)n0 * ldb + k0 : (int64_t)k0 * ldb + n0) * SZ;
        pa_step = kAKc ? 128 : (int64_t)BK * lda * SZ;
        pb_step = kBKc ? 128 : (int64_t)BK * ldb * SZ;
        ba = ra_rows <= 0 ? 0 : (kAKc ? (ra_rows - 1) * lda + krem : (krem - 1) * lda + ra_rows) * SZ;
        bb = brem <= 0 || rb_rows <= 0 ? 0 : (kBKc ? (rb_rows - 1) * ldb + brem : (brem - 1) * ldb + rb_rows) * SZ;
        const int pieces = krem < BK ? (krem * SZ) >> 4 : 8;
        la.init(wave, lane, lda, 0, pieces);
        lb.init(wave, lane, ldb, second ? BN / 2 : 0, pieces);
        // whole steps of this term for both operands, then the next turn
        const int whole = (kBKc || K < KB ? K : KB) / BK + (seg ? st0 : 0);
        const int end = seg || kMode != kSeg2 ? steps : st0;
        turn = fs < whole ? whole : fs + 1 < end ? fs + 1 : end;
        turn = turn < f_end ? turn : f_end;
    };
    auto enter = [&](int id) __attribute__((always_inline)) {  // the first step of an item
        f_id = id;
        if (id >= id_end) {
            ba = bb = 0;
            pa_step = pb_step = 0;
            turn = f_end = 0x7fffffff;
            return;
        }
        const GemmItem it = item_of(id);
        const GemmArgs a = args_of(it.prob);
        const int steps = gemm_steps_of<kMode, BK>(a);
        fs = gemm_first_step(steps, a.splits, it.split);
        f_end = gemm_first_step(steps, a.splits, it.split + 1);
        set_up();
    };
    auto advance = [&]() __attribute__((always_inline)) {
        ++fs;
        if (fs == turn) {
            if (fs == f_end) enter(f_id + grid);
            else set_up();
        } else {
            pa += pa_step;
            pb += pb_step;
        }
    };
    const unsigned lds0 = (unsigned)reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)gemm_smem);
    auto fetch = [&](int i, int slot) __attribute__((always_inline)) {  // instruction i of NLD
        const unsigned sl = lds0 + slot * Tile::kStageBytes;
        if (i < LA::NI) la.issue(i, pa, ba, sl, wave);
        else lb.issue(i - LA::NI, pb, bb, sl + BM * 128, wave);
    };

    GemmReader<T, kAKc, BM, MF> ra;
    GemmReader<T, kBKc, BN, MF> rb;
    ra.init(lane);
    rb.init(lane);
    const int wm = wave / Tile::WGN, wn = wave % Tile::WGN;
    auto unit_b = [&](int fn) __attribute__((always_inline)) {
        if constexpr (kMode == kGated)
            return fn < FN / 2 ? wn * (FN / 2) + fn : BN / (2 * MF) + wn * (FN / 2) + fn - FN / 2;
        else
            return wn * FN + fn;
    };
    typename Type::Acc acc[FM][FN];
    // fp32 tiles of few rows, where a library cuts k: every 512 k are summed apart, so that the error of a long
    // k does not grow with the square root of its length (16384 random terms: 2.4e-6 of the sum in one chain, below
    // 5.7e-7 so; 1% more time). The 128 x 128 tile would need 64 more registers a lane; over the lengths that it
    // serves it is as near as a library (dW of 1000 rows: 9.2e-7, 9.4e-7).
    constexpr bool kFold = sizeof(T) == 4 && BM == 64;
    constexpr int kFoldSteps = 16;
    typename Type::Acc total[kFold ? FM : 1][kFold ? FN : 1];

    // A step is two halves of KH k steps. While one half's fragments are multiplied, the next half's
    // are read from LDS. A barrier in front of a half says that all waves have read what lies before it,
    // and that the next half's data has landed; what has been read makes room for the step ST further
    // on. With rows of m or n a half of the copies fetches a half of the k, so each half has its
    // barrier and refills its own place: copies then have one and a half steps to land. Rows of k
    // would come in pieces of 64 bytes that way, which costs more than it gives (8192^3 x W^T 783 ->
    // 827 us; dy^T x 823 -> 800): there the whole step's place is refilled halfway through it.
    // Copies and reads are issued between groups of FN MFMAs, which cover them.
    constexpr bool kHalves = !kAKc && !kBKc && LA::NI > 1 && LB::NI > 1;
    typedef typename Type::Frag Frag;
    constexpr int KH = MF == 16 ? 1 : 2;
    constexpr int kGroups = KH * FM, kReads = KH * (FM + FN);
    Frag fa[2][KH][FM], fb[2][KH][FN];
    auto read = [&](int half, int slot, int i) __attribute__((always_inline)) {  // fragment i of a half
        const char* ta = gemm_smem + slot * Tile::kStageBytes;
        const int ks = i / (FM + FN), r = i % (FM + FN);
        if (r < FN) fb[half][ks][r] = rb.read(ta + BM * 128, unit_b(r), half * KH + ks);
        else fa[half][ks][r - FN] = ra.read(ta, wm * FM + r - FN, half * KH + ks);
    };
    auto group = [&](int half, int g) __attribute__((always_inline)) {
        const int ks = g / FM, i = g % FM;
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = Type::mma(fb[half][ks][j], fa[half][ks][i], acc[i][j]);
    };
    // Reads and copies between two groups: two, and with B in rows of n as few copies as fit the half
    // (256 x 256 tiles, 8192^3: dy W 786 us at two copies, 765 at one; dy^T x 781 us, and 813 at three
    // reads; x W^T 777, and 760 at three reads and one copy, which over short k is slower: cross
    // entropy of 8192 x 768 against 32000 tokens, forward and backward, 1609 us and 1627).
    constexpr int kPer = (kReads + kGroups - 1) / kGroups < 2 ? 2 : (kReads + kGroups - 1) / kGroups;
    constexpr int kLd = kHalves ? NLD / 2 : NLD;  // copies behind a barrier
    constexpr int kPerLd = (kLd + kGroups - 1) / kGroups < 2 && kBKc ? 2 : (kLd + kGroups - 1) / kGroups;
    auto fetch_half = [&](int half, int i, int slot) __attribute__((always_inline)) {  // copy i of the kLd behind the barrier before `half`
        if constexpr (kHalves) {
            constexpr int A = LA::NI / 2;
            fetch(i < A ? half * A + i : LA::NI + half * (LB::NI / 2) + i - A, slot);
        } else {
            fetch(i, slot);
        }
    };

    enter(id0);
#pragma unroll
    for (int s = 0; s < ST; ++s) {
        if (s) advance();
#pragma unroll
        for (int i = 0; i < NLD; ++i) fetch(i, s);
    }
    int slot = 0;
    // The steps of all items form one row: an item's last steps already fetch the next one's first,
    // which land during the epilogue.
    for (int id = id0; id < id_end; id += grid) {
        const GemmItem it = item_of(id);
        int n_steps;
        {
            const GemmArgs a = args_of(it.prob);
            const int steps = gemm_steps_of<kMode, BK>(a);
            n_steps = gemm_first_step(steps, a.splits, it.split + 1) - gemm_first_step(steps, a.splits, it.split);
        }
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j)
#pragma unroll
                for (int e = 0; e < MF * MF / 64; ++e) acc[i][j][e] = 0.f;
        if constexpr (kFold) {
#pragma unroll
            for (int i = 0; i < FM; ++i)
#pragma unroll
                for (int j = 0; j < FN; ++j) total[i][j] = typename Type::Acc{};
        }
        wait_vm_lds<0>();  // also the last epilogue's stores, which count with the copies
        M3_LDS_FENCE();
        __builtin_amdgcn_s_barrier();
        M3_LDS_FENCE();
#pragma unroll
        for (int i = 0; i < kReads; ++i) read(0, slot, i);
        for (int n = n_steps; n > 0; --n) {
            const int next = slot + 1 == ST ? 0 : slot + 1;
            M3_FENCE();
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                if (half == (kHalves ? 0 : 1)) advance();
                if (kHalves || half == 1) {
                    wait_vm_lds<NLD * (kHalves ? ST - 1 : ST - 2)>();
                    M3_LDS_FENCE();
                    __builtin_amdgcn_s_barrier();
                    M3_LDS_FENCE();
                }
#pragma unroll
                for (int g = 0; g < kGroups; ++g) {
                    if (kHalves || half == 1) {
#pragma unroll
                        for (int i = g * kPerLd; i < (g + 1) * kPerLd && i < kLd; ++i) fetch_half(half, i, slot);
                    }
#pragma unroll
                    for (int i = g * kPer; i < (g + 1) * kPer && i < kReads; ++i) read(half ^ 1, half ? next : slot, i);
                    M3_FENCE();
                    group(half, g);
                    M3_FENCE();
                }
            }
            slot = next;
            if constexpr (kFold) {
                if (n_steps > kFoldSteps && (n & (kFoldSteps - 1)) == 1) {
                    asm volatile("");  // a branch: as selections the sums would wait for the products of every step
#pragma unroll
                    for (int i = 0; i < FM; ++i)
#pragma unroll
                        for (int j = 0; j < FN; ++j) {
                            total[i][j] += acc[i][j];
                            acc[i][j] = n > 1 ? typename Type::Acc{} : total[i][j];
                        }
                }
            }
        }
        const GemmPlace<Tile, kMode> at{it.tm * BM, it.tn * (kMode == kGated ? BN / 2 : BN), wm, wn, lane};
        epi.template run<T, Tile, kMode>(at, acc, gemm_smem + Tile::kStages, it);
    }
    // no copy outlives its block, and none meets what the block does next in LDS
    wait_vm_lds<0>();
    M3_LDS_FENCE();
    __builtin_amdgcn_s_barrier();
    M3_LDS_FENCE();
}

template <typename T, typename Tile, bool kAKc, bool kBKc, int kMode, typename Epi>
__global__ __launch_bounds__(Tile::NT, 2) void gemm_kernel(GemmGroup<1> grp, Epi epi) {
    gemm_run<T, Tile, kAKc, kBKc, kMode, 0, 1>(grp, epi);
}

}  // namespace m3
