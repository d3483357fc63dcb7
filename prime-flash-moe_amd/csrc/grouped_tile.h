// Tiles of the ragged expert products, gfx950: out[i][j] = sum over k of P[i][k] Q[j][k] for a tile of 64 FM rows i
// (FM = 1 .. 4) and 256 columns j, on four waves.
//
// The same engine serves the product of rows with their expert's weights (P: rows, Q: weights), its gradient with
// respect to the rows (Q read across) and with respect to the weights (both read across).  An operand is either
// "along": the contraction is its contiguous dimension, or "across": i (or j) is, and its k rows lie one pitch apart.
//
// Why four waves: wave (wm, wn) owns a 32 FM x 128 part of the tile, so a slab's operands are read from LDS
// (64 FM + 256) x 2 times 128 bytes in all; eight waves of 32 FM x 64 would read half as much again, and under the
// card's power limit every byte moved costs clock.  One wave per SIMD holds 256 accumulators (FM = 4) and two sets of
// operand fragments; the next 16-wide step's fragments are read under the current step's matrix instructions.
//
// LDS: a ring of stages, each a slab of 128 bytes of contraction (64 elements of 16 bits, 128 of 8): the tile's P rows,
// then the 256 Q rows.  Along: rows of 128 B, chunk c (16 B) of row r in slot c ^ ((r >> 1) & 7).  Across (16-bit types
// only): one row per k of 2 bytes per i, 32-byte group c of row k in slot c ^ 2 (k & 3), read through the transposing
// LDS read: four k rows x 16 columns per 16 lanes, which the swizzle spreads over all banks.  The copies go straight to
// LDS, 1 KB per wave instruction; the swizzle is applied to the lanes' addresses.
//
// One barrier per slab, in the last step, where the slab's last fragments are in registers: it certifies that the next
// slab has landed and hands this slab's stage to the copies of the slab S behind it.
//
// Ends: rows and columns outside the operand are read from its last one inside (they only reach outputs that are not
// stored); contraction elements outside it come from a page of zeros, in both operands, so that nothing that lies there
// (a NaN in the next group's rows) reaches a sum.
#pragma once
#include <type_traits>

#include "moe_ring.h"

namespace pmoe {
namespace gmm {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef int i32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256;
constexpr int kWaves = 4;
constexpr int kCols = 256;                       // Q rows of a tile
constexpr int kSlab = 128;                       // bytes of contraction of a slab
constexpr int kQBytes = kCols * kSlab;
constexpr int kScratchBytes = 32 * 256;          // per wave: 32 rows of 256 B on their way out
constexpr int kScratchOff = 160 * 1024 - kWaves * kScratchBytes;
constexpr int kLdsBytes = 160 * 1024;

struct Bf16 {
    using Acc = f32x16;
    static constexpr int kBytes = 2;
    static __device__ __forceinline__ Acc mfma(i32x4 a, i32x4 b, Acc c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
};
struct F16 {
    using Acc = f32x16;
    static constexpr int kBytes = 2;
    static __device__ __forceinline__ Acc mfma(i32x4 a, i32x4 b, Acc c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
};
struct I8 {  // sums in 32-bit integers: exact
    using Acc = i32x16;
    static constexpr int kBytes = 1;
    static __device__ __forceinline__ Acc mfma(i32x4 a, i32x4 b, Acc c) {
        return __builtin_amdgcn_mfma_i32_32x32x32_i8(a, b, c, 0, 0, 0);
    }
};

template <int FM>
struct Geo {
    static constexpr int kRows = 64 * FM;
    static constexpr int kPBytes = kRows * kSlab;
    static constexpr int kStageBytes = kPBytes + kQBytes;
    static constexpr int kFit = kScratchOff / kStageBytes;
    static constexpr int kStages = kFit < 4 ? kFit : 4;
    static constexpr int kPPieces = kPBytes / 1024 / kWaves, kQPieces = kQBytes / 1024 / kWaves;  // copies per wave
    static constexpr int kCopies = kPPieces + kQPieces;
    static_assert(kStages >= 2, "a stage to compute on and one to fill");
};

// What lies behind the end of a contraction.
__device__ const uint4 g_zeros = {0, 0, 0, 0};

__device__ __forceinline__ void copy16_at(const char *src, const char *lds_dst) {
    asm volatile("s_mov_b32 m0, %1\n\tglobal_load_lds_dwordx4 %0, off" : : "v"(src), "s"(ring::lds_addr(lds_dst)) : "memory");
}

// An operand of a tile.  ROWS: its rows (64 FM or 256) in a stage.
template <int ROWS, bool ACROSS>
struct Operand {
    static constexpr int kPieces = ROWS * kSlab / 1024 / kWaves;
    static constexpr int kRowBytes = ACROSS ? ROWS * 2 : kSlab;  // of a row in LDS
    static constexpr int kPerPiece = 1024 / kRowBytes;           // rows that a copy moves
    static constexpr int kLanes = kRowBytes / 16;                // lanes of a row
    const char *base;         // wave-uniform: row 0 of the tile, slab 0
    uint32_t off[kPieces];    // of this lane's chunk, slab 0
    int64_t step;             // bytes between slabs

    // `pitch`: bytes between rows (along) or between k rows (across).  `live`: rows of the tile inside the operand (>= 1;
    // across: a multiple of 8).
    __device__ __forceinline__ void setup(int tid, const char *src, int64_t pitch, int live) {
        base = ring::uniform_ptr(src);
        step = ACROSS ? 64 * pitch : kSlab;
        const int wave = tid >> 6, lane = tid & 63, sub = lane / kLanes, slot = lane % kLanes;
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            const int row = (wave + kWaves * i) * kPerPiece + sub;
            if constexpr (ACROSS) {
                const int chunk = slot ^ ((row & 3) << 2);  // 2 (row & 3) in groups of two chunks
                off[i] = (uint32_t)row * (uint32_t)pitch + (uint32_t)min(chunk, live / 8 - 1) * 16u;
            } else {
                off[i] = (uint32_t)min(row, live - 1) * (uint32_t)pitch + (uint32_t)(slot ^ ((row >> 1) & 7)) * 16u;
            }
        }
    }
    // Copy `i` of this wave's share of a slab.  END: the contraction may end inside the slab; `left` of it remains from the slab
    // on, in bytes (along) or k rows (across).
    template <bool END>
    __device__ __forceinline__ void issue(int i, int tid, char *at, int64_t slab_off, int left) const {
        const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
        char *dst = at + (wave + kWaves * i) * 1024;
        if constexpr (!END) {
            ring::copy16(base + slab_off, off[i], dst);
        } else {
            const int lane = tid & 63, row = (wave + kWaves * i) * kPerPiece + lane / kLanes;
            const int k = ACROSS ? row : ((lane % kLanes) ^ ((row >> 1) & 7)) * 16;
            uint32_t o = off[i];
            asm volatile("" : "+v"(o));  // (the 64-bit addresses of all pieces, kept through the whole contraction otherwise)
            copy16_at(k < left ? base + slab_off + o : reinterpret_cast<const char *>(&g_zeros), dst);
        }
    }
};

// Where this lane reads its fragments: `at[j]` for an operand along (step j of a slab, fragment f at f * 4 KB), `at[f & 3]`
// for one across (step j at 16 j rows).
template <int ROWS, bool ACROSS>
struct Reader {
    int at[4];
    // `first`: the wave's first fragment in the operand
    __device__ __forceinline__ void setup(int lane, int first) {
        if constexpr (ACROSS) {
            const int q = lane >> 4, i = lane & 15, k = 8 * (q >> 1) + (i >> 2);
#pragma unroll
            for (int f = 0; f < 4; ++f) {
                const int group = ((first + f) * 2 + (q & 1)) ^ ((k & 3) << 1);
                at[f] = k * (ROWS * 2) + group * 32 + (i & 3) * 8;
            }
        } else {
            const int r = lane & 31, half = lane >> 5, sx = (lane >> 1) & 7;
#pragma unroll
            for (int j = 0; j < 4; ++j) at[j] = (first * 32 + r) * kSlab + (((2 * j + half) ^ sx) << 4);
        }
    }
    __device__ __forceinline__ i32x4 read(const char *stage, int f, int j) const {
        if constexpr (ACROSS) {
            typedef __attribute__((address_space(3))) s16x4 *lds4;
            char *p = const_cast<char *>(stage) + at[f] + j * 16 * (ROWS * 2);
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)p);
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(p + 4 * (ROWS * 2)));
            typedef short s16x8 __attribute__((ext_vector_type(8)));
            return __builtin_bit_cast(i32x4, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        } else {
            return *reinterpret_cast<const i32x4 *>(stage + at[j] + f * 32 * kSlab);
        }
    }
};

// Nothing crosses this point in the instruction schedule.
#define PMOE_GMM_FENCE() __builtin_amdgcn_sched_barrier(0)

// A tile's operands and its place in the contraction.
template <int FM, bool PX, bool QX>
struct Feed {
    using G = Geo<FM>;
    Operand<G::kRows, PX> p;
    Operand<kCols, QX> q;
    int n_slabs, full;  // slabs, and how many of them are whole
    int len_p, len_q;   // contraction in bytes (along) or elements (across)

    __device__ __forceinline__ void set_length(int elements, int bytes_per) {
        len_p = PX ? elements : elements * bytes_per;
        len_q = QX ? elements : elements * bytes_per;
        full = elements * bytes_per / kSlab;
        n_slabs = (elements * bytes_per + kSlab - 1) / kSlab;
    }
    template <bool END>
    __device__ __forceinline__ void issue(int c, int tid, char *stage, int slab) const {
        if (c < G::kQPieces) q.template issue<END>(c, tid, stage + G::kPBytes, slab * q.step, len_q - slab * (QX ? 64 : kSlab));
        else p.template issue<END>(c - G::kQPieces, tid, stage, slab * p.step, len_p - slab * (PX ? 64 : kSlab));
    }
    template <bool END>
    __device__ __forceinline__ void issue_all(int tid, char *stage, int slab) const {
#pragma unroll
        for (int c = 0; c < G::kCopies; ++c) issue<END>(c, tid, stage, slab);
    }
    // The first slabs, up to all stages.
    __device__ __forceinline__ void start(int tid, char *lds) const {
#pragma unroll 1
        for (int s = 0; s < G::kStages; ++s) {
            if (s < full) issue_all<false>(tid, lds + s * G::kStageBytes, s);
            else if (s < n_slabs) issue_all<true>(tid, lds + s * G::kStageBytes, s);
        }
    }
};

// Waits until at most `slabs` (wave-uniform, <= 3) slabs of copies are in flight and this wave's LDS reads have returned,
// then joins the barrier.
template <int COPIES>
__device__ __forceinline__ void landed(int slabs) {
    if (slabs <= 0) ring::wait_and_barrier<0>();
    else if (slabs == 1) ring::wait_and_barrier<COPIES>();
    else if (slabs == 2) ring::wait_and_barrier<2 * COPIES>();
    else ring::wait_and_barrier<3 * COPIES>();
}

// The contraction of one tile whose first slabs are on their way (Feed::start).  acc[f][t]: column fragment 4 wn + f
// against row fragment FM wm + t.  Every wave is past the reads
// of the last slab when one returns (n_slabs > 0): the stages may be filled again.
template <class T, int FM, bool PX, bool QX>
__device__ __forceinline__ void contract(typename T::Acc (&acc)[4][FM], const Feed<FM, PX, QX> &feed, char *lds, int tid) {
    using G = Geo<FM>;
    constexpr int S = G::kStages, READS = 4 + FM, MM = 4 * FM;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    Reader<G::kRows, PX> rp;
    Reader<kCols, QX> rq;
    rp.setup(lane, (wave >> 1) * FM);
    rq.setup(lane, (wave & 1) * 4);
    const int n = feed.n_slabs;
    landed<G::kCopies>(min(S, n) - 1);

    i32x4 a[2][4], b[2][FM];
    auto read = [&](int r, int set, const char *stage, int j) {
        if (r < 4) a[set][r] = rq.read(stage + G::kPBytes, r, j);
        else b[set][r - 4] = rp.read(stage, r - 4, j);
    };
#pragma unroll
    for (int r = 0; r < READS; ++r) read(r, 0, lds, 0);

    // Straight-line code for a slab, with branches around copies only: with the matrix instructions themselves in
    // branches the compiler keeps a second set of accumulators and spills.
    int cur = 0;
    for (int k = 0; k < n; ++k) {
        char *stage = lds + cur * G::kStageBytes;
        cur = cur + 1 == S ? 0 : cur + 1;
        const char *next = lds + cur * G::kStageBytes;
        const bool fill = k + S < feed.full;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int set = j & 1;
            if (j == 3) {
                landed<G::kCopies>(min(S - 2, n - 2 - k));
                if (k + S < n && !fill) feed.template issue_all<true>(tid, stage, k + S);
            }
            PMOE_GMM_FENCE();
#pragma unroll
            for (int m = 0; m < MM; ++m) {
                const int t = m >> 2, f = m & 3;
                acc[f][t] = T::mfma(a[set][f], b[set][t], acc[f][t]);
                // the next step's fragments behind the first half of this step's instructions (behind the last slab:
                // whatever the stage holds, which nobody uses)
#pragma unroll
                for (int r = 0; r < READS; ++r)
                    if (r * MM / (2 * READS) == m) read(r, set ^ 1, j < 3 ? stage : next, (j + 1) & 3);
                if (j == 3 && m % 2 == 1 && fill) {
#pragma unroll
                    for (int c = 0; c < G::kCopies; ++c)
                        if (c * (MM / 2) / G::kCopies == m / 2) feed.template issue<false>(c, tid, stage, k + S);
                }
                PMOE_GMM_FENCE();
            }
        }
    }
}

}  // namespace gmm
}  // namespace pmoe
