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
// LDS: two stages, each a slab of 128 bytes of contraction (64 elements of 16 bits, 128 of 8): the tile's P rows,
// then the 256 Q rows.  Along: rows of 128 B, chunk c (16 B) of row r in slot c ^ ((r >> 1) & 7).  Across (16-bit types
// only): one row per k of 2 bytes per i, 32-byte group c of row k in slot c ^ 2 (k & 3), read through the transposing
// LDS read: four k rows x 16 columns per 16 lanes, which the swizzle spreads over all banks.  The copies go straight to
// LDS, 1 KB per wave instruction; the swizzle is applied to the lanes' addresses.
//
// One barrier per slab, in the last step, where the slab's last fragments are in registers: it certifies that the next
// slab has landed and hands this slab's stage to the copies of the slab two behind it, which may be the next tile's.
//
// Bound by the matrix pipe and the card's power: in a long contraction a slab of the tallest tile takes 2130 cycles, 2048 of
// them matrix instructions, and the clock falls as they fill up (8192 x 8192 x 8192 in bf16: 1.40 PFLOP/s along, with one
// operand across and with both; the library's on the same card 1.57, 1.34 and 1.16).  A tile costs about 10 000 cycles besides: the way out
// (7000, the L2's writes), the first fragments, the next tile's addresses.  Where weights are read by two or three tiles (128
// experts of 512 rows) the slabs wait for memory, 700 cycles a step of 64 rows instead of 512.
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

constexpr int kStageStride = 64 * 1024;  // of the tallest tile, so that tiles of different height follow each other in the ring
template <int FM>
struct Geo {
    static constexpr int kRows = 64 * FM;
    static constexpr int kPBytes = kRows * kSlab;
    static constexpr int kPPieces = kPBytes / 1024 / kWaves, kQPieces = kQBytes / 1024 / kWaves;  // copies per wave
    static constexpr int kCopies = kPPieces + kQPieces;
    static_assert(kPBytes + kQBytes <= kStageStride && 2 * kStageStride <= kScratchOff, "two stages fit in front of the scratch");
};

// What lies behind the end of a contraction.
__device__ const uint4 g_zeros = {0, 0, 0, 0};

// Copies to `lds` (wave-uniform byte address) + OFF.  One scalar instruction in front of each: what stands between two matrix
// instructions of the only wave of a SIMD has 32 cycles, and a longer chain of dependent scalar instructions (a wave number
// read, shifted and added for every copy) cost 50 cycles a copy.
// (The wait state behind it is the one that the instruction set asks for between a scalar write of M0 and a load to LDS.)
template <int OFF>
__device__ __forceinline__ void copy16(const char *base, uint32_t voff, uint32_t lds) {
    asm volatile("s_add_u32 m0, %2, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" : : "v"(voff), "s"(base), "s"(lds), "n"(OFF) : "memory", "scc");
}
// The same with the non-temporal hint, for what no other workgroup reads.
template <int OFF>
__device__ __forceinline__ void copy16_once(const char *base, uint32_t voff, uint32_t lds) {
    asm volatile("s_add_u32 m0, %2, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1 nt" : : "v"(voff), "s"(base), "s"(lds), "n"(OFF) : "memory", "scc");
}
template <int OFF>
__device__ __forceinline__ void copy16_at(const char *src, uint32_t lds) {
    asm volatile("s_add_u32 m0, %1, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" : : "v"(src), "s"(lds), "n"(OFF) : "memory", "scc");
}
__device__ __forceinline__ void copy4_at(const char *src, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" : : "v"(src), "s"(lds) : "memory");
}
// Calls f(integral_constant<int, 0>) ... f(integral_constant<int, N - 1>).
template <int N, class F>
__device__ __forceinline__ void unrolled(F f) {
    if constexpr (N > 0) {
        unrolled<N - 1>(f);
        f(std::integral_constant<int, N - 1>());
    }
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
        const int row = wave * kPerPiece + sub;  // of the first piece; the swizzle is the same for all
        const uint32_t first = (uint32_t)row * (uint32_t)pitch, next = (uint32_t)(kWaves * kPerPiece) * (uint32_t)pitch;
        // (a slot holds chunk slot ^ 4 (row & 3): 2 (row & 3) in groups of two chunks)
        const uint32_t last = ACROSS ? ~0u : (uint32_t)(live - 1) * (uint32_t)pitch;
        const uint32_t chunk = ACROSS ? (uint32_t)min(slot ^ ((row & 3) << 2), live / 8 - 1) * 16u : (uint32_t)(slot ^ ((row >> 1) & 7)) * 16u;
#pragma unroll
        for (int i = 0; i < kPieces; ++i) off[i] = min(first + i * next, last) + chunk;
    }
    // Byte offset of line `i` of a slab (ROWS lines of 128 B).
    static __device__ __forceinline__ uint32_t line(int i, int64_t pitch, int live) {
        if constexpr (ACROSS) return (uint32_t)(i / (ROWS / 64)) * (uint32_t)pitch + (uint32_t)min(i % (ROWS / 64) * 128, live * 2 - 4);
        return (uint32_t)min(i, live - 1) * (uint32_t)pitch;
    }
    // Copy I of this wave's share of a slab to `at` (the wave's first piece) + AT.  END: the contraction may end inside the slab;
    // `left` of it remains from the slab on, in bytes (along) or k rows (across).
    template <int I, int AT>
    __device__ __forceinline__ void issue(const char *slab, uint32_t at) const {
        copy16<AT + I * kWaves * 1024>(slab, off[I], at);
    }
    template <int I, int AT>
    __device__ __forceinline__ void issue_end(int tid, const char *slab, uint32_t at, int left) const {
        const int wave = tid >> 6, lane = tid & 63, row = (wave + kWaves * I) * kPerPiece + lane / kLanes;
        const int k = ACROSS ? row : ((lane % kLanes) ^ ((row >> 1) & 7)) * 16;
        uint32_t o = off[I];
        asm volatile("" : "+v"(o));  // (the 64-bit addresses of all pieces, kept through the whole contraction otherwise)
        copy16_at<AT + I * kWaves * 1024>(k < left ? slab + o : reinterpret_cast<const char *>(&g_zeros), at);
    }
};

// Where this lane reads its fragments, as LDS byte addresses in the current stage: `at[j]` for an operand along (step j of a
// slab, fragment f 4 KB f behind), `at[f]` for one across (step j 16 j rows behind).
template <int ROWS, bool ACROSS>
struct Reader {
    uint32_t at[4];
    // `first`: the wave's first fragment in the operand, `lds`: the operand in the first stage
    __device__ __forceinline__ void setup(int lane, int first, uint32_t lds) {
        if constexpr (ACROSS) {
            const int q = lane >> 4, i = lane & 15, k = 8 * (q >> 1) + (i >> 2);
#pragma unroll
            for (int f = 0; f < 4; ++f) {
                const int group = ((first + f) * 2 + (q & 1)) ^ ((k & 3) << 1);
                at[f] = lds + k * (ROWS * 2) + group * 32 + (i & 3) * 8;
            }
        } else {
            const int r = lane & 31, half = lane >> 5, sx = (lane >> 1) & 7;
#pragma unroll
            for (int j = 0; j < 4; ++j) at[j] = lds + (first * 32 + r) * kSlab + (((2 * j + half) ^ sx) << 4);
        }
    }
    __device__ __forceinline__ i32x4 read(int f, int j) const {
        if constexpr (ACROSS) {
            typedef __attribute__((address_space(3))) s16x4 *lds4;
            typedef short s16x8 __attribute__((ext_vector_type(8)));
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(uintptr_t)(at[f] + j * 16 * (ROWS * 2)));
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(uintptr_t)(at[f] + j * 16 * (ROWS * 2) + 4 * (ROWS * 2)));
            return __builtin_bit_cast(i32x4, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        } else {
            typedef const __attribute__((address_space(3))) i32x4 *lds16;
            return *(lds16)(uintptr_t)(at[j] + f * 32 * kSlab);
        }
    }
};

// Nothing crosses this point in the instruction schedule.
#define PMOE_GMM_FENCE() __builtin_amdgcn_sched_barrier(0)

constexpr int kAhead = 1;  // slabs that lines are asked for in front of their copies (0, 2 and 3 are slower by 0.5 - 1 %)

// A tile's operands and its place in the contraction.
template <int FM, bool PX, bool QX>
struct Feed {
    using G = Geo<FM>;
    Operand<G::kRows, PX> p;
    Operand<kCols, QX> q;
    int n_slabs, full;  // slabs (two at least: what is behind the end is zeros), and how many of them are whole
    int len_p, len_q;   // contraction in bytes (along) or elements (across)
    // Lines of a slab that this workgroup asks the L2 for, kAhead slabs in front of its copies: of the row tile that its eight
    // neighbours on the XCD share an eighth, of the column tile that four share a quarter, 24 lines per wave.  (The barrier
    // of a slab waits for the slowest of 512 lines: without this, nearly always for one that missed the L2.)
    const char *ahead;
    int64_t ahead_step;
    int ahead_slab;

    __device__ __forceinline__ void set_ahead(int tid, int64_t p_pitch, int p_live, int64_t q_pitch, int q_live) {
        const int slot = blockIdx.x / 8, wave = tid >> 6, lane = min(tid & 63, 23);
        const bool is_p = lane < 8;
        ahead = is_p ? p.base + Operand<G::kRows, PX>::line((slot & 7) * 8 * FM + wave * 2 * FM + min(lane, 2 * FM - 1), p_pitch, p_live)
                     : q.base + Operand<kCols, QX>::line(((slot >> 3) & 3) * 64 + wave * 16 + lane - 8, q_pitch, q_live);
        ahead_step = is_p ? p.step : q.step;
        ahead_slab = min(2 + kAhead, full - 1);
        ahead += ahead_slab * ahead_step;
        if (full == 0) ahead = reinterpret_cast<const char *>(&g_zeros);
    }
    // Behind the copies of a slab: one more copy, into the wave's scratch, which is free during a contraction.
    __device__ __forceinline__ void ask_ahead(uint32_t sink) {
        copy4_at(ahead, sink);
        if (++ahead_slab < full) ahead += ahead_step;
    }
    __device__ __forceinline__ void set_length(int elements, int bytes_per) {
        len_p = PX ? elements : elements * bytes_per;
        len_q = QX ? elements : elements * bytes_per;
        const int per = kSlab / bytes_per;  // (the bytes of a group's rows may pass 32 bits; an operand's along do not)
        full = elements / per;
        n_slabs = max(full + (elements % per > 0), 2);
    }
    // `at`: the wave's first piece in the stage.
    template <int C>
    __device__ __forceinline__ void issue(uint32_t at, const char *p_slab, const char *q_slab) const {
        if constexpr (C < G::kQPieces) q.template issue<C, G::kPBytes>(q_slab, at);
        else p.template issue<C - G::kQPieces, 0>(p_slab, at);
    }
    __device__ __forceinline__ void issue_all(int tid, uint32_t at, int slab) const {
        const char *p_slab = p.base + slab * p.step, *q_slab = q.base + slab * q.step;
        if (slab < full) {
            unrolled<G::kCopies>([&](auto c) { issue<c.value>(at, p_slab, q_slab); });
        } else {
            unrolled<G::kQPieces>([&](auto c) { q.template issue_end<c.value, G::kPBytes>(tid, q_slab, at, len_q - slab * (QX ? 64 : kSlab)); });
            unrolled<G::kPPieces>([&](auto c) { p.template issue_end<c.value, 0>(tid, p_slab, at, len_p - slab * (PX ? 64 : kSlab)); });
        }
    }
};

template <int N>
__device__ __forceinline__ void wait_copies() {
    asm volatile("s_waitcnt vmcnt(%0)" : : "n"(N) : "memory");
}

// The contraction of one tile.  acc[f][t]: column fragment 4 wn + f against row fragment FM wm + t.  The copies run through
// from tile to tile: slab k is in stage (stage + k) % 2, slabs 0 and 1 are on their way (slab 0 of this wave has landed) when a
// tile begins, and while its last two slabs are computed, the first two of the next tile follow them into the ring.
//   next.post()          behind the first barrier: looks for the next tile
//   next.pin()           before the first slab but one is waited for: loads of the caller's have landed
//   next.take(feed)      behind a later barrier, when the last copy of this tile is out: 0: there is none; 1: one of the same
//                        height, which `feed` is now; 2: one of another, which next.other(slab, at) copies
// Returns what take() did.  Every wave is past the last slab's reads when one returns: the scratch may be used.
template <class T, int FM, bool PX, bool QX, class Next>
__device__ __forceinline__ int contract(typename T::Acc (&acc)[4][FM], Feed<FM, PX, QX> &feed, const char *lds, int tid, uint32_t &stage,
                                        Next &next) {
    using G = Geo<FM>;
    constexpr int READS = 4 + FM, MM = 4 * FM;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6), base = ring::lds_addr(lds);
    const uint32_t sink = base + kScratchOff + wave * kScratchBytes + kScratchBytes - 256;
    const int lane = tid & 63, n = feed.n_slabs;
    Reader<G::kRows, PX> rp;
    Reader<kCols, QX> rq;
    rp.setup(lane, (wave >> 1) * FM, base + stage * kStageStride);
    rq.setup(lane, (wave & 1) * 4, base + stage * kStageStride + G::kPBytes);
    ring::all_read();  // every wave's share of slab 0 has landed; the scratch is free

    i32x4 a[2][4], b[2][FM];
    auto read = [&](int r, int set, int j) {
        if (r < 4) a[set][r] = rq.read(r, j);
        else b[set][r - 4] = rp.read(r - 4, j);
    };
#pragma unroll
    for (int r = 0; r < READS; ++r) read(r, 0, 0);
    next.post();

    // Where the next copies go: the wave's first piece in the stage of slab k, and slab k + 2 of the operands.
    uint32_t into = base + stage * kStageStride + wave * 1024;
    const char *p_slab = feed.p.base + 2 * feed.p.step, *q_slab = feed.q.base + 2 * feed.q.step;
    uint32_t by = 0;
    // Step J of a slab: its matrix instructions, the reads of the next step's fragments behind the first half of them, and
    // copies FROM .. TO - 1 of a slab spread over all of them, if `go`.  `more(m)` runs behind instruction m.  J == 4: step 0 of
    // the first slab, where the sums begin.
    auto step = [&](auto J, auto read_next, auto from, auto to, bool go, auto more) {
        constexpr int j = J.value % 4, set = j & 1, FROM = from.value, COUNT = to.value - from.value;
        unrolled<MM>([&](auto M) {
            constexpr int m = M.value, t = m >> 2, f = m & 3;
            acc[f][t] = T::mfma(a[set][f], b[set][t], J.value == 4 ? typename T::Acc{} : acc[f][t]);
            if constexpr (read_next.value) {
#pragma unroll
                for (int r = 0; r < READS; ++r)
                    if (r * MM / (2 * READS) == m) read(r, set ^ 1, (j + 1) & 3);
            }
            unrolled<COUNT>([&](auto c) {
                if constexpr ((c.value * MM + MM / 2) / COUNT == m) {
                    if (go) feed.template issue<FROM + c.value>(into, p_slab, q_slab);
                }
            });
            more(M);
            PMOE_GMM_FENCE();
        });
    };
    using Yes = std::integral_constant<bool, true>;
    using No = std::integral_constant<bool, false>;
#define PMOE_INT(v) std::integral_constant<int, (v)>()
    // Copies are spread over two steps: in one, the four waves ask the address path of the CU for more than it takes (16 cycles
    // a copy) and stand still; in three, the last ones have too little time to land.
    constexpr int C1 = G::kCopies / 2, C2 = G::kCopies;
    auto nothing = [](auto) {};
    // The readers on to the other stage, among the last instructions of step 2, whose reads are the stage's last.
    auto move = [&](auto M) {
        constexpr int m = M.value;
        if constexpr (m == MM / 2) {
            by = stage == 0 ? kStageStride : 0u - kStageStride;
            stage ^= 1;
        } else if constexpr (m > MM / 2) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (MM / 2 + 1 + i * (MM / 2 - 1) / 8 == m) (i < 4 ? rp.at[i & 3] : rq.at[i & 3]) += by;
        }
    };
    // The slabs of the loops begin with step 3 of slab k and end with step 2 of slab k + 1.  Matrix instructions stand in no
    // branch: with them in branches the compiler keeps a second set of accumulators and spills.
    step(PMOE_INT(4), Yes(), PMOE_INT(0), PMOE_INT(0), false, nothing);
    step(PMOE_INT(1), Yes(), PMOE_INT(0), PMOE_INT(0), false, nothing);
    step(PMOE_INT(2), Yes(), PMOE_INT(0), PMOE_INT(0), false, move);
    wait_copies<0>();
    next.pin();
    int k = 0;
    for (; k + 2 < feed.full; ++k) {
        ring::wait_and_barrier<1>();  // slab k + 1 has landed (behind it is the line asked for ahead)
        PMOE_GMM_FENCE();
        step(PMOE_INT(3), Yes(), PMOE_INT(0), PMOE_INT(C1), true, nothing);
        step(PMOE_INT(0), Yes(), PMOE_INT(C1), PMOE_INT(C2), true, nothing);
        step(PMOE_INT(1), Yes(), PMOE_INT(0), PMOE_INT(0), false, [&](auto M) {  // (no copy of the slab may follow)
            if constexpr (M.value == MM / 2) feed.ask_ahead(sink);
            if constexpr (M.value == MM / 2 + 1) {
                p_slab += feed.p.step;
                q_slab += feed.q.step;
                into = base + stage * kStageStride + wave * 1024;
            }
        });
        step(PMOE_INT(2), Yes(), PMOE_INT(0), PMOE_INT(0), false, move);
    }
    int kind = 0;
    for (; k + 1 < n; ++k) {
        ring::wait_and_barrier<0>();
        bool go = false;
        if (k + 2 < n) {
            feed.issue_all(tid, into, k + 2);  // the slab with the end, or behind it
        } else {
            kind = next.take(feed);
            go = kind == 1 && feed.full >= 1;
            if (kind == 1 && !go) feed.issue_all(tid, into, 0);
            if (kind == 2) next.other(0, into);
            p_slab = feed.p.base;
            q_slab = feed.q.base;
        }
        PMOE_GMM_FENCE();
        step(PMOE_INT(3), Yes(), PMOE_INT(0), PMOE_INT(C1), go, nothing);
        step(PMOE_INT(0), Yes(), PMOE_INT(C1), PMOE_INT(C2), go, nothing);
        step(PMOE_INT(1), Yes(), PMOE_INT(0), PMOE_INT(0), false, nothing);
        into = base + stage * kStageStride + wave * 1024;
        step(PMOE_INT(2), Yes(), PMOE_INT(0), PMOE_INT(0), false, move);
    }
    ring::all_read();
    const bool go = kind == 1 && feed.full >= 2;
    if (kind == 1 && !go) feed.issue_all(tid, into, 1);
    if (kind == 2) next.other(1, into);
    p_slab = feed.p.base + feed.p.step;
    q_slab = feed.q.base + feed.q.step;
    PMOE_GMM_FENCE();
    step(PMOE_INT(3), No(), PMOE_INT(0), PMOE_INT(C2), go, nothing);
#undef PMOE_INT
    // Slab 0 of the next tile took the place of the last slab but one, which `stage` is back at.  It has landed once at most
    // the copies of its slab 1 are under way (10 in the lowest tile).
    if (kind == 1) wait_copies<G::kCopies>();
    else wait_copies<Geo<1>::kCopies>();
    return kind;
}

}  // namespace gmm
}  // namespace pmoe
