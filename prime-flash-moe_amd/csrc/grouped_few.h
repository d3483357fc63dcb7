// Ragged expert products for few rows per group, gfx950: out[r] = x[r] times its group's weights, streamed once.
//
// Bound by the stream of the touched groups' weights from HBM and, for the smallest calls, by how soon it starts and over how
// many CUs it is spread.  So a workgroup takes one group and 16 U of its weight rows, nothing is planned ahead, and every wave
// works alone until the last sum: the waves share the contraction in chunks of 128 bytes per row by turns, and each copies
// its chunks (weight rows, then the rows of x that are live) into a ring of its own in LDS, whole lines at a time, and waits
// for nobody.  (Straight into registers a matrix instruction's operand is 64 bytes of 16 rows, half a line: 4.3 TB/s.)
// 8 experts of 28672 x 4096 in bf16, 58 rows: 287 us, 6.6 TB/s; 64 tokens on 256 experts of 4096 x 7168 in 8 bits, 512 rows:
// 590 us, 6.3 TB/s.  Rings of 20 KB (eight waves per CU) or weights without the non-temporal hint lose 10 - 20 %.
// Whether rows are few is a matter of their average: a group with many of them is one workgroup's per 16 U weight rows, which
// it reads once per 32 rows (1536 x 2048 in bf16: 2048 rows on one of 128 experts 437 us, spread evenly 146).
//
// Matrix instructions of 16 x 16: lane l holds weight row l % 16 and row l % 16 of x, 16 bytes at 16 (l / 16).  Rows of a
// stage are 8 chunks of 16 B, chunk c of row r in slot c ^ (r / 2) % 8: the reads of 16 rows cover all banks once.  The waves'
// sums meet in LDS and are added in wave order.
#pragma once
#include <algorithm>

#include "grouped_kernel.h"

namespace pmoe {
namespace gmm {
namespace few {

typedef float f32x4 __attribute__((ext_vector_type(4)));

template <class T>
struct Mini;
template <>
struct Mini<Bf16> {
    using Acc = f32x4;
    static __device__ __forceinline__ Acc mfma(i32x4 a, i32x4 b, Acc c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
};
template <>
struct Mini<F16> {
    using Acc = f32x4;
    static __device__ __forceinline__ Acc mfma(i32x4 a, i32x4 b, Acc c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
};
template <>
struct Mini<I8> {
    using Acc = i32x4;
    static __device__ __forceinline__ Acc mfma(i32x4 a, i32x4 b, Acc c) { return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0); }
};

struct Span {
    int group, begin, end;
    bool zero;  // rows behind the last group
};

// The `slot`-th block of up to BLOCK rows of a group (0: all of them); behind those, the rows behind the last group; begin ==
// end: neither.  A wave at a time, lane l looks at groups c l .. c l + c - 1.  As Walk: a group begins at the furthest end in
// front of it.
template <int BLOCK>
__device__ __forceinline__ int blocks_of(int rows) {
    return BLOCK > 0 ? (rows + BLOCK - 1) / max(BLOCK, 1) : rows > 0;
}
template <int BLOCK>
__device__ __forceinline__ Span find_span(const RowsArgs &a, int slot) {
    Span s = {0, 0, a.rows, false};
    if (a.offsets == nullptr) {
        if (BLOCK > 0) s.begin = min(slot * BLOCK, a.rows), s.end = min(s.begin + BLOCK, a.rows);
        else if (slot != 0) s.end = 0;
        return s;
    }
    const int lane = threadIdx.x & 63, c = (a.n_groups + 63) / 64, g0 = c * lane;
    int far = 0;
    for (int i = 0; i < c; ++i) far = max(far, g0 + i < a.n_groups ? group_end(a, g0 + i) : 0);
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const int v = __shfl_up(far, d, 64);
        if (lane >= d) far = max(far, v);
    }
    const int before = __shfl_up(far, 1, 64), first = lane == 0 ? 0 : before;
    int count = 0, begin = first;
    for (int i = 0; i < c; ++i) {
        const int end = g0 + i < a.n_groups ? max(group_end(a, g0 + i), begin) : begin;
        count += blocks_of<BLOCK>(end - begin);
        begin = end;
    }
    int incl = count;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const int v = __shfl_up(incl, d, 64);
        if (lane >= d) incl += v;
    }
    const int total = __shfl(incl, 63, 64), live_rows = __shfl(far, 63, 64);
    if (slot >= total) {
        s.begin = live_rows;
        s.end = slot == total ? a.rows : live_rows;
        s.zero = true;
    } else {
        const bool mine = incl - count <= slot && slot < incl;
        if (mine) {
            int left = slot - (incl - count);
            begin = first;
            for (int i = 0; i < c; ++i) {
                const int end = g0 + i < a.n_groups ? max(group_end(a, g0 + i), begin) : begin;
                const int blocks = blocks_of<BLOCK>(end - begin);
                if (left >= 0 && left < blocks) {
                    const int from = BLOCK > 0 ? begin + left * BLOCK : begin;
                    s = {g0 + i, from, BLOCK > 0 ? min(from + BLOCK, end) : end, false};
                }
                left -= blocks;
                begin = end;
            }
        }
        const int owner = __builtin_ctzll(__ballot(mine));
        s.group = __shfl(s.group, owner, 64);
        s.begin = __shfl(s.begin, owner, 64);
        s.end = __shfl(s.end, owner, 64);
    }
    s.group = uniform(s.group);
    s.begin = uniform(s.begin);
    s.end = uniform(s.end);
    return s;
}

// Waits until at most `n` (wave-uniform, 0 .. 40) of this wave's copies are in flight.
__device__ __forceinline__ void wait_copies(int n) {
#define PMOE_W(k) case k: asm volatile("s_waitcnt vmcnt(" #k ")" : : : "memory"); break;
    switch (n) {
        PMOE_W(1) PMOE_W(2) PMOE_W(3) PMOE_W(4) PMOE_W(5) PMOE_W(6) PMOE_W(7) PMOE_W(8) PMOE_W(9) PMOE_W(10)
        PMOE_W(11) PMOE_W(12) PMOE_W(13) PMOE_W(14) PMOE_W(15) PMOE_W(16) PMOE_W(17) PMOE_W(18) PMOE_W(19) PMOE_W(20)
        PMOE_W(21) PMOE_W(22) PMOE_W(23) PMOE_W(24) PMOE_W(25) PMOE_W(26) PMOE_W(27) PMOE_W(28) PMOE_W(29) PMOE_W(30)
        PMOE_W(31) PMOE_W(32) PMOE_W(33) PMOE_W(34) PMOE_W(35) PMOE_W(36) PMOE_W(37) PMOE_W(38) PMOE_W(39) PMOE_W(40)
        default: asm volatile("s_waitcnt vmcnt(0)" : : : "memory"); break;
    }
#undef PMOE_W
}

constexpr int kMaxStages = 4;
constexpr int kCH = 128;          // bytes of a row that a wave copies at a time
constexpr int kRing = 10 * 1024;  // of a wave: sixteen waves per CU
constexpr int kBlockRing = 20 * 1024, kBlock = 64;  // blocks of 64 rows: eight waves per CU

// LDS of a workgroup: a ring per wave; the waves' sums lie where their own rings were.
template <int U, int WAVES, int RING>
struct Shared {
    char ring[WAVES][RING];
    static_assert(RING >= U * 64 * 16, "a wave's sums of one fragment of rows fit its ring");
};

// One pass of up to 16 R rows over the workgroup's 16 U weight rows.
template <class T, class OUT, int U, int R, int WAVES, int RING>
__device__ __forceinline__ void pass(const RowsArgs &a, int group, int row0, int live, int col0, Shared<U, WAVES, RING> &sh) {
    static_assert(RING >= 16 * (U + R) * kCH, "a stage fits the ring");
    constexpr int CH = kCH;
    using Acc = typename Mini<T>::Acc;
    constexpr int CHUNKS = CH / 16, PER = 1024 / CH;      // chunks of a row; rows that a copy moves
    constexpr int W_COPIES = 16 * U / PER, X_COPIES = 16 * R / PER;
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
    const int depth = a.depth * T::kBytes, chunks = (depth + CH - 1) / CH;
    auto swizzle = [](int row) { return (row >> 1) % CHUNKS; };

    const char *w = ring::uniform_ptr(a.w + group * a.w_group + col0 * a.w_pitch), *x = ring::uniform_ptr(a.x + row0 * a.x_pitch);
    const int sub = lane / CHUNKS, slot = lane % CHUNKS;
    uint32_t w_off[W_COPIES], x_off[X_COPIES];
#pragma unroll
    for (int i = 0; i < W_COPIES; ++i) {
        const int row = i * PER + sub;
        w_off[i] = (uint32_t)min(row, a.cols - 1 - col0) * (uint32_t)a.w_pitch + (uint32_t)(slot ^ swizzle(row)) * 16u;
    }
#pragma unroll
    for (int i = 0; i < X_COPIES; ++i) {
        const int row = i * PER + sub;
        x_off[i] = (uint32_t)min(row, live - 1) * (uint32_t)a.x_pitch + (uint32_t)(slot ^ swizzle(row)) * 16u;
    }
    const int x_copies = (live + PER - 1) / PER;
    const int copies = W_COPIES + x_copies, stage_bytes = copies * 1024;
    const int stages = min(min(RING / stage_bytes, kMaxStages), 40 / copies + 1);
    const uint32_t base = ring::lds_addr(sh.ring[wave]);
    const int n = (chunks - wave + WAVES - 1) / WAVES;  // chunks of this wave
    // Each workgroup begins at another chunk of its rows: workgroups that run side by side read the same place in rows that lie a
    // multiple of some KB apart, few HBM channels at a time (8 experts of 28672 x 4096 in bf16: 308 -> 287 us).
    const int rot = n > 0 ? (int)blockIdx.x % n : 0;
    auto issue = [&](int j, uint32_t at) {
        const int turn = j + rot >= n ? j + rot - n : j + rot;
        const int64_t k = (int64_t)(wave + turn * WAVES) * CH;
        if (k + CH <= depth) {
            unrolled<W_COPIES>([&](auto i) {
                copy16_once<i.value * 1024>(w + k, w_off[i.value], at);
            });
            unrolled<X_COPIES>([&](auto i) {
                if (i.value < x_copies) copy16<(W_COPIES + i.value) * 1024>(x + k, x_off[i.value], at);
            });
        } else {
            auto from = [&](const char *src, uint32_t off, int row) {
                return (slot ^ swizzle(row)) * 16 < depth - (int)k ? src + k + off : reinterpret_cast<const char *>(&g_zeros);
            };
            unrolled<W_COPIES>([&](auto i) { copy16_at<i.value * 1024>(from(w, w_off[i.value], i.value * PER + sub), at); });
            unrolled<X_COPIES>([&](auto i) {
                if (i.value < x_copies) copy16_at<(W_COPIES + i.value) * 1024>(from(x, x_off[i.value], i.value * PER + sub), at);
            });
        }
    };
    const int first = min(stages, n);
    for (int j = 0; j < first; ++j) issue(j, base + j * stage_bytes);

    Acc acc[U][R] = {};
    // This lane's first chunk of its weight row and of its rows of x (one that was copied where its own was not, which reaches no
    // output); step s: chunk 4 s on, exclusive or.
    const int r = lane & 15, q = lane >> 4;
    const uint32_t w_at = r * CH + ((q ^ swizzle(r)) << 4);
    uint32_t x_at[R];
#pragma unroll
    for (int t = 0; t < R; ++t) {
        const int row = min(t * 16 + r, x_copies * PER - 1);
        x_at[t] = row * CH + ((q ^ swizzle(row)) << 4);
    }
    uint32_t at = base;
    for (int j = 0; j < n; ++j) {
        wait_copies(copies * min(n - 1 - j, stages - 1));
        i32x4 wv[U][CH / 64], xv[R][CH / 64];
        typedef const __attribute__((address_space(3))) i32x4 *lds16;
#pragma unroll
        for (int s = 0; s < CH / 64; ++s) {
#pragma unroll
            for (int u = 0; u < U; ++u) wv[u][s] = *(lds16)(uintptr_t)(at + (w_at ^ s << 6) + u * 16 * CH);
#pragma unroll
            for (int t = 0; t < R; ++t) xv[t][s] = *(lds16)(uintptr_t)(at + (x_at[t] ^ s << 6) + 16 * U * CH);
        }
        asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");  // the stage is in registers
        if (j + stages < n) issue(j + stages, at);
        at = at + stage_bytes == base + stages * stage_bytes ? base : at + stage_bytes;
#pragma unroll
        for (int s = 0; s < CH / 64; ++s)
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int t = 0; t < R; ++t) acc[u][t] = Mini<T>::mfma(wv[u][s], xv[t][s], acc[u][t]);
    }

#pragma unroll
    for (int t = 0; t < R; ++t) {
        if (t > 0) __syncthreads();
#pragma unroll
        for (int u = 0; u < U; ++u) reinterpret_cast<f32x4 *>(sh.ring[wave])[u * 64 + lane] = __builtin_bit_cast(f32x4, acc[u][t]);
        __syncthreads();
        const int row = t * 16 + r, u = wave, col = col0 + u * 16 + q * 4;
        if (u < U && row < live && col < a.cols) {
            Acc sum = __builtin_bit_cast(Acc, reinterpret_cast<const f32x4 *>(sh.ring[0])[u * 64 + lane]);
#pragma unroll
            for (int v = 1; v < WAVES; ++v) sum += __builtin_bit_cast(Acc, reinterpret_cast<const f32x4 *>(sh.ring[v])[u * 64 + lane]);
            float4 f = make_float4((float)sum[0], (float)sum[1], (float)sum[2], (float)sum[3]);
            if constexpr (std::is_same<T, I8>::value) {
                const float xs = a.x_scale[row0 + row];
                const float *ws = a.w_scale + (int64_t)group * a.cols + col;
                f = make_float4(f.x * xs * ws[0], f.y * xs * ws[1], f.z * xs * ws[2], f.w * xs * ws[3]);
            }
            const auto v = Pack<OUT>::four(f.x, f.y, f.z, f.w);
            *reinterpret_cast<std::remove_const_t<decltype(v)> *>(a.out + (row0 + row) * a.out_pitch + (int64_t)col * Pack<OUT>::kBytes) = v;
        }
    }
    __syncthreads();  // the rings may be filled again
}

// BLOCK == 0: a job is all rows of a group, 32 at a time; otherwise one block of up to BLOCK rows.
template <class T, class OUT, int U, int WAVES, int RING, int BLOCK>
__global__ __launch_bounds__(64 * WAVES) void grouped_mm_few_kernel(RowsArgs a, int strips) {
    static_assert(U <= WAVES, "a wave adds up the sums of one unit");
    __shared__ __attribute__((aligned(1024))) Shared<U, WAVES, RING> sh;
    const int slot = (int)blockIdx.x / strips, col0 = ((int)blockIdx.x - slot * strips) * 16 * U;
    const Span s = find_span<BLOCK>(a, slot);
    if (s.zero) {
        constexpr int PER = 16 / Pack<OUT>::kBytes;
        const int chunks = min(16 * U, a.cols - col0) / PER;
        for (int64_t i = threadIdx.x; i < (int64_t)(s.end - s.begin) * chunks; i += 64 * WAVES)
            *reinterpret_cast<uint4 *>(a.out + (s.begin + i / chunks) * a.out_pitch + (int64_t)col0 * Pack<OUT>::kBytes + i % chunks * 16) = make_uint4(0, 0, 0, 0);
        return;
    }
    for (int row0 = s.begin; row0 < s.end;) {
        const int left = s.end - row0;
        if (left <= 16) {
            pass<T, OUT, U, 1, WAVES, RING>(a, s.group, row0, left, col0, sh);
            row0 += 16;
        } else if (BLOCK == 0 || left <= 32) {
            pass<T, OUT, U, 2, WAVES, RING>(a, s.group, row0, min(left, 32), col0, sh);
            row0 += 32;
        } else if constexpr (BLOCK > 0) {
            pass<T, OUT, U, BLOCK / 16, WAVES, RING>(a, s.group, row0, left, col0, sh);
            row0 += BLOCK;
        }
    }
}

template <class T, class OUT, int U, int WAVES, int RING, int BLOCK>
void launch_as(const RowsArgs &a, int64_t slots, hipStream_t stream) {
    const int strips = (a.cols + 16 * U - 1) / (16 * U);
    hipLaunchKernelGGL((grouped_mm_few_kernel<T, OUT, U, WAVES, RING, BLOCK>), dim3((uint32_t)(strips * slots)), dim3(64 * WAVES), 0, stream,
                       a, strips);
}

// Launches these kernels if they are the faster ones.  (Both ways are right for any rows.)
template <class T, class OUT>
bool launch(const RowsArgs &a, hipStream_t stream) {
    const int64_t cus = resident_grid(), behind = a.offsets != nullptr ? 1 : 0;
    const int64_t slots = std::min(a.rows, a.n_groups) + behind, strips = (a.cols + 15) / 16;
    // (A launch has less than 2^32 threads: 256 a job of 32 weight rows where jobs are many.)
    if (a.rows <= 16 * (int64_t)a.n_groups && (strips + 1) / 2 * slots <= UINT32_MAX / 256) {
        // Few jobs: eight waves share one, so that a CU's share is under way at once (one row through 4096 x 7168 in 8 bits: 7.5
        // us instead of 10.4 with four); with more than two jobs per CU four (8 of 128 experts of 1536 x 2048: 12.3 us instead
        // of 14.9).  Wider jobs read x less often: 32 weight rows where there are many (64 tokens on 256 experts of 4096 x
        // 7168 in 8 bits: 590 us instead of 664).
        if (strips * slots <= 2 * cus) launch_as<T, OUT, 1, 8, kRing, 0>(a, slots, stream);
        else if (strips * slots <= 8 * cus) launch_as<T, OUT, 1, 4, kRing, 0>(a, slots, stream);
        else launch_as<T, OUT, 2, 4, kRing, 0>(a, slots, stream);
        return true;
    }
    // Blocks of 64 rows x 32 columns (16, with at most one such job per CU), where tiles of 256 columns would leave CUs idle: a
    // tile's contraction is one workgroup's, a block's is shared by eight waves, and so up to three jobs per CU are faster (8
    // experts of 512 x 4096 in bf16, beside tiles of the height that suits them best: 1.4 jobs per CU 24 us instead of 48, 2.4 37
    // instead of 48; 8 of 1024 x 4096: 2.9 38 instead of 49, but 4.9 65 instead of 48).
    const int64_t blocks = a.rows / kBlock + slots, block_jobs = (strips + 1) / 2 * blocks;
    const int64_t tiles = (a.rows / 256 + std::min(a.rows, a.n_groups)) * ((a.cols + kCols - 1) / kCols);
    if (tiles <= cus && block_jobs <= 3 * cus) {
        if (block_jobs <= cus) launch_as<T, OUT, 1, 8, kBlockRing, kBlock>(a, blocks, stream);
        else launch_as<T, OUT, 2, 8, kBlockRing, kBlock>(a, blocks, stream);
        return true;
    }
    return false;
}

}  // namespace few
}  // namespace gmm
}  // namespace pmoe
