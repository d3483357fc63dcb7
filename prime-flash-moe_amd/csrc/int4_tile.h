// Weights of 4 bits with a scale per 32, 64 or 128 values of a row, gfx950: their layout in memory, and how a wave multiplies
// them with rows of 16-bit numbers.
//
// A weight is q s, q an integer in -8 .. 7, s a 16-bit number.  A matrix (N, K) is held in tiles of 16 rows x 128 columns, 1 KB
// each, [N / 16][K / 128]; lane l of the wave that takes a tile reads its 16 bytes at 16 l, so that a load of the wave is 1 KB in
// one piece (rows of their own would be 64 bytes of 16 rows per load).  With r = l % 16, c = l / 16: dword j of the lane holds row
// r, columns 32 j + 8 c .. + 7, which is what a matrix instruction of 16 x 16 x 32 wants of the lane.  In the dword, as q + 8,
// columns 0, 2, 4, 6, 1, 3, 5, 7 from the lowest bits up: a shift and a mask leave two neighbours in the halves of a register.
// Scales: [N / 16][K / 128][16 rows][128 / group].  What a last tile has behind column K is q = 0, s = 0.
//
// To 16 bits without arithmetic: q + 8 in the highest bits of the mantissa of 16.0 is the number 24 + q.  The 24 too much leaves
// the sum again as a matrix instruction of its own, with -24 in place of the weights, once per row of x and group for all strips
// of weights of a wave.  (Products and sums are fp32: what cancels costs two bits of 24, where the result keeps 8 or 11.  A row of
// x with an infinity comes out as NaN, where the exact weights would leave an infinity.)  Eight weights are four shifts and four
// and-ors; conversions to fp32 and back would be twenty instructions, which is more than there is time for at the rate of the memory:
// 21 weights a cycle and CU.
//
// bf16 reaches as far as fp32, and 24 times a sum of 128 of it further.  So bf16 weights are 2^-12 (24 + q), from 2^-8 in place of 16.0: no
// sum of a group passes 24 x 128 x 2^-12 = 0.75 of the largest |x|, and the 2^12 come back in the wave's sum, where all rows of weights
// have been scaled.  Powers of two change no bit of what stays above 2^-126; the products of the least numbers are subnormal, which
// the matrix instructions keep.  (What is left of it: scaled sums have steps of 2^-149, so that those of outputs below 2^-114 are
// rounded to multiples of 2^-137.)
//
// Sums of a group are scaled in fp32, by four multiply-adds per 128 / group tiles.
#pragma once
#include "grouped_few.h"

namespace pmoe {
namespace int4 {

using gmm::Bf16;
using gmm::F16;
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kTileRows = 16, kTileCols = 128, kTileBytes = 1024;

__host__ __device__ inline int tiles_of(int k) { return (k + kTileCols - 1) / kTileCols; }

// The two constants of the way to 16 bits, one in a scalar and one in a vector register, which the compiler is not told the values of: an
// and-or has no room for a constant of 32 bits, and for known ones it makes an and and an or, half as many instructions again.
struct Masks {
    uint32_t mask, sixteen;
    __device__ __forceinline__ Masks(uint32_t m, uint32_t s) : mask(m), sixteen(s) {
        asm("" : "+s"(mask));
        asm("" : "+v"(sixteen));
    }
};

template <class T>
struct Num;
template <>
struct Num<Bf16> {
    static constexpr uint32_t kMask = 0x00780078u, kSixteen = 0x41804180u;
    // of a product: 16 and -24, both over kUnit
    static constexpr uint32_t kBase = 0x3b803b80u, kMinus24 = 0xbbc0bbc0u;
    static constexpr float kUnit = 0x1p12f;
    static __device__ __forceinline__ i32x4 wide(uint32_t w, Masks m) {
        return i32x4{(int)((w << 3 & m.mask) | m.sixteen), (int)((w >> 1 & m.mask) | m.sixteen), (int)((w >> 5 & m.mask) | m.sixteen), (int)((w >> 9 & m.mask) | m.sixteen)};
    }
    static __device__ __forceinline__ float to_f32(uint16_t v) { return __uint_as_float((uint32_t)v << 16); }
    static __device__ __forceinline__ uint16_t from_f32(float v) { return (uint16_t)pack2_bf16(v, 0.f); }
    static __device__ __forceinline__ bool finite(uint16_t v) { return (v & 0x7f80u) != 0x7f80u; }
    static constexpr uint16_t kNan = 0x7fc0;
    static constexpr float kLeastScale = 0x1p-126f;
};
template <>
struct Num<F16> {
    static constexpr uint32_t kMask = 0x03c003c0u, kSixteen = 0x4c004c00u;
    static constexpr uint32_t kBase = kSixteen, kMinus24 = 0xce00ce00u;
    static constexpr float kUnit = 1.0f;
    static __device__ __forceinline__ i32x4 wide(uint32_t w, Masks m) {
        return i32x4{(int)((w << 6 & m.mask) | m.sixteen), (int)((w << 2 & m.mask) | m.sixteen), (int)((w >> 2 & m.mask) | m.sixteen), (int)((w >> 6 & m.mask) | m.sixteen)};
    }
    static __device__ __forceinline__ float to_f32(uint16_t v) { return (float)__builtin_bit_cast(_Float16, v); }
    static __device__ __forceinline__ uint16_t from_f32(float v) { return __builtin_bit_cast(uint16_t, (_Float16)v); }
    static __device__ __forceinline__ bool finite(uint16_t v) { return (v & 0x7c00u) != 0x7c00u; }
    static constexpr uint16_t kNan = 0x7e00;
    static constexpr float kLeastScale = 0x1p-24f;
};

__device__ __forceinline__ i32x4 load_once16(const char *p) { return __builtin_nontemporal_load(reinterpret_cast<const i32x4 *>(p)); }

// A piece of memory of up to 4 GB, wave-uniform: a load takes an offset per lane and one for the wave; behind `bytes` it reads zeros.
typedef __amdgpu_buffer_rsrc_t Buffer;
__device__ __forceinline__ Buffer buffer(const char *p, uint32_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<char *>(ring::uniform_ptr(p)), 0, (int)bytes, 0x00020000);  // (raw bytes, no stride)
}
__device__ __forceinline__ i32x4 load(Buffer b, uint32_t lane, uint32_t wave) { return __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(b, lane, wave, 0)); }
// The same with the non-temporal hint, for what no other workgroup reads.  (The workgroup itself does, of experts with more rows than it takes at
// a time.)
__device__ __forceinline__ i32x4 load_once(Buffer b, uint32_t lane, uint32_t wave) { return __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(b, lane, wave, 2)); }

// The same, as it stands in memory now, whatever the caches of the XCD hold.
__device__ __forceinline__ i32x4 load_now(Buffer b, uint32_t lane, uint32_t wave) { return __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(b, lane, wave, 16)); }

// The scales of a lane's row in a tile.
template <int GROUP>
struct TileScales {
    static constexpr int kCount = kTileCols / GROUP, kBytes = kTileRows * kCount * 2;  // of a row, of a tile
    uint16_t v[kCount];
    __device__ __forceinline__ void load(const char *tile, int r) {
        const char *p = tile + r * kCount * 2;
        if constexpr (kCount == 4) {
            const uint2 u = *reinterpret_cast<const uint2 *>(p);
            v[0] = (uint16_t)u.x, v[1] = (uint16_t)(u.x >> 16), v[2] = (uint16_t)u.y, v[3] = (uint16_t)(u.y >> 16);
        } else if constexpr (kCount == 2) {
            const uint32_t u = *reinterpret_cast<const uint32_t *>(p);
            v[0] = (uint16_t)u, v[1] = (uint16_t)(u >> 16);
        } else {
            v[0] = *reinterpret_cast<const uint16_t *>(p);
        }
    }
};

// Rows of x on their way to a wave: S tiles of up to M rows, in LDS of the wave's own.  A load of the wave is 1 KB, four rows
// of a tile, where the operands of its matrix instructions would be 64 bytes of 16 rows each, most of them the same row again: one
// load per tile instead of four for up to four rows.  Row q of tile i is 256 bytes, its chunk of 16 bytes k in slot k ^ q % 16: the
// reads of 16 rows cover all banks.
template <int M, int S>
struct Rows {
    static_assert(M % 4 == 0, "four rows a load");
    static constexpr int kBytes = S * M * 256;
    i32x4 v[S][M / 4];
    // f(tile, load) for what there is of `n` rows and tiles t .. t1 - 1.
    template <class F>
    static __device__ __forceinline__ void each(int n, int t, int t1, F f) {
#pragma unroll
        for (int i = 0; i < S; ++i)
            if (i == 0 || t + i < t1) {
#pragma unroll
                for (int g = 0; g < M / 4; ++g)
                    if (g == 0 || 4 * g < n) f(i, g);
            }
    }
    // `at[g]`: where this lane's 16 bytes of row 4 g + lane / 16 are in tile 0; `n`: rows, from 1 to M; `k`: columns; get(at, what to add): 16
    // bytes.
    template <class Get>
    __device__ __forceinline__ void load(Get get, const uint32_t (&at)[M / 4], int n, int t, int t1, int k) {
        each(n, t, t1, [&](int i, int g) {
            if ((t + i + 1) * kTileCols <= k) {
                v[i][g] = get(at[g], (t + i) * (kTileCols * 2));
            } else {
                v[i][g] = i32x4{0, 0, 0, 0};
                if ((t + i) * kTileCols + (int)(threadIdx.x & 15) * 8 < k) v[i][g] = get(at[g], (t + i) * (kTileCols * 2));
            }
        });
    }
    // The largest of the words that were loaded.
    __device__ __forceinline__ uint32_t most(int n, int t, int t1) const {
        uint32_t m = 0;
        each(n, t, t1, [&](int i, int g) {
#pragma unroll
            for (int d = 0; d < 4; ++d) m = max(m, (uint32_t)v[i][g][d]);
        });
        return m;
    }
    __device__ __forceinline__ void store(char *lds, int n, int t, int t1) const {
        const int lane = threadIdx.x & 63, sub = lane >> 4;
        each(n, t, t1, [&](int i, int g) {
            *reinterpret_cast<i32x4 *>(lds + ((i * M + 4 * g + sub) * 256 + (((lane & 15) ^ (4 * g + sub)) & 15) * 16)) = v[i][g];
        });
    }
    // Operand of row 16 q + r, columns 32 j + 8 c .. + 7 of tile i.
    static __device__ __forceinline__ i32x4 read(const char *lds, int n, int i, int q, int j) {
        const int lane = threadIdx.x & 63, row = min(16 * q + (lane & 15), n - 1);
        return *reinterpret_cast<const i32x4 *>(lds + (i * M + row) * 256 + (((4 * j + (lane >> 4)) ^ row) & 15) * 16);
    }
};

// acc[u][q] = n rows of x times the weights of tiles t0 .. t1 - 1 of U strips (16 weight rows each), for one wave.  Lane l, r = l %
// 16, c = l / 16: `w[u]`, `s[u]` begin strip u, row q of x is row(q) bytes behind `x`.  acc[u][q][i]: weight row r, row 16 q + 4 c + i of x (any of the n where there are fewer).
// `k`: columns; nothing of x is read behind them.  M: rows at most, `lds`: Rows<M, S>::kBytes of the wave's own.  S: tiles whose loads are in flight
// together; what hides the rest of their latency is other waves.  X: type of the rows, T: of the scales.  wait(most): called with the largest word of what was loaded of x, for
// rows that may not all be there yet: true until they are.
struct NoWait {
    static constexpr bool kWaits = false;
};
template <class X, class T, int GROUP, int U, int R, int S, int M = 16 * R, class Row, class Wait = NoWait>
__device__ __forceinline__ void dots(f32x4 (&acc)[U][R], const char *const (&w)[U], const char *const (&s)[U], const char *x, Row row, int n, int t0, int t1, int k, char *lds, Wait wait = {}) {
    using Sc = TileScales<GROUP>;
    constexpr int PER = GROUP / 32;
    const int lane = threadIdx.x & 63, r = lane & 15;
    const Buffer xb = buffer(x, ~0u);
    uint32_t at[M / 4];
#pragma unroll
    for (int g = 0; g < M / 4; ++g) at[g] = row(min(4 * g + (lane >> 4), n - 1)) + r * 16;
    const Masks masks(Num<X>::kMask, Num<X>::kBase);
    const i32x4 minus = {(int)Num<X>::kMinus24, (int)Num<X>::kMinus24, (int)Num<X>::kMinus24, (int)Num<X>::kMinus24};
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int q = 0; q < R; ++q) acc[u][q] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int t = t0; t < t1; t += S) {
        i32x4 wv[S][U];
        Sc sc[S][U];
        Rows<M, S> rows;
        rows.load([&](uint32_t l, uint32_t w) { return load(xb, l, w); }, at, n, t, t1, k);
#pragma unroll
        for (int i = 0; i < S; ++i)
            if (i == 0 || t + i < t1) {
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    wv[i][u] = load_once16(w[u] + (int64_t)(t + i) * kTileBytes + lane * 16);
                    sc[i][u].load(s[u] + (int64_t)(t + i) * Sc::kBytes, r);
                }
            }
        if constexpr (Wait::kWaits)
            while (wait(rows.most(n, t, t1))) rows.load([&](uint32_t l, uint32_t w) { return load_now(xb, l, w); }, at, n, t, t1, k);
        wave_lds_order();  // (the reads of the tiles before are done)
        rows.store(lds, n, t, t1);
        wave_lds_order();
#pragma unroll
        for (int i = 0; i < S; ++i)
            if (i == 0 || t + i < t1) {
#pragma unroll
                for (int g = 0; g < Sc::kCount; ++g) {
                    i32x4 xv[R][PER];
                    f32x4 less[R];  // -24 times the sums of the group's part of x
#pragma unroll
                    for (int q = 0; q < R; ++q) {
                        less[q] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int j = 0; j < PER; ++j) {
                            xv[q][j] = Rows<M, S>::read(lds, n, i, q, g * PER + j);
                            less[q] = gmm::few::Mini<X>::mfma(xv[q][j], minus, less[q]);
                        }
                    }
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        f32x4 sum[R];
#pragma unroll
                        for (int q = 0; q < R; ++q) sum[q] = less[q];
#pragma unroll
                        for (int j = 0; j < PER; ++j) {
                            const i32x4 b = Num<X>::wide((uint32_t)wv[i][u][g * PER + j], masks);
#pragma unroll
                            for (int q = 0; q < R; ++q) sum[q] = gmm::few::Mini<X>::mfma(xv[q][j], b, sum[q]);
                        }
                        const float f = Num<T>::to_f32(sc[i][u].v[g]);
#pragma unroll
                        for (int q = 0; q < R; ++q)
#pragma unroll
                            for (int e = 0; e < 4; ++e) acc[u][q][e] = fmaf(sum[q][e], f, acc[u][q][e]);
                    }
                }
            }
    }
    if constexpr (Num<X>::kUnit != 1.0f)
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int q = 0; q < R; ++q)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[u][q][e] *= Num<X>::kUnit;
}

}  // namespace int4
}  // namespace pmoe
