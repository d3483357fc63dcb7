// To 4 bits and back (layout: int4_tile.h).
//
// scale = the 16-bit number nearest to max(amax c, least) with c = 1 / 7 in fp32; q = the integer nearest to the exact quotient of
// value and scale, ties to even, from -8 to 7.  A group with an infinity, a NaN, or a scale beyond the 16-bit type
// gets the scale NaN and q = 0.
//
// Bound by memory: 402 M weights in bf16 to 4 bits 212 us, back 165 us, 4.9 and 6.2 TB/s (a large copy: 5.0).  A wave takes a tile,
// which lies in LDS between the rows of the matrix, 256 bytes of four rows a load or store, and the lanes' shares of the tile.  (Straight
// to and from registers a load is 64 bytes of sixteen rows: 217 and 284 us.)
#include <algorithm>

#include "grouped_host.h"
#include "int4_tile.h"

namespace {

using namespace pmoe;
using namespace pmoe::int4;

struct F32 {};
// Eight values from registers as they were loaded, and the largest magnitude among them as the bits of a float: infinity and the
// NaNs are above all numbers.
template <class FROM>
struct Load {
    static constexpr int kWords = 1;      // of 16 bytes, that hold eight values
    static constexpr bool kShort = true;  // 11 bits of mantissa at most
    static __device__ __forceinline__ uint32_t eight(const i32x4 (&p)[kWords], float (&v)[8]) {
        typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
        const i32x4 w = p[0];
        u16x2 m = {0, 0};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = Num<FROM>::to_f32((uint16_t)w[i]), v[2 * i + 1] = Num<FROM>::to_f32((uint16_t)((uint32_t)w[i] >> 16));
            m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, w[i] & 0x7fff7fffu));
        }
        return __float_as_uint(Num<FROM>::to_f32(m[0] > m[1] ? m[0] : m[1]));
    }
};
template <>
struct Load<F32> {
    static constexpr int kWords = 2;
    static constexpr bool kShort = false;
    static __device__ __forceinline__ uint32_t eight(const i32x4 (&p)[kWords], float (&v)[8]) {
        uint32_t m = 0;
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = __int_as_float(p[k / 4][k % 4]), m = max(m, (uint32_t)p[k / 4][k % 4] & 0x7fffffffu);
        return m;
    }
};

// The integer nearest to x / scale, ties to even, from -8 to 7; plus 8, in the lowest bits of kBias + it.
// The quotient is corrected by its remainder, which an fma gives without rounding.  For 16-bit values that leaves the exact
// quotient where it is half way between two integers, and nothing else is near: with up to 11 bits of mantissa in both, a
// quotient that is not half an odd number is 2^-13 or more away from it.  A float's may be nearer than its last place: there the
// remainder of the integer decides.
constexpr uint32_t kBias = 0x4b400000u;  // bits of 1.5 2^23, whose last place is 1
template <bool SHORT>
__device__ __forceinline__ uint32_t nearest(float x, float scale, float inv) {
    float q = x * inv;
    if constexpr (SHORT) {
        q = fmaf(fmaf(-q, scale, x), inv, q);
    } else {
        q = rintf(q);
        const float rest = fmaf(-q, scale, x), twice = 2.0f * fabsf(rest);
        const bool odd = ((int)q & 1) != 0;
        if (twice > scale || (twice == scale && odd)) q += copysignf(1.0f, rest);
    }
    return __float_as_uint(__builtin_amdgcn_fmed3f(q, -8.0f, 7.0f) + 12582920.0f);
}

// Position of column k (0 .. 7) of a dword, in nibbles.
__device__ __forceinline__ constexpr int nibble(int k) { return k / 2 + k % 2 * 4; }

template <class FROM, class T, int GROUP>
__global__ __launch_bounds__(256) void quantize_int4_kernel(const char *__restrict__ src, char *__restrict__ q, char *__restrict__ scales,
                                                            int64_t n_tiles, int tiles, int cols) {
    using Sc = TileScales<GROUP>;
    constexpr int PER = GROUP / 32, W = Load<FROM>::kWords;
    // A tile of each wave's own, chunk k of row r in slot k ^ r: in by 256 bytes of four rows a load instead of 64 of
    // sixteen
    __shared__ i32x4 lds[4][W][256];
    const int lane = threadIdx.x & 63, r = lane & 15, c = lane >> 4;
    i32x4(&mine)[W][256] = lds[threadIdx.x >> 6];
    for (int64_t tile = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); tile < n_tiles; tile += (int64_t)gridDim.x * 4) {
        const int64_t strip = tile / tiles;
        const int col0 = (int)(tile - strip * tiles) * kTileCols;
        const i32x4 *p = reinterpret_cast<const i32x4 *>(src) + ((strip * 16 + c) * cols + col0 + 8 * r) / 8 * W;
        i32x4 in[4][W];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int k = 0; k < W; ++k) {
                in[i][k] = i32x4{0, 0, 0, 0};
                if (col0 + 8 * r < cols) in[i][k] = p[(int64_t)i * cols / 2 * W + k];
            }
        wave_lds_order();
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int k = 0; k < W; ++k) mine[k][(4 * i + c) * 16 + (r ^ (4 * i + c))] = in[i][k];
        wave_lds_order();
        float v[4][8];
        uint32_t peaks[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            i32x4 raw[W];
#pragma unroll
            for (int k = 0; k < W; ++k) raw[k] = mine[k][r * 16 + ((4 * j + c) ^ r)];
            peaks[j] = Load<FROM>::eight(raw, v[j]);
        }
        uint32_t out[4];
#pragma unroll
        for (int g = 0; g < Sc::kCount; ++g) {
            uint32_t peak = peaks[g * PER];
#pragma unroll
            for (int j = 1; j < PER; ++j) peak = max(peak, peaks[g * PER + j]);
            peak = max(peak, (uint32_t)__shfl_xor((int)peak, 16, 64));
            peak = max(peak, (uint32_t)__shfl_xor((int)peak, 32, 64));
            uint16_t s16 = Num<T>::from_f32(fmaxf(__uint_as_float(peak) * (1.0f / 7.0f), Num<T>::kLeastScale));
            const bool fine = peak < 0x7f800000u && Num<T>::finite(s16), inside = col0 + g * GROUP < cols;
            if (!fine) s16 = Num<T>::kNan;
            const float scale = Num<T>::to_f32(s16), inv = 1.0f / scale;
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                uint32_t word = 0, bias = 0;  // (the sum of the biases leaves in one subtraction)
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    word += nearest<Load<FROM>::kShort>(v[g * PER + j][k], scale, inv) << (4 * nibble(k));
                    bias += kBias << (4 * nibble(k));
                }
                out[g * PER + j] = fine ? word - bias : 0x88888888u;
            }
            if (c == 0) reinterpret_cast<uint16_t *>(scales + tile * Sc::kBytes)[r * Sc::kCount + g] = inside ? s16 : 0;
        }
        *reinterpret_cast<uint4 *>(q + tile * kTileBytes + lane * 16) = make_uint4(out[0], out[1], out[2], out[3]);
    }
}

template <class T, int GROUP>
__global__ __launch_bounds__(256) void dequantize_int4_kernel(const char *__restrict__ q, const char *__restrict__ scales, char *__restrict__ out,
                                                              int64_t n_tiles, int tiles, int cols) {
    using Sc = TileScales<GROUP>;
    __shared__ __attribute__((aligned(16))) char lds[4][4096];  // a tile of each wave's own: chunk k of row r in slot k ^ r
    const int lane = threadIdx.x & 63, r = lane & 15, c = lane >> 4;
    const Masks masks(Num<T>::kMask, Num<T>::kSixteen);
    for (int64_t tile = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); tile < n_tiles; tile += (int64_t)gridDim.x * 4) {
        const int64_t strip = tile / tiles;
        const int col0 = (int)(tile - strip * tiles) * kTileCols;
        const uint4 u = *reinterpret_cast<const uint4 *>(q + tile * kTileBytes + lane * 16);
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
        Sc sc;
        sc.load(scales + tile * Sc::kBytes, r);
        char *const mine = lds[threadIdx.x >> 6];
        wave_lds_order();
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float s = Num<T>::to_f32(sc.v[j / (GROUP / 32)]);
            // (24 is taken off before the product: the difference is exact, where 24 s may be beyond fp32 and q s is not)
            const i32x4 wide = Num<T>::wide(w[j], masks);
            float v[8];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                v[2 * k] = (Num<T>::to_f32((uint16_t)wide[k]) - 24.0f) * s;
                v[2 * k + 1] = (Num<T>::to_f32((uint16_t)((uint32_t)wide[k] >> 16)) - 24.0f) * s;
            }
            const uint2 lo = gmm::Pack<T>::four(v[0], v[1], v[2], v[3]), hi = gmm::Pack<T>::four(v[4], v[5], v[6], v[7]);
            *reinterpret_cast<uint4 *>(mine + r * 256 + ((4 * j + c) ^ r) * 16) = make_uint4(lo.x, lo.y, hi.x, hi.y);
        }
        wave_lds_order();
        // (out by 256 bytes of four rows a store)
        const int col = col0 + (lane & 15) * 8;
        char *p = out + ((strip * 16 + c) * cols + col) * 2;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint4 v = *reinterpret_cast<const uint4 *>(mine + (4 * i + c) * 256 + (r ^ (4 * i + c)) * 16);
            if (col < cols) *reinterpret_cast<uint4 *>(p + (int64_t)i * 8 * cols) = v;
        }
    }
}

int grid_for(int64_t tiles) { return (int)std::min<int64_t>((tiles + 3) / 4, 16384); }

template <class FROM, class T>
int quantize(const void *src, void *q, void *scales, int64_t n_tiles, int tiles, int cols, int group, hipStream_t s) {
    const char *from = static_cast<const char *>(src);
    char *to = static_cast<char *>(q), *sc = static_cast<char *>(scales);
    const dim3 grid(grid_for(n_tiles)), block(256);
    if (group == 32) hipLaunchKernelGGL((quantize_int4_kernel<FROM, T, 32>), grid, block, 0, s, from, to, sc, n_tiles, tiles, cols);
    else if (group == 64) hipLaunchKernelGGL((quantize_int4_kernel<FROM, T, 64>), grid, block, 0, s, from, to, sc, n_tiles, tiles, cols);
    else hipLaunchKernelGGL((quantize_int4_kernel<FROM, T, 128>), grid, block, 0, s, from, to, sc, n_tiles, tiles, cols);
    return check_launch("quantize_int4 launch");
}
template <class T>
int dequantize(const void *q, const void *scales, void *out, int64_t n_tiles, int tiles, int cols, int group, hipStream_t s) {
    const char *from = static_cast<const char *>(q), *sc = static_cast<const char *>(scales);
    char *to = static_cast<char *>(out);
    const dim3 grid(grid_for(n_tiles)), block(256);
    if (group == 32) hipLaunchKernelGGL((dequantize_int4_kernel<T, 32>), grid, block, 0, s, from, sc, to, n_tiles, tiles, cols);
    else if (group == 64) hipLaunchKernelGGL((dequantize_int4_kernel<T, 64>), grid, block, 0, s, from, sc, to, n_tiles, tiles, cols);
    else hipLaunchKernelGGL((dequantize_int4_kernel<T, 128>), grid, block, 0, s, from, sc, to, n_tiles, tiles, cols);
    return check_launch("dequantize_int4 launch");
}

int check_sizes(const char *what, int64_t rows, int cols, int group) {
    PMOE_REQUIRE(group == 32 || group == 64 || group == 128, "%s: group must be 32, 64 or 128, got %d", what, group);
    PMOE_REQUIRE(rows >= 0 && rows % 16 == 0 && cols > 0 && cols % group == 0 && cols <= gmm::kMaxSide,
                 "%s: rows (%lld) must be a multiple of 16, cols (%d) a positive multiple of group (%d) up to 2^28", what, (long long)rows, cols, group);
    return PMOE_OK;
}

}  // namespace

extern "C" int pmoe_quantize_int4(const void *src, int dtype, void *q, void *scales, int scale_dtype, int64_t rows, int cols, int group,
                                  void *stream) {
    PMOE_REQUIRE(dtype == PMOE_DTYPE_BF16 || dtype == PMOE_DTYPE_F16 || dtype == PMOE_DTYPE_F32, "quantize_int4: dtype must be bf16, fp16 or fp32");
    PMOE_REQUIRE(scale_dtype == PMOE_DTYPE_BF16 || scale_dtype == PMOE_DTYPE_F16, "quantize_int4: scale_dtype must be bf16 or fp16");
    if (int rc = check_sizes("quantize_int4", rows, cols, group)) return rc;
    if (rows == 0) return PMOE_OK;
    PMOE_REQUIRE(src && q && scales, "quantize_int4: null pointer");
    PMOE_REQUIRE_ALIGNED("quantize_int4", src, q, scales);
    const int tiles = tiles_of(cols);
    const int64_t n_tiles = rows / 16 * tiles;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const bool to_bf16 = scale_dtype == PMOE_DTYPE_BF16;
    if (dtype == PMOE_DTYPE_BF16) return to_bf16 ? quantize<Bf16, Bf16>(src, q, scales, n_tiles, tiles, cols, group, s) : quantize<Bf16, F16>(src, q, scales, n_tiles, tiles, cols, group, s);
    if (dtype == PMOE_DTYPE_F16) return to_bf16 ? quantize<F16, Bf16>(src, q, scales, n_tiles, tiles, cols, group, s) : quantize<F16, F16>(src, q, scales, n_tiles, tiles, cols, group, s);
    return to_bf16 ? quantize<F32, Bf16>(src, q, scales, n_tiles, tiles, cols, group, s) : quantize<F32, F16>(src, q, scales, n_tiles, tiles, cols, group, s);
}

extern "C" int pmoe_dequantize_int4(const void *q, const void *scales, void *out, int dtype, int64_t rows, int cols, int group, void *stream) {
    PMOE_REQUIRE(dtype == PMOE_DTYPE_BF16 || dtype == PMOE_DTYPE_F16, "dequantize_int4: dtype must be bf16 or fp16");
    if (int rc = check_sizes("dequantize_int4", rows, cols, group)) return rc;
    if (rows == 0) return PMOE_OK;
    PMOE_REQUIRE(q && scales && out, "dequantize_int4: null pointer");
    PMOE_REQUIRE_ALIGNED("dequantize_int4", q, scales, out);
    const int tiles = tiles_of(cols);
    const int64_t n_tiles = rows / 16 * tiles;
    hipStream_t s = static_cast<hipStream_t>(stream);
    return dtype == PMOE_DTYPE_BF16 ? dequantize<Bf16>(q, scales, out, n_tiles, tiles, cols, group, s)
                                    : dequantize<F16>(q, scales, out, n_tiles, tiles, cols, group, s);
}
