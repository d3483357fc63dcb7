// Quantiser per row to 8-bit integers: scale = max(amax c, 2^-126) with c = 1 / 127 in fp32, q = the integer nearest to x / scale, ties to even.
// (The product and not the quotient amax / 127, as torch divides by a number on the GPU: they differ by a unit in the last place
// in 5 % of rows.)
//
// The result is that of exact arithmetic on the fp32 scale: a first guess x (1 / scale) is off by at most one, and the
// remainder x - q scale, which one fma gives without rounding (it has at most 24 bits at the weight of scale's last bit),
// tells which way.  A row with an infinity or a NaN gets the scale NaN and zeros, so that what is computed from it is NaN.
//
// Bound by memory: a row is read once and held in registers between its maximum and its quantisation (131071 x 2048 in bf16:
// 153 - 159 us, 5.1 - 5.3 TB/s of reads and writes; a large copy 4.8).  64 rows of 7168: 6 us, of which a launch with a dependent
// read is 2; the rest is a workgroup's loads, its two barriers and 32 values a lane.
#include <algorithm>

#include "grouped_host.h"
#include "moe_tile.h"

namespace {

using namespace pmoe;

struct FromBf16 {
    static constexpr int kBytes = 2;
    static __device__ __forceinline__ void eight(const uint4 *p, float (&v)[8]) {
        const uint4 r = p[0];
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) v[2 * j] = bf16_bits_to_f32(w[j] & 0xffffu), v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
    }
};
struct FromF16 {
    static constexpr int kBytes = 2;
    static __device__ __forceinline__ void eight(const uint4 *p, float (&v)[8]) {
        typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
        const f16x8 r = __builtin_bit_cast(f16x8, p[0]);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = (float)r[j];
    }
};
struct FromF32 {
    static constexpr int kBytes = 4;
    static __device__ __forceinline__ void eight(const uint4 *p, float (&v)[8]) {
        const uint4 a = p[0], b = p[1];
        const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = __uint_as_float(w[j]);
    }
};

// Largest magnitude as its bits: these order like the numbers, with infinity and the NaNs above all of them.
__device__ __forceinline__ uint32_t peak8(const float (&v)[8], uint32_t m) {
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(v[j]) & 0x7fffffffu);
    return m;
}

__device__ __forceinline__ uint32_t quantize4(float a, float b, float c, float d, float scale, float inv) {
    const float x[4] = {a, b, c, d};
    uint32_t out = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        float q = rintf(x[j] * inv);
        const float r = fmaf(-q, scale, x[j]), twice = 2.0f * fabsf(r);  // (half of the smallest scales would be rounded)
        const bool odd = ((int)q & 1) != 0;
        if (twice > scale || (twice == scale && odd)) q += copysignf(1.0f, r);
        out |= ((uint32_t)(int)q & 0xffu) << (8 * j);
    }
    return out;
}

// WAVES waves per row (1 or 4), HELD groups of eight per lane in registers; what a row has beyond that is read again.
template <class FROM, int WAVES, int HELD>
__global__ __launch_bounds__(256) void quantize_int8_kernel(const char *__restrict__ src, int64_t pitch, uint2 *__restrict__ q,
                                                            float *__restrict__ scales, int64_t rows, int cols) {
    constexpr int LANES = 64 * WAVES, ROWS = 4 / WAVES;
    const int lane = threadIdx.x % LANES, n8 = cols / 8;
    __shared__ uint32_t peaks[4];
    for (int64_t r0 = (int64_t)blockIdx.x * ROWS; r0 < rows; r0 += (int64_t)gridDim.x * ROWS) {
        const int64_t row = r0 + threadIdx.x / LANES;
        const bool live = row < rows;
        const char *p = src + (live ? row : rows - 1) * pitch;
        float v[HELD][8];
        uint32_t peak = 0;
#pragma unroll
        for (int i = 0; i < HELD; ++i) {
            const int at = lane + i * LANES;
            if (at < n8) {
                FROM::eight(reinterpret_cast<const uint4 *>(p + (int64_t)at * 8 * FROM::kBytes), v[i]);
                peak = peak8(v[i], peak);
            }
        }
        for (int at = lane + HELD * LANES; at < n8; at += LANES) {
            float more[8];
            FROM::eight(reinterpret_cast<const uint4 *>(p + (int64_t)at * 8 * FROM::kBytes), more);
            peak = peak8(more, peak);
        }
#pragma unroll
        for (int d = 32; d > 0; d /= 2) peak = max(peak, (uint32_t)__shfl_xor((int)peak, d, 64));
        if constexpr (WAVES > 1) {
            if ((threadIdx.x & 63) == 0) peaks[threadIdx.x >> 6] = peak;
            __syncthreads();
            peak = max(max(peaks[0], peaks[1]), max(peaks[2], peaks[3]));
            __syncthreads();
        }
        const bool finite = peak < 0x7f800000u;
        const float scale = finite ? fmaxf(__uint_as_float(peak) * (1.0f / 127.0f), 0x1p-126f) : __uint_as_float(0x7fc00000u);
        const float inv = 1.0f / scale;
        if (!live) continue;
        uint2 *out = q + row * n8;
        auto put = [&](int at, const float (&x)[8]) {
            uint2 o = make_uint2(0, 0);
            if (finite) o = make_uint2(quantize4(x[0], x[1], x[2], x[3], scale, inv), quantize4(x[4], x[5], x[6], x[7], scale, inv));
            out[at] = o;
        };
#pragma unroll
        for (int i = 0; i < HELD; ++i)
            if (lane + i * LANES < n8) put(lane + i * LANES, v[i]);
        for (int at = lane + HELD * LANES; at < n8; at += LANES) {
            float more[8];
            FROM::eight(reinterpret_cast<const uint4 *>(p + (int64_t)at * 8 * FROM::kBytes), more);
            put(at, more);
        }
        if (lane == 0) scales[row] = scale;
    }
}

template <class FROM>
void launch(const void *src, int64_t pitch, void *q, float *scales, int64_t rows, int cols, hipStream_t stream) {
    const char *s = static_cast<const char *>(src);
    uint2 *o = static_cast<uint2 *>(q);
    // A wave per row where rows are many and fit its registers, a workgroup per row otherwise.
    if (rows >= 4096 && cols <= 4096) {
        const int grid = (int)std::min<int64_t>((rows + 3) / 4, 16384);
        if (cols <= 2048) hipLaunchKernelGGL((quantize_int8_kernel<FROM, 1, 4>), dim3(grid), dim3(256), 0, stream, s, pitch, o, scales, rows, cols);
        else hipLaunchKernelGGL((quantize_int8_kernel<FROM, 1, 8>), dim3(grid), dim3(256), 0, stream, s, pitch, o, scales, rows, cols);
    } else {
        const int grid = (int)std::min<int64_t>(rows, 16384);
        hipLaunchKernelGGL((quantize_int8_kernel<FROM, 4, 4>), dim3(grid), dim3(256), 0, stream, s, pitch, o, scales, rows, cols);
    }
}

}  // namespace

extern "C" int pmoe_quantize_int8(const void *src, int dtype, void *q, float *scales, int64_t rows, int cols, int64_t stride, void *stream) {
    PMOE_REQUIRE(dtype == PMOE_DTYPE_BF16 || dtype == PMOE_DTYPE_F16 || dtype == PMOE_DTYPE_F32, "quantize_int8: dtype must be bf16, fp16 or fp32");
    PMOE_REQUIRE(rows >= 0 && cols > 0 && cols % 8 == 0, "quantize_int8: cols (%d) must be a positive multiple of 8", cols);
    PMOE_REQUIRE(stride >= cols && stride % 8 == 0, "quantize_int8: rows %lld elements apart (supported: multiples of 8 from %d on)", (long long)stride, cols);
    if (rows == 0) return PMOE_OK;
    PMOE_REQUIRE(src && q && scales, "quantize_int8: null pointer");
    PMOE_REQUIRE_ALIGNED("quantize_int8", src, q);
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (dtype == PMOE_DTYPE_BF16) launch<FromBf16>(src, stride * 2, q, scales, rows, cols, s);
    else if (dtype == PMOE_DTYPE_F16) launch<FromF16>(src, stride * 2, q, scales, rows, cols, s);
    else launch<FromF32>(src, stride * 4, q, scales, rows, cols, s);
    return check_launch("quantize_int8 launch");
}
