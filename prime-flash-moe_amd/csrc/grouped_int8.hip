// Ragged (or dense) products of 8-bit integers with a scale per row of each operand, on the tiles of grouped_tile.h.
// Sums are exact in 32 bits (the depth is limited to what cannot overflow); scales are applied in fp32 on the way out.
#include <algorithm>

#include "grouped_few.h"
#include "grouped_host.h"
#include "grouped_kernel.h"

namespace {

using namespace pmoe;
using namespace pmoe::gmm;

template <class OUT>
void launch(const RowsArgs &a, int grid, hipStream_t stream) {
    if (few::launch<I8, OUT>(a, stream)) return;
    // A dense product whose last round of tiles would be a few rows high: these go to the kernels for few rows, which spread their
    // contraction over the whole chip (4097 rows x 4096 x 7168: 147 -> 104 us; the 4097th alone took a workgroup 40 us) unless
    // they are wide (73 rows of 28672 columns: 70 us there, 50 in tiles).
    const int col_tiles = (a.cols + kCols - 1) / kCols, round = resident_grid() / col_tiles * 256;
    const int rest = a.offsets == nullptr && round > 0 && a.rows > round ? a.rows % round : 0;
    if (rest > 0 && (int64_t)(rest / few::kBlock + 1) * ((a.cols + 31) / 32) <= 4 * resident_grid()) {
        RowsArgs last = a;
        last.rows = rest;
        last.x += (a.rows - rest) * a.x_pitch;
        last.x_scale += a.rows - rest;
        last.out += (a.rows - rest) * a.out_pitch;
        if (few::launch<I8, OUT>(last, stream)) {
            RowsArgs first = a;
            first.rows = a.rows - rest;
            hipLaunchKernelGGL((grouped_mm_kernel<I8, false, OUT>), dim3(grid), dim3(kThreads), 0, stream, first);
            return;
        }
    }
    hipLaunchKernelGGL((grouped_mm_kernel<I8, false, OUT>), dim3(grid), dim3(kThreads), 0, stream, a);
}

}  // namespace

extern "C" int pmoe_grouped_mm_int8(const void *x, const void *w, const float *x_scale, const float *w_scale, void *out,
                                    const int32_t *offsets, int n_groups, int64_t M, int N, int K, int64_t x_stride,
                                    int64_t w_stride, int64_t w_group_stride, int out_dtype, void *stream) {
    PMOE_REQUIRE(out_dtype == PMOE_DTYPE_BF16 || out_dtype == PMOE_DTYPE_F16 || out_dtype == PMOE_DTYPE_F32, "grouped_mm_int8: out_dtype must be bf16, fp16 or fp32");
    PMOE_REQUIRE(n_groups > 0 && n_groups <= kMaxGroups, "grouped_mm_int8 supports 1..%d groups, got %d", kMaxGroups, n_groups);
    PMOE_REQUIRE(offsets || n_groups == 1, "grouped_mm_int8: without offsets there is one group, got %d", n_groups);
    PMOE_REQUIRE(M >= 0 && M <= kMaxRows && N > 0 && N % 8 == 0 && N <= kMaxSide, "grouped_mm_int8: N (%d) must be a positive multiple of 8, M (%lld) below 2^31 - 512", N, (long long)M);
    // (131072 products of -128 and -128 are 2^31)
    PMOE_REQUIRE(K > 0 && K % 16 == 0 && K < 131072, "grouped_mm_int8: K (%d) must be a positive multiple of 16 below 131072", K);
    PMOE_REQUIRE_STRIDE("grouped_mm_int8: x", x_stride, K, 16, 2 * kMaxStride);
    PMOE_REQUIRE_STRIDE("grouped_mm_int8: w", w_stride, K, 16, 2 * kMaxStride);
    PMOE_REQUIRE(w_group_stride % 16 == 0 && w_group_stride >= 0, "grouped_mm_int8: the stride of w between groups must be a multiple of 16");
    if (M == 0) return PMOE_OK;
    PMOE_REQUIRE(x && w && x_scale && w_scale && out, "grouped_mm_int8: null pointer");
    PMOE_REQUIRE_ALIGNED("grouped_mm_int8", x, w, out);
    const int64_t tiles = most_tiles(M, N, n_groups);
    PMOE_REQUIRE(tiles > 0, "grouped_mm_int8: too many tiles");
    RowsArgs a = {};
    a.x = static_cast<const char *>(x);
    a.w = static_cast<const char *>(w);
    a.out = static_cast<char *>(out);
    a.x_pitch = x_stride;
    a.w_pitch = w_stride;
    a.w_group = w_group_stride;
    a.out_pitch = (int64_t)N * (out_dtype == PMOE_DTYPE_F32 ? 4 : 2);
    a.offsets = offsets;
    a.n_groups = n_groups;
    a.rows = (int)M;
    a.cols = N;
    a.depth = K;
    a.once = stores_once(M * a.out_pitch);
    a.x_scale = x_scale;
    a.w_scale = w_scale;
    a.fills = fills(M, N);
    const int grid = grid_of(a.fills ? tiles : 4 * tiles);  // (a tile of 256 rows may be four of 64)
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (out_dtype == PMOE_DTYPE_BF16) launch<Bf16>(a, grid, s);
    else if (out_dtype == PMOE_DTYPE_F16) launch<F16>(a, grid, s);
    else launch<F32>(a, grid, s);
    return check_launch("grouped_mm_int8 launch");
}
