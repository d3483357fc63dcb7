// Ragged expert products in bf16 and fp16: rows by their expert's weights, and the gradient of the weights.
#include <algorithm>

#include "grouped_few.h"
#include "grouped_host.h"
#include "grouped_kernel.h"

namespace {

using namespace pmoe;
using namespace pmoe::gmm;

template <class T, bool QX>
void launch_rows(const RowsArgs &a, int grid, hipStream_t stream) {
    if constexpr (!QX)
        if (few::launch<T, T>(a, stream)) return;
    hipLaunchKernelGGL((grouped_mm_kernel<T, QX, T>), dim3(grid), dim3(kThreads), 0, stream, a);
}

}  // namespace

namespace pmoe {
namespace gmm {

int64_t most_tiles(int64_t rows, int cols, int n_groups) {
    const int64_t t = (rows / 256 + n_groups + 2) * ((cols + kCols - 1) / kCols);
    return t < (1ll << 31) - 8192 ? t : -1;
}
bool fills(int64_t rows, int cols) { return rows / 128 * ((cols + kCols - 1) / kCols) > resident_grid(); }
int grid_of(int64_t tiles) { return (int)std::min<int64_t>(resident_grid(), (tiles + 7) / 8 * 8); }

}  // namespace gmm
}  // namespace pmoe

// The ends of the groups of a sorted schedule: entry i - 1 of `ids` and entry i differ exactly where the groups in between
// end.  Every end is written by one thread.  One pass without a search: 2 us for 1020 rows, 5 us for 65541.
namespace {
__global__ __launch_bounds__(256) void expert_offsets_kernel(const int32_t *__restrict__ ids, const int32_t *__restrict__ total,
                                                             int32_t *__restrict__ offsets, int n, int n_groups) {
    const int count = min(max(total[0], 0), n);
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i <= count; i += (int64_t)gridDim.x * 256) {
        const int from = i == 0 ? 0 : min(max(ids[i - 1], 0), n_groups), to = i == count ? n_groups : min(max(ids[i], 0), n_groups);
        for (int g = from; g < to; ++g) offsets[g] = (int)i;
    }
}
}  // namespace

extern "C" int pmoe_expert_offsets(const int32_t *expert_ids, const int32_t *num_tokens_post_padded, int32_t *offsets, int n, int n_groups,
                                   void *stream) {
    PMOE_REQUIRE(n >= 0 && n_groups > 0, "expert_offsets: n (%d) must not be negative, num_experts (%d) must be positive", n, n_groups);
    PMOE_REQUIRE((n == 0 || expert_ids) && num_tokens_post_padded && offsets, "expert_offsets: null pointer");
    const int grid = std::min(n / 256 + 1, 1024);
    hipLaunchKernelGGL(expert_offsets_kernel, dim3(grid), dim3(256), 0, static_cast<hipStream_t>(stream), expert_ids,
                       num_tokens_post_padded, offsets, n, n_groups);
    return check_launch("expert_offsets launch");
}

extern "C" int pmoe_grouped_mm(const void *x, const void *w, void *out, const int32_t *offsets, int n_groups, int64_t M, int N,
                               int K, int64_t x_stride, int64_t w_stride, int64_t w_group_stride, int w_across, int dtype,
                               void *stream) {
    PMOE_REQUIRE(dtype == PMOE_DTYPE_BF16 || dtype == PMOE_DTYPE_F16, "grouped_mm: dtype must be bf16 or fp16");
    PMOE_REQUIRE(n_groups > 0 && n_groups <= kMaxGroups, "grouped_mm supports 1..%d groups, got %d", kMaxGroups, n_groups);
    PMOE_REQUIRE(M >= 0 && M <= kMaxRows && N > 0 && K > 0 && N % 8 == 0 && K % 8 == 0, "grouped_mm: N (%d) and K (%d) must be positive multiples of 8, M (%lld) below 2^31 - 512", N, K, (long long)M);
    PMOE_REQUIRE(K <= kMaxSide && N <= kMaxSide, "grouped_mm: N and K must be at most 2^28");
    PMOE_REQUIRE_STRIDE("grouped_mm: x", x_stride, K, 8, kMaxStride);
    PMOE_REQUIRE_STRIDE("grouped_mm: w", w_stride, w_across ? N : K, 8, kMaxStride);
    PMOE_REQUIRE(w_group_stride % 8 == 0 && w_group_stride >= 0, "grouped_mm: the stride of w between groups must be a multiple of 8");
    if (M == 0) return PMOE_OK;
    PMOE_REQUIRE(x && w && out && offsets, "grouped_mm: null pointer");
    PMOE_REQUIRE_ALIGNED("grouped_mm", x, w, out);
    const int64_t tiles = most_tiles(M, N, n_groups);
    PMOE_REQUIRE(tiles > 0, "grouped_mm: too many tiles");
    RowsArgs a = {};
    a.x = static_cast<const char *>(x);
    a.w = static_cast<const char *>(w);
    a.out = static_cast<char *>(out);
    a.x_pitch = x_stride * 2;
    a.w_pitch = w_stride * 2;
    a.w_group = w_group_stride * 2;
    a.out_pitch = (int64_t)N * 2;
    a.offsets = offsets;
    a.n_groups = n_groups;
    a.rows = (int)M;
    a.cols = N;
    a.depth = K;
    a.once = stores_once(M * N * 2);
    a.fills = fills(M, N);
    const int grid = grid_of(a.fills ? tiles : 4 * tiles);  // (a tile of 256 rows may be four of 64)
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (dtype == PMOE_DTYPE_BF16) w_across ? launch_rows<Bf16, true>(a, grid, s) : launch_rows<Bf16, false>(a, grid, s);
    else w_across ? launch_rows<F16, true>(a, grid, s) : launch_rows<F16, false>(a, grid, s);
    return check_launch("grouped_mm launch");
}

extern "C" int pmoe_grouped_mm_wgrad(const void *dy, const void *x, void *dw, const int32_t *offsets, int n_groups, int64_t M, int N,
                                     int K, int64_t dy_stride, int64_t x_stride, int dtype, void *stream) {
    PMOE_REQUIRE(dtype == PMOE_DTYPE_BF16 || dtype == PMOE_DTYPE_F16, "grouped_mm_wgrad: dtype must be bf16 or fp16");
    PMOE_REQUIRE(n_groups > 0 && n_groups <= kMaxGroups, "grouped_mm_wgrad supports 1..%d groups, got %d", kMaxGroups, n_groups);
    PMOE_REQUIRE(M >= 0 && M <= kMaxRows && N > 0 && K > 0 && N % 8 == 0 && K % 8 == 0, "grouped_mm_wgrad: N (%d) and K (%d) must be positive multiples of 8, M (%lld) below 2^31 - 512", N, K, (long long)M);
    PMOE_REQUIRE(K <= kMaxSide && N <= kMaxSide, "grouped_mm_wgrad: N and K must be at most 2^28");
    PMOE_REQUIRE_STRIDE("grouped_mm_wgrad: dy", dy_stride, N, 8, kMaxStride);
    PMOE_REQUIRE_STRIDE("grouped_mm_wgrad: x", x_stride, K, 8, kMaxStride);
    PMOE_REQUIRE(dw && offsets && (M == 0 || (dy && x)), "grouped_mm_wgrad: null pointer");
    PMOE_REQUIRE_ALIGNED("grouped_mm_wgrad", dy, x, dw);
    const int64_t tiles = (int64_t)n_groups * ((N + 127) / 128) * ((K + kCols - 1) / kCols);
    PMOE_REQUIRE(tiles < (1ll << 31) - 8192, "grouped_mm_wgrad: too many tiles");
    WgradArgs a = {};
    a.dy = static_cast<const char *>(dy);
    a.x = static_cast<const char *>(x);
    a.dw = static_cast<char *>(dw);
    a.dy_pitch = dy_stride * 2;
    a.x_pitch = x_stride * 2;
    a.offsets = offsets;
    a.n_groups = n_groups;
    a.rows = (int)M;
    a.out_rows = N;
    a.cols = K;
    a.once = stores_once((int64_t)n_groups * N * K * 2);
    hipStream_t s = static_cast<hipStream_t>(stream);
    // (tiles of 128 rows where those of 256 would leave CUs idle)
    const int64_t tall = (int64_t)n_groups * ((N + 255) / 256) * ((K + kCols - 1) / kCols);
    const bool small = tall < resident_grid();
    const int grid = grid_of(small ? tiles : tall);
    if (dtype == PMOE_DTYPE_BF16) {
        if (small) hipLaunchKernelGGL((grouped_mm_wgrad_kernel<Bf16, 2>), dim3(grid), dim3(kThreads), 0, s, a);
        else hipLaunchKernelGGL((grouped_mm_wgrad_kernel<Bf16, 4>), dim3(grid), dim3(kThreads), 0, s, a);
    } else {
        if (small) hipLaunchKernelGGL((grouped_mm_wgrad_kernel<F16, 2>), dim3(grid), dim3(kThreads), 0, s, a);
        else hipLaunchKernelGGL((grouped_mm_wgrad_kernel<F16, 4>), dim3(grid), dim3(kThreads), 0, s, a);
    }
    return check_launch("grouped_mm_wgrad launch");
}
