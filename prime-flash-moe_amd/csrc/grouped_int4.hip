// Products with weights of 4 bits (int4_tile.h): rows by their group's matrix, or by a single one.
//
// Bound by the stream of the touched groups' weights.  A workgroup takes one group and 16 U of its weight rows; its waves share
// the contraction, each in one run of tiles, and add their sums in LDS in the order of the waves.  Rows of x come from the L2 straight
// into registers, 16 (or 32) at a time; a group with more rows streams its weights again for every 32.
#include <algorithm>

#include "grouped_host.h"
#include "int4_tile.h"

namespace {

using namespace pmoe;
using namespace pmoe::int4;
using gmm::RowsArgs;
using gmm::few::Span;

struct Int4Args {
    RowsArgs rows;      // x, w, out, offsets, n_groups, rows, cols, depth; w_group: bytes of a group's weights
    const char *scale;
    int64_t scale_group;
};

template <int U, int R, int WAVES>
struct Shared {
    f32x4 sum[WAVES][U * R][64];
};

template <class T, int GROUP, int U, int R, int WAVES>
__device__ __forceinline__ void pass(const Int4Args &a, int group, int row0, int live, int strip0, int strips, Shared<U, 2, WAVES> &sh) {
    const int tid = threadIdx.x, lane = tid & 63, wave = gmm::uniform(tid >> 6), r = lane & 15, c = lane >> 4;
    const int tiles = tiles_of(a.rows.depth), t0 = wave * tiles / WAVES, t1 = (wave + 1) * tiles / WAVES;
    const char *w[U], *s[U], *x[R];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int64_t strip = min(strip0 + u, strips - 1);
        w[u] = a.rows.w + group * a.rows.w_group + strip * tiles * kTileBytes;
        s[u] = a.scale + group * a.scale_group + strip * tiles * TileScales<GROUP>::kBytes;
    }
#pragma unroll
    for (int t = 0; t < R; ++t) x[t] = a.rows.x + (row0 + min(16 * t + r, live - 1)) * a.rows.x_pitch;
    f32x4 acc[U][R] = {};
    dots<T, GROUP, U, R, 2>(acc, w, s, x, t0, t1, a.rows.depth);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int t = 0; t < R; ++t) sh.sum[wave][u * R + t][lane] = acc[u][t];
    __syncthreads();
    // element (row m, column n) of the U x R fragments: lane n + 16 (m / 4), component m % 4
    for (int i = tid; i < U * R * 256; i += 64 * WAVES) {
        const int n = i & 15, m = i / 16 % 16, f = i / 256, u = f / R, row = f % R * 16 + m, col = (strip0 + u) * 16 + n;
        if (row < live && col < a.rows.cols) {
            float v = 0.f;
#pragma unroll
            for (int k = 0; k < WAVES; ++k) v += sh.sum[k][f][n + m / 4 * 16][m & 3];
            *reinterpret_cast<uint16_t *>(a.rows.out + (row0 + row) * a.rows.out_pitch + (int64_t)col * 2) = Num<T>::from_f32(v);
        }
    }
    __syncthreads();  // the sums may be overwritten
}

template <class T, int GROUP, int U, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void grouped_mm_int4_kernel(Int4Args a, int strips, int jobs) {
    __shared__ Shared<U, 2, WAVES> sh;
    const int slot = (int)blockIdx.x / jobs, strip0 = ((int)blockIdx.x - slot * jobs) * U;
    const Span s = gmm::few::find_span<0>(a.rows, slot);
    if (s.zero) {
        const int chunks = min(16 * U, a.rows.cols - 16 * strip0) / 8;
        for (int64_t i = threadIdx.x; i < (int64_t)(s.end - s.begin) * chunks; i += 64 * WAVES)
            *reinterpret_cast<uint4 *>(a.rows.out + (s.begin + i / chunks) * a.rows.out_pitch + strip0 * 32 + i % chunks * 16) = make_uint4(0, 0, 0, 0);
        return;
    }
    for (int row0 = s.begin; row0 < s.end; row0 += 32) {
        const int live = min(s.end - row0, 32);
        if (live <= 16) pass<T, GROUP, U, 1, WAVES>(a, s.group, row0, live, strip0, strips, sh);
        else pass<T, GROUP, U, 2, WAVES>(a, s.group, row0, live, strip0, strips, sh);
    }
}

template <class T, int GROUP>
int launch(const Int4Args &a, hipStream_t stream) {
    constexpr int U = 1, WAVES = 8;
    const int strips = a.rows.cols / 16, jobs = (strips + U - 1) / U;
    const int64_t slots = std::min(a.rows.rows, a.rows.n_groups) + (a.rows.offsets != nullptr ? 1 : 0);
    PMOE_REQUIRE(jobs * slots * (64 * WAVES) <= UINT32_MAX, "grouped_mm_int4: too many tiles");
    hipLaunchKernelGGL((grouped_mm_int4_kernel<T, GROUP, U, WAVES>), dim3((uint32_t)(jobs * slots)), dim3(64 * WAVES), 0, stream, a, strips, jobs);
    return check_launch("grouped_mm_int4 launch");
}
template <class T>
int launch(const Int4Args &a, int group, hipStream_t stream) {
    return group == 32 ? launch<T, 32>(a, stream) : group == 64 ? launch<T, 64>(a, stream) : launch<T, 128>(a, stream);
}

}  // namespace

extern "C" int pmoe_grouped_mm_int4(const void *x, const void *w, const void *w_scale, void *out, const int32_t *offsets, int n_groups,
                                    int64_t M, int N, int K, int group, int64_t x_stride, int dtype, void *stream) {
    PMOE_REQUIRE(dtype == PMOE_DTYPE_BF16 || dtype == PMOE_DTYPE_F16, "grouped_mm_int4: dtype must be bf16 or fp16");
    PMOE_REQUIRE(n_groups > 0 && n_groups <= gmm::kMaxGroups, "grouped_mm_int4 supports 1..%d groups, got %d", gmm::kMaxGroups, n_groups);
    PMOE_REQUIRE(offsets || n_groups == 1, "grouped_mm_int4: without offsets there is one matrix, got %d", n_groups);
    PMOE_REQUIRE(group == 32 || group == 64 || group == 128, "grouped_mm_int4: group must be 32, 64 or 128, got %d", group);
    PMOE_REQUIRE(M >= 0 && M <= gmm::kMaxRows && N > 0 && N % 16 == 0 && N <= gmm::kMaxSide, "grouped_mm_int4: N (%d) must be a positive multiple of 16 up to 2^28, M (%lld) below 2^31 - 512", N, (long long)M);
    PMOE_REQUIRE(K > 0 && K % group == 0 && K <= gmm::kMaxSide, "grouped_mm_int4: K (%d) must be a positive multiple of group (%d) up to 2^28", K, group);
    PMOE_REQUIRE_STRIDE("grouped_mm_int4: x", x_stride, K, 8, gmm::kMaxStride);
    if (M == 0) return PMOE_OK;
    PMOE_REQUIRE(x && w && w_scale && out, "grouped_mm_int4: null pointer");
    PMOE_REQUIRE_ALIGNED("grouped_mm_int4", x, w, w_scale, out);
    Int4Args a = {};
    const int64_t tiles = (int64_t)(N / 16) * tiles_of(K);
    a.rows.x = static_cast<const char *>(x);
    a.rows.w = static_cast<const char *>(w);
    a.rows.out = static_cast<char *>(out);
    a.rows.x_pitch = x_stride * 2;
    a.rows.w_group = tiles * kTileBytes;
    a.rows.out_pitch = (int64_t)N * 2;
    a.rows.offsets = offsets;
    a.rows.n_groups = n_groups;
    a.rows.rows = (int)M;
    a.rows.cols = N;
    a.rows.depth = K;
    a.scale = static_cast<const char *>(w_scale);
    a.scale_group = tiles * (kTileRows * (kTileCols / group) * 2);
    hipStream_t s = static_cast<hipStream_t>(stream);
    return dtype == PMOE_DTYPE_BF16 ? launch<Bf16>(a, group, s) : launch<F16>(a, group, s);
}
