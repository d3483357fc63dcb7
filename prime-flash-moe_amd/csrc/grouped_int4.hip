// Products with weights of 4 bits (int4_tile.h): rows by their group's matrix, or by a single one.
//
// Bound by the stream of the touched groups' weights, 64 tokens on half of 256 experts of 4096 x 7168 by 387 us, 5.2 TB/s, with the vector
// units busy for half of the time (the way to 16 bits).  A workgroup takes one
// group and 16 U of its weight rows at a time; its waves share the contraction, each in one run of tiles, and add their sums in LDS
// in the order of the waves.  Rows of x come 16 (or 32) at a time; a group with more rows streams its weights again for them.
#include <algorithm>

#include "grouped_host.h"
#include "int4_tile.h"

namespace {

using namespace pmoe;
using namespace pmoe::int4;
using gmm::RowsArgs;

struct Int4Args {
    RowsArgs rows;      // x, w, out, offsets, n_groups, rows, cols, depth; w_group: bytes of a group's weights
    const char *scale;
    int64_t scale_group;
};

template <int U, int R, int S, int WAVES>
union Shared {
    f32x4 sum[WAVES][U * R][64];
    char rows[WAVES][Rows<16 * R, S>::kBytes];
};

template <class T, int GROUP, int U, int R, int S, int WAVES>
__device__ __forceinline__ void pass(const Int4Args &a, int group, int row0, int live, int strip0, int strips, Shared<U, R, S, WAVES> &sh) {
    const int tid = threadIdx.x, lane = tid & 63, wave = gmm::uniform(tid >> 6);
    const int tiles = tiles_of(a.rows.depth), t0 = wave * tiles / WAVES, t1 = (wave + 1) * tiles / WAVES;
    const char *w[U], *s[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int64_t strip = min(strip0 + u, strips - 1);
        w[u] = a.rows.w + group * a.rows.w_group + strip * tiles * kTileBytes;
        s[u] = a.scale + group * a.scale_group + strip * tiles * TileScales<GROUP>::kBytes;
    }
    const char *const x = a.rows.x + row0 * a.rows.x_pitch;
    f32x4 acc[U][R];
    dots<T, T, GROUP, U, R, S>(acc, w, s, x, [&](int q) { return (uint32_t)q * (uint32_t)a.rows.x_pitch; }, live, t0, t1, a.rows.depth, sh.rows[wave]);
    __syncthreads();  // the sums lie where the rows were
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

// The groups that have rows, in their order: what a group's rows are follows Walk (a group begins at the furthest end in front of it).
struct Spans {
    int n, live_rows;
    int group[gmm::kMaxGroups], begin[gmm::kMaxGroups + 1];
    int scan[2][8];
};
template <int WAVES>
__device__ __forceinline__ void find_spans(const RowsArgs &a, Spans &s) {
    constexpr int PER = gmm::kMaxGroups / (64 * WAVES);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    if (a.offsets == nullptr) {
        if (tid == 0) s.n = 1, s.live_rows = a.rows, s.group[0] = 0, s.begin[0] = 0, s.begin[1] = a.rows;
        __syncthreads();
        return;
    }
    int end[PER], far = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int g = tid * PER + i;
        far = max(far, g < a.n_groups ? gmm::group_end(a, g) : 0);
        end[i] = far;
    }
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const int v = __shfl_up(far, d, 64);
        if (lane >= d) far = max(far, v);
    }
    if (lane == 63) s.scan[0][wave] = far;
    __syncthreads();
    int before = __shfl_up(far, 1, 64);
    if (lane == 0) before = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w)
        if (w < wave) before = max(before, s.scan[0][w]);
    int count = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        end[i] = max(end[i], before);
        count += end[i] > (i == 0 ? before : end[i - 1]);
    }
    int incl = count;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const int v = __shfl_up(incl, d, 64);
        if (lane >= d) incl += v;
    }
    if (lane == 63) s.scan[1][wave] = incl;
    __syncthreads();
    int at = incl - count;
#pragma unroll
    for (int w = 0; w < WAVES; ++w)
        if (w < wave) at += s.scan[1][w];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int begin = i == 0 ? before : end[i - 1];
        if (end[i] > begin) s.group[at] = tid * PER + i, s.begin[at] = begin, s.begin[at + 1] = end[i], ++at;
    }
    if (tid == 64 * WAVES - 1) {
        s.n = at;
        s.live_rows = end[PER - 1];
    }
    __syncthreads();
}

// Resident: a workgroup takes every grid-th job, a group and U strips of its weights, then its part of the rows behind the last group.
// (A workgroup per job spends more on starting, finding its group and filling its pipeline than on its weights.)
template <class T, int GROUP, int U, int R, int S, int WAVES, int PER_SIMD>
__global__ __launch_bounds__(64 * WAVES, PER_SIMD) void grouped_mm_int4_kernel(Int4Args a, int strips, int jobs) {
    __shared__ __attribute__((aligned(1024))) Shared<U, R, S, WAVES> sh;
    __shared__ Spans sp;
    find_spans<WAVES>(a.rows, sp);
    const int64_t total = (int64_t)sp.n * jobs;
    for (int64_t job = blockIdx.x; job < total; job += gridDim.x) {
        const int slot = (int)(job / jobs), strip0 = (int)(job - (int64_t)slot * jobs) * U;
        const int group = gmm::uniform(sp.group[slot]), begin = gmm::uniform(sp.begin[slot]), end = gmm::uniform(sp.begin[slot + 1]);
        for (int row0 = begin; row0 < end; row0 += 16 * R) pass<T, GROUP, U, R, S, WAVES>(a, group, row0, min(end - row0, 16 * R), strip0, strips, sh);
    }
    const int64_t from = sp.live_rows * a.rows.out_pitch / 16, to = a.rows.rows * a.rows.out_pitch / 16;
    for (int64_t i = from + (int64_t)blockIdx.x * 64 * WAVES + threadIdx.x; i < to; i += (int64_t)gridDim.x * 64 * WAVES)
        reinterpret_cast<uint4 *>(a.rows.out)[i] = make_uint4(0, 0, 0, 0);
}

template <class T, int GROUP, int U, int R, int S, int WAVES, int PER_SIMD>
int launch_as(const Int4Args &a, int64_t slots, hipStream_t stream) {
    const int strips = a.rows.cols / 16, jobs = (strips + U - 1) / U;
    const int64_t grid = std::min<int64_t>(jobs * slots, resident_grid() * (4 * PER_SIMD / WAVES));
    hipLaunchKernelGGL((grouped_mm_int4_kernel<T, GROUP, U, R, S, WAVES, PER_SIMD>), dim3((uint32_t)grid), dim3(64 * WAVES), 0, stream, a, strips, jobs);
    return check_launch("grouped_mm_int4 launch");
}
template <class T, int GROUP>
int launch(const Int4Args &a, hipStream_t stream) {
    const int64_t slots = std::min(a.rows.rows, a.rows.n_groups), strips = a.rows.cols / 16;
    // Rows are taken 16 at a time, or 32 where there are more, or on average nearly as many as that in a group, so that some have more (27 rows x
    // 28672 x 4096: 22 us instead of 30; 16 on average of 8 groups 125 instead of 137, 14 the same).  The registers of 32 rows cost
    // those with fewer half of their waves: 12 on average 123 us instead of 104, 4 (128 experts of 1536 x 2048) 51 instead of 41.
    // A wave with more strips reads x less often; few strips are shared by more waves instead, so that all CUs have some.  Strips
    // of one, two, four, us: 256 (a row through 4096 x 7168) 7.8, 9.8, 18; 1024 (8 of 128 experts of 2048 x 768) 8.0, 6.5, 7.8; 1536 (16
    // of 128 of 1536 x 2048) 11.8, 10.2, 11.1; 1792 (a row through 28672 x 4096) 16.8, 17.2, 15.6; 7900 (16 tokens on 128 of 1536 x 2048) 37, 30,
    // 26.
    const int64_t all = strips * slots, cus = resident_grid();
    if (a.rows.rows > (a.rows.offsets != nullptr ? 14 : 16) * (int64_t)a.rows.n_groups)
        return all <= 2 * cus ? launch_as<T, GROUP, 1, 2, 1, 8, 2>(a, slots, stream) : launch_as<T, GROUP, 4, 2, 1, 4, 2>(a, slots, stream);
    if (all <= 2 * cus) return launch_as<T, GROUP, 1, 1, 2, 8, 4>(a, slots, stream);
    if (all <= 6 * cus) return launch_as<T, GROUP, 2, 1, 1, 8, 4>(a, slots, stream);
    return launch_as<T, GROUP, 4, 1, 1, 4, 4>(a, slots, stream);
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
