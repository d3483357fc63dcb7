// Entry points and kernels of the whole layer for a few tokens (moe_layer.h).
#include "grouped_host.h"
#include "moe_layer.h"

namespace {

using namespace pmoe;
using namespace pmoe::layer;

// Workgroups that run at a time.
int slots() { return std::min(2 * resident_grid(), kMaxGroups); }

// logits[t][e]: four experts and up to four tokens per workgroup, whose waves share the contraction.  Beside that, the queues begin and the
// activation is marked as absent.
constexpr int kRouterTokens = 4;
template <class T>
__global__ __launch_bounds__(kThreads) void moe_layer_router_kernel(Args a) {
    __shared__ float part[kWaves][kRouterTokens][4];
    const int lane = threadIdx.x & 63, wave = gmm::uniform(threadIdx.x >> 6), sub = lane >> 4, t0 = blockIdx.y * kRouterTokens, rows = min(a.T - t0, kRouterTokens);
    const int steps = (a.K + 127) / 128, s0 = wave * steps >> kWavesLog, s1 = (wave + 1) * steps >> kWavesLog;
    const char *const w[1] = {a.gate + (int64_t)blockIdx.x * 4 * a.K * 2};
    auto some = [&](auto n) {
        constexpr int N = decltype(n)::value;
        uint32_t xo[N];
        float acc[1][N] = {};
#pragma unroll
        for (int j = 0; j < N; ++j) xo[j] = (uint32_t)(t0 + min(j, rows - 1)) * (uint32_t)a.K * 2;
        row_dots<T, 1, N, 4, 4>(acc, w, a.K * 2, a.x, (uint32_t)a.T * a.K * 2, xo, s0, s1, a.K, 1, min(a.E - 1 - (int)blockIdx.x * 4, 3));
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const float v = row_sum(acc[0][j]);
            if ((lane & 15) == 0) part[wave][j][sub] = v;
        }
    };
    if (rows == 1) some(std::integral_constant<int, 1>{});
    else some(std::integral_constant<int, kRouterTokens>{});
    const int block = blockIdx.y * gridDim.x + blockIdx.x;
    if (block == 0)
        for (int i = threadIdx.x; i < (int)(sizeof(Sync) / 4); i += kThreads) reinterpret_cast<int32_t *>(a.sync)[i] = 0;
    const int64_t words = (int64_t)a.T * a.top_k * 2 * a.act_pitch / 16;
#pragma unroll 1
    for (int64_t i = (int64_t)block * kThreads + threadIdx.x; i < words; i += (int64_t)gridDim.x * gridDim.y * kThreads)
        reinterpret_cast<i32x4 *>(a.act)[i] = i32x4{(int)kAbsent, (int)kAbsent, (int)kAbsent, (int)kAbsent};
    __syncthreads();
    const int t = threadIdx.x >> 2, e = blockIdx.x * 4 + (threadIdx.x & 3);
    if (t < rows && e < a.E) {
        float v = 0.f;
#pragma unroll
        for (int k = 0; k < kWaves; ++k) v += part[k][t][threadIdx.x & 3];
        a.logits[(int64_t)(t0 + t) * a.E + e] = v;
    }
}

template <class W, bool ONE>
__global__ __launch_bounds__(kThreads, 4) void moe_layer_kernel(Args a) {
    __shared__ Plan p;
    __shared__ __attribute__((aligned(1024))) Sums sums;
    int ticket = 0;
    if (threadIdx.x == 0) ticket = next_ticket(&a.sync->ticket[blockIdx.x % kQueues][0]);
    find_plan<ONE>(a, p, blockIdx.x == 0);
    const int each = W::down_steps(a), all = gmm::uniform(p.n) * each;
    const Place from = place_of<W>(a, blockIdx.x, all), to = place_of<W>(a, blockIdx.x + 1, all);
    const bool down_too = (int)blockIdx.x < a.down_groups;
    up_jobs<W, ONE>(a, p, sums, ticket, from, Steps(from, to, from.strip, all), each, down_too);
    if (!down_too) return;
    for (int strip = from.strip; strip <= to.strip; ++strip) {
        const Steps mine(from, to, strip, all);
        if (mine.from < mine.to) down_job<W, ONE>(a, p, sums, strip, mine, each, all);
    }
}

template <class W>
int launch(Args a, hipStream_t s) {
    hipLaunchKernelGGL((moe_layer_router_kernel<typename W::Type>), dim3((a.E + 3) / 4, (a.T + kRouterTokens - 1) / kRouterTokens), dim3(kThreads), 0, s, a);
    const int64_t up_jobs = (int64_t)std::min(a.E, a.T * a.top_k) * ((a.H + a.up_cols - 1) / a.up_cols);
    const dim3 grid((uint32_t)std::min<int64_t>(std::max<int64_t>(up_jobs, a.down_groups), slots())), block(kThreads);
    if (a.T == 1) hipLaunchKernelGGL((moe_layer_kernel<W, true>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((moe_layer_kernel<W, false>), grid, block, 0, s, a);
    return check_launch("moe_layer launch");
}
template <class T>
int launch(const Args &a, int group, hipStream_t s) {
    return group == 0 ? (a.up_cols == 4 ? launch<Wide<T, 1>>(a, s) : launch<Wide<T, 4>>(a, s)) : group == 32 ? launch<Narrow<T, 32>>(a, s) : group == 64 ? launch<Narrow<T, 64>>(a, s) : launch<Narrow<T, 128>>(a, s);
}

// How the jobs of a layer are cut.
void cut_jobs(Args &a, int group) {
    const int64_t most = std::min(a.E, a.T * a.top_k), rows = group != 0 ? 16 : 4, jobs = most * ((a.H + rows - 1) / rows);
    if (group != 0) {
        // As many columns as leave every workgroup a job: fewer jobs of a wave's longer reads.  16, 32, 64 columns, us: 12288 jobs of 16
        // (16 tokens on 256 experts of 7168 x 2048) 514, 496, 489; 3936 (16 on 128 of 2048 x 768) 64, 59, 58; 1024 (one on the 256) 55,
        // 53, 68; 384 (one on the 128) 17, 18, 21.
        while (a.up_log < Narrow<Bf16, 128>::kMaxUpLog && jobs >> (a.up_log + 1) >= slots()) ++a.up_log;
        a.up_cols = 16 << a.up_log;
    } else {
        // One round of the grid where jobs of up to 16 columns do that, otherwise the 16: a row of x is read less often.  (One token on 128
        // experts of 2048 x 768, 12 columns: 22.6 us, 25.5 with 4; 16 tokens 138, 166 with 4.)
        a.up_cols = 4 * (int)std::min<int64_t>(4, (jobs + slots() - 1) / slots());
    }
    // Strips of out are shared where that takes enough steps from the wave that has the most: joining takes two microseconds.  Shared, not
    // shared, us: 4 bits, 16 tokens on 128 experts of 2048 x 768 62, 79, three 31, 34, one (4 steps) 19.4, 17.0; 16 bits, 16 tokens 138,
    // 143, four (12 steps) 64.2, 63.2.
    const int64_t strips = group != 0 ? a.K / 16 : (a.K + 7) / 8, steps = most * ((a.H + 127) / 128);
    a.split = ((strips + slots() - 1) / slots() * steps - strips * steps / slots()) / kWaves >= (group != 0 ? 8 : 16);
    a.down_groups = (int)std::min<int64_t>(slots(), a.split ? strips * most : strips);
}
size_t act_pitch(int H) { return align_up((size_t)H * 2, 128); }
size_t logits_bytes(int T, int E) { return align_up((size_t)T * E * 4, 256); }
static_assert(sizeof(Sync) % 256 == 0, "what follows is aligned");

}  // namespace

extern "C" size_t pmoe_moe_layer_workspace_bytes(int T, int H, int num_experts, int top_k) {
    if (T <= 0 || H <= 0 || num_experts <= 0 || top_k <= 0) return 0;
    return sizeof(Sync) + logits_bytes(T, num_experts) + (size_t)2 * kMaxGroups * 16 * T * 4 + (size_t)T * top_k * 2 * act_pitch(H);
}

extern "C" int pmoe_moe_layer(const void *x, const void *gate, const float *bias, const void *w1, const void *w1_scale, const void *w2,
                              const void *w2_scale, int group, void *out, int32_t *topk_ids, float *topk_weights, int T, int K, int H,
                              int num_experts, int top_k, int dtype, void *workspace, size_t workspace_bytes, void *stream) {
    PMOE_REQUIRE(dtype == PMOE_DTYPE_BF16 || dtype == PMOE_DTYPE_F16, "moe_layer: dtype must be bf16 or fp16");
    PMOE_REQUIRE(T >= 0 && T <= kMaxTokens, "moe_layer takes up to %d tokens, got %d (more: %s)", kMaxTokens, T,
                 group != 0 ? "route and grouped_mm_int4" : dtype == PMOE_DTYPE_F16 ? "route and grouped_mm" : "route and fused_moe_bf16");
    PMOE_REQUIRE(num_experts > 0 && num_experts <= kMaxExperts, "moe_layer supports 1..%d experts, got %d", kMaxExperts, num_experts);
    PMOE_REQUIRE(top_k > 0 && top_k <= kMaxTopK && top_k <= num_experts, "moe_layer: top_k must be in 1..min(%d, num_experts), got %d", kMaxTopK, top_k);
    PMOE_REQUIRE(group == 0 || group == 32 || group == 64 || group == 128, "moe_layer: group must be 0 (16-bit weights), 32, 64 or 128, got %d", group);
    const int unit = group == 0 ? 8 : std::max(group, 16);
    PMOE_REQUIRE(K > 0 && H > 0 && K % unit == 0 && H % unit == 0 && K <= 1 << 20 && H <= 1 << 20,
                 "moe_layer: K (%d) and H (%d) must be positive multiples of %d up to 2^20", K, H, unit);
    if (T == 0) return PMOE_OK;
    PMOE_REQUIRE(x && gate && w1 && w2 && out && topk_ids && topk_weights && workspace && (group == 0 || (w1_scale && w2_scale)), "moe_layer: null pointer");
    PMOE_REQUIRE_ALIGNED("moe_layer", x, gate, w1, w2, out, w1_scale, w2_scale);
    PMOE_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 256 == 0, "moe_layer: the workspace must be 256-byte aligned");
    const size_t need = pmoe_moe_layer_workspace_bytes(T, H, num_experts, top_k);
    PMOE_REQUIRE(workspace_bytes >= need, "moe_layer: workspace of %zu bytes, %zu needed", workspace_bytes, need);
    Args a = {};
    a.x = static_cast<const char *>(x);
    a.gate = static_cast<const char *>(gate);
    a.bias = bias;
    a.w1 = static_cast<const char *>(w1);
    a.w1_scale = static_cast<const char *>(w1_scale);
    a.w2 = static_cast<const char *>(w2);
    a.w2_scale = static_cast<const char *>(w2_scale);
    a.out = static_cast<char *>(out);
    a.topk_ids = topk_ids;
    a.topk_weights = topk_weights;
    a.sync = static_cast<Sync *>(workspace);
    a.logits = reinterpret_cast<float *>(a.sync + 1);
    a.shares = reinterpret_cast<float *>(reinterpret_cast<char *>(a.logits) + logits_bytes(T, num_experts));
    a.act = reinterpret_cast<char *>(a.shares + (size_t)2 * kMaxGroups * 16 * T);
    a.act_pitch = (int)act_pitch(H);
    a.T = T;
    a.K = K;
    a.H = H;
    a.E = num_experts;
    a.top_k = top_k;
    cut_jobs(a, group);
    hipStream_t s = static_cast<hipStream_t>(stream);
    return dtype == PMOE_DTYPE_BF16 ? launch<Bf16>(a, group, s) : launch<F16>(a, group, s);
}
