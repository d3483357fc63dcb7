// Entry points and kernels of the whole layer for a few tokens (moe_layer.h).
#include "grouped_host.h"
#include "moe_layer.h"

namespace {

using namespace pmoe;
using namespace pmoe::layer;

// logits[t][e], four experts per workgroup; its waves share the contraction.
template <class T>
__global__ __launch_bounds__(256) void moe_layer_router_kernel(Args a) {
    __shared__ float part[4][kMaxTokens][4];
    const int lane = threadIdx.x & 63, wave = gmm::uniform(threadIdx.x >> 6), sub = lane >> 4;
    const int steps = (a.K + 127) / 128, s0 = wave * steps / 4, s1 = (wave + 1) * steps / 4;
    const char *const w[1] = {a.gate + (int64_t)min((int)blockIdx.x * 4 + sub, a.E - 1) * a.K * 2};
    by_rows(a.T, [&](auto n, int row0) {
        constexpr int N = decltype(n)::value;
        const char *x[N];
        float acc[1][N] = {};
#pragma unroll
        for (int j = 0; j < N; ++j) x[j] = a.x + (int64_t)min(row0 + j, a.T - 1) * a.K * 2;
        row_dots<T, 1, N, (N <= 4 ? 4 : 2)>(acc, w, x, s0, s1, a.K);
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const float v = row_sum(acc[0][j]);
            if ((lane & 15) == 0 && row0 + j < a.T) part[wave][row0 + j][sub] = v;
        }
    });
    __syncthreads();
    const int t = threadIdx.x >> 2, e = blockIdx.x * 4 + (threadIdx.x & 3);
    if (t < a.T && e < a.E) {
        float v = 0.f;
#pragma unroll
        for (int k = 0; k < 4; ++k) v += part[k][t][threadIdx.x & 3];
        a.logits[(int64_t)t * a.E + e] = v;
    }
}

template <class W>
__global__ __launch_bounds__(kThreads) void moe_layer_up_kernel(Args a) {
    __shared__ Plan p;
    __shared__ __attribute__((aligned(1024))) Sums sums;
    find_plan(a, p, blockIdx.x == 0);
    const int strips = (a.H + kUpCols - 1) / kUpCols, u = (int)blockIdx.x / strips;
    if (u < p.n) W::up(a, p, sums, u, (int)blockIdx.x - u * strips);
}

template <class W>
__global__ __launch_bounds__(kThreads) void moe_layer_down_kernel(Args a) {
    __shared__ Plan p;
    __shared__ __attribute__((aligned(1024))) Sums sums;
    find_plan(a, p, false);
    down_job<W>(a, p, sums, (int)blockIdx.x);
}

template <class W>
int launch(const Args &a, hipStream_t s) {
    hipLaunchKernelGGL((moe_layer_router_kernel<typename W::Type>), dim3((a.E + 3) / 4), dim3(256), 0, s, a);
    const int most = std::min(a.E, a.T * a.top_k);
    hipLaunchKernelGGL((moe_layer_up_kernel<W>), dim3(most * ((a.H + kUpCols - 1) / kUpCols)), dim3(kThreads), 0, s, a);
    hipLaunchKernelGGL((moe_layer_down_kernel<W>), dim3((a.K + W::kDownCols - 1) / W::kDownCols), dim3(kThreads), 0, s, a);
    return check_launch("moe_layer launch");
}
template <class T>
int launch(const Args &a, int group, hipStream_t s) {
    return group == 0 ? launch<Wide<T>>(a, s) : group == 32 ? launch<Narrow<T, 32>>(a, s) : group == 64 ? launch<Narrow<T, 64>>(a, s) : launch<Narrow<T, 128>>(a, s);
}

size_t act_pitch(int H) { return align_up((size_t)H * 2, 128); }
size_t logits_bytes(int T, int E) { return align_up((size_t)T * E * 4, 256); }

}  // namespace

extern "C" size_t pmoe_moe_layer_workspace_bytes(int T, int H, int num_experts, int top_k) {
    if (T <= 0 || H <= 0 || num_experts <= 0 || top_k <= 0) return 0;
    return logits_bytes(T, num_experts) + (size_t)T * top_k * 2 * act_pitch(H);
}

extern "C" int pmoe_moe_layer(const void *x, const void *gate, const float *bias, const void *w1, const void *w1_scale, const void *w2,
                              const void *w2_scale, int group, void *out, int32_t *topk_ids, float *topk_weights, int T, int K, int H,
                              int num_experts, int top_k, int dtype, void *workspace, size_t workspace_bytes, void *stream) {
    PMOE_REQUIRE(dtype == PMOE_DTYPE_BF16 || dtype == PMOE_DTYPE_F16, "moe_layer: dtype must be bf16 or fp16");
    PMOE_REQUIRE(T >= 0 && T <= kMaxTokens, "moe_layer takes up to %d tokens, got %d (more: route and fused_moe_bf16)", kMaxTokens, T);
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
    a.logits = static_cast<float *>(workspace);
    a.act = static_cast<char *>(workspace) + logits_bytes(T, num_experts);
    a.act_pitch = (int)act_pitch(H);
    a.T = T;
    a.K = K;
    a.H = H;
    a.E = num_experts;
    a.top_k = top_k;
    hipStream_t s = static_cast<hipStream_t>(stream);
    return dtype == PMOE_DTYPE_BF16 ? launch<Bf16>(a, group, s) : launch<F16>(a, group, s);
}
