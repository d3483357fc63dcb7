// Host side of the Python package: argument checks, output and workspace allocation, and the calls into
// libprime_moe_hip.so.  Registers the CUDA-key implementations of the prime_moe:: ops (their schemas are defined in
// prime_moe/__init__.py) and exposes what is not an op (route, quantize_mx, the checks) as Python functions.
//
// Replaces the stubs of the reference's prime_moe/csrc/torch_interface.cpp:82-268; the conditions are those of its
// TORCH_CHECKs (:85-87, :132-155, :208-241) and the ones the kernels need on top.  No device code.
//
// In C++ because the calls a decode step makes are short: checks, allocations and ctypes in Python cost 25 - 30 us a
// call, which the device spends less than on a single token.
#include <limits>

#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/utils/pybind.h>
#include <torch/library.h>
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include "../../include/prime_moe_hip.h"

namespace {

using at::Tensor;

#define REQUIRE(cond, ...)                                            \
    do {                                                              \
        if (C10_UNLIKELY(!(cond))) fail(c10::str(__VA_ARGS__));       \
    } while (0)

[[noreturn]] void fail(const std::string &msg) { throw std::runtime_error(msg); }

void check_status(int rc) {
    if (C10_UNLIKELY(rc != PMOE_OK)) {
        const char *msg = pmoe_last_error();
        fail(msg != nullptr && *msg ? msg : c10::str("prime_moe native error ", rc));
    }
}

void *stream_of(const c10::Device &dev) {
    return c10::hip::getCurrentHIPStream(dev.index()).stream();
}

Tensor empty(at::IntArrayRef size, at::ScalarType dtype, const c10::Device &dev) {
    return at::empty(size, at::TensorOptions().dtype(dtype).device(dev));
}
// Scratch of one call, from torch's caching allocator: stream ordered, no hipMalloc in steady state, capturable.
Tensor workspace(size_t bytes, const c10::Device &dev) {
    return empty({(int64_t)std::max<size_t>(bytes, 256)}, at::kByte, dev);
}

struct Arg {
    const char *name;
    const Tensor *t;
};

// Every tensor must live on the GPU of the first one: the kernels take raw device pointers, so a CPU tensor (or one on
// another GPU) would be a memory fault on the device, not an exception.
void require_same_device(const char *op, std::initializer_list<Arg> args) {
    const Arg &anchor = *args.begin();
    const c10::Device dev = anchor.t->device();
    REQUIRE(dev.is_cuda(), op, ": ", anchor.name, " must be a GPU tensor, got device ", dev);
    for (const Arg &a : args)
        REQUIRE(a.t->device() == dev, op, ": ", a.name, " is on ", a.t->device(), ", expected ", dev, " (the device of ",
                anchor.name, ")");
}
// The kernels read these with `align`-byte vector loads from the start of the tensor.
void require_aligned(const char *op, std::initializer_list<Arg> args, uintptr_t align) {
    for (const Arg &a : args)
        REQUIRE(reinterpret_cast<uintptr_t>(a.t->const_data_ptr()) % align == 0, op, ": ", a.name, " must start at a ", align,
                "-byte aligned address");
}
void require_contiguous(const char *op, std::initializer_list<Arg> args) {
    for (const Arg &a : args) REQUIRE(a.t->is_contiguous(), op, ": ", a.name, " must be contiguous");
}
void require_dtype(const char *op, std::initializer_list<Arg> args, at::ScalarType dtype, const char *dtype_name) {
    for (const Arg &a : args) REQUIRE(a.t->scalar_type() == dtype, op, ": ", a.name, " must be ", dtype_name);
}

void check_tuning(const char *what, int64_t block_m, int64_t block_n, int64_t warp_n, int64_t stages, int64_t max_stages) {
    REQUIRE((block_n == 64 && warp_n == 4) || (block_n == 32 && warp_n == 8), what,
            ": (block_n, warp_n) must be (64, 4) or (32, 8), got (", block_n, ", ", warp_n, ")");
    REQUIRE(stages > 0 && stages <= max_stages, what, " supports stages in 1..", max_stages, ", got ", stages);
    REQUIRE(block_m == 128, what, " requires block_m=128, got ", block_m);
}

// ------------------------------------------------------------------------------- moe_align

// (pad_to, max_padded, max_blocks) as torch_interface.cpp:88-91 computes them.  Ids, positions and sizes are int32 in the
// kernels and the C ABI: what does not fit is an error here (block_m, bpc > 0, num_experts <= 1024: no step overflows).
struct AlignSizes {
    int64_t pad_to, max_padded, max_blocks;
    AlignSizes(int64_t n, int64_t num_experts, int64_t block_m, int64_t bpc) {
        constexpr int64_t kMax = std::numeric_limits<int32_t>::max();
        REQUIRE(n <= kMax, "moe_align: ", n, " ids do not fit 32 bits");
        REQUIRE(block_m <= kMax && bpc <= kMax / block_m, "moe_align: block_m * bpc does not fit 32 bits (", block_m, " * ", bpc, ")");
        pad_to = block_m * bpc;
        max_padded = (n + num_experts * (pad_to - 1) + pad_to - 1) / pad_to * pad_to;
        REQUIRE(max_padded <= kMax, "moe_align: a schedule of ", max_padded, " rows does not fit 32 bits");
        max_blocks = max_padded / block_m;
    }
};

// `placement`: false leaves out the device check (what is left can then be exercised with CPU tensors).
void validate_align(const Tensor &topk_ids, int64_t num_experts, int64_t block_m, int64_t bpc, bool placement) {
    REQUIRE(topk_ids.is_cuda() || !placement, "moe_align: topk_ids must be a GPU tensor, got device ", topk_ids.device());
    REQUIRE(topk_ids.is_contiguous(), "moe_align: topk_ids must be contiguous");
    REQUIRE(topk_ids.scalar_type() == at::kInt, "moe_align: topk_ids must be int32");
    REQUIRE(block_m > 0 && bpc > 0 && num_experts > 0, "moe_align: block_m, bpc and num_experts must be positive");
    REQUIRE(num_experts <= 1024, "moe_align supports at most 1024 experts, got ", num_experts);
    AlignSizes(topk_ids.numel(), num_experts, block_m, bpc);
}

struct Schedule {
    Tensor sorted_token_ids, expert_ids, num_tokens_post_padded, ws;
    size_t ws_bytes;
    Schedule(const AlignSizes &sz, int64_t n, int64_t num_experts, const c10::Device &dev)
        : sorted_token_ids(empty({sz.max_padded}, at::kInt, dev)),
          expert_ids(empty({sz.max_blocks}, at::kInt, dev)),
          num_tokens_post_padded(empty({1}, at::kInt, dev)) {
        // many ids: scratch for the multi-workgroup sort (0 bytes when one workgroup does it)
        ws_bytes = pmoe_moe_align_workspace_bytes_fast((int)n, (int)num_experts);
        if (ws_bytes > 0) ws = workspace(ws_bytes, dev);
    }
    void *ws_ptr() const { return ws_bytes > 0 ? ws.data_ptr() : nullptr; }
};

std::tuple<Tensor, Tensor, Tensor> moe_align(const Tensor &topk_ids, int64_t num_experts, int64_t block_m, int64_t bpc) {
    validate_align(topk_ids, num_experts, block_m, bpc, true);
    const c10::Device dev = topk_ids.device();
    const c10::DeviceGuard guard(dev);
    const int64_t n = topk_ids.numel();
    const AlignSizes sz(n, num_experts, block_m, bpc);
    Schedule s(sz, n, num_experts, dev);
    check_status(pmoe_moe_align_ws(topk_ids.const_data_ptr<int32_t>(), s.sorted_token_ids.data_ptr<int32_t>(),
                                   s.expert_ids.data_ptr<int32_t>(), s.num_tokens_post_padded.data_ptr<int32_t>(), (int)n,
                                   (int)num_experts, (int)block_m, (int)sz.pad_to, (int)sz.max_padded, (int)sz.max_blocks,
                                   s.ws_ptr(), s.ws_bytes, stream_of(dev)));
    return {s.sorted_token_ids, s.expert_ids, s.num_tokens_post_padded};
}

// ------------------------------------------------------------------------------- fused_moe_bf16

void validate_bf16(const Tensor &x, const Tensor &w, const Tensor &w2, const Tensor &sorted_token_ids, const Tensor &expert_ids,
                   const Tensor &num_tokens_post_padded, const Tensor &topk_weights, const Tensor &out, int64_t top_k,
                   int64_t block_m, int64_t block_n, int64_t warp_n, int64_t stages, int64_t bpc, int64_t cpc, bool split,
                   bool placement) {
    const char *op = "fused_moe_bf16";
    REQUIRE(x.dim() == 2 && w.dim() == 3 && w2.dim() == 3, op, ": x must be 2-D, w and w2 3-D");
    REQUIRE(x.size(0) > 0, op, ": x has no rows");
    REQUIRE(x.size(1) == w.size(2), op, ": x.size(1) must equal w.size(2)");
    REQUIRE(x.size(1) % 128 == 0, "K dimension must be a multiple of 128");
    REQUIRE(w.size(1) % 256 == 0, op, ": N must be a multiple of 256, got ", w.size(1));
    REQUIRE(w2.size(0) == w.size(0) && w2.size(1) == x.size(1) && w2.size(2) == w.size(1) / 2, op,
            ": w2 must have shape (E, K, N/2)");
    check_tuning(op, block_m, block_n, warp_n, stages, 5);
    REQUIRE(bpc == 1 && cpc == 1, "bpc=cpc=1 is the only supported configuration");
    REQUIRE(!split || stages <= 4, "split=True requires stages<=4, got stages=", stages);
    REQUIRE(top_k > 0, op, ": top_k must be positive");
    const Arg ax{"x", &x}, aw{"w", &w}, aw2{"w2", &w2}, as{"sorted_token_ids", &sorted_token_ids}, ae{"expert_ids", &expert_ids},
        an{"num_tokens_post_padded", &num_tokens_post_padded}, at_{"topk_weights", &topk_weights}, ao{"out", &out};
    if (placement) {
        require_same_device(op, {ax, aw, aw2, as, ae, an, at_, ao});
        require_aligned(op, {ax, aw, aw2, ao}, 16);
        require_aligned(op, {as, ae, an, at_}, 4);
    }
    require_contiguous(op, {ax, aw, aw2, as, ae, an, at_, ao});
    require_dtype(op, {ax, aw, aw2, ao}, at::kBFloat16, "bfloat16");
    require_dtype(op, {at_}, at::kFloat, "float32");
    require_dtype(op, {as, ae, an}, at::kInt, "int32");
    REQUIRE(out.sizes() == x.sizes(), op, ": out must have the shape of x");
    REQUIRE(num_tokens_post_padded.numel() >= 1, op, ": num_tokens_post_padded is empty");
    REQUIRE(expert_ids.numel() * block_m >= sorted_token_ids.numel(), op,
            ": expert_ids is shorter than sorted_token_ids / block_m");
}

void fused_moe_bf16(const Tensor &x, const Tensor &w, const Tensor &w2, const Tensor &sorted_token_ids, const Tensor &expert_ids,
                    const Tensor &num_tokens_post_padded, const Tensor &topk_weights, Tensor &out, int64_t top_k, int64_t block_m,
                    int64_t block_n, int64_t warp_n, int64_t stages, int64_t bpc, int64_t cpc, bool split) {
    validate_bf16(x, w, w2, sorted_token_ids, expert_ids, num_tokens_post_padded, topk_weights, out, top_k, block_m, block_n,
                  warp_n, stages, bpc, cpc, split, true);
    const c10::Device dev = x.device();
    const c10::DeviceGuard guard(dev);
    const int M = (int)x.size(0), K = (int)x.size(1), E = (int)w.size(0), N = (int)w.size(1), S = (int)sorted_token_ids.size(0);
    const Tensor ws = workspace(pmoe_fused_moe_bf16_workspace_bytes(M, K, N, E, S, (int)top_k, split), dev);
    check_status(pmoe_fused_moe_bf16(
        x.const_data_ptr(), w.const_data_ptr(), w2.const_data_ptr(), out.data_ptr(), sorted_token_ids.const_data_ptr<int32_t>(),
        expert_ids.const_data_ptr<int32_t>(), num_tokens_post_padded.const_data_ptr<int32_t>(),
        topk_weights.const_data_ptr<float>(), (int)top_k, M, K, N, E, S, (int)block_m, (int)block_n, (int)warp_n, (int)stages,
        (int)bpc, (int)cpc, split, ws.data_ptr(), (size_t)ws.numel(), stream_of(dev)));
}

// ------------------------------------------------------------------------------- fused_moe_mxfp8

void validate_mxfp8(const Tensor &x, const Tensor &x_scales, const Tensor &w, const Tensor &w_scales, const Tensor &w2,
                    const Tensor &w2_scales, const Tensor &sorted_token_ids, const Tensor &expert_ids,
                    const Tensor &num_tokens_post_padded, const Tensor &topk_weights, const Tensor &out, int64_t top_k,
                    int64_t block_m, int64_t block_n, int64_t warp_n, int64_t stages, int64_t bpc, bool split, bool placement) {
    const char *op = "fused_moe_mxfp8";
    REQUIRE(x.dim() == 2 && w.dim() == 3 && w2.dim() == 3, op, ": x must be 2-D, w and w2 3-D");
    const int64_t M = x.size(0), K = x.size(1), E = w.size(0), N = w.size(1);
    REQUIRE(M > 0, op, ": x has no rows");
    REQUIRE(K == w.size(2), op, ": x.size(1) must equal w.size(2)");
    REQUIRE(K % 256 == 0, "K dimension must be a multiple of 256 on the mxfp8 path");
    REQUIRE(N % 256 == 0, "N dimension must be a multiple of 256 on the mxfp8 path");
    REQUIRE(w2.size(0) == E && w2.size(1) == K && w2.size(2) == N / 2, op, ": w2 must have shape (E, K, N/2)");
    check_tuning("mxfp8", block_m, block_n, warp_n, stages, 4);
    REQUIRE(bpc == 1, "mxfp8 supports bpc=1 only");
    REQUIRE(top_k > 0, op, ": top_k must be positive");
    REQUIRE(x_scales.numel() == M * (K / 32), "x_scales must be a row major (M, K/32) e8m0 tensor");
    REQUIRE(w_scales.numel() == E * N * (K / 32), "w_scales must hold E*N*K/32 e8m0 values in the blocked layout");
    REQUIRE(w2_scales.numel() == E * K * ((N / 2) / 32), "w2_scales must hold E*K*(N/2)/32 e8m0 values in the blocked layout");
    const Arg ax{"x", &x}, axs{"x_scales", &x_scales}, aw{"w", &w}, aws{"w_scales", &w_scales}, aw2{"w2", &w2},
        aw2s{"w2_scales", &w2_scales}, as{"sorted_token_ids", &sorted_token_ids}, ae{"expert_ids", &expert_ids},
        an{"num_tokens_post_padded", &num_tokens_post_padded}, at_{"topk_weights", &topk_weights}, ao{"out", &out};
    if (placement) {
        require_same_device(op, {ax, axs, aw, aws, aw2, aw2s, as, ae, an, at_, ao});
        require_aligned(op, {ax, aw, aw2, ao}, 16);
        require_aligned(op, {axs, aws, aw2s, as, ae, an, at_}, 4);
    }
    require_contiguous(op, {ax, axs, aw, aws, aw2, aw2s, as, ae, an, at_, ao});
    require_dtype(op, {ax, aw, aw2}, at::kFloat8_e4m3fn, "float8_e4m3fn");
    require_dtype(op, {axs, aws, aw2s}, at::kFloat8_e8m0fnu, "float8_e8m0fnu");
    require_dtype(op, {at_}, at::kFloat, "float32");
    require_dtype(op, {as, ae, an}, at::kInt, "int32");
    require_dtype(op, {ao}, at::kBFloat16, "bfloat16");
    REQUIRE(out.dim() == 2 && out.size(0) == M && out.size(1) == K, op, ": out must have shape (M, K)");
    REQUIRE(num_tokens_post_padded.numel() >= 1, op, ": num_tokens_post_padded is empty");
    REQUIRE(expert_ids.numel() * block_m >= sorted_token_ids.numel(), op,
            ": expert_ids is shorter than sorted_token_ids / block_m");
}

void fused_moe_mxfp8(const Tensor &x, const Tensor &x_scales, const Tensor &w, const Tensor &w_scales, const Tensor &w2,
                     const Tensor &w2_scales, const Tensor &sorted_token_ids, const Tensor &expert_ids,
                     const Tensor &num_tokens_post_padded, const Tensor &topk_weights, Tensor &out, int64_t top_k,
                     int64_t block_m, int64_t block_n, int64_t warp_n, int64_t stages, int64_t bpc, bool split) {
    validate_mxfp8(x, x_scales, w, w_scales, w2, w2_scales, sorted_token_ids, expert_ids, num_tokens_post_padded, topk_weights,
                   out, top_k, block_m, block_n, warp_n, stages, bpc, split, true);
    const c10::Device dev = x.device();
    const c10::DeviceGuard guard(dev);
    const int M = (int)x.size(0), K = (int)x.size(1), E = (int)w.size(0), N = (int)w.size(1), S = (int)sorted_token_ids.size(0);
    const Tensor ws = workspace(pmoe_fused_moe_mxfp8_workspace_bytes(M, K, N, E, S, (int)top_k, split), dev);
    check_status(pmoe_fused_moe_mxfp8(
        x.const_data_ptr(), x_scales.const_data_ptr(), w.const_data_ptr(), w_scales.const_data_ptr(), w2.const_data_ptr(),
        w2_scales.const_data_ptr(), out.data_ptr(), sorted_token_ids.const_data_ptr<int32_t>(),
        expert_ids.const_data_ptr<int32_t>(), num_tokens_post_padded.const_data_ptr<int32_t>(),
        topk_weights.const_data_ptr<float>(), (int)top_k, M, K, N, E, S, (int)block_m, (int)block_n, (int)warp_n, (int)stages,
        (int)bpc, split, ws.data_ptr(), (size_t)ws.numel(), stream_of(dev)));
}

// ------------------------------------------------------------------------------- ragged expert products

// What the checks below find out about a matrix, or a stack of them, whose rows are `stride` elements apart.
struct Rows {
    int64_t stride = 0;        // between rows
    int64_t group_stride = 0;  // between matrices
    bool across = false;       // stored transposed
};
// A stride that no access uses (a single row) may be anything: it is taken as the least that the kernels accept.
int64_t stride_of(const Tensor &t, int64_t dim, int64_t least) {
    return t.size(dim) > 1 ? t.stride(dim) : (least + 15) / 16 * 16;
}
void require_rows(const char *op, const char *name, const Tensor &t, int64_t unit, int64_t stride, int64_t width) {
    REQUIRE(stride >= width && stride % unit == 0 && stride <= (8 << 20) / t.element_size(), op, ": the rows of ", name, " are ", stride,
            " elements apart; supported are multiples of ", unit, " from ", width, " to ", (8 << 20) / t.element_size());
}
Rows rows_of(const char *op, const char *name, const Tensor &t, int64_t unit) {
    Rows r;
    REQUIRE(t.size(1) == 1 || t.stride(1) == 1, op, ": the last dimension of ", name, " must be contiguous");
    r.stride = stride_of(t, 0, t.size(1));
    if (t.numel() > 0) require_rows(op, name, t, unit, r.stride, t.size(1));
    return r;
}
// `w` (E, N, K): K contiguous, or (`transposed`) N.
Rows stack_of(const char *op, const Tensor &w, int64_t unit, bool transposed) {
    Rows r;
    r.across = transposed && w.stride(2) != 1 && w.stride(1) == 1;
    REQUIRE(r.across || w.stride(2) == 1, op, ": ", transposed ? "one of the last two dimensions" : "the last dimension", " of w must be contiguous");
    const int64_t along = r.across ? 1 : 2;
    r.stride = stride_of(w, 3 - along, w.size(along));
    require_rows(op, "w", w, unit, r.stride, w.size(along));
    r.group_stride = w.size(0) > 1 ? w.stride(0) : 0;
    REQUIRE(r.group_stride % unit == 0, op, ": the matrices of w are ", r.group_stride, " elements apart, which is not a multiple of ", unit);
    return r;
}
int dtype_code(at::ScalarType t) {
    return t == at::kFloat ? PMOE_DTYPE_F32 : t == at::kBFloat16 ? PMOE_DTYPE_BF16 : t == at::kHalf ? PMOE_DTYPE_F16 : -1;
}
void require_16bit(const char *op, const char *name, const Tensor &t) {
    REQUIRE(t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf, op, ": ", name, " must be bfloat16 or float16");
}
constexpr int64_t kMostGroups = 1024, kMostRows = std::numeric_limits<int32_t>::max() - 512, kMostSide = 1 << 28;
void require_groups(const char *op, const Tensor &offsets, int64_t groups) {
    REQUIRE(offsets.dim() == 1 && offsets.is_contiguous() && offsets.scalar_type() == at::kInt, op, ": offsets must be a contiguous int32 (E,) tensor");
    REQUIRE(groups < 0 || offsets.size(0) == groups, op, ": offsets must have one entry per matrix of w (", groups, "), got ", offsets.size(0));
    REQUIRE(offsets.size(0) > 0 && offsets.size(0) <= kMostGroups, op, " supports 1..", kMostGroups, " experts, got ", offsets.size(0));
}
void require_side(const char *op, const char *name, int64_t n, int64_t unit) {
    REQUIRE(n > 0 && n % unit == 0 && n <= kMostSide, op, ": ", name, " must be a positive multiple of ", unit, " up to 2^28, got ", n);
}

struct MmPlan {
    Rows x, w;
};
MmPlan check_grouped_mm(const Tensor &x, const Tensor &w, const Tensor &offsets, bool placement) {
    const char *op = "grouped_mm";
    REQUIRE(x.dim() == 2 && w.dim() == 3, op, ": x must be 2-D (M, K), w 3-D (E, N, K)");
    REQUIRE(x.size(1) == w.size(2), op, ": x.size(1) must equal w.size(2), got ", x.size(1), " and ", w.size(2));
    require_16bit(op, "x", x);
    REQUIRE(w.scalar_type() == x.scalar_type(), op, ": x and w must have the same dtype");
    REQUIRE(x.size(0) <= kMostRows, op, ": too many rows");
    require_side(op, "N", w.size(1), 8);
    require_side(op, "K", w.size(2), 8);
    require_groups(op, offsets, w.size(0));
    const MmPlan p{rows_of(op, "x", x, 8), stack_of(op, w, 8, true)};
    if (placement) {
        require_same_device(op, {{"x", &x}, {"w", &w}, {"offsets", &offsets}});
        require_aligned(op, {{"x", &x}, {"w", &w}}, 16);
    }
    return p;
}
Tensor grouped_mm(const Tensor &x, const Tensor &w, const Tensor &offsets) {
    const MmPlan p = check_grouped_mm(x, w, offsets, true);
    const c10::Device dev = x.device();
    const c10::DeviceGuard guard(dev);
    Tensor out = empty({x.size(0), w.size(1)}, x.scalar_type(), dev);
    check_status(pmoe_grouped_mm(x.const_data_ptr(), w.const_data_ptr(), out.data_ptr(), offsets.const_data_ptr<int32_t>(), (int)w.size(0),
                                 x.size(0), (int)w.size(1), (int)w.size(2), p.x.stride, p.w.stride, p.w.group_stride, p.w.across,
                                 dtype_code(x.scalar_type()), stream_of(dev)));
    return out;
}

MmPlan check_grouped_mm_wgrad(const Tensor &dy, const Tensor &x, const Tensor &offsets, bool placement) {
    const char *op = "grouped_mm_wgrad";
    REQUIRE(dy.dim() == 2 && x.dim() == 2 && dy.size(0) == x.size(0), op, ": dy (M, N) and x (M, K) must be 2-D with the same number of rows");
    require_16bit(op, "x", x);
    REQUIRE(dy.scalar_type() == x.scalar_type(), op, ": dy and x must have the same dtype");
    REQUIRE(x.size(0) <= kMostRows, op, ": too many rows");
    require_side(op, "N", dy.size(1), 8);
    require_side(op, "K", x.size(1), 8);
    require_groups(op, offsets, -1);
    const MmPlan p{rows_of(op, "dy", dy, 8), rows_of(op, "x", x, 8)};
    if (placement) {
        require_same_device(op, {{"dy", &dy}, {"x", &x}, {"offsets", &offsets}});
        require_aligned(op, {{"dy", &dy}, {"x", &x}}, 16);
    }
    return p;
}
Tensor grouped_mm_wgrad(const Tensor &dy, const Tensor &x, const Tensor &offsets) {
    const MmPlan p = check_grouped_mm_wgrad(dy, x, offsets, true);
    const c10::Device dev = x.device();
    const c10::DeviceGuard guard(dev);
    Tensor dw = empty({offsets.size(0), dy.size(1), x.size(1)}, x.scalar_type(), dev);
    check_status(pmoe_grouped_mm_wgrad(dy.const_data_ptr(), x.const_data_ptr(), dw.data_ptr(), offsets.const_data_ptr<int32_t>(),
                                       (int)offsets.size(0), x.size(0), (int)dy.size(1), (int)x.size(1), p.x.stride, p.w.stride,
                                       dtype_code(x.scalar_type()), stream_of(dev)));
    return dw;
}

// Gradients.  Each of the two operators has its gradients in terms of both, so gradients of gradients exist too.  What
// comes back from a loss may have any strides (an expanded scalar): it is laid out first where the kernels need it.
using Product = Tensor(const Tensor &, const Tensor &, const Tensor &);
Tensor call_mm(const Tensor &x, const Tensor &w, const Tensor &offsets) {
    static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("prime_moe::grouped_mm", "").typed<Product>();
    return op.call(x, w, offsets);
}
Tensor call_wgrad(const Tensor &dy, const Tensor &x, const Tensor &offsets) {
    static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("prime_moe::grouped_mm_wgrad", "").typed<Product>();
    return op.call(dy, x, offsets);
}

// (contiguous() would return a contiguous tensor that begins at an odd element, such as a piece of a flat gradient, as it is)
Tensor laid_out(const Tensor &t) {
    const bool rows = t.dim() == 2 && (t.size(1) == 1 || t.stride(1) == 1) &&
                      (t.size(0) <= 1 || (t.stride(0) >= t.size(1) && t.stride(0) % 8 == 0 && t.stride(0) <= 4 << 20));
    return (rows || t.is_contiguous()) && t.storage_offset() % 8 == 0 ? t : t.clone(at::MemoryFormat::Contiguous);
}

struct GroupedMm : torch::autograd::Function<GroupedMm> {
    static Tensor forward(torch::autograd::AutogradContext *ctx, const Tensor &x, const Tensor &w, const Tensor &offsets) {
        at::AutoDispatchBelowADInplaceOrView below;
        ctx->save_for_backward({x, w, offsets});
        return call_mm(x, w, offsets);
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx, torch::autograd::variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        Tensor dx, dw;
        if (grads[0].defined()) {
            const Tensor dy = laid_out(grads[0]);
            if (ctx->needs_input_grad(0)) dx = call_mm(dy, saved[1].transpose(1, 2), saved[2]);
            if (ctx->needs_input_grad(1)) dw = call_wgrad(dy, saved[0], saved[2]);
        }
        return {dx, dw, Tensor()};
    }
};
struct GroupedMmWgrad : torch::autograd::Function<GroupedMmWgrad> {
    static Tensor forward(torch::autograd::AutogradContext *ctx, const Tensor &dy, const Tensor &x, const Tensor &offsets) {
        at::AutoDispatchBelowADInplaceOrView below;
        ctx->save_for_backward({dy, x, offsets});
        return call_wgrad(dy, x, offsets);
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx, torch::autograd::variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        Tensor ddy, dx;
        if (grads[0].defined()) {
            const Tensor g = laid_out(grads[0]);  // (E, N, K)
            if (ctx->needs_input_grad(0)) ddy = call_mm(saved[1], g, saved[2]);
            if (ctx->needs_input_grad(1)) dx = call_mm(saved[0], g.transpose(1, 2), saved[2]);
        }
        return {ddy, dx, Tensor()};
    }
};
// A dual tensor has a tangent and need not require gradients: without a tangent of its own the output would stand for one that
// does not change.
bool differentiated(const char *op, const Tensor &a, const Tensor &b) {
    REQUIRE(!a._fw_grad(0).defined() && !b._fw_grad(0).defined(), op, ": forward-mode derivatives are not implemented");
    return at::GradMode::is_enabled() && (a.requires_grad() || b.requires_grad());
}
Tensor grouped_mm_autograd(const Tensor &x, const Tensor &w, const Tensor &offsets) {
    if (differentiated("grouped_mm", x, w)) return GroupedMm::apply(x, w, offsets);
    at::AutoDispatchBelowADInplaceOrView below;
    return call_mm(x, w, offsets);
}
Tensor grouped_mm_wgrad_autograd(const Tensor &dy, const Tensor &x, const Tensor &offsets) {
    if (differentiated("grouped_mm_wgrad", dy, x)) return GroupedMmWgrad::apply(dy, x, offsets);
    at::AutoDispatchBelowADInplaceOrView below;
    return call_wgrad(dy, x, offsets);
}

MmPlan check_grouped_mm_int8(const Tensor &x, const Tensor &w, const Tensor &x_scale, const Tensor &w_scale, const std::optional<Tensor> &offsets,
                             at::ScalarType out_dtype, bool placement) {
    const char *op = "grouped_mm_int8";
    const bool dense = !offsets.has_value();
    REQUIRE(x.dim() == 2 && w.dim() == (dense ? 2 : 3), op, ": x must be 2-D (M, K), w 3-D (E, N, K) with offsets and 2-D (N, K) without");
    REQUIRE(x.size(1) == w.size(-1), op, ": x.size(1) must equal w.size(-1), got ", x.size(1), " and ", w.size(-1));
    REQUIRE(x.scalar_type() == at::kChar && w.scalar_type() == at::kChar, op, ": x and w must be int8");
    REQUIRE(dtype_code(out_dtype) >= 0, op, ": out_dtype must be bfloat16, float16 or float32");
    REQUIRE(x.size(0) <= kMostRows, op, ": too many rows");
    require_side(op, "N", w.size(-2), 8);
    require_side(op, "K", w.size(-1), 16);
    REQUIRE(x.size(1) < 131072, op, ": K must be below 131072 (exact sums in 32 bits), got ", x.size(1));
    if (!dense) require_groups(op, *offsets, w.size(0));
    REQUIRE(x_scale.scalar_type() == at::kFloat && x_scale.is_contiguous() && x_scale.dim() == 1 && x_scale.size(0) == x.size(0), op,
            ": x_scale must be a contiguous float32 (M,) tensor");
    REQUIRE(w_scale.scalar_type() == at::kFloat && w_scale.is_contiguous() && w_scale.sizes() == w.sizes().slice(0, w.dim() - 1), op,
            ": w_scale must be a contiguous float32 tensor of shape ", dense ? "(N,)" : "(E, N)");
    const MmPlan p{rows_of(op, "x", x, 16), dense ? rows_of(op, "w", w, 16) : stack_of(op, w, 16, false)};
    if (placement) {
        require_same_device(op, {{"x", &x}, {"w", &w}, {"x_scale", &x_scale}, {"w_scale", &w_scale}});
        if (!dense) require_same_device(op, {{"x", &x}, {"offsets", &*offsets}});
        require_aligned(op, {{"x", &x}, {"w", &w}}, 16);
    }
    return p;
}
Tensor grouped_mm_int8(const Tensor &x, const Tensor &w, const Tensor &x_scale, const Tensor &w_scale, const std::optional<Tensor> &offsets,
                       at::ScalarType out_dtype) {
    const MmPlan p = check_grouped_mm_int8(x, w, x_scale, w_scale, offsets, out_dtype, true);
    const c10::Device dev = x.device();
    const c10::DeviceGuard guard(dev);
    Tensor out = empty({x.size(0), w.size(-2)}, out_dtype, dev);
    check_status(pmoe_grouped_mm_int8(x.const_data_ptr(), w.const_data_ptr(), x_scale.const_data_ptr<float>(), w_scale.const_data_ptr<float>(),
                                      out.data_ptr(), offsets.has_value() ? offsets->const_data_ptr<int32_t>() : nullptr,
                                      offsets.has_value() ? (int)w.size(0) : 1, x.size(0), (int)w.size(-2), (int)x.size(1), p.x.stride,
                                      p.w.stride, p.w.group_stride, dtype_code(out_dtype), stream_of(dev)));
    return out;
}

// `x` (..., K): rows of the last dimension; a 2-D view may have rows any multiple of 8 elements apart.
int64_t check_quantize_int8(const Tensor &x, bool placement) {
    const char *op = "quantize_int8";
    REQUIRE(dtype_code(x.scalar_type()) >= 0, op, ": x must be bfloat16, float16 or float32");
    REQUIRE(x.dim() > 0, op, ": x must have a dimension");
    const int64_t cols = x.size(-1);
    require_side(op, "the last dimension", cols, 8);
    REQUIRE(x.is_contiguous() || (x.dim() == 2 && x.stride(1) == 1), op, ": x must be contiguous, or 2-D with a contiguous last dimension");
    const int64_t stride = x.is_contiguous() || x.size(0) <= 1 ? cols : x.stride(0);
    REQUIRE(stride >= cols && stride % 8 == 0, op, ": the rows of x are ", stride, " elements apart; supported are multiples of 8 from ", cols, " on");
    if (placement) {
        require_same_device(op, {{"x", &x}});
        require_aligned(op, {{"x", &x}}, 16);
    }
    return stride;
}
std::tuple<Tensor, Tensor> quantize_int8(const Tensor &x) {
    const int64_t stride = check_quantize_int8(x, true);
    const c10::Device dev = x.device();
    const c10::DeviceGuard guard(dev);
    Tensor q = empty(x.sizes(), at::kChar, dev), scale = empty(x.sizes().slice(0, x.dim() - 1), at::kFloat, dev);
    check_status(pmoe_quantize_int8(x.const_data_ptr(), dtype_code(x.scalar_type()), q.data_ptr(), scale.data_ptr<float>(),
                                    x.numel() / x.size(-1), (int)x.size(-1), stride, stream_of(dev)));
    return {q, scale};
}

// ------------------------------------------------------------------------------- weights of 4 bits, whole layers

// A stack of matrices in tiles of 16 x 128 with its scales (see prime_moe_hip.h); `lead`: dimensions in front of a matrix.
struct Int4 {
    int64_t rows = 0, tiles = 0, group = 0;
};
Int4 int4_of(const char *op, const char *name, const Tensor &q, const Tensor &scale, int64_t lead, bool placement) {
    REQUIRE(q.scalar_type() == at::kByte && q.dim() == lead + 3 && q.size(-1) == 1024, op, ": ", name, " must be uint8 of shape (",
            lead ? "E, " : "", "N/16, ceil(K/128), 1024), as quantize_int4 makes it");
    const int64_t per = scale.dim() == lead + 4 ? scale.size(-1) : 0;
    REQUIRE((per == 1 || per == 2 || per == 4) && scale.size(-2) == 16 && scale.sizes().slice(0, lead + 2) == q.sizes().slice(0, lead + 2), op,
            ": the scales of ", name, " must have the shape (", lead ? "E, " : "", "N/16, ceil(K/128), 16, 128/group), as quantize_int4 makes them");
    require_16bit(op, "the scales", scale);
    require_contiguous(op, {{name, &q}, {"the scales", &scale}});
    if (placement) require_aligned(op, {{name, &q}, {"the scales", &scale}}, 16);
    return {q.size(-3) * 16, q.size(-2), 128 / per};
}
void require_columns(const char *op, const char *name, const Int4 &w, int64_t k) {
    REQUIRE(k > 0 && k % w.group == 0 && (k + 127) / 128 == w.tiles, op, ": ", name, " has ", w.tiles, " tiles of 128 columns in groups of ",
            w.group, ", which does not fit ", k, " columns");
}

struct Int4Mm {
    Rows x;
    Int4 w;
};
Int4Mm check_grouped_mm_int4(const Tensor &x, const Tensor &w, const Tensor &w_scale, const std::optional<Tensor> &offsets, bool placement) {
    const char *op = "grouped_mm_int4";
    const bool dense = !offsets.has_value();
    REQUIRE(x.dim() == 2, op, ": x must be 2-D (M, K)");
    require_16bit(op, "x", x);
    const Int4 m = int4_of(op, "w", w, w_scale, dense ? 0 : 1, placement);
    REQUIRE(w_scale.scalar_type() == x.scalar_type(), op, ": x and w_scale must have the same dtype");
    REQUIRE(x.size(0) <= kMostRows, op, ": too many rows");
    require_side(op, "N", m.rows, 16);
    require_side(op, "K", x.size(1), 32);
    require_columns(op, "w", m, x.size(1));
    if (!dense) require_groups(op, *offsets, w.size(0));
    const Int4Mm p{rows_of(op, "x", x, 8), m};
    if (placement) {
        require_same_device(op, {{"x", &x}, {"w", &w}, {"w_scale", &w_scale}});
        if (!dense) require_same_device(op, {{"x", &x}, {"offsets", &*offsets}});
        require_aligned(op, {{"x", &x}}, 16);
    }
    return p;
}
Tensor grouped_mm_int4(const Tensor &x, const Tensor &w, const Tensor &w_scale, const std::optional<Tensor> &offsets) {
    const Int4Mm p = check_grouped_mm_int4(x, w, w_scale, offsets, true);
    const c10::Device dev = x.device();
    const c10::DeviceGuard guard(dev);
    Tensor out = empty({x.size(0), p.w.rows}, x.scalar_type(), dev);
    check_status(pmoe_grouped_mm_int4(x.const_data_ptr(), w.const_data_ptr(), w_scale.const_data_ptr(), out.data_ptr(),
                                      offsets.has_value() ? offsets->const_data_ptr<int32_t>() : nullptr, offsets.has_value() ? (int)w.size(0) : 1,
                                      x.size(0), (int)p.w.rows, (int)x.size(1), (int)p.w.group, p.x.stride, dtype_code(x.scalar_type()),
                                      stream_of(dev)));
    return out;
}

void check_quantize_int4(const Tensor &w, int64_t group, at::ScalarType scale_dtype, bool placement) {
    const char *op = "quantize_int4";
    REQUIRE(dtype_code(w.scalar_type()) >= 0, op, ": w must be bfloat16, float16 or float32");
    REQUIRE(scale_dtype == at::kBFloat16 || scale_dtype == at::kHalf, op, ": scale_dtype must be bfloat16 or float16");
    REQUIRE(w.dim() >= 2, op, ": w must have two dimensions or more");
    REQUIRE(group == 32 || group == 64 || group == 128, op, ": group must be 32, 64 or 128, got ", group);
    require_side(op, "N", w.size(-2), 16);
    require_side(op, "K", w.size(-1), group);
    require_contiguous(op, {{"w", &w}});
    if (placement) {
        require_same_device(op, {{"w", &w}});
        require_aligned(op, {{"w", &w}}, 16);
    }
}
std::tuple<Tensor, Tensor> quantize_int4(const Tensor &w, int64_t group, at::ScalarType scale_dtype) {
    check_quantize_int4(w, group, scale_dtype, true);
    const c10::Device dev = w.device();
    const c10::DeviceGuard guard(dev);
    std::vector<int64_t> size = w.sizes().slice(0, w.dim() - 2).vec();
    const int64_t cols = w.size(-1);
    size.insert(size.end(), {w.size(-2) / 16, (cols + 127) / 128, 1024});
    Tensor q = empty(size, at::kByte, dev);
    size.back() = 16;
    size.push_back(128 / group);
    Tensor scale = empty(size, scale_dtype, dev);
    check_status(pmoe_quantize_int4(w.const_data_ptr(), dtype_code(w.scalar_type()), q.data_ptr(), scale.data_ptr(), dtype_code(scale_dtype),
                                    w.numel() / cols, (int)cols, (int)group, stream_of(dev)));
    return {q, scale};
}

Int4 check_dequantize_int4(const Tensor &q, const Tensor &scale, int64_t columns, bool placement) {
    const char *op = "dequantize_int4";
    REQUIRE(q.dim() >= 3, op, ": q must be uint8 of shape (..., N/16, ceil(K/128), 1024), as quantize_int4 makes it");
    const Int4 w = int4_of(op, "q", q, scale, q.dim() - 3, placement);
    require_side(op, "columns", columns, w.group);
    require_columns(op, "q", w, columns);
    if (placement) require_same_device(op, {{"q", &q}, {"scale", &scale}});
    return w;
}
Tensor dequantize_int4(const Tensor &q, const Tensor &scale, int64_t columns) {
    const Int4 w = check_dequantize_int4(q, scale, columns, true);
    const c10::Device dev = q.device();
    const c10::DeviceGuard guard(dev);
    std::vector<int64_t> size = q.sizes().slice(0, q.dim() - 3).vec();
    size.insert(size.end(), {w.rows, columns});
    Tensor out = empty(size, scale.scalar_type(), dev);
    check_status(pmoe_dequantize_int4(q.const_data_ptr(), scale.const_data_ptr(), out.data_ptr(), dtype_code(scale.scalar_type()),
                                      out.numel() / columns, (int)columns, (int)w.group, stream_of(dev)));
    return out;
}

struct Layer {
    const Tensor &x, &gate, &w1, &w2;
    const Tensor *w1_scale, *w2_scale;  // null: weights of 16 bits
    int64_t top_k;
    const std::optional<Tensor> &bias;
};
struct LayerSizes {
    int64_t hidden, group;  // columns of the activation
};
constexpr int64_t kMostTokens = 16, kMostExperts = 512, kMostTopK = 32;
LayerSizes check_layer(const char *op, const Layer &l, bool placement) {
    REQUIRE(l.x.dim() == 2 && l.gate.dim() == 2 && l.gate.size(1) == l.x.size(1), op, ": x must be 2-D (T, K), gate 2-D (E, K)");
    const int64_t T = l.x.size(0), K = l.x.size(1), E = l.gate.size(0);
    require_16bit(op, "x", l.x);
    REQUIRE(l.gate.scalar_type() == l.x.scalar_type(), op, ": x and gate must have the same dtype");
    REQUIRE(T <= kMostTokens, op, " takes up to ", kMostTokens, " tokens, got ", T, " (more: ",
            l.w1_scale != nullptr ? "route, expert_offsets and grouped_mm_int4, or grouped_mm on what dequantize_int4 returns"
            : l.x.scalar_type() == at::kHalf ? "route, expert_offsets and grouped_mm" : "route and fused_moe_bf16", ")");
    REQUIRE(E > 0 && E <= kMostExperts, op, " supports 1..", kMostExperts, " experts, got ", E);
    REQUIRE(l.top_k > 0 && l.top_k <= std::min(kMostTopK, E), op, ": top_k must be in 1..min(", kMostTopK, ", E), got ", l.top_k);
    LayerSizes z{0, 0};
    if (l.w1_scale != nullptr) {
        const Int4 up = int4_of(op, "w1", l.w1, *l.w1_scale, 1, placement), down = int4_of(op, "w2", l.w2, *l.w2_scale, 1, placement);
        z = {up.rows / 2, up.group};
        REQUIRE(up.group == down.group, op, ": w1 and w2 must have groups of the same size");
        REQUIRE(l.w1_scale->scalar_type() == l.x.scalar_type() && l.w2_scale->scalar_type() == l.x.scalar_type(), op, ": x and the scales must have the same dtype");
        REQUIRE(l.w1.size(0) == E && l.w2.size(0) == E, op, ": w1 and w2 must hold the experts of gate (", E, ")");
        REQUIRE(up.rows % 32 == 0, op, ": the rows of w1, 2H, must be a multiple of 32, got ", up.rows);
        require_columns(op, "w1", up, K);
        require_columns(op, "w2", down, z.hidden);
        REQUIRE(down.rows == K, op, ": w2 must have K (", K, ") rows, got ", down.rows);
    } else {
        REQUIRE(l.w1.dim() == 3 && l.w1.size(0) == E && l.w1.size(2) == K && l.w1.size(1) % 2 == 0, op, ": w1 must have shape (E, 2H, K)");
        z.hidden = l.w1.size(1) / 2;
        REQUIRE(l.w2.dim() == 3 && l.w2.size(0) == E && l.w2.size(1) == K && l.w2.size(2) == z.hidden, op, ": w2 must have shape (E, K, H)");
        REQUIRE(l.w1.scalar_type() == l.x.scalar_type() && l.w2.scalar_type() == l.x.scalar_type(), op, ": x, w1 and w2 must have the same dtype");
        require_contiguous(op, {{"w1", &l.w1}, {"w2", &l.w2}});
    }
    REQUIRE(K > 0 && K % 8 == 0 && K <= 1 << 20 && z.hidden > 0 && z.hidden % 8 == 0 && z.hidden <= 1 << 20, op, ": K (", K, ") and H (", z.hidden,
            ") must be positive multiples of 8 up to 2^20");
    require_contiguous(op, {{"x", &l.x}, {"gate", &l.gate}});
    if (l.bias.has_value())
        REQUIRE(l.bias->scalar_type() == at::kFloat && l.bias->is_contiguous() && l.bias->dim() == 1 && l.bias->size(0) == E, op,
                ": bias must be a contiguous float32 (E,) tensor");
    if (placement) {
        require_same_device(op, {{"x", &l.x}, {"gate", &l.gate}, {"w1", &l.w1}, {"w2", &l.w2}});
        if (l.w1_scale != nullptr) require_same_device(op, {{"x", &l.x}, {"w1_scale", l.w1_scale}, {"w2_scale", l.w2_scale}});
        if (l.bias.has_value()) require_same_device(op, {{"x", &l.x}, {"bias", &*l.bias}});
        require_aligned(op, {{"x", &l.x}, {"gate", &l.gate}, {"w1", &l.w1}, {"w2", &l.w2}}, 16);
    }
    return z;
}
std::tuple<Tensor, Tensor, Tensor> run_layer(const char *op, const Layer &l) {
    const LayerSizes z = check_layer(op, l, true);
    const c10::Device dev = l.x.device();
    const c10::DeviceGuard guard(dev);
    const int64_t T = l.x.size(0), E = l.gate.size(0);
    Tensor out = empty(l.x.sizes(), l.x.scalar_type(), dev), ids = empty({T, l.top_k}, at::kInt, dev), weights = empty({T, l.top_k}, at::kFloat, dev);
    const Tensor ws = workspace(pmoe_moe_layer_workspace_bytes((int)T, (int)z.hidden, (int)E, (int)l.top_k), dev);
    check_status(pmoe_moe_layer(l.x.const_data_ptr(), l.gate.const_data_ptr(), l.bias.has_value() ? l.bias->const_data_ptr<float>() : nullptr,
                                l.w1.const_data_ptr(), l.w1_scale ? l.w1_scale->const_data_ptr() : nullptr, l.w2.const_data_ptr(),
                                l.w2_scale ? l.w2_scale->const_data_ptr() : nullptr, (int)z.group, out.data_ptr(), ids.data_ptr<int32_t>(),
                                weights.data_ptr<float>(), (int)T, (int)l.x.size(1), (int)z.hidden, (int)E, (int)l.top_k,
                                dtype_code(l.x.scalar_type()), ws.data_ptr(), (size_t)ws.numel(), stream_of(dev)));
    return {out, ids, weights};
}
std::tuple<Tensor, Tensor, Tensor> moe_layer(const Tensor &x, const Tensor &gate, const Tensor &w1, const Tensor &w2, int64_t top_k,
                                             const std::optional<Tensor> &bias) {
    return run_layer("moe_layer", {x, gate, w1, w2, nullptr, nullptr, top_k, bias});
}
std::tuple<Tensor, Tensor, Tensor> moe_layer_int4(const Tensor &x, const Tensor &gate, const Tensor &w1, const Tensor &w1_scale, const Tensor &w2,
                                                  const Tensor &w2_scale, int64_t top_k, const std::optional<Tensor> &bias) {
    return run_layer("moe_layer_int4", {x, gate, w1, w2, &w1_scale, &w2_scale, top_k, bias});
}

void check_expert_offsets(const Tensor &expert_ids, const Tensor &total, int64_t num_experts, bool placement) {
    const char *op = "expert_offsets";
    const Arg ae{"expert_ids", &expert_ids}, at_{"num_tokens_post_padded", &total};
    require_dtype(op, {ae, at_}, at::kInt, "int32");
    require_contiguous(op, {ae, at_});
    REQUIRE(num_experts > 0 && num_experts <= kMostGroups, op, " supports 1..", kMostGroups, " experts, got ", num_experts);
    REQUIRE(expert_ids.numel() <= kMostRows, op, ": too many rows");
    REQUIRE(total.numel() >= 1, op, ": num_tokens_post_padded is empty");
    if (placement) require_same_device(op, {ae, at_});
}
Tensor expert_offsets(const Tensor &expert_ids, const Tensor &total, int64_t num_experts) {
    check_expert_offsets(expert_ids, total, num_experts, true);
    const c10::Device dev = expert_ids.device();
    const c10::DeviceGuard guard(dev);
    Tensor offsets = empty({num_experts}, at::kInt, dev);
    check_status(pmoe_expert_offsets(expert_ids.const_data_ptr<int32_t>(), total.const_data_ptr<int32_t>(), offsets.data_ptr<int32_t>(),
                                     (int)expert_ids.numel(), (int)num_experts, stream_of(dev)));
    return offsets;
}

// ------------------------------------------------------------------------------- helpers that are not ops

std::tuple<Tensor, Tensor> quantize_mx(const Tensor &t) {
    REQUIRE(t.is_cuda(), "quantize_mx: a GPU tensor is required");
    REQUIRE(t.scalar_type() == at::kBFloat16, "quantize_mx: bfloat16 input required");
    REQUIRE(t.is_contiguous(), "quantize_mx: input must be contiguous");
    REQUIRE(t.dim() > 0, "quantize_mx: input must have a dimension");
    const int64_t cols = t.size(-1);
    REQUIRE(cols > 0 && cols % 32 == 0, "quantize_mx: last dim ", cols, " must be a multiple of 32");
    const c10::Device dev = t.device();
    const c10::DeviceGuard guard(dev);
    Tensor q = empty(t.sizes(), at::kFloat8_e4m3fn, dev);
    std::vector<int64_t> size = t.sizes().vec();
    size.back() = cols / 32;
    Tensor s = empty(size, at::kFloat8_e8m0fnu, dev);
    check_status(pmoe_quantize_mx(t.const_data_ptr(), q.data_ptr(), s.data_ptr(), t.numel() / cols, (int)cols, stream_of(dev)));
    return {q, s};
}

std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> route(const Tensor &logits, int64_t top_k, int64_t block_m, int64_t bpc,
                                                         const std::optional<Tensor> &bias) {
    REQUIRE(logits.is_cuda(), "route: logits must be a GPU tensor, got device ", logits.device());
    REQUIRE(logits.dim() == 2 && logits.is_contiguous(), "route: logits must be a contiguous (T, E) tensor");
    REQUIRE(logits.scalar_type() == at::kFloat || logits.scalar_type() == at::kBFloat16, "route: logits must be float32 or bfloat16");
    const int64_t T = logits.size(0), E = logits.size(1);
    REQUIRE(E > 0 && E <= 1024, "route supports 1..1024 experts, got ", E);
    REQUIRE(top_k > 0 && top_k <= std::min<int64_t>(32, E), "route: top_k must be in 1..min(32, E), got ", top_k);
    REQUIRE(block_m > 0 && bpc > 0, "route: block_m and bpc must be positive");
    const c10::Device dev = logits.device();
    if (bias.has_value())
        REQUIRE(bias->device() == dev && bias->scalar_type() == at::kFloat && bias->is_contiguous() && bias->numel() == E,
                "route: bias must be a contiguous float32 (E,) tensor on the device of logits");
    const c10::DeviceGuard guard(dev);
    const int64_t n = T * top_k;
    const AlignSizes sz(n, E, block_m, bpc);
    Tensor topk_ids = empty({T, top_k}, at::kInt, dev), topk_weights = empty({T, top_k}, at::kFloat, dev);
    Schedule s(sz, n, E, dev);
    check_status(pmoe_route(logits.const_data_ptr(), logits.scalar_type() == at::kFloat ? PMOE_DTYPE_F32 : PMOE_DTYPE_BF16,
                            bias.has_value() ? bias->const_data_ptr<float>() : nullptr, topk_ids.data_ptr<int32_t>(),
                            topk_weights.data_ptr<float>(), s.sorted_token_ids.data_ptr<int32_t>(),
                            s.expert_ids.data_ptr<int32_t>(), s.num_tokens_post_padded.data_ptr<int32_t>(), (int)T, (int)E,
                            (int)top_k, (int)block_m, (int)sz.pad_to, (int)sz.max_padded, (int)sz.max_blocks, s.ws_ptr(),
                            s.ws_bytes, stream_of(dev)));
    return {topk_ids, topk_weights, s.sorted_token_ids, s.expert_ids, s.num_tokens_post_padded};
}

}  // namespace

TORCH_LIBRARY_IMPL(prime_moe, CUDA, m) {
    m.impl("moe_align", &moe_align);
    m.impl("fused_moe_bf16", &fused_moe_bf16);
    m.impl("fused_moe_mxfp8", &fused_moe_mxfp8);
    m.impl("grouped_mm", &grouped_mm);
    m.impl("grouped_mm_wgrad", &grouped_mm_wgrad);
    m.impl("grouped_mm_int8", &grouped_mm_int8);
    m.impl("quantize_int8", &quantize_int8);
    m.impl("expert_offsets", &expert_offsets);
    m.impl("grouped_mm_int4", &grouped_mm_int4);
    m.impl("quantize_int4", &quantize_int4);
    m.impl("dequantize_int4", &dequantize_int4);
    m.impl("moe_layer", &moe_layer);
    m.impl("moe_layer_int4", &moe_layer_int4);
}

TORCH_LIBRARY_IMPL(prime_moe, AutogradCUDA, m) {
    m.impl("grouped_mm", &grouped_mm_autograd);
    m.impl("grouped_mm_wgrad", &grouped_mm_wgrad_autograd);
}

PYBIND11_MODULE(_torch_ops, m) {
    namespace py = pybind11;
    const auto nogil = py::call_guard<py::gil_scoped_release>();
    m.def("validate_align", &validate_align, nogil);
    m.def("validate_bf16", &validate_bf16, nogil);
    m.def("validate_mxfp8", &validate_mxfp8, nogil);
    m.def("validate_grouped_mm", [](const Tensor &x, const Tensor &w, const Tensor &o) { check_grouped_mm(x, w, o, false); }, nogil);
    m.def("validate_grouped_mm_wgrad", [](const Tensor &dy, const Tensor &x, const Tensor &o) { check_grouped_mm_wgrad(dy, x, o, false); }, nogil);
    m.def("validate_grouped_mm_int8", [](const Tensor &x, const Tensor &w, const Tensor &xs, const Tensor &ws, const std::optional<Tensor> &o,
                                         at::ScalarType t) { check_grouped_mm_int8(x, w, xs, ws, o, t, false); }, nogil);
    m.def("validate_quantize_int8", [](const Tensor &x) { check_quantize_int8(x, false); }, nogil);
    m.def("validate_grouped_mm_int4", [](const Tensor &x, const Tensor &w, const Tensor &ws, const std::optional<Tensor> &o) {
        check_grouped_mm_int4(x, w, ws, o, false); }, nogil);
    m.def("validate_quantize_int4", [](const Tensor &w, int64_t g, at::ScalarType t) { check_quantize_int4(w, g, t, false); }, nogil);
    m.def("validate_dequantize_int4", [](const Tensor &q, const Tensor &s, int64_t c) { check_dequantize_int4(q, s, c, false); }, nogil);
    m.def("validate_moe_layer", [](const Tensor &x, const Tensor &g, const Tensor &w1, const Tensor &w2, int64_t k, const std::optional<Tensor> &b) {
        check_layer("moe_layer", {x, g, w1, w2, nullptr, nullptr, k, b}, false); }, nogil);
    m.def("validate_moe_layer_int4", [](const Tensor &x, const Tensor &g, const Tensor &w1, const Tensor &s1, const Tensor &w2, const Tensor &s2,
                                        int64_t k, const std::optional<Tensor> &b) { check_layer("moe_layer_int4", {x, g, w1, w2, &s1, &s2, k, b}, false); }, nogil);
    m.def("validate_expert_offsets", [](const Tensor &e, const Tensor &n, int64_t k) { check_expert_offsets(e, n, k, false); }, nogil);
    m.def("quantize_mx", &quantize_mx, nogil);
    m.def("route", &route, nogil);
}
