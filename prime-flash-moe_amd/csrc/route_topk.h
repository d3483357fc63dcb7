// Top-k and softmax of one token's gate logits by one wave, gfx950.
//
// Lane l holds experts l, l + 64, l + 128, ... (EPL of them) as order-preserving 32-bit keys.
// A round takes the largest key (a maximum over the lane's keys, then over the wave by DPP moves: register to
// register, where shuffles through LDS cost ten times the latency), finds the lowest expert that holds it with a ballot
// per key register, and retires it.  The softmax of the top_k winners is computed by the lanes that keep them.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace pmoe {
namespace route {

__device__ __forceinline__ float load_logit(const float *p, int64_t i) { return p[i]; }
__device__ __forceinline__ float load_logit(const uint16_t *p, int64_t i) { return __uint_as_float((uint32_t)p[i] << 16); }

// Monotone map float -> uint32 (a < b <=> key(a) < key(b)); -0 counts as +0, NaN lands above +inf.
__device__ __forceinline__ uint32_t order_key(float v) {
    v += 0.0f;  // -0 -> +0
    uint32_t u = __float_as_uint(v);
    if (v != v) u = 0x7fffffffu;  // every NaN: the largest positive pattern
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
    const uint32_t u = (k & 0x80000000u) ? (k & 0x7fffffffu) : ~k;
    return __uint_as_float(u);
}

// Maximum over the wave, in every lane.  Row shifts by 1, 2, 4, 8 and the two row broadcasts leave it in lane 63.
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
#define PMOE_DPP_MAX(ctrl, rows) v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, ctrl, rows, 0xf, false))
    PMOE_DPP_MAX(0x111, 0xf);  // row_shr:1
    PMOE_DPP_MAX(0x112, 0xf);  // row_shr:2
    PMOE_DPP_MAX(0x114, 0xf);  // row_shr:4
    PMOE_DPP_MAX(0x118, 0xf);  // row_shr:8
    PMOE_DPP_MAX(0x142, 0xa);  // row_bcast:15
    PMOE_DPP_MAX(0x143, 0xc);  // row_bcast:31
#undef PMOE_DPP_MAX
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}

// Top-k and softmax of token t; lane r < top_k returns winner r (id, weight).
template <int EPL, typename T>
__device__ __forceinline__ void topk_of_token(const T *__restrict__ logits, const float *__restrict__ bias, int64_t t, int E, int top_k,
                                              int lane, int &my_id, float &my_weight) {
    uint32_t key[EPL];
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
        const int e = lane + 64 * j;
        key[j] = 0u;  // below every real key: never selected before a real element
        if (e < E) {
            float v = load_logit(logits, t * E + e);
            if (bias != nullptr) v += bias[e];
            key[j] = order_key(v);
        }
    }
    float my_val = 0.f;  // lane r keeps the value of winner r
    my_id = 0;
    for (int r = 0; r < top_k; ++r) {
        uint32_t best = key[0];
#pragma unroll
        for (int j = 1; j < EPL; ++j) best = max(best, key[j]);
        best = wave_max(best);
        int win = -1;
#pragma unroll
        for (int j = EPL - 1; j >= 0; --j) {
            const uint64_t m = __ballot(key[j] == best);
            if (m != 0) win = 64 * j + __builtin_ctzll(m);
        }
#pragma unroll
        for (int j = 0; j < EPL; ++j)
            if (lane + 64 * j == win) key[j] = 0u;
        if (lane == r) {
            my_val = key_value(best);
            my_id = win;
        }
    }
    // softmax over the winners: lanes 0 .. top_k - 1 hold them, winner 0 is the maximum
    const float vmax = __shfl(my_val, 0, 64);
    const float ex = lane < top_k ? expf(my_val - vmax) : 0.f;
    float sum = ex;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) sum += __shfl_xor(sum, d, 64);
    my_weight = ex / sum;
}

}  // namespace route
}  // namespace pmoe
