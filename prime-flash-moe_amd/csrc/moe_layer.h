// A whole layer of experts for up to 16 tokens, gfx950: what its kernels (moe_layer.hip) are made of.
//
//   l[t][e] = x[t] . gate[e] (+ bias[e]);  S(t): the top_k largest, ties to the lower index;  a[t][.] = softmax over S(t)
//   out[t]  = sum over e in S(t) of a[t][e] W2[e] (silu(G[e] x[t]) * (U[e] x[t])),  G: rows 0 .. H - 1 of W1[e], U: rows H .. 2H - 1
//
// With so few tokens most experts have a row or two: the stream of the touched experts' weights from HBM bounds the large
// layers (16 tokens on 128 experts of 2048 x 768, 778 MB: 138 us, 5.6 TB/s), a chain of latencies the small ones (one token on
// them, 76 MB: 22.7 us, of which the logits take 2, the next kernel's start 1, the plan 2.5, the up jobs and the wait for the last 9,
// the down projection 6).  Nothing is sorted or padded: a workgroup finds the touched experts and their tokens by itself, from the
// logits, in LDS.  Two kernels: the logits, and everything else by resident workgroups that take up jobs from queues and then go
// over to their part of the down projection.  (A kernel for each projection: 27.7 us for one token, 225 for 16: the tails of the
// first were idle, and the second began with its weights' latency.)
//
// Weights of 16 bits, rows of (E, 2H, K) and (E, K, H): sixteen lanes share a weight row, a step of theirs is 128 elements, 256
// contiguous bytes, straight into registers, and a lane multiplies its eight with those of up to four tokens (eight in jobs of four columns) by
// dot products of two elements with fp32 sums.  An expert with more rows has its weights loaded again for the next ones, which is what
// bounds layers of few small experts (16 tokens, 4 of 8 experts of 4096 x 256: 44 us for 50 MB).  Weights of 4 bits: int4_tile.h.
//
// The activation keeps the range of fp32 and 16 bits of mantissa or more, so that the output is rounded once, in 32 bits a value.  With fp16
// weights of 16 bits it is fp32: an instruction multiplies half of a register of fp16 with fp32, as many of them as dot products of two halves.
// Otherwise it is the sum of two bf16 numbers, the rounded value and the rounded rest, of which the down projection
// multiplies both, at two dot products (or two rows of a matrix instruction that has rows to spare) instead of one; integers of 4 bits are
// whole in bf16 whatever the layer's type is.  (Two fp16 numbers end at 65504, where activations of fp16 layers do not, and lose the rest's bits
// below 2^-9.)
#pragma once
#include "int4_tile.h"
#include "route_topk.h"

namespace pmoe {
namespace layer {

using gmm::Bf16;
using gmm::F16;
using int4::f32x4;
using int4::Num;

constexpr int kMaxTokens = 16, kMaxTopK = 32, kMaxPairs = kMaxTokens * kMaxTopK, kMaxExperts = 512;
constexpr int kThreads = 512, kWaves = 8, kWavesLog = 3;
constexpr int kUpCols = 16;       // activation columns that waves share the contraction of, at most
constexpr int kMaxGroups = 512;   // workgroups at most
constexpr int64_t kMostTries = 1 << 24;  // of a wait, about a microsecond each: then the outputs are NaN

// Queues of the up jobs, a line of 128 bytes each (an atomic of the device takes 11 ns per address).
constexpr int kQueues = 8;  // as many as XCDs, which workgroups go round
struct Sync {
    int32_t ticket[kQueues][32];
    int32_t arrived[kMaxGroups];  // of the strip of out that begins with this workgroup: steps of its contraction that are done
};
struct Args {
    Sync *sync;
    const char *x, *gate, *w1, *w1_scale, *w2, *w2_scale;
    const float *bias;
    char *out;
    int32_t *topk_ids;
    float *topk_weights;
    float *logits;  // (T, E)
    char *act;      // [pair][2][act_pitch bytes]: values, rests; or whole ones: columns 8 c .. + 3, columns 8 c + 4 .. + 7 behind byte 16 c
    int act_pitch;
    float *shares;  // [workgroup][2: of its first strip, of its last one][token][column]: sums of workgroups that share a strip of out
    int T, K, H, E, top_k;
    int up_cols;    // columns of an up job: 4, 8, 12 or 16, or 16 << up_log (weights of 4 bits)
    int up_log;     // 8 >> up_log waves share the contraction of 16 columns
    int down_groups;  // workgroups of the down projection
    int split;        // whether they share strips of out
};

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
template <class T>
__device__ __forceinline__ float dot2(int a, int b, float c);
template <>
__device__ __forceinline__ float dot2<Bf16>(int a, int b, float c) {
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, a), __builtin_bit_cast(bf16x2, b), c, false);
}
template <>
__device__ __forceinline__ float dot2<F16>(int a, int b, float c) {
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, a), __builtin_bit_cast(f16x2, b), c, false);
}

// Sum over the 16 lanes of a row, in all of them.
__device__ __forceinline__ float row_sum(float v) {
#define PMOE_DPP_ADD(ctrl) v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), ctrl, 0xf, 0xf, true))
    PMOE_DPP_ADD(0xb1);   // quad_perm [1, 0, 3, 2]
    PMOE_DPP_ADD(0x4e);   // quad_perm [2, 3, 0, 1]
    PMOE_DPP_ADD(0x141);  // row_half_mirror
    PMOE_DPP_ADD(0x140);  // row_mirror
#undef PMOE_DPP_ADD
    return v;
}

// What a word of the activation holds until its up job has written it: a NaN, or two, that no job writes.  So a word says by
// itself whether it is there, and where a cached one says that it is not, memory is asked again: nothing else is needed between
// the up jobs and the down jobs, no counter behind the stores, no cache to be emptied.
constexpr uint32_t kAbsent = 0xffffffffu;
struct Arrival {
    static constexpr bool kWaits = true;
    int *failed;  // LDS
    int64_t tries = 0;
    // Whether this wave has to load again.
    __device__ __forceinline__ bool operator()(uint32_t most) {
        if (__ballot(most == kAbsent) == 0) return false;
        if (++tries > kMostTries || __hip_atomic_load(failed, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP) != 0) {
            __hip_atomic_store(failed, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
            return false;
        }
        __builtin_amdgcn_s_sleep(2);
        return true;
    }
};

// acc[q][n] += this lane's share of a weight row times row n of x: steps s0 .. s1 - 1 of 128 elements.  `w[q]` begins four weight rows,
// `pitch` bytes apart, of which a lane has number lane / 16, `last` at most; row n begins at byte xo[n] of `x`, which holds `x_bytes`
// (all wave-uniform).  `k`: elements of a row, a multiple of 8; nothing is read behind them.  Only the first `live` of the Q are there.  The
// weights of S steps are in flight together, of x SX steps of NX rows.  WHOLE: two rows of x are one of fp32, the first four of every eight
// columns and the others (T is F16).  wait: see int4::dots.
template <class T, int Q, int N, int S, int SX, int NX = N, bool WHOLE = false, class Wait = int4::NoWait>
__device__ __forceinline__ void row_dots(float (&acc)[Q][N], const char *const (&w)[Q], int pitch, const char *x, uint32_t x_bytes, const uint32_t (&xo)[N], int s0,
                                         int s1, int k, int live = Q, int last = 3, Wait wait = {}) {
    const int lane = threadIdx.x & 63;
    const uint32_t own = (lane & 15) * 16, wo = (uint32_t)min(lane >> 4, last) * (uint32_t)pitch + own;
    // (buffer loads take a step's offset from a scalar register, where pointers of their own per step fill the vector registers)
    int4::Buffer wb[Q];
#pragma unroll
    for (int q = 0; q < Q; ++q)
        if (q < live) wb[q] = int4::buffer(w[q], 4u * (uint32_t)pitch);
    const int4::Buffer xb = int4::buffer(x, x_bytes);
    auto multiply = [&](const i32x4 (&wv)[Q], const i32x4 (&xv)[NX], int n0) {
        if constexpr (WHOLE) {
            // (by columns, so that no sum waits for the one before it)
#pragma unroll
            for (int d = 0; d < 4; ++d)
#pragma unroll
                for (int q = 0; q < Q; ++q)
                    if (q < live)
#pragma unroll
                        for (int n = 0; n < NX; ++n) {
                            const int word = wv[q][n % 2 * 2 + d / 2];  // (a value: of an element of a vector the cast would take the first)
                            const f16x2 pair = __builtin_bit_cast(f16x2, word);
                            acc[q][n0 + n] = fmaf((float)pair[d % 2], __int_as_float(xv[n][d]), acc[q][n0 + n]);
                        }
            return;
        }
#pragma unroll
        for (int q = 0; q < Q; ++q)
            if (q < live)
#pragma unroll
                for (int n = 0; n < NX; ++n) {
#pragma unroll
                    for (int d = 0; d < 4; ++d) acc[q][n0 + n] = dot2<T>(wv[q][d], xv[n][d], acc[q][n0 + n]);
                }
    };
    const int whole = min(s1, k / 128);
    for (int s = s0; s < whole; s += S) {
        i32x4 wv[S][Q];
#pragma unroll
        for (int i = 0; i < S; ++i)
            if (s + i < whole) {
#pragma unroll
                for (int q = 0; q < Q; ++q)
                    if (q < live) wv[i][q] = int4::load_once(wb[q], wo, (s + i) * 256);
            }
#pragma unroll
        for (int i0 = 0; i0 < S; i0 += SX)
            if (s + i0 < whole) {
#pragma unroll
                for (int n0 = 0; n0 < N; n0 += NX) {
                    i32x4 xv[SX][NX];
#pragma unroll
                    for (int i = 0; i < SX; ++i)
                        if (s + i0 + i < whole) {
#pragma unroll
                            for (int n = 0; n < NX; ++n) xv[i][n] = int4::load(xb, own, xo[n0 + n] + (s + i0 + i) * 256);
                        }
                    if constexpr (Wait::kWaits)
                        for (;;) {
                            uint32_t most = 0;
#pragma unroll
                            for (int i = 0; i < SX; ++i)
                                if (s + i0 + i < whole) {
#pragma unroll
                                    for (int n = 0; n < NX; ++n)
#pragma unroll
                                        for (int d = 0; d < 4; ++d) most = max(most, (uint32_t)xv[i][n][d]);
                                }
                            if (!wait(most)) break;
#pragma unroll
                            for (int i = 0; i < SX; ++i)
                                if (s + i0 + i < whole) {
#pragma unroll
                                    for (int n = 0; n < NX; ++n) xv[i][n] = int4::load_now(xb, own, xo[n0 + n] + (s + i0 + i) * 256);
                                }
                        }
#pragma unroll
                    for (int i = 0; i < SX; ++i)
                        if (s + i0 + i < whole) multiply(wv[i0 + i], xv[i], n0);
                }
            }
    }
    if (s1 > k / 128 && s0 < s1 && (lane & 15) * 8 < k % 128) {  // a step in part (the last one)
        i32x4 wv[Q];
#pragma unroll
        for (int q = 0; q < Q; ++q)
            if (q < live) wv[q] = int4::load_once(wb[q], wo, k / 128 * 256);
#pragma unroll
        for (int n0 = 0; n0 < N; n0 += NX) {
            i32x4 xv[NX];
#pragma unroll
            for (int n = 0; n < NX; ++n) xv[n] = int4::load(xb, own, xo[n0 + n] + k / 128 * 256);
            if constexpr (Wait::kWaits)
                for (;;) {
                    uint32_t most = 0;
#pragma unroll
                    for (int n = 0; n < NX; ++n)
#pragma unroll
                        for (int d = 0; d < 4; ++d) most = max(most, (uint32_t)xv[n][d]);
                    if (!wait(most)) break;
#pragma unroll
                    for (int n = 0; n < NX; ++n) xv[n] = int4::load_now(xb, own, xo[n0 + n] + k / 128 * 256);
                }
            multiply(wv, xv, n0);
        }
    }
}

// The touched experts and their tokens, by every workgroup for itself.
struct Plan {
    int n;                              // touched experts
    int job;                            // the workgroup's
    int failed;                         // a wait was given up
    uint32_t touched[kMaxExperts / 32];
    uint16_t expert[kMaxPairs];
    uint32_t tokens[kMaxPairs];         // bit t: token t is the expert's
    uint8_t slot[kMaxPairs][kMaxTokens];  // which of the token's top_k the expert is
    float weight[kMaxPairs];            // of pair t top_k + r
    int16_t id[kMaxPairs];
    __attribute__((aligned(16))) uint32_t key[kMaxExperts];
    int32_t rank[kMaxExperts];
};

// One token: top-k by ranks.  A thread counts, for one expert, how many of a part of the logits are in front of it (rounds of a wave, one
// winner after the other, take 0.7 us longer).  Every chosen expert is the token's, in the order of the ranks.
__device__ __forceinline__ void plan_one(const Args &a, Plan &p, bool publish) {
    const int tid = threadIdx.x, log = a.E <= 64 ? 6 : a.E <= 128 ? 7 : a.E <= 256 ? 8 : 9, stride = 1 << log;
    const int parts_log = min(9 - log, log - 2), e = tid & (stride - 1), part = tid >> log;  // (a part is a multiple of four)
    if (tid == 0) p.failed = 0, p.n = a.top_k;
    if (tid < stride) {
        uint32_t key = 0;
        if (tid < a.E) {
            float v = a.logits[tid];
            if (a.bias != nullptr) v += a.bias[tid];
            key = route::order_key(v);
        }
        p.key[tid] = key;
        p.rank[tid] = 0;
    }
    __syncthreads();
    if (part < 1 << parts_log && e < a.E) {
        const uint32_t mine = p.key[e];
        const int each = stride >> 2 >> parts_log;
        int before = 0;
#pragma unroll 2
        for (int i = part * each; i < (part + 1) * each; ++i) {
            const i32x4 k = reinterpret_cast<const i32x4 *>(p.key)[i];
#pragma unroll
            for (int j = 0; j < 4; ++j) before += (uint32_t)k[j] > mine || ((uint32_t)k[j] == mine && 4 * i + j < e);
        }
        atomicAdd(&p.rank[e], before);
    }
    __syncthreads();
    if (tid < a.E && p.rank[tid] < a.top_k) {
        p.expert[p.rank[tid]] = (uint16_t)tid;
        p.weight[p.rank[tid]] = route::key_value(p.key[tid]);
    }
    __syncthreads();
    if (tid < 64) {  // softmax over the winners, the first of which is the largest; read behind a later barrier
        const float v = tid < a.top_k ? p.weight[tid] : 0.f, most = __int_as_float(gmm::uniform(__float_as_int(v)));
        const float ex = tid < a.top_k ? expf(v - most) : 0.f;
        float sum = row_sum(ex);
        sum += __shfl_xor(sum, 16, 64);
        if (tid < a.top_k) {
            p.weight[tid] = ex / sum;
            if (publish) {
                a.topk_ids[tid] = p.expert[tid];
                a.topk_weights[tid] = ex / sum;
            }
        }
    }
}

template <bool ONE>
__device__ __forceinline__ void find_plan(const Args &a, Plan &p, bool publish) {
    if constexpr (ONE) {
        plan_one(a, p, publish);
        return;
    }
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n_pairs = a.T * a.top_k;
    if (tid == 0) p.failed = 0;
    if (tid < kMaxExperts / 32) p.touched[tid] = 0;
    if (tid < kMaxPairs) p.tokens[tid] = 0;
    for (int t = wave; t < a.T; t += kWaves) {
        int id;
        float w;
        if (a.E <= 64) route::topk_of_token<1, float>(a.logits, a.bias, t, a.E, a.top_k, lane, id, w);
        else if (a.E <= 128) route::topk_of_token<2, float>(a.logits, a.bias, t, a.E, a.top_k, lane, id, w);
        else if (a.E <= 256) route::topk_of_token<4, float>(a.logits, a.bias, t, a.E, a.top_k, lane, id, w);
        else route::topk_of_token<8, float>(a.logits, a.bias, t, a.E, a.top_k, lane, id, w);
        if (lane < a.top_k) {
            p.id[t * a.top_k + lane] = (int16_t)id;
            p.weight[t * a.top_k + lane] = w;
            if (publish) {
                a.topk_ids[t * a.top_k + lane] = id;
                a.topk_weights[t * a.top_k + lane] = w;
            }
        }
    }
    __syncthreads();
    if (tid < n_pairs) atomicOr(&p.touched[p.id[tid] >> 5], 1u << (p.id[tid] & 31));
    __syncthreads();
    if (tid < n_pairs) {
        const int e = p.id[tid], t = tid / a.top_k;
        int u = 0;
        for (int i = 0; i < e >> 5; ++i) u += __popc(p.touched[i]);
        u += __popc(p.touched[e >> 5] & ((1u << (e & 31)) - 1u));
        p.expert[u] = (uint16_t)e;
        p.slot[u][t] = (uint8_t)(tid - t * a.top_k);
        atomicOr(&p.tokens[u], 1u << t);
    }
    if (wave == kWaves - 1) {
        int n = lane < kMaxExperts / 32 ? __popc(p.touched[lane]) : 0;
#pragma unroll
        for (int d = 8; d > 0; d /= 2) n += __shfl_xor(n, d, 64);
        if (lane == 0) p.n = n;
    }
    __syncthreads();
}

// Token of an expert's row j (the j-th set bit).
__device__ __forceinline__ int token_of(uint32_t tokens, int j) {
    for (int i = 0; i < j; ++i) tokens &= tokens - 1;
    return __builtin_ctz(tokens);
}

// The tokens of an expert, the token of row j, and what number of its experts this is.  ONE: the layer has one token.
template <bool ONE>
__device__ __forceinline__ uint32_t tokens_of(const Plan &p, int u) {
    return ONE ? 1u : (uint32_t)gmm::uniform((int)p.tokens[u]);
}
template <bool ONE>
__device__ __forceinline__ int pair_of(const Args &a, const Plan &p, int u, int t) {
    return ONE ? u : t * a.top_k + p.slot[u][t];
}

// The rows of an expert one, two, four or eight (MOST) at a time: f(integral N, first row).
// (Eight in jobs of four columns: 9 tokens, 4 of 8 experts of 4096 x 256, 30.7 us instead of 34.0; other jobs lack the registers.)
template <bool ONE, int MOST, class F>
__device__ __forceinline__ void by_rows(int n, F f) {
    if (ONE || n == 1) return f(std::integral_constant<int, 1>{}, 0);
    if constexpr (!ONE) {
        if (n == 2) return f(std::integral_constant<int, 2>{}, 0);
        if (MOST > 4 && n <= 4) return f(std::integral_constant<int, 4>{}, 0);
        for (int j = 0; j < n; j += MOST) f(std::integral_constant<int, MOST>{}, j);
    }
}

// How many rows at most a wave's piece of LDS is laid out for (4, 8 or 16; the fewer, the more tiles are on their way at a time).
template <bool ONE, class F>
__device__ __forceinline__ void by_height(int n, F f) {
    if (ONE || n <= 4) return f(std::integral_constant<int, 4>{});
    if constexpr (!ONE) {
        if (n <= 8) f(std::integral_constant<int, 8>{});
        else f(std::integral_constant<int, 16>{});
    }
}

// Two bf16 numbers that add up to v (infinity and NaN the first alone; one NaN for all, see kAbsent).  What would round to infinity has the
// largest number in front of its rest.
__device__ __forceinline__ uint32_t split(float v) {
    using N = Num<Bf16>;
    uint16_t hi = v != v ? N::kNan : N::from_f32(v);
    if (!N::finite(hi) && fabsf(v) <= 0x1.fffffep127f) --hi;
    const uint16_t lo = N::finite(hi) ? N::from_f32(v - N::to_f32(hi)) : 0;
    return hi | (uint32_t)lo << 16;
}

struct UpSums {
    float part[kWaves][2][kMaxTokens][kUpCols];  // [part of the contraction][gate, up][row][column]
};
struct DownSums {
    float y[kWaves][kMaxTokens][16];  // [wave][token][column]
};
struct Sums {
    union {
        UpSums up;
        DownSums down;
    };
    char rows[kWaves][4096];  // rows of x or of the activation on their way to a wave (int4::Rows: 16 of a tile, 8 of two, 4 of four)
};

// What the columns of an up job have from every wave -> activation, two columns a thread.  The stores go through to where all XCDs see
// them.  LOG: see Args::up_log.
template <class W, bool ONE, int LOG>
__device__ __forceinline__ void finish_up(const Args &a, const Plan &p, const UpSums &s, int u, int col0) {
    constexpr int WAVES = kWaves >> LOG;
    const uint32_t tokens = tokens_of<ONE>(p, u);
    const int rows = __popc(tokens), c = (threadIdx.x & 7) * 2, j = threadIdx.x >> 3 & 15, strip = threadIdx.x >> 7;
    col0 += strip * kUpCols;
    if (strip < 1 << LOG && j < rows && strip * kUpCols + c < a.up_cols && col0 + c < a.H) {
        float gate[2] = {}, up[2] = {};
#pragma unroll
        for (int k = 0; k < WAVES; ++k)
#pragma unroll
            for (int i = 0; i < 2; ++i) gate[i] += s.part[strip * WAVES + k][0][j][c + i], up[i] += s.part[strip * WAVES + k][1][j][c + i];
        const int t = ONE ? 0 : token_of(tokens, j);
        // (the gate's curve first: gate * up may be beyond fp32 where what is left of it is not)
        float v[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) v[i] = gate[i] * __builtin_amdgcn_rcpf(1.0f + __expf(-gate[i])) * up[i];
        char *const row = a.act + (int64_t)pair_of<ONE>(a, p, u, t) * 2 * a.act_pitch;
        const int col = col0 + c;
        if constexpr (W::kWhole) {
            uint32_t *const at = reinterpret_cast<uint32_t *>(row + (col & 4 ? a.act_pitch : 0) + col / 8 * 16 + col % 4 * 4);
#pragma unroll
            for (int i = 0; i < 2; ++i) __hip_atomic_store(at + i, v[i] != v[i] ? 0x7fc00000u : __float_as_uint(v[i]), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        } else {
            const uint32_t v0 = split(v[0]), v1 = split(v[1]);
            char *const at = row + col * 2;
            __hip_atomic_store(reinterpret_cast<uint32_t *>(at), (v0 & 0xffffu) | v1 << 16, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            __hip_atomic_store(reinterpret_cast<uint32_t *>(at + a.act_pitch), v0 >> 16 | (v1 & 0xffff0000u), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
    }
}

// Weights of 16 bits.  QUADS: of four columns, that an up job has at most.
template <class T, int QUADS>
struct Wide {
    using Type = T;
    static constexpr int kDownCols = 8, kMaxUpLog = 0;
    static constexpr bool kWhole = std::is_same<T, F16>::value;  // the activation is fp32

    // The waves share the contraction; each has the gate and up rows of all columns, so that a row of x is read for up to 32 of them.
    template <bool ONE>
    static __device__ __forceinline__ void up(const Args &a, const Plan &p, Sums &sh, int u, int strip) {
        const int lane = threadIdx.x & 63, wave = gmm::uniform(threadIdx.x >> 6), sub = lane >> 4, quads = a.up_cols / 4;
        const int steps = (a.K + 127) / 128, s0 = wave * steps >> kWavesLog, s1 = (wave + 1) * steps >> kWavesLog;
        const uint32_t tokens = tokens_of<ONE>(p, u);
        const char *const gate = a.w1 + (int64_t)gmm::uniform(p.expert[u]) * 2 * a.H * a.K * 2;
        const char *w[2 * QUADS];
#pragma unroll
        for (int q = 0; q < QUADS; ++q) {
            const int col = min(strip * a.up_cols + 4 * q, a.H - 4);  // (H is a multiple of 4: all four are inside or none)
            w[2 * q] = gate + (int64_t)col * a.K * 2;
            w[2 * q + 1] = gate + (int64_t)(a.H + col) * a.K * 2;
        }
        by_rows<ONE, (QUADS == 1 ? 8 : 4)>(__popc(tokens), [&](auto n, int row0) {
            constexpr int N = decltype(n)::value;
            const int last = __popc(tokens) - 1;
            uint32_t xo[N];
            float acc[2 * QUADS][N] = {};
#pragma unroll
            for (int j = 0; j < N; ++j) xo[j] = ONE ? 0 : (uint32_t)token_of(tokens, min(row0 + j, last)) * (uint32_t)a.K * 2;
            constexpr int S = QUADS == 1 ? (N == 1 ? 8 : N == 2 ? 6 : N == 4 ? 4 : 2) : N <= 2 ? 2 : 1, SX = QUADS == 1 ? (N == 1 ? 8 : N == 2 ? 3 : N == 4 ? 2 : 1) : S;
            row_dots<T, 2 * QUADS, N, S, SX, (N == 8 ? 4 : N)>(acc, w, a.K * 2, a.x, (uint32_t)a.T * a.K * 2, xo, s0, s1, a.K, 2 * quads);
#pragma unroll
            for (int q = 0; q < QUADS; ++q)
                if (q < quads)
#pragma unroll
                    for (int j = 0; j < N; ++j) {
                        const float g = row_sum(acc[2 * q][j]), v = row_sum(acc[2 * q + 1][j]);
                        if ((lane & 15) == 0 && row0 + j <= last) sh.up.part[wave][0][row0 + j][4 * q + sub] = g, sh.up.part[wave][1][row0 + j][4 * q + sub] = v;
                    }
        });
    }

    static __device__ __forceinline__ int down_steps(const Args &a) { return (a.H + 127) / 128; }
    // Address of line `lane` of steps s0 .. s1 - 1 of a strip of out (null: there are fewer).
    static __device__ __forceinline__ const char *down_line(const Args &a, const Plan &p, int u, int strip, int s0, int s1, int lane) {
        const int row = lane % 8, line = lane / 8, at = s0 * 256 + line * 128;
        const char *const first = down_weights(a, p, u, strip);
        return line < (s1 - s0) * 2 && at < a.H * 2 ? first + (int64_t)row * a.H * 2 + at : nullptr;
    }
    static __device__ __forceinline__ const char *down_weights(const Args &a, const Plan &p, int u, int strip) {
        return a.w2 + ((int64_t)gmm::uniform(p.expert[u]) * a.K + strip * kDownCols) * a.H * 2;
    }

    // y[.][.] += steps s0 .. s1 - 1 of expert u's share of a strip of out.
    template <bool ONE>
    static __device__ __forceinline__ void down(const Args &a, Plan &p, float (&y)[kMaxTokens][16], char *rows, int u, int strip, int s0, int s1) {
        const int lane = threadIdx.x & 63, sub = lane >> 4;
        const uint32_t tokens = tokens_of<ONE>(p, u);
        const char *const first = down_weights(a, p, u, strip);
        const char *const w[2] = {first, first + (int64_t)4 * a.H * 2};
        auto some = [&](auto n, int row0) {
            constexpr int N = decltype(n)::value;
            const int last = __popc(tokens) - 1;
            uint32_t xo[2 * N];
            float acc[2][2 * N] = {};
            int t[N], pair[N];
#pragma unroll
            for (int j = 0; j < N; ++j) {
                t[j] = ONE ? 0 : token_of(tokens, min(row0 + j, last));
                pair[j] = gmm::uniform(pair_of<ONE>(a, p, u, t[j]));
                xo[2 * j] = (uint32_t)pair[j] * 2u * (uint32_t)a.act_pitch;
                xo[2 * j + 1] = xo[2 * j] + a.act_pitch;
            }
            row_dots<T, 2, 2 * N, (N == 1 ? 6 : N == 2 ? 4 : 2), (N == 1 ? 3 : N == 2 ? 2 : 1), 2 * N, kWhole>(acc, w, a.H * 2, a.act, (uint32_t)(a.T * a.top_k) * 2u * (uint32_t)a.act_pitch, xo, s0, s1, a.H, 2, 3, Arrival{&p.failed});
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const float v0 = row_sum(acc[0][2 * j] + acc[0][2 * j + 1]), v1 = row_sum(acc[1][2 * j] + acc[1][2 * j + 1]);
                const float wt = p.weight[pair[j]];
                if ((lane & 15) == 0 && row0 + j <= last) y[t[j]][sub] += wt * v0, y[t[j]][4 + sub] += wt * v1;
            }
        };
        by_rows<ONE, 4>(__popc(tokens), some);
    }
};

// Weights of 4 bits.
template <class T, int GROUP>
struct Narrow {
    using Type = T;
    static constexpr int kDownCols = 16, kMaxUpLog = 2;
    static constexpr bool kWhole = false;

    // 8 >> up_log waves share the contraction of a strip of gate rows and the matching one of up rows.
    template <bool ONE>
    static __device__ __forceinline__ void up(const Args &a, const Plan &p, Sums &sh, int u, int job) {
        UpSums &sums = sh.up;
        const int lane = threadIdx.x & 63, wave = gmm::uniform(threadIdx.x >> 6), r = lane & 15, c = lane >> 4;
        char *const rows = sh.rows[wave];
        const int tiles = int4::tiles_of(a.K), log = kWavesLog - a.up_log, part = wave & ((1 << log) - 1), t0 = part * tiles >> log, t1 = (part + 1) * tiles >> log;
        const int strips = a.H / 16, strip = (job << a.up_log) + (wave >> log);
        if (strip >= strips) return;
        const uint32_t tokens = tokens_of<ONE>(p, u);
        const int last = __popc(tokens) - 1;
        constexpr int SB = int4::TileScales<GROUP>::kBytes;
        const int64_t first = (int64_t)gmm::uniform(p.expert[u]) * 2 * strips + strip;
        const char *const w[2] = {a.w1 + first * tiles * int4::kTileBytes, a.w1 + (first + strips) * tiles * int4::kTileBytes};
        const char *const s[2] = {a.w1_scale + first * tiles * SB, a.w1_scale + (first + strips) * tiles * SB};
        f32x4 acc[2][1];
        auto row = [&](int q) { return ONE ? 0u : (uint32_t)token_of(tokens, q) * (uint32_t)a.K * 2; };
        by_height<ONE>(last + 1, [&](auto m) {
            constexpr int M = decltype(m)::value, S = M == 4 || (M == 8 && GROUP > 32) ? 2 : 1;  // (what registers there are)
            int4::dots<T, T, GROUP, 2, 1, S, M>(acc, w, s, a.x, row, last + 1, t0, t1, a.K, rows);
        });
#pragma unroll
        for (int i = 0; i < 4; ++i) sums.part[wave][0][4 * c + i][r] = acc[0][0][i], sums.part[wave][1][4 * c + i][r] = acc[1][0][i];
    }

    static __device__ __forceinline__ int down_steps(const Args &a) { return int4::tiles_of(a.H); }
    static __device__ __forceinline__ const char *down_line(const Args &a, const Plan &p, int u, int strip, int s0, int s1, int lane) {
        const char *const first = down_weights(a, p, u, strip);
        return lane < (s1 - s0) * (int4::kTileBytes / 128) ? first + (int64_t)s0 * int4::kTileBytes + lane * 128 : nullptr;
    }
    static __device__ __forceinline__ const char *down_weights(const Args &a, const Plan &p, int u, int strip) {
        return a.w2 + ((int64_t)gmm::uniform(p.expert[u]) * (a.K / 16) + strip) * int4::tiles_of(a.H) * int4::kTileBytes;
    }

    template <bool ONE>
    static __device__ __forceinline__ void down(const Args &a, Plan &p, float (&y)[kMaxTokens][16], char *rows, int u, int strip, int s0, int s1) {
        const int lane = threadIdx.x & 63, r = lane & 15, c = lane >> 4;
        const int tiles = int4::tiles_of(a.H);
        const uint32_t tokens = tokens_of<ONE>(p, u);
        const int last = __popc(tokens) - 1;
        constexpr int SB = int4::TileScales<GROUP>::kBytes;
        const int64_t first = (int64_t)gmm::uniform(p.expert[u]) * (a.K / 16) + strip;
        const char *const w[1] = {down_weights(a, p, u, strip)};
        const char *const s[1] = {a.w2_scale + first * tiles * SB};
        // row m of the matrix instructions: value (m even) or rest of the expert's row m / 2
        for (int row0 = 0; row0 <= last; row0 += 8) {
            f32x4 acc[1][1];
            auto row = [&](int q) {
                const int t = ONE ? 0 : token_of(tokens, row0 + q / 2);
                return ((uint32_t)pair_of<ONE>(a, p, u, t) * 2 + (q & 1)) * (uint32_t)a.act_pitch;
            };
            const int n = 2 * min(last + 1 - row0, 8);
            by_height<ONE>(n, [&](auto m) {
                constexpr int M = decltype(m)::value, S = 16 / M;
                int4::dots<Bf16, T, GROUP, 1, 1, S, M>(acc, w, s, a.act, row, n, s0, s1, a.H, rows, Arrival{&p.failed});
            });
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int j = row0 + 2 * c + i;
                if (j <= last) {
                    const int t = ONE ? 0 : token_of(tokens, j);
                    y[t][r] += p.weight[pair_of<ONE>(a, p, u, t)] * (acc[0][0][2 * i] + acc[0][0][2 * i + 1]);
                }
            }
        }
    }
};

__device__ __forceinline__ int load_device(const int32_t *p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ int add_device(int32_t *p, int n) { return __hip_atomic_fetch_add(p, n, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

// The same with the answer on its way: what stands behind it does not wait.  (An add would be gathered over the wave by the compiler, which
// waits at once.)
__device__ __forceinline__ int next_ticket(int32_t *p) { return (int)__builtin_amdgcn_atomic_inc32(reinterpret_cast<uint32_t *>(p), ~0u, __ATOMIC_RELAXED, "agent"); }

// Who does what of the down projection.  A strip of out, kDownCols columns, is n `down_steps` steps: those of the touched experts, one
// behind the other.  All strips in a row are cut into `down_groups` pieces of one length (or of whole strips), and what a workgroup has of a
// strip into one for each wave, wherever that is in an expert: no wave has more than one step more than others, whatever the numbers of strips
// and experts.
struct Place {
    int strip, step;  // of the strip
};
template <class W>
__device__ __forceinline__ Place place_of(const Args &a, int group, int all) {
    const uint32_t strips = (a.K + W::kDownCols - 1) / W::kDownCols, at = (uint32_t)group * strips, g = (uint32_t)a.down_groups, strip = at / g;
    return {(int)strip, a.split ? (int)((at - strip * g) * (uint32_t)all / g) : 0};
}
// The steps of a strip that are between two places.
struct Steps {
    int from, to;
    __device__ __forceinline__ Steps(Place p0, Place p1, int strip, int all) : from(strip == p0.strip ? p0.step : 0), to(strip == p1.strip ? p1.step : all) {}
};

// A workgroup's share of a strip.  A wave's sums are its own; they are added up in the order of the waves, and those of the workgroups that
// share a strip, by the last of them to arrive, in the order of the workgroups.
template <class W, bool ONE>
__device__ __forceinline__ void down_job(const Args &a, Plan &p, Sums &sh, int strip, Steps mine, int each, int all) {
    DownSums &sums = sh.down;
    const int tid = threadIdx.x, wave = gmm::uniform(tid >> 6), lane = tid & 63;
    float(&y)[kMaxTokens][16] = sums.y[wave];
#pragma unroll
    for (int i = 0; i < (ONE ? 1 : kMaxTokens * 16 / 64); ++i) (&y[0][0])[i * 64 + lane] = 0.f;
    wave_lds_order();
    const int n = mine.to - mine.from, end = mine.from + ((wave + 1) * n >> kWavesLog);
    int at = mine.from + (wave * n >> kWavesLog), u = at / each, s0 = at - u * each;
    while (at < end) {
        const int s1 = min(each, s0 + end - at);
        W::template down<ONE>(a, p, y, sh.rows[wave], u, strip, s0, s1);
        wave_lds_order();  // (the next expert's tokens may be other lanes')
        at += s1 - s0, ++u, s0 = 0;
    }
    __syncthreads();
    constexpr int C = W::kDownCols;
    const int t = tid / C, c = tid % C;
    const bool has = tid < a.T * C;
    float v = 0.f;
    if (has) {
#pragma unroll
        for (int k = 0; k < kWaves; ++k) v += sums.y[k][t][c];
    }
    bool last = true;
    if (n < all) {
        // (what begins a strip is its workgroup's last share, everything else the first)
        const int64_t size = a.T * C;
        if (has) __hip_atomic_store(a.shares + (2 * (int)blockIdx.x + (mine.from == 0)) * size + tid, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        asm volatile("s_waitcnt vmcnt(0)" : : : "memory");
        __syncthreads();
        const int strips = (a.K + C - 1) / C, g0 = (int)((uint32_t)strip * (uint32_t)a.down_groups / (uint32_t)strips);
        if (tid == 0) p.job = add_device(&a.sync->arrived[g0], n) + n;
        __syncthreads();
        last = p.job == all;
        if (last && has) {
            v = 0.f;
            Place from = place_of<W>(a, g0, all);
            for (int g = g0; g < a.down_groups && from.strip <= strip; ++g) {
                const Place to = place_of<W>(a, g + 1, all);
                const Steps s(from, to, strip, all);
                if (s.from < s.to) v += __hip_atomic_load(a.shares + (2 * g + (s.from == 0)) * size + tid, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                from = to;
            }
        }
    }
    if (last && has && strip * C + c < a.K)
        reinterpret_cast<uint16_t *>(a.out)[(int64_t)t * a.K + strip * C + c] = Num<typename W::Type>::from_f32(p.failed ? __uint_as_float(0x7fc00000u) : v);
    __syncthreads();  // the sums may be cleared again
}

// The up jobs, (touched expert, up_cols columns), job j in queue j % 8; a workgroup takes those of its own queue, `ticket` its first, and then
// what other queues have left.  Returns when all have been taken: what a workgroup waits for then is with workgroups that run and do not
// wait, so that a wait ends whatever else is on the device and however few workgroups fit on it.
// Meanwhile the first weights of the workgroup's part of the down projection, if it has one, are brought into the L2.
template <class W, bool ONE>
__device__ __forceinline__ void up_jobs(const Args &a, Plan &p, Sums &sh, int ticket, Place down, Steps mine, int each, bool down_too) {
    const int tid = threadIdx.x, lane = tid & 63, home = blockIdx.x % kQueues;
    const int strips = (a.H + a.up_cols - 1) / a.up_cols, jobs = p.n * strips;
    bool own = true;
    uint32_t ahead = 0;
    for (;;) {
        if (tid < 64) {
            int job = -1;
            if (own) {
                const int j = gmm::uniform(ticket) * kQueues + home;
                if (j < jobs) {
                    job = j;
                    if (lane == 0) ticket = next_ticket(&a.sync->ticket[home][0]);  // (on its way while the job runs)
                }
            } else {
                for (;;) {  // lane q: queue q
                    const uint64_t open = __ballot(lane < kQueues && load_device(&a.sync->ticket[lane % kQueues][0]) < (jobs - lane + kQueues - 1) / kQueues);
                    if (open == 0) break;
                    const int victim = __builtin_ctzll(open);
                    int t = 0;
                    if (lane == 0) t = add_device(&a.sync->ticket[victim][0], 1);
                    const int j = gmm::uniform(t) * kQueues + victim;
                    if (j < jobs) {
                        job = j;
                        break;
                    }
                }
            }
            if (lane == 0) p.job = job;
        }
        __syncthreads();
        const int job = gmm::uniform(p.job);
        if (job >= 0) {
            const int u = job / strips;
            W::template up<ONE>(a, p, sh, u, job - u * strips);
            __syncthreads();
            const int col0 = (job - u * strips) * a.up_cols;
            if (W::kMaxUpLog == 0 || a.up_log == 0) finish_up<W, ONE, 0>(a, p, sh.up, u, col0);
            else if (a.up_log == 1) finish_up<W, ONE, (W::kMaxUpLog > 0)>(a, p, sh.up, u, col0);
            else finish_up<W, ONE, W::kMaxUpLog>(a, p, sh.up, u, col0);
        } else if (own && down_too) {
            own = false;
            const int wave = gmm::uniform(tid >> 6), n = mine.to - mine.from, at = mine.from + (wave * n >> kWavesLog), end = mine.from + ((wave + 1) * n >> kWavesLog);
            const int eu = at / each, s0 = at - eu * each;
            const char *line = at < end ? W::down_line(a, p, eu, down.strip, s0, min(each, s0 + end - at), lane) : nullptr;
            if (line != nullptr) ahead = *reinterpret_cast<const uint32_t *>(line);
            __syncthreads();
        } else {
            break;
        }
    }
    // (The last word of the last job: most others are there when it is, and lines that are not would be in the L2 for nothing.)
    if (tid == 0 && down_too) {
        const int u = p.n - 1, t = ONE ? 0 : __builtin_ctz(p.tokens[u]);
        const int32_t *word = reinterpret_cast<const int32_t *>(a.act + ((int64_t)pair_of<ONE>(a, p, u, t) * 2 + 1) * a.act_pitch + a.H * 2 - 4);
#pragma unroll 1
        for (int64_t tries = 0; (uint32_t)load_device(word) == kAbsent; ++tries) {
            if (tries >= kMostTries) {
                p.failed = 1;
                break;
            }
            __builtin_amdgcn_s_sleep(2);
        }
    }
    asm volatile("" : : "v"(ahead));
    __syncthreads();
}

}  // namespace layer
}  // namespace pmoe
