// A whole layer of experts for up to 16 tokens, gfx950: what its kernels (moe_layer.hip) are made of.
//
//   l[t][e] = x[t] . gate[e] (+ bias[e]);  S(t): the top_k largest, ties to the lower index;  a[t][.] = softmax over S(t)
//   out[t]  = sum over e in S(t) of a[t][e] W2[e] (silu(G[e] x[t]) * (U[e] x[t])),  G: rows 0 .. H - 1 of W1[e], U: rows H .. 2H - 1
//
// With so few tokens every weight is used a few times at most: the stream of the touched experts' weights from HBM bounds the large
// layers, a chain of latencies (router, top-k, up, down) the small ones.  Nothing is sorted or padded: a workgroup finds the
// touched experts and their tokens by itself, from the logits, in LDS.
//
// Weights of 16 bits, rows of (E, 2H, K) and (E, K, H): sixteen lanes share a weight row, a step of theirs is 128 elements, 256
// contiguous bytes, straight into registers, and a lane multiplies its eight with those of up to eight tokens by dot products
// of two elements with fp32 sums.  (No matrix instruction wants its operands in whole lines of 128 bytes.)  Weights of 4 bits: int4_tile.h.
//
// The activation is kept as the sum of two 16-bit numbers, the rounded value and the rounded rest, of which the down
// projection multiplies both: 16 bits or more of mantissa at two dot products (or two rows of a matrix instruction that has rows to
// spare) instead of one, so that the output is rounded once.
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
constexpr int kThreads = 512, kWaves = 8;
constexpr int kUpCols = 16;  // activation columns of an up job

struct Args {
    const char *x, *gate, *w1, *w1_scale, *w2, *w2_scale;
    const float *bias;
    char *out;
    int32_t *topk_ids;
    float *topk_weights;
    float *logits;  // (T, E)
    char *act;      // [pair][2: value, rest][act_pitch bytes]
    int act_pitch;
    int T, K, H, E, top_k;
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

// acc[q][n] += this lane's share of weight row w[q] times row x[n]: steps s0 .. s1 - 1 of 128 elements.  The pointers begin
// the rows; `k`: their elements, a multiple of 8; nothing is read behind them.
template <class T, int Q, int N, int S>
__device__ __forceinline__ void row_dots(float (&acc)[Q][N], const char *const (&w)[Q], const char *const (&x)[N], int s0, int s1, int k) {
    const int at = (threadIdx.x & 15) * 8;
    for (int s = s0; s < s1; s += S) {
        i32x4 wv[Q][S], xv[N][S];
#pragma unroll
        for (int i = 0; i < S; ++i)
            if (s + i < s1) {
                const int e = (s + i) * 128 + at;
#pragma unroll
                for (int q = 0; q < Q; ++q) {
                    wv[q][i] = i32x4{0, 0, 0, 0};
                    if (e < k) wv[q][i] = int4::load_once16(w[q] + (int64_t)e * 2);
                }
#pragma unroll
                for (int n = 0; n < N; ++n) {
                    xv[n][i] = i32x4{0, 0, 0, 0};
                    if (e < k) xv[n][i] = *reinterpret_cast<const i32x4 *>(x[n] + (int64_t)e * 2);
                }
            }
#pragma unroll
        for (int i = 0; i < S; ++i)
            if (s + i < s1) {
#pragma unroll
                for (int n = 0; n < N; ++n)
#pragma unroll
                    for (int q = 0; q < Q; ++q)
#pragma unroll
                        for (int d = 0; d < 4; ++d) acc[q][n] = dot2<T>(wv[q][i][d], xv[n][i][d], acc[q][n]);
            }
    }
}

// The touched experts and their tokens, by every workgroup for itself.
struct Plan {
    int n;                              // touched experts
    uint32_t touched[kMaxExperts / 32];
    uint16_t expert[kMaxPairs];
    uint32_t tokens[kMaxPairs];         // bit t: token t is the expert's
    uint8_t slot[kMaxPairs][kMaxTokens];  // which of the token's top_k the expert is
    float weight[kMaxPairs];            // of pair t top_k + r
    int16_t id[kMaxPairs];
};

__device__ __forceinline__ void find_plan(const Args &a, Plan &p, bool publish) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n_pairs = a.T * a.top_k;
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
        for (int d = 32; d > 0; d /= 2) n += __shfl_xor(n, d, 64);
        if (lane == 0) p.n = n;
    }
    __syncthreads();
}

// Token of an expert's row j (the j-th set bit).
__device__ __forceinline__ int token_of(uint32_t tokens, int j) {
    for (int i = 0; i < j; ++i) tokens &= tokens - 1;
    return __builtin_ctz(tokens);
}

// The rows of an expert one, two, four or eight at a time: f(integral N, first row).
template <class F>
__device__ __forceinline__ void by_rows(int n, F f) {
    if (n == 1) f(std::integral_constant<int, 1>{}, 0);
    else if (n == 2) f(std::integral_constant<int, 2>{}, 0);
    else if (n <= 4) f(std::integral_constant<int, 4>{}, 0);
    else
        for (int j = 0; j < n; j += 8) f(std::integral_constant<int, 8>{}, j);
}

// Two 16-bit numbers that add up to v.
template <class T>
__device__ __forceinline__ uint32_t split(float v) {
    const uint16_t hi = Num<T>::from_f32(v), lo = Num<T>::from_f32(v - Num<T>::to_f32(hi));
    return hi | (uint32_t)lo << 16;
}

using Rows = int4::Rows<1, 1>;
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
    char rows[kWaves][Rows::kBytes];  // rows of x or of the activation on their way to a wave
};

// What the 16 columns of an up job have in `parts` parts -> activation.
template <class T>
__device__ __forceinline__ void finish_up(const Args &a, const Plan &p, const UpSums &s, int u, int col0, int parts) {
    const uint32_t tokens = p.tokens[u];
    const int rows = __popc(tokens), c = threadIdx.x & 15, j = threadIdx.x >> 4;
    if (j < rows && col0 + c < a.H) {
        float gate = 0.f, up = 0.f;
        for (int k = 0; k < parts; ++k) gate += s.part[k][0][j][c], up += s.part[k][1][j][c];
        const int t = token_of(tokens, j);
        const uint32_t v = split<T>(swiglu(gate, up));
        char *at = a.act + (int64_t)(t * a.top_k + p.slot[u][t]) * 2 * a.act_pitch + (col0 + c) * 2;
        *reinterpret_cast<uint16_t *>(at) = (uint16_t)v;
        *reinterpret_cast<uint16_t *>(at + a.act_pitch) = (uint16_t)(v >> 16);
    }
}

// Weights of 16 bits.
template <class T>
struct Wide {
    using Type = T;
    static constexpr int kDownCols = 8;

    // Waves: four groups of four columns (a column's gate and up row on 16 lanes) x two halves of the contraction.
    static __device__ __forceinline__ void up(const Args &a, const Plan &p, Sums &sh, int u, int strip) {
        UpSums &sums = sh.up;
        const int lane = threadIdx.x & 63, wave = gmm::uniform(threadIdx.x >> 6), quad = wave & 3, half = wave >> 2, sub = lane >> 4;
        const int steps = (a.K + 127) / 128, s0 = half * steps / 2, s1 = (half + 1) * steps / 2;
        const int c = 4 * quad + sub, col = min(strip * kUpCols + c, a.H - 1);
        const uint32_t tokens = gmm::uniform(p.tokens[u]);
        const char *gate = a.w1 + ((int64_t)p.expert[u] * 2 * a.H + col) * a.K * 2;
        const char *const w[2] = {gate, gate + (int64_t)a.H * a.K * 2};
        by_rows(__popc(tokens), [&](auto n, int row0) {
            constexpr int N = decltype(n)::value;
            const int last = __popc(tokens) - 1;
            const char *x[N];
            float acc[2][N] = {};
#pragma unroll
            for (int j = 0; j < N; ++j) x[j] = a.x + (int64_t)token_of(tokens, min(row0 + j, last)) * a.K * 2;
            row_dots<T, 2, N, (N <= 2 ? 8 : N == 4 ? 4 : 2)>(acc, w, x, s0, s1, a.K);
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const float g = row_sum(acc[0][j]), v = row_sum(acc[1][j]);
                if ((lane & 15) == 0 && row0 + j <= last) sums.part[half][0][row0 + j][c] = g, sums.part[half][1][row0 + j][c] = v;
            }
        });
        __syncthreads();
        finish_up<T>(a, p, sums, u, strip * kUpCols, 2);
    }

    // sums[.][.] += expert u's share, steps part / parts, of 8 columns of out.
    static __device__ __forceinline__ void down(const Args &a, const Plan &p, float (&y)[kMaxTokens][16], char *rows, int u, int strip, int part, int parts) {
        const int lane = threadIdx.x & 63, sub = lane >> 4;
        const int steps = (a.H + 127) / 128, s0 = part * steps / parts, s1 = (part + 1) * steps / parts;
        const uint32_t tokens = gmm::uniform(p.tokens[u]);
        const char *w2 = a.w2 + (int64_t)p.expert[u] * a.K * a.H * 2;
        const char *const w[2] = {w2 + (int64_t)(strip * 8 + sub) * a.H * 2, w2 + (int64_t)(strip * 8 + 4 + sub) * a.H * 2};
        auto some = [&](auto n, int row0) {
            constexpr int N = decltype(n)::value;
            const int last = __popc(tokens) - 1;
            const char *x[2 * N];
            float acc[2][2 * N] = {};
            int t[N];
#pragma unroll
            for (int j = 0; j < N; ++j) {
                t[j] = token_of(tokens, min(row0 + j, last));
                x[2 * j] = a.act + (int64_t)(t[j] * a.top_k + p.slot[u][t[j]]) * 2 * a.act_pitch;
                x[2 * j + 1] = x[2 * j] + a.act_pitch;
            }
            row_dots<T, 2, 2 * N, (N <= 1 ? 8 : N == 2 ? 4 : 2)>(acc, w, x, s0, s1, a.H);
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const float v0 = row_sum(acc[0][2 * j] + acc[0][2 * j + 1]), v1 = row_sum(acc[1][2 * j] + acc[1][2 * j + 1]);
                const float wt = p.weight[t[j] * a.top_k + p.slot[u][t[j]]];
                if ((lane & 15) == 0 && row0 + j <= last) y[t[j]][sub] += wt * v0, y[t[j]][4 + sub] += wt * v1;
            }
        };
        const int n = __popc(tokens);
        if (n == 1) some(std::integral_constant<int, 1>{}, 0);
        else if (n == 2) some(std::integral_constant<int, 2>{}, 0);
        else
            for (int j = 0; j < n; j += 4) some(std::integral_constant<int, 4>{}, j);
    }
};

// Weights of 4 bits.
template <class T, int GROUP>
struct Narrow {
    using Type = T;
    static constexpr int kDownCols = 16;

    // The waves share the contraction; a strip of gate rows and the matching one of up rows.
    static __device__ __forceinline__ void up(const Args &a, const Plan &p, Sums &sh, int u, int strip) {
        UpSums &sums = sh.up;
        const int lane = threadIdx.x & 63, wave = gmm::uniform(threadIdx.x >> 6), r = lane & 15, c = lane >> 4;
        char *const rows = sh.rows[wave];
        const int tiles = int4::tiles_of(a.K), t0 = wave * tiles / kWaves, t1 = (wave + 1) * tiles / kWaves, strips = a.H / 16;
        const uint32_t tokens = gmm::uniform(p.tokens[u]);
        const int last = __popc(tokens) - 1;
        constexpr int SB = int4::TileScales<GROUP>::kBytes;
        const int64_t first = (int64_t)p.expert[u] * 2 * strips + strip;
        const char *const w[2] = {a.w1 + first * tiles * int4::kTileBytes, a.w1 + (first + strips) * tiles * int4::kTileBytes};
        const char *const s[2] = {a.w1_scale + first * tiles * SB, a.w1_scale + (first + strips) * tiles * SB};
        f32x4 acc[2][1] = {};
        int4::dots<T, GROUP, 2, 1, 1>(acc, w, s, [&](int q) { return a.x + (int64_t)token_of(tokens, q) * a.K * 2; }, last + 1, t0, t1, a.K, rows);
        __syncthreads();  // the sums may lie where the rows were
#pragma unroll
        for (int i = 0; i < 4; ++i) sums.part[wave][0][4 * c + i][r] = acc[0][0][i], sums.part[wave][1][4 * c + i][r] = acc[1][0][i];
        __syncthreads();
        finish_up<T>(a, p, sums, u, strip * kUpCols, kWaves);
    }

    static __device__ __forceinline__ void down(const Args &a, const Plan &p, float (&y)[kMaxTokens][16], char *rows, int u, int strip, int part, int parts) {
        const int lane = threadIdx.x & 63, r = lane & 15, c = lane >> 4;
        const int tiles = int4::tiles_of(a.H), t0 = part * tiles / parts, t1 = (part + 1) * tiles / parts;
        const uint32_t tokens = gmm::uniform(p.tokens[u]);
        const int last = __popc(tokens) - 1;
        constexpr int SB = int4::TileScales<GROUP>::kBytes;
        const int64_t first = (int64_t)p.expert[u] * (a.K / 16) + strip;
        const char *const w[1] = {a.w2 + first * tiles * int4::kTileBytes};
        const char *const s[1] = {a.w2_scale + first * tiles * SB};
        // row m of the matrix instructions: value (m even) or rest of the expert's row m / 2
        for (int row0 = 0; row0 <= last; row0 += 8) {
            f32x4 acc[1][1] = {};
            auto row = [&](int q) {
                const int t = token_of(tokens, row0 + q / 2);
                return a.act + ((int64_t)(t * a.top_k + p.slot[u][t]) * 2 + (q & 1)) * a.act_pitch;
            };
            int4::dots<T, GROUP, 1, 1, 1>(acc, w, s, row, 2 * min(last + 1 - row0, 8), t0, t1, a.H, rows);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int j = row0 + 2 * c + i;
                if (j <= last) {
                    const int t = token_of(tokens, j);
                    y[t][r] += p.weight[t * a.top_k + p.slot[u][t]] * (acc[0][0][2 * i] + acc[0][0][2 * i + 1]);
                }
            }
        }
    }
};

// kDownCols columns of out.  A wave takes experts wave, wave + 8, ...; of four experts or fewer two waves or more share the contraction
// of each.  Its sums are its own; they are added up in the order of the waves.
template <class W>
__device__ __forceinline__ void down_job(const Args &a, const Plan &p, Sums &sh, int strip) {
    DownSums &sums = sh.down;
    const int tid = threadIdx.x, wave = gmm::uniform(tid >> 6), lane = tid & 63;
    const int parts = p.n > 4 ? 1 : p.n > 2 ? 2 : p.n == 2 ? 4 : 8;
    float(&y)[kMaxTokens][16] = sums.y[wave];
#pragma unroll
    for (int i = 0; i < kMaxTokens * 16 / 64; ++i) (&y[0][0])[i * 64 + lane] = 0.f;
    for (int u = wave / parts; u < p.n; u += kWaves / parts) W::down(a, p, y, sh.rows[wave], u, strip, wave & (parts - 1), parts);
    __syncthreads();
    constexpr int C = W::kDownCols;
    if (tid < a.T * C) {
        const int t = tid / C, c = tid % C;
        float v = 0.f;
#pragma unroll
        for (int k = 0; k < kWaves; ++k) v += sums.y[k][t][c];
        if (strip * C + c < a.K) reinterpret_cast<uint16_t *>(a.out)[(int64_t)t * a.K + strip * C + c] = Num<typename W::Type>::from_f32(v);
    }
}

}  // namespace layer
}  // namespace pmoe
