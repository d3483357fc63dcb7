// Kernels of the ragged expert products on the tiles of grouped_tile.h: argument blocks, the walk over the tiles, the way
// out.  Resident: one workgroup per CU, which takes its tiles one after the other and has the next tile's first slabs on
// their way while the current one is stored.
#pragma once
#include "grouped_tile.h"
#include "pmoe_common.h"

namespace pmoe {

int resident_grid();

namespace gmm {

constexpr int kMaxGroups = 4 * kThreads;
constexpr int kWalkCols = 8;  // column tiles that are walked side by side

// out[r] = sum over k of x[r][k] w[g(r)][.][k]; strides in bytes.
struct RowsArgs {
    const char *x, *w;
    char *out;
    int64_t x_pitch, w_pitch, w_group, out_pitch;
    const int32_t *offsets;  // null: one group of all rows
    int n_groups, rows, cols;
    int depth;               // contraction, elements
    const float *x_scale, *w_scale;  // 8-bit integers: (rows), (groups, cols)
};
// dw[g] = sum over the group's rows of dy[r] x[r]^T; strides in bytes.
struct WgradArgs {
    const char *dy, *x;
    char *dw;
    int64_t dy_pitch, x_pitch;
    const int32_t *offsets;
    int n_groups, rows, out_rows, cols;
};

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// Ends outside 0 .. rows are taken as the nearest inside, so that whatever the offsets hold, no access leaves x.
__device__ __forceinline__ int group_end(const RowsArgs &a, int g) {
    return a.offsets == nullptr ? a.rows : min(max(a.offsets[g], 0), a.rows);
}

struct Tile {
    int group, fm;
    int row0, live;  // first row and how many
    int col0;
    bool zero;       // rows behind the last group: their outputs are zero
};

// Walk over the tiles of a launch.  A group's rows are cut into as few tiles as there can be, of even height (in
// steps of 64 rows); tile number t runs through [group][8 column tiles][row tile][column tile], and the rows behind the
// last group follow.  Thread i holds groups 4 i .. 4 i + 3 in registers.
struct Walk {
    int begin[5];   // first rows of the thread's groups, and the end of the last one
    int before[5];  // row tiles in front of them
    int row_tiles, col_tiles, live_rows, total;

    __device__ __forceinline__ void setup(const RowsArgs &a, int tid, int *words) {
        const int g0 = 4 * tid, lane = tid & 63, wave = tid >> 6;
        // A group begins where the furthest end in front of it is (its predecessor's, if the ends are in order), so that
        // whatever the offsets hold no two groups share a row.
#pragma unroll
        for (int i = 0; i < 4; ++i) begin[i + 1] = max(g0 + i < a.n_groups ? group_end(a, g0 + i) : 0, i == 0 ? 0 : begin[i]);
        int far = begin[4];
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const int v = __shfl_up(far, d, 64);
            if (lane >= d) far = max(far, v);
        }
        if (lane == 63) words[wave] = far;
        const int up = __shfl_up(far, 1, 64);
        begin[0] = lane == 0 ? 0 : up;
        ring::all_read();
        live_rows = 0;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            if (w < wave) begin[0] = max(begin[0], words[w]);
            live_rows = max(live_rows, words[w]);
        }
        live_rows = uniform(live_rows);
        int sum = 0, count[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            begin[i + 1] = max(begin[i + 1], begin[i]);
            count[i] = (begin[i + 1] - begin[i] + 255) / 256;
            sum += count[i];
        }
        int incl = sum;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const int v = __shfl_up(incl, d, 64);
            if (lane >= d) incl += v;
        }
        if (lane == 63) words[kWaves + wave] = incl;
        ring::all_read();
        int lower = 0;
        row_tiles = 0;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            if (w < wave) lower += words[kWaves + w];
            row_tiles += words[kWaves + w];
        }
        ring::all_read();  // the words may be written again
        before[0] = lower + incl - sum;
#pragma unroll
        for (int i = 0; i < 4; ++i) before[i + 1] = before[i] + count[i];
        row_tiles = uniform(row_tiles);
        col_tiles = (a.cols + kCols - 1) / kCols;
        total = (row_tiles + (a.rows - live_rows + 255) / 256) * col_tiles;
    }

    // Tile t < total, through five words of LDS that nobody else uses meanwhile.  Two barriers.
    __device__ __forceinline__ Tile find(const RowsArgs &a, int t, int tid, int *words) const {
        Tile r;
        if (t < row_tiles * col_tiles) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int rt = before[i + 1] - before[i], local = t - before[i] * col_tiles;
                if (local >= 0 && local < rt * col_tiles) {
                    const int band = local / (rt * kWalkCols), width = min(kWalkCols, col_tiles - band * kWalkCols);
                    const int rem = local - band * rt * kWalkCols, m = rem / width;
                    const int rows = begin[i + 1] - begin[i];
                    const int height = ((rows + rt - 1) / rt + 63) & ~63;
                    words[0] = 4 * tid + i;
                    words[1] = begin[i] + m * height;
                    words[2] = min(height, rows - m * height);
                    words[3] = band * kWalkCols + rem - m * width;
                }
            }
            ring::all_read();
            r.group = uniform(words[0]);
            r.row0 = uniform(words[1]);
            r.live = uniform(words[2]);
            r.col0 = uniform(words[3]) * kCols;
            r.zero = false;
            ring::all_read();
        } else {
            const int local = t - row_tiles * col_tiles, m = local / col_tiles;
            r.group = 0;
            r.row0 = live_rows + m * 256;
            r.live = min(256, a.rows - r.row0);
            r.col0 = (local - m * col_tiles) * kCols;
            r.zero = true;
        }
        r.fm = (r.live + 63) / 64;
        return r;
    }
};

// Place of this workgroup's `i`-th tile in the walk: a round of the resident grid is dealt to the XCDs (workgroup id mod 8)
// in runs of consecutive tiles, so that what runs side by side on an XCD shares rows and weights in its L2.
__device__ __forceinline__ int walk_place(int i) {
    const int per = gridDim.x / 8;
    return i * (int)gridDim.x + ((int)blockIdx.x % 8) * per + (int)blockIdx.x / 8;
}

template <class OUT>
struct Pack;
template <>
struct Pack<Bf16> {
    static constexpr int kBytes = 2;
    static __device__ __forceinline__ uint2 four(float a, float b, float c, float d) {
        return make_uint2(pack2_bf16(a, b), pack2_bf16(c, d));
    }
};
template <>
struct Pack<F16> {
    static constexpr int kBytes = 2;
    static __device__ __forceinline__ uint32_t two(float a, float b) {
        typedef float f32x2 __attribute__((ext_vector_type(2)));
        typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, f16x2));
    }
    static __device__ __forceinline__ uint2 four(float a, float b, float c, float d) { return make_uint2(two(a, b), two(c, d)); }
};
struct F32 {};
template <>
struct Pack<F32> {
    static constexpr int kBytes = 4;
    static __device__ __forceinline__ uint4 four(float a, float b, float c, float d) {
        return make_uint4(__float_as_uint(a), __float_as_uint(b), __float_as_uint(c), __float_as_uint(d));
    }
};

// Scales of an 8-bit product: a row's in a register of its lane, the wave's 128 columns' in the upper half of its scratch
// (64 registers otherwise, which spill).  Nothing for the other types.
template <class T, int FM>
struct Scales {
    static constexpr int kRowBytes = 256;  // of a row in scratch
    __device__ __forceinline__ void load(const RowsArgs &, const Tile &, int) {}
    __device__ __forceinline__ void keep(char *, int) const {}
    __device__ __forceinline__ float4 apply(const typename T::Acc &acc, int, int, int i4, const char *, int) const {
        return make_float4(acc[4 * i4], acc[4 * i4 + 1], acc[4 * i4 + 2], acc[4 * i4 + 3]);
    }
};
template <int FM>
struct Scales<I8, FM> {
    static constexpr int kRowBytes = 128;
    float x[FM];
    float2 w;
    __device__ __forceinline__ void load(const RowsArgs &a, const Tile &tile, int tid) {
        const int wave = uniform(tid >> 6), lane = tid & 63;
#pragma unroll
        for (int t = 0; t < FM; ++t) x[t] = a.x_scale[tile.row0 + min(((wave >> 1) * FM + t) * 32 + (lane & 31), tile.live - 1)];
        const float *p = a.w_scale + (int64_t)tile.group * a.cols + min(tile.col0 + (wave & 1) * 128 + lane * 2, a.cols - 2);
        w = make_float2(p[0], p[1]);
        if (tile.zero) {  // (a scale that is not finite)
#pragma unroll
            for (int t = 0; t < FM; ++t) x[t] = 0.f;
            w = make_float2(0.f, 0.f);
        }
    }
    __device__ __forceinline__ void keep(char *scratch, int lane) const {
        *reinterpret_cast<float2 *>(scratch + kScratchBytes / 2 + lane * 8) = w;
    }
    // The sum is rounded to 24 bits, then each product: 1.5 units in the last place of fp32 in all.
    __device__ __forceinline__ float4 apply(const i32x16 &acc, int f, int t, int i4, const char *scratch, int half) const {
        const float4 c = *reinterpret_cast<const float4 *>(scratch + kScratchBytes / 2 + (f * 32 + i4 * 8 + half * 4) * 4);
        return make_float4((float)acc[4 * i4] * x[t] * c.x, (float)acc[4 * i4 + 1] * x[t] * c.y, (float)acc[4 * i4 + 2] * x[t] * c.z,
                           (float)acc[4 * i4 + 3] * x[t] * c.w);
    }
};

// A tile's way out: 32 rows x 256 B (8-bit products: 128 B) at a time through the wave's scratch, chunk c of row r in slot
// c ^ r (modulo the chunks of a row), and from there in whole rows.  `out`: the tile's first element.  `live`, `cols`: rows and
// columns to store.
template <class T, class OUT, int FM>
__device__ __forceinline__ void store_tile(const typename T::Acc (&acc)[4][FM], const Scales<T, FM> &scales, char *lds, char *out,
                                           int64_t pitch, int live, int cols, int tid) {
    using P = Pack<OUT>;
    constexpr int ROW = Scales<T, FM>::kRowBytes, CHUNKS = ROW / 16;
    constexpr int FRAGS = ROW / (32 * P::kBytes);  // column fragments that go through at a time
    constexpr int PER = 16 / P::kBytes;            // columns of a chunk
    const int wave = uniform(tid >> 6), lane = tid & 63;
    char *scratch = lds + kScratchOff + wave * kScratchBytes;
    const int r = lane & 31, half = lane >> 5, sx = r % CHUNKS;
#pragma unroll
    for (int t = 0; t < FM; ++t)
#pragma unroll
        for (int h = 0; h < 4 / FRAGS; ++h) {
#pragma unroll
            for (int f = 0; f < FRAGS; ++f)
#pragma unroll
                for (int i4 = 0; i4 < 4; ++i4) {
                    const float4 v = scales.apply(acc[h * FRAGS + f][t], h * FRAGS + f, t, i4, scratch, half);
                    if constexpr (P::kBytes == 2)
                        *reinterpret_cast<uint2 *>(scratch + r * ROW + (((4 * f + i4) ^ sx) << 4) + half * 8) = P::four(v.x, v.y, v.z, v.w);
                    else
                        *reinterpret_cast<uint4 *>(scratch + r * ROW + (((8 * f + 2 * i4 + half) ^ sx) << 4)) = P::four(v.x, v.y, v.z, v.w);
                }
            __builtin_amdgcn_wave_barrier();
            const int chunk = lane % CHUNKS, col = ((wave & 1) * 4 + h * FRAGS) * 32 + chunk * PER;
#pragma unroll
            for (int it = 0; it < CHUNKS / 2; ++it) {
                const int row = it * (64 / CHUNKS) + lane / CHUNKS, at = ((wave >> 1) * FM + t) * 32 + row;
                const uint4 v = *reinterpret_cast<const uint4 *>(scratch + row * ROW + ((chunk ^ (row % CHUNKS)) << 4));
                if (at < live && col < cols) *reinterpret_cast<uint4 *>(out + at * pitch + col * P::kBytes) = v;
            }
            __builtin_amdgcn_wave_barrier();
        }
}

// ------------------------------------------------------------------------------- rows by their expert's weights

template <class T, bool QX, int FM>
__device__ __forceinline__ void rows_feed(Feed<FM, false, QX> &feed, const RowsArgs &a, const Tile &tile, int tid) {
    feed.p.setup(tid, a.x + tile.row0 * a.x_pitch, a.x_pitch, tile.live);
    feed.q.setup(tid, a.w + tile.group * a.w_group + tile.col0 * (QX ? (int64_t)T::kBytes : a.w_pitch), a.w_pitch, min(kCols, a.cols - tile.col0));
    feed.set_length(tile.zero ? 0 : a.depth, T::kBytes);
    feed.set_ahead(tid, a.x_pitch, tile.live, a.w_pitch, min(kCols, a.cols - tile.col0));
}
template <class T, bool QX>
__device__ __forceinline__ void rows_start(const RowsArgs &a, const Tile &tile, char *lds, int tid) {
    auto start = [&](auto &feed) {
        rows_feed<T>(feed, a, tile, tid);
        feed.start(tid, lds);
    };
    switch (tile.fm) {
        case 1: { Feed<1, false, QX> feed; start(feed); break; }
        case 2: { Feed<2, false, QX> feed; start(feed); break; }
        case 3: { Feed<3, false, QX> feed; start(feed); break; }
        default: { Feed<4, false, QX> feed; start(feed); break; }
    }
}
template <class T, bool QX, class OUT, int FM>
__device__ __forceinline__ bool rows_tile(const RowsArgs &a, const Walk &walk, Tile &tile, int next, char *lds, int tid) {
    typename T::Acc acc[4][FM] = {};
    {
        Feed<FM, false, QX> feed;
        rows_feed<T>(feed, a, tile, tid);
        contract<T>(acc, feed, lds, tid);
    }
    Scales<T, FM> scales;
    scales.load(a, tile, tid);
    char *out = a.out + tile.row0 * a.out_pitch + (int64_t)tile.col0 * Pack<OUT>::kBytes;
    const int live = tile.live, cols = a.cols - tile.col0;
    const bool more = next < walk.total;
    if (more) {
        tile = walk.find(a, next, tid, reinterpret_cast<int *>(lds + kScratchOff));
    }
    scales.keep(lds + kScratchOff + uniform(tid >> 6) * kScratchBytes, tid & 63);
    if (more) rows_start<T, QX>(a, tile, lds, tid);
    store_tile<T, OUT, FM>(acc, scales, lds, out, a.out_pitch, live, cols, tid);
    return more;
}

template <class T, bool QX, class OUT>
__global__ __launch_bounds__(kThreads, 1) void grouped_mm_kernel(RowsArgs a) {
    __shared__ __attribute__((aligned(1024))) char lds[kLdsBytes];
    const int tid = threadIdx.x;
    int *words = reinterpret_cast<int *>(lds + kScratchOff);
    Walk walk;
    walk.setup(a, tid, words);
    int i = 0;
    if (walk_place(0) >= walk.total) return;
    Tile tile = walk.find(a, walk_place(0), tid, words);
    rows_start<T, QX>(a, tile, lds, tid);
    bool more = true;
    while (more) {
        const int next = walk_place(++i);
        switch (tile.fm) {
            case 1: more = rows_tile<T, QX, OUT, 1>(a, walk, tile, next, lds, tid); break;
            case 2: more = rows_tile<T, QX, OUT, 2>(a, walk, tile, next, lds, tid); break;
            case 3: more = rows_tile<T, QX, OUT, 3>(a, walk, tile, next, lds, tid); break;
            default: more = rows_tile<T, QX, OUT, 4>(a, walk, tile, next, lds, tid); break;
        }
    }
}

// ------------------------------------------------------------------------------- gradient of the weights

template <class T, int FM>
__global__ __launch_bounds__(kThreads, 1) void grouped_mm_wgrad_kernel(WgradArgs a) {
    __shared__ __attribute__((aligned(1024))) char lds[kLdsBytes];
    const int tid = threadIdx.x;
    const int row_tiles = (a.out_rows + 64 * FM - 1) / (64 * FM), col_tiles = (a.cols + kCols - 1) / kCols;
    const int per = row_tiles * col_tiles, total = per * a.n_groups;
    struct Place {
        int group, row0, col0;
    };
    auto place = [&](int t) {
        Place p;
        p.group = t / per;
        const int local = t - p.group * per, band = local / (row_tiles * kWalkCols);
        const int width = min(kWalkCols, col_tiles - band * kWalkCols), rem = local - band * row_tiles * kWalkCols;
        p.row0 = rem / width * (64 * FM);
        p.col0 = (band * kWalkCols + rem % width) * kCols;
        return p;
    };
    auto set = [&](Feed<FM, true, true> &feed, const Place &p) {
        const int begin = p.group == 0 ? 0 : min(max(a.offsets[p.group - 1], 0), a.rows);
        const int end = max(min(max(a.offsets[p.group], 0), a.rows), begin);
        feed.p.setup(tid, a.dy + begin * a.dy_pitch + p.row0 * T::kBytes, a.dy_pitch, min(64 * FM, a.out_rows - p.row0));
        feed.q.setup(tid, a.x + begin * a.x_pitch + p.col0 * T::kBytes, a.x_pitch, min(kCols, a.cols - p.col0));
        feed.set_length(uniform(end - begin), T::kBytes);
        feed.set_ahead(tid, a.dy_pitch, min(64 * FM, a.out_rows - p.row0), a.x_pitch, min(kCols, a.cols - p.col0));
    };
    int i = 0, t = walk_place(0);
    if (t >= total) return;
    Place p = place(t);
    Feed<FM, true, true> feed;
    set(feed, p);
    feed.start(tid, lds);
    while (true) {
        typename T::Acc acc[4][FM] = {};
        contract<T>(acc, feed, lds, tid);
        const int64_t pitch = (int64_t)a.cols * T::kBytes;
        char *out = a.dw + ((int64_t)p.group * a.out_rows + p.row0) * pitch + (int64_t)p.col0 * T::kBytes;
        const int live = a.out_rows - p.row0, cols = a.cols - p.col0;
        t = walk_place(++i);
        const bool more = t < total;
        if (more) {
            p = place(t);
            set(feed, p);
            feed.start(tid, lds);
        }
        store_tile<T, T, FM>(acc, Scales<T, FM>(), lds, out, pitch, live, cols, tid);
        if (!more) return;
    }
}

}  // namespace gmm
}  // namespace pmoe
