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
    bool once;               // see stores_once
    bool fills;              // even tiles of 128 rows are more than one round of the grid
};
// dw[g] = sum over the group's rows of dy[r] x[r]^T; strides in bytes.
struct WgradArgs {
    const char *dy, *x;
    char *dw;
    int64_t dy_pitch, x_pitch;
    const int32_t *offsets;
    int n_groups, rows, out_rows, cols;
    bool once;  // see stores_once
};

// Whether outputs are stored with the non-temporal hint: they leave the L2 to the operands, but lose where they are larger than
// what the last cache in front of the memory takes (268 MB of 8-bit products: 1646 -> 1607 us, of gradients of rows 450 -> 440
// us, 33 MB of weights' 15.0 -> 13.4 us; 470 MB of bf16 products: 1582 -> 1627 us, 805 MB of weights' gradients 463 -> 473 us).
inline bool stores_once(int64_t bytes) { return bytes <= 320ll << 20; }

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

// Walk over the tiles of a launch.  A group's rows are cut into as few tiles as there can be, of their even share rounded up to
// 64 rows (the last one has what is left: 1025 rows are four tiles of 256 and one of a row).  The walk takes the tallest tiles first: tile number t runs through [height, 4 to 1][group][8 column tiles][row
// tile][column tile], and the rows behind the last group follow.  The workgroups, which take every grid-th tile, then have
// equal shares of every height (in the order of the groups: the largest share 16 % above the mean with 128 groups of 512
// rows on average), and a tile is nearly always followed by one of its own height.  Thread i holds groups 4 i .. 4 i + 3.
struct Walk {
    int begin[5];   // first rows of the thread's groups, and the end of the last one
    int before[4];  // row tiles in front of each
    int row_tiles, col_tiles, live_rows, total;
    int shift;  // a tile has at most 2^shift rows

    __device__ __forceinline__ int tiles_of(int rows) const { return (rows + (1 << shift) - 1) >> shift; }
    // Tiles of 128 or 64 rows where they still are one round of the grid: so many CUs would stand still beside taller ones, and a
    // slab of fewer rows is over sooner (8 experts of 512 columns, contraction 4096, bf16: 1020 rows 67 -> 49 us, 8192 rows 69 ->
    // 63; 512 rows of one group x 4096 x 4096: 71 -> 42; 510 rows whose tiles are short, contraction 512: 16.2 -> 14.6).
    // (Between its words and setup's furthest ends, which a wave may still be reading, there is no barrier: they are others.)
    __device__ __forceinline__ void choose_height(const RowsArgs &a, int tid, int *words) {
        shift = 8;
        if (a.fills) return;
        int *const counts = words + kWaves;
        int n[2] = {};
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int c = 0; c < 2; ++c) n[c] += (begin[i + 1] - begin[i] + (64 << c) - 1) >> (6 + c);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
#pragma unroll
            for (int d = 32; d > 0; d /= 2) n[c] += __shfl_xor(n[c], d, 64);
            if ((tid & 63) == 0) counts[kWaves * c + (tid >> 6)] = n[c];
        }
        ring::all_read();
#pragma unroll
        for (int c = 1; c >= 0; --c) {
            int sum = 0;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) sum += counts[kWaves * c + w];
            if ((int64_t)sum * col_tiles <= gridDim.x) shift = 6 + c;
        }
        ring::all_read();  // the words may be written again
        shift = uniform(shift);
    }
    static __device__ __forceinline__ int height_of(int rows, int tiles) { return ((rows - 1) / tiles + 64) & ~63; }  // rows >= 1
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
#pragma unroll
        for (int i = 0; i < 4; ++i) begin[i + 1] = max(begin[i + 1], begin[i]);
        col_tiles = (a.cols + kCols - 1) / kCols;
        choose_height(a, tid, words);
        int count[4], fm[4], sum[4] = {}, incl[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int rows = begin[i + 1] - begin[i];
            count[i] = tiles_of(rows);
            fm[i] = rows > 0 ? height_of(rows, count[i]) / 64 : 0;
#pragma unroll
            for (int c = 0; c < 4; ++c) sum[c] += fm[i] == c + 1 ? count[i] : 0;
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) incl[c] = sum[c];
#pragma unroll
        for (int d = 1; d < 64; d *= 2)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int v = __shfl_up(incl[c], d, 64);
                if (lane >= d) incl[c] += v;
            }
        if (lane == 63)
#pragma unroll
            for (int c = 0; c < 4; ++c) words[kWaves + 4 * wave + c] = incl[c];
        ring::all_read();
        row_tiles = 0;
#pragma unroll
        for (int c = 3; c >= 0; --c) {
            int at = row_tiles + incl[c] - sum[c];
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                const int v = words[kWaves + 4 * w + c];
                if (w < wave) at += v;
                row_tiles += v;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (fm[i] == c + 1) {
                    before[i] = at;
                    at += count[i];
                }
        }
        ring::all_read();  // the words may be written again
        row_tiles = uniform(row_tiles);
        total = (row_tiles + (a.rows - live_rows + 255) / 256) * col_tiles;
    }

    // Tile t < total, through four words of LDS: post(), a barrier, get().
    __device__ __forceinline__ void post(int t, int tid, int *words) const {
        int mine = -1, from = 0, rows = 0, local = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int n = begin[i + 1] - begin[i], at = t - before[i] * col_tiles;
            const bool hit = (n > 0) & (at >= 0) & (at < tiles_of(n) * col_tiles);
            mine = hit ? i : mine;
            from = hit ? begin[i] : from;
            rows = hit ? n : rows;
            local = hit ? at : local;
        }
        if (mine >= 0) {
            const int rt = tiles_of(rows), band = local / (rt * kWalkCols), width = min(kWalkCols, col_tiles - band * kWalkCols);
            const int rem = local - band * rt * kWalkCols, m = rem / width, height = height_of(rows, rt);
            words[0] = 4 * tid + mine;
            words[1] = from + m * height;
            words[2] = min(height, rows - m * height);
            words[3] = band * kWalkCols + rem - m * width;
        }
    }
    __device__ __forceinline__ Tile get(const RowsArgs &a, int t, const int *words) const {
        Tile r;
        if (t < row_tiles * col_tiles) {
            r.group = uniform(words[0]);
            r.row0 = uniform(words[1]);
            r.live = uniform(words[2]);
            r.col0 = uniform(words[3]) * kCols;
            r.zero = false;
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
    __device__ __forceinline__ void pin() {}
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
    // Waits for them here, where few copies are under way, and not in front of their first use.
    __device__ __forceinline__ void pin() {
#pragma unroll
        for (int t = 0; t < FM; ++t) asm volatile("" : "+v"(x[t]));
        asm volatile("" : "+v"(w.x), "+v"(w.y));
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
// columns to store.  A part is read back while the next one is converted and written behind it (the LDS serves a wave in order),
// and stored behind that; `once`: past the caches (see stores_once).
template <class T, class OUT, int FM>
__device__ __forceinline__ void store_tile(const typename T::Acc (&acc)[4][FM], const Scales<T, FM> &scales, char *lds, char *out,
                                           int64_t pitch, int live, int cols, bool once, int tid) {
    using P = Pack<OUT>;
    constexpr int ROW = Scales<T, FM>::kRowBytes, CHUNKS = ROW / 16, PER_READ = 64 / CHUNKS, READS = 32 / PER_READ;
    constexpr int FRAGS = ROW / (32 * P::kBytes);  // column fragments that go through at a time
    constexpr int PARTS = FM * 4 / FRAGS;
    const int wave = uniform(tid >> 6), lane = tid & 63;
    char *scratch = lds + kScratchOff + wave * kScratchBytes;
    const int r = lane & 31, half = lane >> 5, sx = r % CHUNKS;
    const int sub = lane / CHUNKS, chunk = lane % CHUNKS;
    // rows and columns of the wave's part of the tile, from its own first ones
    const int first_row = (wave >> 1) * FM * 32, first_col = (wave & 1) * 128;
    out += first_row * pitch + first_col * P::kBytes;
    live -= first_row;
    cols -= first_col;
    // (32 bits hold three rows of 2^29 bytes, or seven of an 8-bit product in 16 bits; seven of 2^30 they do not)
    using Offset = std::conditional_t<P::kBytes == 4, int64_t, uint32_t>;
    const Offset lane_off = (Offset)sub * (Offset)pitch + chunk * 16;
    const bool whole = live >= 32 * FM && cols >= 128;
    auto put = [&](auto part) {
        constexpr int t = part.value / (4 / FRAGS), h = part.value % (4 / FRAGS);
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
    };
    put(std::integral_constant<int, 0>());
    unrolled<PARTS>([&](auto part) {
        constexpr int t = part.value / (4 / FRAGS), h = part.value % (4 / FRAGS);
        i32x4 v[READS];
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int it = 0; it < READS; ++it) {
            const int row = it * PER_READ + sub;
            v[it] = *reinterpret_cast<const i32x4 *>(scratch + row * ROW + ((chunk ^ (row % CHUNKS)) << 4));
        }
        __builtin_amdgcn_wave_barrier();
        if constexpr (part.value + 1 < PARTS) put(std::integral_constant<int, part.value + 1>());
        PMOE_GMM_FENCE();
        char *to = out + t * 32 * pitch + h * ROW;  // wave-uniform
        if (whole && !once) {
#pragma unroll
            for (int it = 0; it < READS; ++it) *reinterpret_cast<i32x4 *>(to + it * PER_READ * pitch + lane_off) = v[it];
        } else if (whole) {
#pragma unroll
            for (int it = 0; it < READS; ++it) {
                __builtin_nontemporal_store(v[it], reinterpret_cast<i32x4 *>(to + it * PER_READ * pitch + lane_off));
                asm volatile("");  // (the compiler makes one branch, without the hint, of the two otherwise)
            }
        } else {
            const int rows = h * (ROW / P::kBytes) + chunk * (16 / P::kBytes) < cols ? live - t * 32 - sub : 0;
#pragma unroll
            for (int it = 0; it < READS; ++it)
                if (it * PER_READ < rows) __builtin_nontemporal_store(v[it], reinterpret_cast<i32x4 *>(to + it * PER_READ * pitch + lane_off));
        }
        PMOE_GMM_FENCE();
    });
}

// ------------------------------------------------------------------------------- rows by their expert's weights

template <class T, bool QX, int FM>
__device__ __forceinline__ void rows_feed(Feed<FM, false, QX> &feed, const RowsArgs &a, const Tile &tile, int tid) {
    feed.p.setup(tid, a.x + tile.row0 * a.x_pitch, a.x_pitch, tile.live);
    feed.q.setup(tid, a.w + tile.group * a.w_group + tile.col0 * (QX ? (int64_t)T::kBytes : a.w_pitch), a.w_pitch, min(kCols, a.cols - tile.col0));
    feed.set_length(tile.zero ? 0 : a.depth, T::kBytes);
    feed.set_ahead(tid, a.x_pitch, tile.live, a.w_pitch, min(kCols, a.cols - tile.col0));
}
// Copies of slab 0 or 1 of a tile of any height, all at once.
template <class T, bool QX>
__device__ __forceinline__ void rows_issue(const RowsArgs &a, const Tile &tile, int slab, uint32_t at, int tid) {
    auto issue = [&](auto &feed) {
        rows_feed<T>(feed, a, tile, tid);
        feed.issue_all(tid, at, slab);
    };
    switch (tile.fm) {
        case 1: { Feed<1, false, QX> feed; issue(feed); break; }
        case 2: { Feed<2, false, QX> feed; issue(feed); break; }
        case 3: { Feed<3, false, QX> feed; issue(feed); break; }
        default: { Feed<4, false, QX> feed; issue(feed); break; }
    }
}

// The walk of a workgroup.
struct RowsState {
    Tile tile;
    int turn;        // of the tile, in this workgroup's list
    uint32_t stage;  // of its slab 0
};

template <class T, bool QX, class OUT, int FM>
struct RowsNext {
    const RowsArgs &a;
    const Walk &walk;
    Scales<T, FM> &scales;
    int *words;
    int tid, place;
    Tile tile;  // the next one, behind take()

    __device__ __forceinline__ void post() const {
        if (place < walk.total) walk.post(place, tid, words);
    }
    __device__ __forceinline__ void pin() { scales.pin(); }
    __device__ __forceinline__ int take(Feed<FM, false, QX> &feed) {
        if (place >= walk.total) return 0;
        tile = walk.get(a, place, words);
        if (tile.fm != FM) return 2;
        rows_feed<T>(feed, a, tile, tid);
        return 1;
    }
    __device__ __forceinline__ void other(int slab, uint32_t at) const { rows_issue<T, QX>(a, tile, slab, at, tid); }
};

// The tiles of height FM that follow each other in the walk, `st.tile` on.  Returns whether one of another height follows.
template <class T, bool QX, class OUT, int FM>
__device__ __forceinline__ bool rows_run(const RowsArgs &a, const Walk &walk, RowsState &st, char *lds, int tid) {
    Feed<FM, false, QX> feed;
    rows_feed<T>(feed, a, st.tile, tid);
    char *scratch = lds + kScratchOff + uniform(tid >> 6) * kScratchBytes;
    while (true) {
        typename T::Acc acc[4][FM];
        Scales<T, FM> scales;
        scales.load(a, st.tile, tid);
        RowsNext<T, QX, OUT, FM> next{a, walk, scales, reinterpret_cast<int *>(lds + kScratchOff), tid, walk_place(++st.turn), Tile()};
        const int kind = contract<T>(acc, feed, lds, tid, st.stage, next);
        scales.keep(scratch, tid & 63);
        store_tile<T, OUT, FM>(acc, scales, lds, a.out + st.tile.row0 * a.out_pitch + (int64_t)st.tile.col0 * Pack<OUT>::kBytes, a.out_pitch,
                               st.tile.live, a.cols - st.tile.col0, a.once, tid);
        st.tile = next.tile;
        if (kind != 1) return kind != 0;
    }
}

template <class T, bool QX, class OUT>
__global__ __launch_bounds__(kThreads, 1) void grouped_mm_kernel(RowsArgs a) {
    __shared__ __attribute__((aligned(1024))) char lds[kLdsBytes];
    const int tid = threadIdx.x;
    int *words = reinterpret_cast<int *>(lds + kScratchOff);
    Walk walk;
    walk.setup(a, tid, words);
    const int place = walk_place(0);
    if (place >= walk.total) return;
    walk.post(place, tid, words);
    ring::all_read();
    RowsState st{walk.get(a, place, words), 0, 0};
    const uint32_t at = ring::lds_addr(lds) + uniform(tid >> 6) * 1024;
    rows_issue<T, QX>(a, st.tile, 0, at, tid);
    rows_issue<T, QX>(a, st.tile, 1, at + kStageStride, tid);
    wait_copies<Geo<1>::kCopies>();
    bool more = true;
    while (more) {
        switch (st.tile.fm) {
            case 1: more = rows_run<T, QX, OUT, 1>(a, walk, st, lds, tid); break;
            case 2: more = rows_run<T, QX, OUT, 2>(a, walk, st, lds, tid); break;
            case 3: more = rows_run<T, QX, OUT, 3>(a, walk, st, lds, tid); break;
            default: more = rows_run<T, QX, OUT, 4>(a, walk, st, lds, tid); break;
        }
    }
}

// ------------------------------------------------------------------------------- gradient of the weights

struct Place {
    int group, begin, rows;  // of x and dy
    int row0, col0;          // of the tile in dw[group]
};

// Walk over the tiles of all groups: [group, the longest first][8 column tiles][row tile][column tile].  The longest first, as
// a tile's time is that of its group's rows (up to kThreads groups; thread i holds the rank of group i).
struct WgradWalk {
    int row_tiles, col_tiles, per, total, rank;

    static __device__ __forceinline__ int end(const WgradArgs &a, int g) { return min(max(a.offsets[g], 0), a.rows); }
    template <int FM>
    __device__ __forceinline__ void setup(const WgradArgs &a, int tid, int *words) {
        row_tiles = (a.out_rows + 64 * FM - 1) / (64 * FM);
        col_tiles = (a.cols + kCols - 1) / kCols;
        per = row_tiles * col_tiles;
        total = per * a.n_groups;
        rank = -1;
        if (a.n_groups <= kThreads) {
            const int mine = tid < a.n_groups ? end(a, tid) - (tid == 0 ? 0 : end(a, tid - 1)) : 0;
            words[8 + tid] = mine;
            ring::all_read();
            rank = 0;
            for (int g = 0; g < a.n_groups; ++g) {
                const int v = words[8 + g];
                rank += v > mine || (v == mine && g < tid) ? 1 : 0;
            }
            ring::all_read();  // the words may be written again
        }
    }
    __device__ __forceinline__ void post(const WgradArgs &a, int t, int tid, int *words) const {
        if (rank == t / per && tid < a.n_groups) words[0] = tid;
    }
    template <int FM>
    __device__ __forceinline__ Place get(const WgradArgs &a, int t, const int *words) const {
        Place p;
        const int turn = t / per, local = t - turn * per, band = local / (row_tiles * kWalkCols);
        const int width = min(kWalkCols, col_tiles - band * kWalkCols), rem = local - band * row_tiles * kWalkCols;
        p.group = a.n_groups <= kThreads ? uniform(words[0]) : turn;
        p.row0 = rem / width * (64 * FM);
        p.col0 = (band * kWalkCols + rem % width) * kCols;
        p.begin = uniform(p.group == 0 ? 0 : end(a, p.group - 1));
        p.rows = uniform(max(end(a, p.group) - p.begin, 0));
        return p;
    }
};

template <class T, int FM>
__device__ __forceinline__ void wgrad_feed(Feed<FM, true, true> &feed, const WgradArgs &a, const Place &p, int tid) {
    feed.p.setup(tid, a.dy + p.begin * a.dy_pitch + p.row0 * T::kBytes, a.dy_pitch, min(64 * FM, a.out_rows - p.row0));
    feed.q.setup(tid, a.x + p.begin * a.x_pitch + p.col0 * T::kBytes, a.x_pitch, min(kCols, a.cols - p.col0));
    feed.set_length(p.rows, T::kBytes);
    feed.set_ahead(tid, a.dy_pitch, min(64 * FM, a.out_rows - p.row0), a.x_pitch, min(kCols, a.cols - p.col0));
}

template <class T, int FM>
struct WgradNext {
    const WgradArgs &a;
    const WgradWalk &walk;
    int *words;
    int tid, t;
    Place place;  // the next one, behind take()

    __device__ __forceinline__ void post() const {
        if (t < walk.total) walk.post(a, t, tid, words);
    }
    __device__ __forceinline__ void pin() {}
    __device__ __forceinline__ int take(Feed<FM, true, true> &feed) {
        if (t >= walk.total) return 0;
        place = walk.template get<FM>(a, t, words);
        wgrad_feed<T>(feed, a, place, tid);
        return 1;
    }
    __device__ __forceinline__ void other(int, uint32_t) const {}
};

template <class T, int FM>
__global__ __launch_bounds__(kThreads, 1) void grouped_mm_wgrad_kernel(WgradArgs a) {
    __shared__ __attribute__((aligned(1024))) char lds[kLdsBytes];
    const int tid = threadIdx.x;
    int *words = reinterpret_cast<int *>(lds + kScratchOff);
    int turn = 0;
    if (walk_place(0) >= (a.out_rows + 64 * FM - 1) / (64 * FM) * ((a.cols + kCols - 1) / kCols) * a.n_groups) return;
    WgradWalk walk;
    walk.setup<FM>(a, tid, words);
    walk.post(a, walk_place(0), tid, words);
    ring::all_read();
    Place p = walk.get<FM>(a, walk_place(0), words);
    Feed<FM, true, true> feed;
    wgrad_feed<T>(feed, a, p, tid);
    const uint32_t at = ring::lds_addr(lds) + uniform(tid >> 6) * 1024;
    feed.issue_all(tid, at, 0);
    feed.issue_all(tid, at + kStageStride, 1);
    wait_copies<Geo<FM>::kCopies>();
    uint32_t stage = 0;
    while (true) {
        typename T::Acc acc[4][FM];
        WgradNext<T, FM> next{a, walk, words, tid, walk_place(++turn), Place()};
        const int kind = contract<T>(acc, feed, lds, tid, stage, next);
        const int64_t pitch = (int64_t)a.cols * T::kBytes;
        store_tile<T, T, FM>(acc, Scales<T, FM>(), lds, a.dw + ((int64_t)p.group * a.out_rows + p.row0) * pitch + (int64_t)p.col0 * T::kBytes,
                             pitch, a.out_rows - p.row0, a.cols - p.col0, a.once, tid);
        p = next.place;
        if (kind == 0) return;
    }
}

}  // namespace gmm
}  // namespace pmoe
