// Runs the walks over tiles (struct Walk, struct WgradWalk) on the CPU: 256 coroutines as the threads of a workgroup, the
// lanes of a wave in step at every shuffle, the waves in any order between two barriers.  What a wave reads from the shared
// words between two barriers must not depend on that order.
// walk.inc (cut out of csrc by the test) holds the walks themselves.
#include <ucontext.h>

#include <algorithm>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <functional>
#include <memory>
#include <vector>

#define __device__
#define __forceinline__ inline

namespace {

constexpr int kLanes = 64, kN = 256, kStack = 128 << 10;

struct Dim {
    int x, y, z;
} threadIdx, blockIdx, gridDim;

struct Thread {
    ucontext_t ctx;
    std::unique_ptr<char[]> stack;
    bool done = false;
    int barriers = 0, shuffles = 0;
    int posted[2];  // what it gave to its last two shuffles
};
std::vector<Thread> threads;
ucontext_t scheduler;
int current;
std::function<void(int)> body;

void yield() { swapcontext(&threads[current].ctx, &scheduler); }
void entry() {
    body(current);
    threads[current].done = true;
    yield();
}
// The value that lane `from` gives to this shuffle: every lane of the wave has to be there.
int exchange(int v, const std::function<int(int)> &from) {
    const int me = current, wave = me / kLanes;
    Thread &t = threads[me];
    const int n = t.shuffles++;
    t.posted[n & 1] = v;
    yield();  // a round of the wave: every lane posts, then every lane reads
    for (int l = 0; l < kLanes; ++l)
        if (threads[wave * kLanes + l].shuffles < n + 1 || threads[wave * kLanes + l].shuffles > n + 2) {
            std::fprintf(stderr, "the lanes of a wave disagree on their shuffles\n");
            std::exit(3);
        }
    return threads[wave * kLanes + from(me % kLanes)].posted[n & 1];
}
int __shfl_up(int v, int d, int) { return exchange(v, [=](int l) { return l >= d ? l - d : l; }); }
int __shfl_xor(int v, int d, int) { return exchange(v, [=](int l) { return l ^ d; }); }
int first_lane(int v) { return exchange(v, [](int) { return 0; }); }
#define __builtin_amdgcn_readfirstlane first_lane

void barrier() {
    const int wanted = ++threads[current].barriers;
    while (true) {
        yield();
        int least = wanted;
        for (const Thread &t : threads)
            if (!t.done) least = std::min(least, t.barriers);
        if (least >= wanted) return;
    }
}

// Runs `f` as all threads.  `order`: the waves' between barriers, each as far as it comes before the next one moves.
void run(const int *order, std::function<void(int)> f) {
    body = std::move(f);
    threads = std::vector<Thread>(kN);
    for (Thread &t : threads) {
        t.stack.reset(new char[kStack]);
        getcontext(&t.ctx);
        t.ctx.uc_stack.ss_sp = t.stack.get();
        t.ctx.uc_stack.ss_size = kStack;
        t.ctx.uc_link = &scheduler;
        makecontext(&t.ctx, entry, 0);
    }
    auto state = [](int wave) {
        long s = 0;
        for (int l = 0; l < kLanes; ++l) {
            const Thread &t = threads[wave * kLanes + l];
            s += t.shuffles + 1000000l * t.barriers + (t.done ? 1000000000l : 0);
        }
        return s;
    };
    for (int idle = 0; idle < 3;) {
        bool moved = false, all = true;
        for (int w = 0; w < kN / kLanes; ++w) {
            const int wave = order[w];
            // until the wave stands still: at a barrier, or at its end (a shuffle takes two rounds)
            for (long seen = -1, still = 0; still < 2;) {
                for (int l = 0; l < kLanes; ++l) {
                    current = wave * kLanes + l;
                    threadIdx = {current, 0, 0};
                    if (!threads[current].done) swapcontext(&scheduler, &threads[current].ctx);
                }
                const long s = state(wave);
                moved |= s != seen && seen >= 0;
                still = s == seen ? still + 1 : 0;
                seen = s;
            }
            for (int l = 0; l < kLanes; ++l) all &= threads[wave * kLanes + l].done;
        }
        if (all) return;
        idle = moved ? 0 : idle + 1;
    }
    std::fprintf(stderr, "waves wait at a barrier that others do not reach\n");
    std::exit(4);
}

using std::max;
using std::min;
namespace ring {
void all_read() { barrier(); }
}  // namespace ring

#include "walk.inc"

const int kOrders[][4] = {{0, 1, 2, 3}, {3, 2, 1, 0}, {1, 0, 3, 2}, {2, 3, 0, 1}, {0, 3, 1, 2}};
constexpr int kPoison = 0x5a5a5a5a;

[[noreturn]] void fail(const char *what, long a = 0, long b = 0) {
    std::fprintf(stderr, "%s (%ld, %ld)\n", what, a, b);
    std::exit(1);
}

// Walks over the tiles of `ends` and checks that they cover every row of its group, and every column, once.
void check_rows(const std::vector<int32_t> &ends, int rows, int cols, int grid, bool fills, const int *order, bool covered) {
    RowsArgs a = {};
    a.offsets = ends.data();
    a.n_groups = (int)ends.size();
    a.rows = rows;
    a.cols = cols;
    a.fills = fills;
    gridDim = {grid, 1, 1};
    std::vector<int> words(64, kPoison);
    std::vector<Walk> walks(kN);
    run(order, [&](int tid) { walks[tid].setup(a, tid, words.data()); });
    int far = 0;
    for (int32_t e : ends) far = max(far, min(max((int)e, 0), rows));
    for (int t = 0; t < kN; ++t) {
        if (walks[t].live_rows != far) fail("live rows: thread, rows", t, walks[t].live_rows);
        if (walks[t].total != walks[0].total || walks[t].row_tiles != walks[0].row_tiles || walks[t].shift != walks[0].shift)
            fail("the threads disagree on the walk: thread, tiles", t, walks[t].total);
    }
    if (!covered) return;
    // a group's rows begin at the furthest end in front of it
    std::vector<int> begin(ends.size()), end(ends.size()), next(ends.size());
    int at = 0;
    for (size_t g = 0; g < ends.size(); ++g) {
        begin[g] = at;
        at = end[g] = max(at, min(max((int)ends[g], 0), rows));
    }
    const int col_tiles = (cols + kCols - 1) / kCols;
    std::vector<std::vector<int>> seen(ends.size());  // first rows of the tiles of a group's first column
    int zero = far;
    for (int t = 0; t < walks[0].total; ++t) {
        // (one thread at a time: post() has no shuffle, and exactly one thread may answer)
        for (int w = 0; w < 4; ++w) words[w] = kPoison;
        int answers = 0;
        for (int tid = 0; tid < kN; ++tid) {
            const int before = words[0];
            words[0] = kPoison;
            walks[tid].post(t, tid, words.data());
            if (words[0] != kPoison) ++answers;
            else words[0] = before;
        }
        if (t >= walks[0].row_tiles * col_tiles) {  // rows behind the last group
            const int local = t - walks[0].row_tiles * col_tiles, m = local / col_tiles;
            if (answers) fail("a tile behind the last group is somebody's", t);
            if (far + m * 256 >= rows) fail("a tile behind the last row", t);
            zero = max(zero, min(rows, far + m * 256 + 256));
            continue;
        }
        const int g = words[0], row0 = words[1], live = words[2], col = words[3];
        if (answers != 1) fail("threads that answer for a tile", t, answers);
        if (g < 0 || g >= (int)ends.size()) fail("a group that is none", t, g);
        if (row0 < begin[g] || live <= 0 || live > 256 || row0 > end[g] - live) fail("rows outside of the group", t, row0);
        if (col < 0 || col >= col_tiles) fail("a column tile that is none", t, col);
        if (col == 0) {
            seen[g].push_back(row0);
            next[g] += live;
        }
    }
    if (zero != rows) fail("rows behind the last group are left out", zero, rows);
    for (size_t g = 0; g < ends.size(); ++g) {
        std::sort(seen[g].begin(), seen[g].end());
        if (next[g] != end[g] - begin[g] || std::adjacent_find(seen[g].begin(), seen[g].end()) != seen[g].end())
            fail("rows of a group that are left out or taken twice", (long)g, next[g]);
    }
}

void check_wgrad(const std::vector<int32_t> &ends, int rows, int out_rows, int cols, const int *order) {
    WgradArgs a = {};
    a.offsets = ends.data();
    a.n_groups = (int)ends.size();
    a.rows = rows;
    a.out_rows = out_rows;
    a.cols = cols;
    std::vector<int> words(1024, kPoison);
    std::vector<WgradWalk> walks(kN);
    run(order, [&](int tid) { walks[tid].setup<4>(a, tid, words.data()); });
    if (a.n_groups > kN) return;  // the groups in their own order
    std::vector<int> rank(ends.size(), 0);
    for (int g = 0; g < a.n_groups; ++g) {
        if (walks[g].rank < 0 || walks[g].rank >= a.n_groups || rank[walks[g].rank]++) fail("ranks of the groups", g, walks[g].rank);
    }
}

}  // namespace

int main(int argc, char **argv) {
    const bool huge = argc > 1;
    if (huge) {  // the largest groups that the entry points take
        const int most = INT32_MAX - 512;
        for (int rows : {most, most - 1, most - 255, 2139127681, 2139127680, 1 << 30})
            for (const int *order : {kOrders[0]}) {
                RowsArgs a = {};
                const int32_t end = rows;
                a.offsets = &end;
                a.n_groups = 1;
                a.rows = rows;
                a.cols = 8;
                a.fills = true;
                gridDim = {256, 1, 1};
                std::vector<int> words(64, kPoison);
                std::vector<Walk> walks(kN);
                run(order, [&](int tid) { walks[tid].setup(a, tid, words.data()); });
                const int tiles = (int)(((int64_t)rows + 255) / 256);
                if (walks[0].total != tiles) fail("tiles of a long group", rows, walks[0].total);
                for (int t : {0, 1, tiles / 2, tiles - 2, tiles - 1}) {
                    walks[0].post(t, 0, words.data());
                    if (words[1] != t * 256 || words[2] != min(256, rows - t * 256)) fail("a tile of a long group", t, words[1]);
                }
            }
        return 0;
    }
    std::srand(1);
    for (const auto &order : kOrders)
        for (int trial = 0; trial < 24; ++trial) {
            static const int sizes[] = {1, 2, 3, 8, 37, 65, 128, 257, 1000, 1024};
            const int n = sizes[trial % 10], most = trial % 3 == 0 ? 5 : trial % 3 == 1 ? 90 : 700;
            std::vector<int32_t> ends(n);
            int at = 0;
            for (int g = 0; g < n; ++g) ends[g] = at += std::rand() % 3 ? std::rand() % (n > 300 ? min(most, 40) : most) : 0;
            const int rows = at + std::rand() % 600;
            for (int cols : {8, 264, 2400})
                for (int grid : {8, 256})
                    check_rows(ends, rows, cols, grid, rows / 128 * ((cols + 255) / 256) > grid, order, true);
            check_wgrad(ends, rows, 520, 264, order);
        }
    // ends that are none: every thread still sees one walk, inside the rows
    for (const auto &order : kOrders) {
        for (const std::vector<int32_t> &ends : {std::vector<int32_t>{50, 20, 120, 90}, std::vector<int32_t>{-7, -1, 1 << 30, 3},
                                                 std::vector<int32_t>{INT32_MAX, INT32_MIN, 0, 60}})
            check_rows(ends, 100, 40, 8, false, order, true), check_wgrad(ends, 100, 40, 64, order);
    }
    return 0;
}
