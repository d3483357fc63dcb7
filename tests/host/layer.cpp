// Runs the whole layer for a few tokens (csrc/moe_layer.hip and what it includes) on the CPU: the host code as it is, its kernels with
// a coroutine for every thread.  The lanes of a wave go in step at every operation across lanes; waves and workgroups take turns at random, a
// limited number of workgroups being resident at a time, the others in line behind them.
//
// What is checked: every buffer ends in front of a page that cannot be touched, arrays of known length are checked by the compiler's traps
// (see the test that builds this); LDS and the workspace hold garbage at first; a cached load of the activation may be as old as the kernel; every
// wait ends; the outputs are the layer's.
// layer.inc (made from csrc by the test) holds the sources themselves.
#include <signal.h>
#include <sys/mman.h>
#include <unistd.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <functional>
#include <memory>
#include <random>
#include <type_traits>
#include <utility>
#include <vector>

#include "prime_moe_hip.h"

#define __device__
#define __host__
#define __global__
#define __forceinline__ inline
#define __launch_bounds__(...)
#define hipLaunchKernelGGL(f, grid, block, lds, stream, ...) emu::launch([=] { f(__VA_ARGS__); }, grid, block)
#define PMOE_REQUIRE(cond, ...) do { if (!(cond)) { std::fprintf(stderr, __VA_ARGS__); return 1; } } while (0)
#define PMOE_REQUIRE_ALIGNED(...) do {} while (0)

// ---- conversions that the compiler calls

extern "C" float __extendhfsf2(_Float16 h) {
    const uint16_t b = __builtin_bit_cast(uint16_t, h);
    const uint32_t sign = (uint32_t)(b & 0x8000) << 16, e = b >> 10 & 31, m = b & 0x3ff;
    if (e == 0) return (sign ? -1.f : 1.f) * std::ldexp((float)m, -24);
    return __builtin_bit_cast(float, sign | (e == 31 ? 255u : e + 112u) << 23 | m << 13);
}
extern "C" _Float16 __truncsfhf2(float f) {
    const uint32_t b = __builtin_bit_cast(uint32_t, f), sign = b >> 16 & 0x8000;
    const float a = std::fabs(f);
    uint32_t r;
    if (f != f) r = 0x7e00;
    else if (a >= 65520.f) r = 0x7c00;
    else if (a < 0x1p-14f) r = (uint32_t)std::nearbyint(a * 0x1p24f);
    else r = ((b & 0x7fffffff) - (112u << 23) + 0xfff + (b >> 13 & 1)) >> 13;
    return __builtin_bit_cast(_Float16, (uint16_t)(r | sign));
}
static uint16_t to_bf16(float f) {
    const uint32_t b = __builtin_bit_cast(uint32_t, f);
    return f != f ? 0x7fc0 : (uint16_t)((b + 0x7fff + (b >> 16 & 1)) >> 16);
}
static float from_bf16(uint16_t v) { return __builtin_bit_cast(float, (uint32_t)v << 16); }
static float from_f16(uint16_t v) { return __extendhfsf2(__builtin_bit_cast(_Float16, v)); }

// ---- threads

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
struct dim3 {
    uint32_t x, y, z;
    dim3(uint32_t a = 1, uint32_t b = 1, uint32_t c = 1) : x(a), y(b), z(c) {}
};
static dim3 threadIdx, blockIdx, gridDim;
struct uint2 { uint32_t x, y; };
typedef void *hipStream_t;

[[noreturn]] static void fail(const char *what) {
    std::fprintf(stderr, "%s\n", what);
    _exit(1);
}

// Saves what a call keeps and goes over to another stack.
extern "C" void switch_stacks(void **from, void *to);
asm(".text\n.globl switch_stacks\nswitch_stacks:\n"
    "push %rbp\npush %rbx\npush %r12\npush %r13\npush %r14\npush %r15\nmov %rsp, (%rdi)\nmov %rsi, %rsp\n"
    "pop %r15\npop %r14\npop %r13\npop %r12\npop %rbx\npop %rbp\nret\n");

namespace emu {

constexpr int kLanes = 64;
constexpr size_t kStack = 96 << 10;
enum State { kReady, kExchange, kDivergent, kBarrier, kAsleep, kDone };
struct Lane {
    void *sp;
    State state;
};
struct Wave {
    Lane lanes[kLanes];
    int ready = kLanes;
    uint64_t given = 0;             // of the last exchange: the lanes that were there and gave something other than 0
    alignas(16) char posted[kLanes][32], seen[kLanes][32];
};
struct Group {
    dim3 block;
    std::vector<Wave> waves;
    std::vector<char> lds[3];
    char *stacks;
};

static std::mt19937 rng;
static void *scheduler;
static Group *group;
static Wave *wave;
static int lane;
static std::function<void()> *body;
static int resident = 4;

static void wait(State s) {
    Lane &l = wave->lanes[lane];
    l.state = s;
    --wave->ready;
    switch_stacks(&l.sp, scheduler);
}
static void entry() {
    (*body)();
    wait(kDone);
    fail("a thread went on behind its end");
}

// Every lane of the wave that is there gives `v` and gets those of all (until the next exchange).
template <class V>
struct Given {
    V operator[](int l) const {
        V v;
        std::memcpy(&v, wave->seen[l], sizeof v);
        return v;
    }
};
template <class V>
static Given<V> exchange(const V &v, State how = kExchange) {
    static_assert(sizeof(V) <= 32, "fits a slot");
    std::memcpy(wave->posted[lane], &v, sizeof v);
    wait(how);
    return {};
}

// Lets the lanes of a wave run until all of them wait.
static void run(Group &g, int w) {
    group = &g;
    wave = &g.waves[w];
    blockIdx = g.block;
    for (int l = 0; l < kLanes; ++l)
        if (wave->lanes[l].state == kReady) {
            lane = l;
            threadIdx = dim3(w * kLanes + l, 0, 0);
            switch_stacks(&scheduler, wave->lanes[l].sp);
        }
}
static void wake(Wave &w, int l) { w.lanes[l].state = kReady, ++w.ready; }

// A step of a wave; whether it did more than to sleep.
static bool step(Group &g, int n) {
    Wave &w = g.waves[n];
    if (w.ready == 0) {
        uint64_t at[kDone + 1] = {};
        for (int l = 0; l < kLanes; ++l) at[w.lanes[l].state] |= 1ull << l;
        const uint64_t how = at[kAsleep] ? at[kAsleep] : at[kDivergent] ? at[kDivergent] : at[kExchange];
        if (how == 0) return false;  // at a barrier or at its end
        if (at[kAsleep] == 0 && at[kDivergent] == 0 && (at[kBarrier] | at[kDone]) != 0) fail("lanes of a wave are at an exchange that others have passed");
        if (at[kAsleep] == 0) {
            std::memcpy(w.seen, w.posted, sizeof w.seen);
            w.given = 0;
            for (int l = 0; l < kLanes; ++l) w.given |= (uint64_t)(w.seen[l][0] != 0 && (how >> l & 1)) << l;
        }
        for (int l = 0; l < kLanes; ++l)
            if (how >> l & 1) wake(w, l);
        run(g, n);
        return at[kAsleep] == 0;
    }
    run(g, n);
    return true;
}
static bool ended(const Group &g) {
    for (const Wave &w : g.waves)
        for (const Lane &l : w.lanes)
            if (l.state != kDone) return false;
    return true;
}
static void barrier(Group &g) {
    for (const Wave &w : g.waves)
        for (const Lane &l : w.lanes)
            if (l.state != kBarrier && l.state != kDone) return;
    for (Wave &w : g.waves)
        for (int l = 0; l < kLanes; ++l)
            if (w.lanes[l].state == kBarrier) wake(w, l);
}

static std::unique_ptr<Group> start(dim3 block, int threads) {
    std::unique_ptr<Group> g(new Group);
    g->block = block;
    g->waves = std::vector<Wave>(threads / kLanes);
    g->stacks = static_cast<char *>(mmap(nullptr, kStack * threads, PROT_READ | PROT_WRITE, MAP_PRIVATE | MAP_ANONYMOUS | MAP_NORESERVE, -1, 0));
    if (g->stacks == MAP_FAILED) fail("no memory for the stacks");
    for (int t = 0; t < threads; ++t) {
        void **top = reinterpret_cast<void **>(g->stacks + kStack * (t + 1) - 16);
        *--top = nullptr;  // (entry never returns)
        *--top = reinterpret_cast<void *>(entry);
        for (int i = 0; i < 6; ++i) *--top = nullptr;
        g->waves[t / kLanes].lanes[t % kLanes] = {top, kReady};
    }
    return g;
}

static void launch(std::function<void()> f, dim3 grid, dim3 block) {
    body = &f;
    gridDim = grid;
    std::vector<std::unique_ptr<Group>> here;
    const int total = (int)(grid.x * grid.y), threads = (int)block.x;
    int next = 0, idle = 0;
    while (next < total || !here.empty()) {
        while ((int)here.size() < resident && next < total) here.push_back(start(dim3(next % grid.x, next / grid.x, 0), threads)), ++next;
        const size_t i = rng() % here.size();
        Group &g = *here[i];
        bool moved = false;
        for (int n = 0; n < (int)g.waves.size(); ++n) moved |= step(g, (int)(rng() % g.waves.size()));
        barrier(g);
        for (const Wave &w : g.waves) moved |= w.ready > 0;
        if (ended(g)) {
            munmap(g.stacks, kStack * threads);
            here.erase(here.begin() + (long)i);
            moved = true;
        }
        idle = moved ? 0 : idle + 1;
        if (idle > 20000) fail("workgroups wait for what nobody does");
    }
}

// LDS of the workgroup, garbage at first.
template <class V>
static V &shared(int which) {
    std::vector<char> &m = group->lds[which];
    if (m.empty()) {
        m.resize(sizeof(V) + 1024);
        for (char &c : m) c = (char)rng();
    }
    return *reinterpret_cast<V *>((reinterpret_cast<uintptr_t>(m.data()) + 1023) / 1024 * 1024);
}

// ---- memory: in front of a page that cannot be touched, and behind one

struct Buffer {
    char *data;
    size_t bytes;
    std::vector<char> before, behind;  // of its own pages, to be left alone
    char *begin, *end;
    Buffer(size_t n, size_t align) : bytes(n) {
        const size_t page = 4096, size = (n + align + page - 1) / page * page;
        char *m = static_cast<char *>(mmap(nullptr, size + 2 * page, PROT_READ | PROT_WRITE, MAP_PRIVATE | MAP_ANONYMOUS, -1, 0));
        if (m == MAP_FAILED) fail("no memory");
        mprotect(m, page, PROT_NONE);
        mprotect(m + page + size, page, PROT_NONE);
        begin = m + page, end = begin + size;
        data = reinterpret_cast<char *>(reinterpret_cast<uintptr_t>(end - n) / align * align);
        for (char *p = begin; p < end; ++p) *p = (char)rng();
        before.assign(begin, data), behind.assign(data + n, end);
    }
    void check() const {
        if (std::memcmp(begin, before.data(), before.size()) != 0 || std::memcmp(data + bytes, behind.data(), behind.size()) != 0) fail("a store beside a buffer");
    }
};
static const char *act_begin, *act_end;

}  // namespace emu

// ---- what kernels call

static void __syncthreads() { emu::wait(emu::kBarrier); }
static uint64_t ballot_of(bool v, emu::State how) {
    emu::exchange((char)v, how);
    return emu::wave->given;
}
static uint64_t __ballot(bool v) { return ballot_of(v, emu::kExchange); }
static uint64_t divergent_ballot(bool v) { return ballot_of(v, emu::kDivergent); }
template <class V>
static V __shfl(V v, int from, int) { return emu::exchange(v)[from]; }
template <class V>
static V __shfl_xor(V v, int d, int) {
    const emu::Given<V> all = emu::exchange(v);
    return all[emu::lane ^ d];
}
static int emu_readlane(int v, int from) { return emu::exchange(v)[from]; }
static int emu_readfirstlane(int v) { return emu::exchange(v)[0]; }
static int emu_update_dpp(int old, int v, int ctrl, int rows, int, bool bound) {
    const emu::Given<int> all = emu::exchange(v);
    const int l = emu::lane, row = l / 16;
    int from = -1;
    if (ctrl < 0x100) from = l / 4 * 4 + (ctrl >> l % 4 * 2 & 3);
    else if (ctrl > 0x110 && ctrl < 0x120) from = l % 16 >= ctrl - 0x110 ? l - (ctrl - 0x110) : -1;
    else if (ctrl == 0x140) from = row * 16 + 15 - l % 16;
    else if (ctrl == 0x141) from = l / 8 * 8 + 7 - l % 8;
    else if (ctrl == 0x142) from = row > 0 ? row * 16 - 1 : -1;
    else if (ctrl == 0x143) from = l >= 32 ? 31 : -1;
    else fail("an unknown move across lanes");
    if (!(rows >> row & 1)) return old;
    return from < 0 ? (bound ? 0 : old) : all[from];
}
static void emu_fence(int, const char *) {}
static void emu_wave_barrier() { emu::exchange((char)0); }
static void emu_s_sleep(int) { emu::wait(emu::kAsleep); }
static float emu_rcpf(float v) { return 1.0f / v; }
static float emu_fmed3f(float a, float b, float c) { return std::max(std::min(a, b), std::min(std::max(a, b), c)); }
static uint32_t emu_atomic_inc32(uint32_t *p, uint32_t most, int, const char *) {
    const uint32_t v = *p;
    *p = v >= most ? 0 : v + 1;
    return v;
}
#undef __HIP_MEMORY_SCOPE_WORKGROUP
#undef __HIP_MEMORY_SCOPE_AGENT
#define __HIP_MEMORY_SCOPE_WORKGROUP 0
#define __HIP_MEMORY_SCOPE_AGENT 0
template <class V, class U>
static void emu_hip_store(V *p, U v, int, int) { *p = (V)v; }
template <class V>
static V emu_hip_load(const V *p, int, int) { return *p; }
template <class V, class U>
static V emu_hip_fetch_add(V *p, U v, int, int) { const V old = *p; *p += (V)v; return old; }
static int atomicAdd(int *p, int v) { const int old = *p; *p += v; return old; }
static uint32_t atomicOr(uint32_t *p, uint32_t v) { const uint32_t old = *p; *p |= v; return old; }
static int __popc(uint32_t v) { return __builtin_popcount(v); }
#define __expf(v) std::exp(v)
static float __int_as_float(int v) { return __builtin_bit_cast(float, v); }
static int __float_as_int(float v) { return __builtin_bit_cast(int, v); }
static float __uint_as_float(uint32_t v) { return __builtin_bit_cast(float, v); }
static uint32_t __float_as_uint(float v) { return __builtin_bit_cast(uint32_t, v); }
using std::max;
using std::min;

// A load by a buffer: inside what the buffer says that it holds, at a multiple of 16.  `aux` 16: past the caches.
struct emu_rsrc {
    const char *base;
    uint32_t bytes;
};
static emu_rsrc emu_make_buffer_rsrc(char *p, int, int bytes, int) { return {p, (uint32_t)bytes}; }
static i32x4 emu_raw_buffer_load_b128(emu_rsrc b, uint32_t at, uint32_t more, int aux) {
    const uint64_t offset = (uint64_t)at + more;
    if (offset + 16 > b.bytes) fail("a load behind the end of its buffer");
    const char *p = b.base + offset;
    if (reinterpret_cast<uintptr_t>(p) % 16 != 0) fail("a load that is not aligned");
    i32x4 v;
    std::memcpy(&v, p, 16);
    if (aux != 16 && p >= emu::act_begin && p < emu::act_end && emu::rng() % 3 == 0) v = i32x4{-1, -1, -1, -1};
    return v;
}

template <class V>
static float emu_fdot2_f32_bf16(V a, V b, float c, bool) {
    const uint32_t x = __builtin_bit_cast(uint32_t, a), y = __builtin_bit_cast(uint32_t, b);
    return from_bf16((uint16_t)x) * from_bf16((uint16_t)y) + from_bf16((uint16_t)(x >> 16)) * from_bf16((uint16_t)(y >> 16)) + c;
}
template <class V>
static float emu_fdot2(V a, V b, float c, bool) {
    const uint32_t x = __builtin_bit_cast(uint32_t, a), y = __builtin_bit_cast(uint32_t, b);
    return from_f16((uint16_t)x) * from_f16((uint16_t)y) + from_f16((uint16_t)(x >> 16)) * from_f16((uint16_t)(y >> 16)) + c;
}

namespace pmoe {
namespace gmm {
struct Bf16 {};
struct F16 {};
namespace few {
// 16 x 16 x 32: lane l holds row l % 16 of both, columns 8 (l / 16) .. + 7; element (m = 4 (l / 16) + i, n = l % 16).
template <class T>
struct Mini {
    static f32x4 mfma(i32x4 a, i32x4 b, f32x4 c) {
        struct Pair {
            i32x4 a, b;
        };
        const emu::Given<Pair> all = emu::exchange(Pair{a, b});
        auto value = [](const i32x4 &v, int k) {
            const uint16_t bits = (uint16_t)((uint32_t)v[k / 2] >> k % 2 * 16);
            return std::is_same<T, Bf16>::value ? from_bf16(bits) : from_f16(bits);
        };
        const int n = emu::lane % 16;
        for (int i = 0; i < 4; ++i) {
            double sum = c[i];
            for (int q = 0; q < 4; ++q)
                for (int k = 0; k < 8; ++k) sum += (double)value(all[4 * (emu::lane / 16) + i + 16 * q].a, k) * value(all[n + 16 * q].b, k);
            c[i] = (float)sum;
        }
        return c;
    }
};
}  // namespace few
}  // namespace gmm
int compute_units = 8;
int resident_grid() { return compute_units; }
int check_launch(const char *) { return 0; }
size_t align_up(size_t v, size_t a) { return (v + a - 1) / a * a; }
}  // namespace pmoe

#include "layer.inc"

// ---- a layer and its outputs in 64 bits

int main(int argc, char **argv) {
    if (argc != 12) fail("usage: group dtype T K H E top_k crowd compute_units resident seed");
    const int group = std::atoi(argv[1]), dtype = std::atoi(argv[2]), T = std::atoi(argv[3]), K = std::atoi(argv[4]), H = std::atoi(argv[5]), E = std::atoi(argv[6]),
              top_k = std::atoi(argv[7]), crowd = std::atoi(argv[8]);
    pmoe::compute_units = std::atoi(argv[9]);
    emu::resident = std::atoi(argv[10]);
    emu::rng.seed((unsigned)std::atoi(argv[11]));
    static char alternate[1 << 16];
    stack_t st = {};
    st.ss_sp = alternate, st.ss_size = sizeof alternate;
    sigaltstack(&st, nullptr);
    struct sigaction sa = {};
    sa.sa_flags = SA_ONSTACK;
    sa.sa_handler = [](int s) {
        const char *what = s == SIGSEGV || s == SIGBUS ? "an access outside of every buffer\n" : "an index outside of its array\n";
        (void)!write(2, what, std::strlen(what));
        _exit(1);
    };
    for (int s : {SIGSEGV, SIGBUS, SIGILL, SIGTRAP}) sigaction(s, &sa, nullptr);

    const bool half = dtype == PMOE_DTYPE_F16;
    std::mt19937 gen((unsigned)std::atoi(argv[11]));
    std::normal_distribution<float> normal;
    auto to16 = [&](float v) { return half ? __builtin_bit_cast(uint16_t, __truncsfhf2(v)) : to_bf16(v); };
    auto from16 = [&](uint16_t v) { return half ? from_f16(v) : from_bf16(v); };
    auto fill16 = [&](emu::Buffer &b, float std) {
        std::vector<float> v(b.bytes / 2);
        for (size_t i = 0; i < v.size(); ++i) {
            const uint16_t w = to16(normal(gen) * std);
            std::memcpy(b.data + 2 * i, &w, 2);
            v[i] = from16(w);
        }
        return v;
    };
    emu::Buffer x((size_t)T * K * 2, 16), gate((size_t)E * K * 2, 16), bias((size_t)E * 4, 4), out((size_t)T * K * 2, 16), ids((size_t)T * top_k * 4, 4), weights((size_t)T * top_k * 4, 4);
    const std::vector<float> xv = fill16(x, 1.f), gv = fill16(gate, 1.f / std::sqrt((float)K));
    std::vector<float> bv((size_t)E);
    for (int e = 0; e < E; ++e) bv[(size_t)e] = normal(gen) * 0.5f + (e < crowd ? 100.f : 0.f);  // (everybody takes the first `crowd`)
    std::memcpy(bias.data, bv.data(), bias.bytes);
    // a matrix of 16-bit weights, or of tiles of 4 bits and their scales; `v`: what it stands for
    struct Matrix {
        std::unique_ptr<emu::Buffer> q, s;
        std::vector<float> v;
    };
    auto matrix = [&](int rows, int cols) {
        Matrix m;
        if (group == 0) {
            m.q.reset(new emu::Buffer((size_t)E * rows * cols * 2, 16));
            m.v = fill16(*m.q, 1.f / std::sqrt((float)cols));
            return m;
        }
        const int tiles = (cols + 127) / 128, per = 128 / group;
        const size_t strips = (size_t)E * rows / 16;
        m.q.reset(new emu::Buffer(strips * tiles * 1024, 16)), m.s.reset(new emu::Buffer(strips * tiles * 16 * per * 2, 16));
        std::memset(m.q->data, 0x88, m.q->bytes), std::memset(m.s->data, 0, m.s->bytes);
        m.v.resize((size_t)E * rows * cols);
        for (size_t row = 0; row < (size_t)E * rows; ++row)
            for (int g = 0; g < cols / group; ++g) {
                const uint16_t sw = to16((0.5f + (float)(gen() % 1000) / 1000.f) * 0.2f / std::sqrt((float)cols));
                std::memcpy(m.s->data + (((row / 16 * tiles + g / per) * 16 + row % 16) * per + g % per) * 2, &sw, 2);
                for (int k = g * group; k < (g + 1) * group; ++k) {
                    const int q = (int)(gen() % 16), j = k % 128 / 32, c = k % 32 / 8, e = k % 8;
                    char &byte = m.q->data[(row / 16 * tiles + k / 128) * 1024 + 16 * (row % 16 + 16 * c) + 4 * j + 2 * (e % 2) + e / 4];
                    byte = (char)(e / 2 % 2 ? (byte & 15) | q << 4 : (byte & 0xf0) | q);
                    m.v[row * cols + k] = (float)(q - 8) * from16(sw);
                }
            }
        return m;
    };
    const Matrix w1 = matrix(2 * H, K), w2 = matrix(K, H);
    emu::Buffer ws(pmoe_moe_layer_workspace_bytes(T, H, E, top_k), 256);
    emu::act_end = ws.data + ws.bytes;
    emu::act_begin = emu::act_end - (size_t)T * top_k * 2 * (((size_t)H * 2 + 127) / 128 * 128);

    for (int turn = 0; turn < 2; ++turn) {  // twice: the second on what the first has left in the workspace
        if (pmoe_moe_layer(x.data, gate.data, reinterpret_cast<float *>(bias.data), w1.q->data, w1.s ? w1.s->data : nullptr, w2.q->data, w2.s ? w2.s->data : nullptr, group, out.data,
                           reinterpret_cast<int32_t *>(ids.data), reinterpret_cast<float *>(weights.data), T, K, H, E, top_k, dtype, ws.data, ws.bytes, nullptr) != 0)
            fail("refused");
        for (emu::Buffer *b : {&x, &gate, &bias, &out, &ids, &weights, &ws, w1.q.get(), w2.q.get()}) b->check();
        for (int t = 0; t < T; ++t) {
            std::vector<std::pair<double, int>> score((size_t)E);
            for (int e = 0; e < E; ++e) {
                double l = bv[(size_t)e];
                for (int k = 0; k < K; ++k) l += (double)xv[(size_t)t * K + k] * gv[(size_t)e * K + k];
                score[(size_t)e] = {-l, e};
            }
            std::vector<std::pair<double, int>> sorted = score;
            std::sort(sorted.begin(), sorted.end());
            double total = 0;
            for (int r = 0; r < top_k; ++r) total += std::exp(sorted[0].first - sorted[(size_t)r].first);
            std::vector<double> y((size_t)K), size((size_t)K);
            for (int r = 0; r < top_k; ++r) {
                int32_t id;
                float weight;
                std::memcpy(&id, ids.data + ((size_t)t * top_k + r) * 4, 4), std::memcpy(&weight, weights.data + ((size_t)t * top_k + r) * 4, 4);
                if (id < 0 || id >= E || std::fabs(score[(size_t)id].first - sorted[(size_t)r].first) > 1e-4) fail("another expert than the definition's");
                const double share = std::exp(sorted[0].first - score[(size_t)id].first) / total;
                if (std::fabs(share - weight) > 1e-4) fail("another weight than the definition's");
                std::vector<double> act((size_t)H);
                for (int h = 0; h < H; ++h) {
                    double g = 0, u = 0;
                    const float *gw = &w1.v[((size_t)id * 2 * H + h) * K], *uw = gw + (size_t)H * K;
                    for (int k = 0; k < K; ++k) g += (double)xv[(size_t)t * K + k] * gw[k], u += (double)xv[(size_t)t * K + k] * uw[k];
                    act[(size_t)h] = g / (1 + std::exp(-g)) * u;
                }
                for (int k = 0; k < K; ++k)
                    for (int h = 0; h < H; ++h) {
                        const double v = share * act[(size_t)h] * w2.v[((size_t)id * K + k) * H + h];
                        y[(size_t)k] += v, size[(size_t)k] += std::fabs(v);
                    }
            }
            for (int k = 0; k < K; ++k) {
                uint16_t got;
                std::memcpy(&got, out.data + ((size_t)t * K + k) * 2, 2);
                // half a step of the output's type, and 2^-10 of the magnitudes for the weights' error and fp32 sums: a column, row or piece that is
                // missing or twice there is many times that
                if (!(std::fabs(from16(got) - y[(size_t)k]) <= std::fabs(y[(size_t)k]) * (half ? 0x1p-11 : 0x1p-8) + size[(size_t)k] * 0x1p-10)) {
                    std::fprintf(stderr, "token %d column %d: %g, not %g\n", t, k, from16(got), y[(size_t)k]);
                    return 1;
                }
            }
        }
    }
    return 0;
}
