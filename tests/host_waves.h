// Runs a kernel's source on the CPU, a workgroup at a time, for what a GPU run cannot be relied on to show: a wave that reads shared
// memory behind a barrier where another wave already writes it again.  Every thread is a fibre.  The waves of a workgroup run one after the
// other, each as far as it can (to the next barrier, or to its end), in an order that the test chooses; a step over the lanes of a wave
// (DPP move, ballot, shuffle) waits for all 64 of them.  Only what sample.hip uses is here.
#pragma once
#include <ucontext.h>

#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <functional>
#include <memory>
#include <random>
#include <vector>

#define __global__
#define __device__
#define __forceinline__ inline
#define __launch_bounds__(...)
#define __shared__ static
#define __align__(n) alignas(n)
#define __HIP_MEMORY_SCOPE_AGENT 0
#define __hip_atomic_load(p, order, scope) (*(p))

struct float4 { float x, y, z, w; };
struct alignas(16) ulonglong2 { unsigned long long x, y; };
inline float4 make_float4(float x, float y, float z, float w) { return {x, y, z, w}; }
inline ulonglong2 make_ulonglong2(unsigned long long x, unsigned long long y) { return {x, y}; }
struct dim3 {
    unsigned x, y, z;
    dim3(unsigned x_ = 1, unsigned y_ = 1, unsigned z_ = 1) : x(x_), y(y_), z(z_) {}
};
inline dim3 threadIdx, blockIdx;

namespace waves {

enum State { kReady, kStep, kBarrier, kDone };
struct Lane {
    ucontext_t ctx;
    State state;
    std::unique_ptr<char[]> stack;
};
inline std::vector<Lane> lanes;
inline std::vector<unsigned long long> words;   // what each lane brings to a step over its wave's lanes
inline std::vector<unsigned long long> given;   // the same, of the step that has been completed last
inline ucontext_t back;
inline unsigned now;
inline int order;                               // 0: waves upwards, 1: downwards, else: the seed of an order by chance
inline std::function<void()> body;
constexpr size_t kStack = 64 << 10;

[[noreturn]] inline void broken(const char* what) {
    std::fprintf(stderr, "workgroup (%u, %u): %s\n", blockIdx.x, blockIdx.y, what);
    std::abort();
}
inline void entry() {
    body();
    lanes[now].state = kDone;
    swapcontext(&lanes[now].ctx, &back);
}
inline void pause(State s) {
    const unsigned me = now;
    lanes[me].state = s;
    swapcontext(&lanes[me].ctx, &back);
    now = me;
}
inline void resume(unsigned l) {
    now = l;
    threadIdx = dim3(l);
    swapcontext(&back, &lanes[l].ctx);
}
// A word from every lane of the wave: those of the 64, in order.
inline const unsigned long long* step(unsigned long long w) {
    words[now] = w;
    pause(kStep);
    return &given[now & ~63u];
}
// One wave as far as it goes.
inline void run_wave(unsigned w) {
    for (;;) {
        unsigned at_step = 0, ready = 0;
        for (unsigned l = w * 64; l < w * 64 + 64; l++) {
            if (lanes[l].state == kReady) resume(l);
            at_step += lanes[l].state == kStep;
            ready += lanes[l].state == kReady;
        }
        if (ready) broken("a fibre came back ready");
        if (at_step == 0) return;
        if (at_step != 64) broken("a step over the lanes of a wave without all of them");
        for (unsigned l = w * 64; l < w * 64 + 64; l++) {
            given[l] = words[l];
            lanes[l].state = kReady;
        }
    }
}
inline void run_group(unsigned threads, std::mt19937& chance) {
    if (threads % 64) broken("a part of a wave");
    lanes.resize(std::max<size_t>(lanes.size(), threads));
    words.assign(lanes.size(), 0);
    given.assign(lanes.size(), 0);
    for (unsigned l = 0; l < threads; l++) {
        Lane& f = lanes[l];
        if (!f.stack) f.stack.reset(new char[kStack]);
        getcontext(&f.ctx);
        f.ctx.uc_stack.ss_sp = f.stack.get();
        f.ctx.uc_stack.ss_size = kStack;
        f.ctx.uc_link = nullptr;
        makecontext(&f.ctx, entry, 0);
        f.state = kReady;
    }
    const unsigned n = threads / 64;
    std::vector<unsigned> turn(n);
    for (;;) {
        for (unsigned i = 0; i < n; i++) turn[i] = order == 1 ? n - 1 - i : i;
        if (order > 1) std::shuffle(turn.begin(), turn.end(), chance);
        for (unsigned w : turn) run_wave(w);
        unsigned done = 0, waiting = 0;
        for (unsigned l = 0; l < threads; l++) {
            done += lanes[l].state == kDone;
            waiting += lanes[l].state == kBarrier;
        }
        if (done == threads) return;
        if (waiting != threads) broken("some threads have ended where others wait at a barrier");
        for (unsigned l = 0; l < threads; l++) lanes[l].state = kReady;
    }
}
template <class F>
void launch(dim3 grid, dim3 block, F&& f) {
    std::mt19937 chance(order);
    body = f;
    for (unsigned y = 0; y < grid.y; y++)
        for (unsigned x = 0; x < grid.x; x++) {
            blockIdx = dim3(x, y);
            run_group(block.x, chance);
        }
}

}  // namespace waves

#define hipLaunchKernelGGL(kernel, grid, block, lds, stream, args) waves::launch(grid, block, [&] { kernel(args); })
inline void __syncthreads() { waves::pause(waves::kBarrier); }

// ---- device functions
template <class T> T max(T a, T b) { return a > b ? a : b; }
template <class T> T min(T a, T b) { return a < b ? a : b; }
inline unsigned min(unsigned a, int b) { return a < (unsigned)b ? a : (unsigned)b; }
inline unsigned __float_as_uint(float f) { unsigned u; std::memcpy(&u, &f, 4); return u; }
inline float __uint_as_float(unsigned u) { float f; std::memcpy(&f, &u, 4); return f; }
inline int __clz(unsigned v) { return v ? __builtin_clz(v) : 32; }
inline int __ffsll(long long v) { return __builtin_ffsll(v); }
inline float __builtin_amdgcn_fmed3f(float a, float b, float c) {   // with a NaN: the smallest of the others
    if (a != a || b != b || c != c) return std::fmin(std::fmin(a, b), c);
    return std::fmax(std::fmin(a, b), std::fmin(std::fmax(a, b), c));
}
template <class T> T atomicAdd(T* p, T v) { const T old = *p; *p += v; return old; }

// ---- steps over the lanes of a wave
inline int __builtin_amdgcn_update_dpp(int old, int v, int ctrl, int rows, int, bool) {
    const int lane = (int)(waves::now & 63), row = lane >> 4;
    const unsigned long long* all = waves::step((unsigned)v);
    int from = -1;
    if (ctrl > 0x110 && ctrl < 0x120) from = (lane & 15) >= ctrl - 0x110 ? lane - (ctrl - 0x110) : -1;   // row_shr
    else if (ctrl == 0x142) from = row > 0 ? row * 16 - 1 : -1;                                            // row_bcast 15
    else if (ctrl == 0x143) from = lane >= 32 ? 31 : -1;                                                   // row_bcast 31
    else waves::broken("a DPP control that is not known here");
    return from >= 0 && (rows >> row & 1) ? (int)(unsigned)all[from] : old;
}
inline int __builtin_amdgcn_readlane(int v, int lane) { return (int)(unsigned)waves::step((unsigned)v)[lane]; }
inline unsigned long long __shfl_xor(unsigned long long v, int o) { const int lane = (int)(waves::now & 63); return waves::step(v)[lane ^ o]; }
inline unsigned long long __ballot(bool b) {
    const unsigned long long* all = waves::step(b);
    unsigned long long m = 0;
    for (int l = 0; l < 64; l++) m |= all[l] << l;
    return m;
}
