// The part of the device language that a workgroup's kernel uses, on the host: one fiber a thread, waves of 64 that run in
// an order the caller chooses.  A wave goes on until all its lanes wait at the same barrier, and only then the next one of
// the order: whatever a kernel leaves to chance between two barriers is decided here, the same way each time.
#pragma once
#include <math.h>
#include <stdint.h>
#include <stdlib.h>
#include <string.h>
#include <ucontext.h>

#include <array>
#include <memory>
#include <type_traits>
#include <vector>

#define __device__
#define __global__
#define __shared__ static
#define __forceinline__ inline
#define __noinline__ __attribute__((noinline))
#define __launch_bounds__(...)
#define __restrict__

struct Uint3 {
    unsigned x, y, z;
};
struct dim3 {
    unsigned x, y, z;
    dim3(unsigned x_ = 1, unsigned y_ = 1, unsigned z_ = 1) : x(x_), y(y_), z(z_) {}
};
struct float4 {
    float x, y, z, w;
};
inline float4 make_float4(float x, float y, float z, float w) { return float4{x, y, z, w}; }
struct __hip_bfloat16 {
    unsigned short bits;
    operator float() const {
        const unsigned u = (unsigned)bits << 16;
        float f;
        memcpy(&f, &u, 4);
        return f;
    }
};
typedef void* hipStream_t;

inline unsigned __float_as_uint(float v) { return __builtin_bit_cast(unsigned, v); }
inline int __float_as_int(float v) { return __builtin_bit_cast(int, v); }
inline float __uint_as_float(unsigned v) { return __builtin_bit_cast(float, v); }
inline float __int_as_float(int v) { return __builtin_bit_cast(float, v); }

namespace waves {

constexpr int kLanes = 64;
enum State { kReady, kCollective, kBarrier, kDone };
struct Thread {
    ucontext_t context;
    State state;
    int where;              // the source line it waits at
    unsigned long long in;  // what it gives a collective
};
inline std::vector<Thread> threads;
inline unsigned long long results[kLanes];  // of the collective that was completed last (one wave runs at a time)
inline ucontext_t scheduler;
inline int current;
inline Uint3 thread_index, block_index, grid_dim;
inline void (*body)(void*);
inline void* body_arg;

inline void wait(State why, int line) {
    Thread& t = threads[current];
    t.state = why, t.where = line;
    swapcontext(&t.context, &scheduler);
}
// every lane's value, once all lanes of the wave have come to the same place
inline const unsigned long long* gather(unsigned long long v, int line) {
    threads[current].in = v;
    wait(kCollective, line);
    return results;
}
inline void entry() {
    body(body_arg);
    wait(kDone, 0);
}
inline void resume(int i) {
    current = i;
    thread_index = Uint3{(unsigned)i, 0, 0};
    swapcontext(&scheduler, &threads[i].context);
}

// Runs `wave` until all its lanes wait at a barrier or have ended: 0, or the line of lanes that wait apart.
inline int run_wave(int wave) {
    const int first = wave * kLanes;
    for (;;) {
        for (int l = 0; l < kLanes; ++l)
            if (threads[first + l].state == kReady) resume(first + l);
        const Thread& lead = threads[first];
        for (int l = 1; l < kLanes; ++l)
            if (threads[first + l].state != lead.state || threads[first + l].where != lead.where) return threads[first + l].where + 1;
        if (lead.state != kCollective) return 0;
        for (int l = 0; l < kLanes; ++l) results[l] = threads[first + l].in;
        for (int l = 0; l < kLanes; ++l) threads[first + l].state = kReady;
    }
}

// A workgroup of size / 64 waves, run in `order` from barrier to barrier.  0: every wave came to every barrier; else a
// negative number: -1 lanes of a wave apart, -2 waves at different barriers, -3 a barrier that some waves never come to.
inline int run_block(int size, const int* order, void (*f)(void*), void* arg) {
    const int n = size / kLanes;
    constexpr size_t kStack = 256 << 10;
    static std::unique_ptr<char[]> stacks(new char[1024 * kStack]);
    threads.assign(size, Thread{});
    body = f, body_arg = arg;
    for (int i = 0; i < size; ++i) {
        Thread& t = threads[i];
        getcontext(&t.context);
        t.context.uc_stack.ss_sp = stacks.get() + i * kStack;
        t.context.uc_stack.ss_size = kStack;
        t.context.uc_link = nullptr;
        makecontext(&t.context, entry, 0);
        t.state = kReady;
    }
    for (;;) {
        for (int w = 0; w < n; ++w)
            if (run_wave(order[w])) return -1;
        int done = 0;
        for (int w = 0; w < n; ++w) done += threads[w * kLanes].state == kDone;
        if (done == n) return 0;
        if (done) return -3;
        for (int w = 1; w < n; ++w)
            if (threads[w * kLanes].where != threads[0].where) return -2;
        for (auto& t : threads) t.state = kReady;
    }
}

inline unsigned long long ballot(bool b, int line) {
    const unsigned long long* r = gather(b, line);
    unsigned long long mask = 0;
    for (int l = 0; l < kLanes; ++l) mask |= r[l] << l;
    return mask;
}
template <typename V>
V read_lane(V v, int lane, int line) {
    unsigned long long bits = 0;
    memcpy(&bits, &v, sizeof(V));
    bits = gather(bits, line)[lane];
    memcpy(&v, &bits, sizeof(V));
    return v;
}
// f over the lanes up to and including `last`, from the first on
template <typename V, typename F>
V fold(V v, int last, int line, F f) {
    unsigned long long bits = 0;
    memcpy(&bits, &v, sizeof(V));
    const unsigned long long* r = gather(bits, line);
    V out{};
    for (int l = 0; l <= last; ++l) {
        V x;
        memcpy(&x, &r[l], sizeof(V));
        out = l ? f(out, x) : x;
    }
    return out;
}
inline int lane() { return (int)(thread_index.x % kLanes); }

}  // namespace waves

#define threadIdx waves::thread_index
#define blockIdx waves::block_index
#define gridDim waves::grid_dim
#define __syncthreads() waves::wait(waves::kBarrier, __LINE__)
#define __ballot(b) waves::ballot(b, __LINE__)
#define __shfl_xor(v, o) waves::read_lane(v, waves::lane() ^ (o), __LINE__)
#define __builtin_amdgcn_readlane(v, l) waves::read_lane(v, l, __LINE__)
#define __builtin_amdgcn_readfirstlane(v) waves::read_lane(v, 0, __LINE__)
#define __builtin_amdgcn_wave_barrier() waves::gather(0, __LINE__)
#define __builtin_amdgcn_fence(...) ((void)0)
#define __builtin_amdgcn_exp2f(x) exp2f(x)
#define __builtin_amdgcn_logf(x) log2f(x)
#define __builtin_amdgcn_permlane16_swap(a, b, c, d) (std::array<unsigned, 2>{a, b})  // (not of a whole wave: not called)

template <typename V>
V atomicAdd(V* p, V v) {
    const V old = *p;
    *p += v;
    return old;
}
template <typename V>
V atomicOr(V* p, V v) {
    const V old = *p;
    *p |= v;
    return old;
}
