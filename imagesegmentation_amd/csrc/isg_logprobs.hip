// Log-probabilities of given classes with the row's entropy and its most probable classes, forward and backward
// (formulas and layout: isg_classes.h).
#include "isg_classes.h"

namespace {

constexpr int kMaxTop = ISG_TOP_MAX;  // classes kept per row
constexpr int kListMax = 1024;        // alternatives a workgroup collects along its part of a row
// ... before it goes back to the best, of which it may keep twice as many as are asked for
constexpr int list_limit(int k) { return 2 * k + 32; }
constexpr int kListKeep = 2 * kMaxTop;

// ---- the `top` first keys of a unit ----------------------------------------------------------------------------------
// The k-th largest of the threads' group maxima is a lower bound of the k-th largest element (k groups hold one at
// least as large), so the elements not below it are few more than k: k + k^2 / (2 groups) for values in any order.
// The bound is found to 16 bits by bisection, the elements above it are put side by side in LDS, and each one's place is
// the number of keys above its own.  Bounds that no finite logit supports and more ties than fit go one class at a time
// instead.

// bits e of a mask: v[FROM + e] >= low, a comparison and an addition with carry each
template <int FROM, int N, int NE>
__device__ __forceinline__ unsigned reach_mask(const float (&v)[NE], float low) {
    unsigned hit = 0;
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int e = FROM + N - 4; e >= FROM; e -= 4) {
            u64 a, b, c, d;  // (four comparisons ahead: a mask is read two states behind its write at the earliest)
            asm("v_cmp_ge_f32_e64 %1, %5, %9\n\t"
                "v_cmp_ge_f32_e64 %2, %6, %9\n\t"
                "v_cmp_ge_f32_e64 %3, %7, %9\n\t"
                "v_cmp_ge_f32_e64 %4, %8, %9\n\t"
                "s_nop 0\n\t"
                "v_addc_co_u32_e64 %0, %1, %0, %0, %1\n\t"
                "v_addc_co_u32_e64 %0, %2, %0, %0, %2\n\t"
                "v_addc_co_u32_e64 %0, %3, %0, %0, %3\n\t"
                "v_addc_co_u32_e64 %0, %4, %0, %0, %4"
                : "+v"(hit), "=&s"(a), "=&s"(b), "=&s"(c), "=&s"(d)
                : "v"(v[e + 3]), "v"(v[e + 2]), "v"(v[e + 1]), "v"(v[e]), "v"(low));
        }
    } else {
#pragma unroll
        for (int e = FROM + N - 1; e >= FROM; --e) hit = hit + hit + (v[e] >= low ? 1u : 0u);
    }
    return hit;
}

// The k first of the list (n keys), through emit(place, key); the G threads of the unit share the work.
template <int G, typename Key, typename Emit>
__device__ __forceinline__ void rank_keys(const Key* keys, int n, int k, Emit emit) {
    for (int r = threadIdx.x & (G - 1); r < n; r += G) {
        const Key own = keys[r];
        int place = 0;
#pragma unroll 4
        for (int o = 0; o < n; ++o) place += keys[o] > own ? 1 : 0;
        if (place < k) emit(place, own);
    }
}

// Lanes of one wave.  Q groups a lane.  (Bisecting between the least and the largest group instead, nine steps for
// sixteen, measured slower: 131,072 x 785 bf16 with five classes 78 us against 69.)
template <int G, int Q>
__device__ __forceinline__ unsigned lanes_bound(const float (&gm)[Q], int k) {
    unsigned g[Q], bound = 0;
#pragma unroll
    for (int q = 0; q < Q; ++q) g[q] = order_bits(gm[q]) >> 16;
    for (int bit = 15; bit >= 0; --bit) {
        const unsigned t = bound | (1u << bit);
        int n = 0;
        if constexpr (G == 64) {
#pragma unroll
            for (int q = 0; q < Q; ++q) n += __builtin_popcountll(__ballot(g[q] >= t));
        } else {
#pragma unroll
            for (int q = 0; q < Q; ++q) n += g[q] >= t ? 1 : 0;
            n = group_sum<G>(n);
        }
        bound = n >= k ? t : bound;
    }
    return bound;
}
template <int Q, int NE>
__device__ __forceinline__ void group_maxima(const float (&v)[NE], float (&gm)[Q]) {
#pragma unroll
    for (int q = 0; q < Q; ++q) {
        gm[q] = v[q];
#pragma unroll
        for (int e = q + Q; e < NE; e += Q) gm[q] = fmaxf(gm[q], v[e]);
    }
}

constexpr int candidates(int lanes) { return lanes == 16 ? 128 : 256; }  // places per unit

// The order of a row's classes in 32 bits where a logit has 16 (bf16) and a class 16: halves what ranking costs.
struct ShortKey {
    typedef unsigned type;
    static __device__ __forceinline__ unsigned of(u64 k) { return (unsigned)(k >> 32 & 0xffff0000u) | ((unsigned)k & 0xffffu); }
    static __device__ __forceinline__ u64 full(unsigned k) {
        // (the lower half of a logit's key: zeros, or ones below 0, whose bits are inverted; NaN is 1)
        const u64 bits = k >> 31 ? k & 0xffff0000u : (k >> 16 ? k | 0xffffu : 1u);
        return bits << 32 | 0xffff0000u | (k & 0xffffu);
    }
};
struct LongKey {
    typedef u64 type;
    static __device__ __forceinline__ u64 of(u64 k) { return k; }
    static __device__ __forceinline__ u64 full(u64 k) { return k; }
};

template <int G, int NE, typename Keys, typename Reload, typename Emit>
__device__ __forceinline__ void select_lanes(const float (&v)[NE], int k, typename Keys::type* cand, Reload reload, Emit emit) {
    constexpr int Q1 = 64 / G < NE ? 64 / G : NE, Q2 = 128 / G < NE ? 128 / G : NE, kCap = candidates(G);
    const int lane = threadIdx.x & (G - 1);
    float gm[Q2];
    group_maxima(v, gm);
    unsigned bound;
    if (k <= 16) {
        float g1[Q1];
        group_maxima(gm, g1);
        bound = lanes_bound<G>(g1, k);
    } else {
        bound = lanes_bound<G>(gm, k);
    }
    int total = kCap + 1;
    if (bound > 0x7fu) {  // (0x7f begins the key of -inf)
        const float low = order_value(bound << 16);
        unsigned hit = reach_mask<0, (NE < 32 ? NE : 32)>(v, low), later = 0;
        if constexpr (NE > 32) later = reach_mask<32, NE - 32>(v, low);
        const int mine = __builtin_popcount(hit) + __builtin_popcount(later);
        int at = group_scan<G>(mine) - mine;
        total = group_sum<G>(mine);
        if (total <= kCap) {
            int add = 0;
            while (hit | later) {
                if (hit == 0) hit = later, later = 0, add = 32;
                const int e = __builtin_ctz(hit);
                hit &= hit - 1;
                cand[at++] = Keys::of(reload(e + add));
            }
            together<G>();
            rank_keys<G>(cand, total, k, [&](int place, typename Keys::type key) { emit(place, Keys::full(key)); });
        }
    }
    if (total > kCap) {
        u64 last = ~0ull;
        for (int j = 0; j < k; ++j) {
            u64 best = 0;
#pragma unroll 1
            for (int e = 0; e < NE; ++e) {
                const u64 x = reload(e);
                if (x < last && x > best) best = x;
            }
            last = best = group_max_key<G>(best);
            if (lane == 0) emit(j, best);
        }
    }
}

// A workgroup.
struct TopShared {
    u64 cand[1024];
    unsigned group[kThreads];
    int count;
    u64 best[4];
};

// where a wave's elements go in a list the workgroup shares: its first place, for the lanes' running total `upto`
__device__ __forceinline__ int wave_places(int* count, int upto) {
    const int all = __builtin_amdgcn_readlane(upto, 63);
    int first = 0;
    if (all && (threadIdx.x & 63) == 0) first = atomicAdd(count, all);
    return __builtin_amdgcn_readfirstlane(first);
}

// (one comparison a group and a count of the wave's mask per bit, the scalar unit's work; every wave for itself)
__device__ __forceinline__ unsigned group_bound(float lane_max, int k, TopShared& sh) {
    const int lane = threadIdx.x & 63;
    sh.group[threadIdx.x] = order_bits(lane_max) >> 16;
    __syncthreads();
    unsigned g[4], bound = 0;
#pragma unroll
    for (int q = 0; q < 4; ++q) g[q] = sh.group[q * 64 + lane];
    for (int bit = 15; bit >= 0; --bit) {
        const unsigned t = bound | (1u << bit);
        int n = 0;
#pragma unroll
        for (int q = 0; q < 4; ++q) n += __builtin_popcountll(__ballot(g[q] >= t));
        if (n >= k) bound = t;
    }
    return bound;
}

template <int NE, typename Reload, typename Emit>
__device__ __forceinline__ void select_workgroup(const float (&v)[NE], int k, TopShared& sh, Reload reload, Emit emit) {
    constexpr int kCap = 1024;
    const int lane = threadIdx.x & 63, tid = threadIdx.x;
    float gm[1];
    group_maxima(v, gm);
    if (tid == 0) sh.count = 0;
    const unsigned bound = group_bound(gm[0], k, sh);
    int total = kCap + 1;
    if (bound > 0x7fu) {
        unsigned hit = reach_mask<0, NE>(v, order_value(bound << 16));
        const int mine = __builtin_popcount(hit), upto = group_scan<64>(mine);
        int at = wave_places(&sh.count, upto) + upto - mine;
        __syncthreads();
        total = sh.count;
        if (total <= kCap) {
            while (hit) {
                const int e = __builtin_ctz(hit);
                hit &= hit - 1;
                sh.cand[at++] = reload(e);
            }
            __syncthreads();
            rank_keys<kThreads>(sh.cand, total, k, emit);
        }
    }
    if (total > kCap) {
        u64 last = ~0ull;
        for (int j = 0; j < k; ++j) {
            u64 best = 0;
#pragma unroll 1
            for (int e = 0; e < NE; ++e) {
                const u64 x = reload(e);
                if (x < last && x > best) best = x;
            }
            best = group_max_key<64>(best);
            __syncthreads();
            if (lane == 0) sh.best[tid >> 6] = best;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < 4; ++w) best = sh.best[w] > best ? sh.best[w] : best;
            last = best;
            if (tid == 0) emit(j, best);
            if (best == 0) {  // (fewer classes than are asked for: the last step of a part)
                for (int o = j + 1 + tid; o < k; o += kThreads) emit(o, 0ull);
                break;
            }
        }
    }
}

// maximum, sum of powers and sum of powers times exponents of a part of a row
struct Sums {
    float m, s, u;
};

__device__ __forceinline__ void add_power(float z, float m, float c, float& s, float& u) {
    const float x = (z - m) * c, p = __builtin_amdgcn_exp2f(x);
    s += p;
    u += p * fmaxf(x, -1000.0f);
}

// (a part without any probability has m = -inf and s = 0)
__device__ __forceinline__ void merge_sums(Sums& t, const Sums& p, float c) {
    const float m = fmaxf(t.m, p.m);
    Sums r{m, 0.0f, 0.0f};
    if (t.s != 0.0f) {
        const float d = (t.m - m) * c, f = __builtin_amdgcn_exp2f(d);
        r.s = f * t.s, r.u = f * (t.u + fmaxf(d, -1000.0f) * t.s);
    }
    if (p.s != 0.0f) {
        const float d = (p.m - m) * c, f = __builtin_amdgcn_exp2f(d);
        r.s += f * p.s, r.u += f * (p.u + fmaxf(d, -1000.0f) * p.s);
    }
    t = r;
}

// What a row's results follow from.  `c_rel`: by how much log2(e) / T exceeds the float c, relative; the logarithm of
// the sum moves with the exponents' scale as their mean does, u / s.
struct RowStats {
    float m, l2s, H, inv_s;
};
__device__ __forceinline__ RowStats row_stats(const Sums& t, float c_rel) {
    RowStats r;
    r.m = t.m == -INFINITY ? 0.0f : t.m;
    const float mean = t.u / t.s;
    r.l2s = t.s == 0.0f ? INFINITY : __builtin_amdgcn_logf(t.s) + c_rel * mean;
    r.H = t.s == 0.0f ? 0.0f : kLn2 * (r.l2s - mean);
    r.inv_s = 1.0f / t.s;
    return r;
}

struct LogprobsArgs {
    const void* tokens;
    const unsigned char* live;
    float* logprobs;
    float* entropy;
    float* top_logprobs;
    int* top_classes;
    float* stats;
    Sums* part;      // [rows][splits]
    u64* part_keys;  // [rows][splits][top]
    long long row_stride, units;
    int token_bytes, cols, splits, per, top;  // a row is cut into `splits` parts of `per` classes
    float c, inv_t, c_rel;
};

// a dead row's outputs, by G threads
template <int G>
__device__ __forceinline__ void dead_row(const LogprobsArgs& a, long long row, int tid) {
    if (tid == 0) {
        if (a.logprobs) a.logprobs[row] = 0.0f;
        a.entropy[row] = 0.0f;
        if (a.stats) *reinterpret_cast<float4*>(a.stats + 4 * row) = make_float4(0.0f, INFINITY, 0.0f, 0.0f);
    }
    for (int j = tid; j < a.top; j += G) a.top_logprobs[row * a.top + j] = 0.0f, a.top_classes[row * a.top + j] = -1;
}

template <typename T>
__device__ __forceinline__ void row_outputs(const LogprobsArgs& a, const T* z, long long row, const RowStats& r) {
    if (a.tokens) {
        const long long t = class_at(a.tokens, a.token_bytes, row);
        a.logprobs[row] = t >= 0 && t < a.cols ? log_prob(ld(z, t), r.m, a.inv_t, r.l2s) : NAN;
    }
    a.entropy[row] = r.H;
    if (a.stats) *reinterpret_cast<float4*>(a.stats + 4 * row) = make_float4(r.m, r.l2s, r.H, r.inv_s);
}

__device__ __forceinline__ void row_alternative(const LogprobsArgs& a, long long row, const RowStats& r, int place, u64 key) {
    a.top_logprobs[row * a.top + place] = log_prob(order_value((unsigned)(key >> 32)), r.m, a.inv_t, r.l2s);
    a.top_classes[row * a.top + place] = (int)~(unsigned)key;
}

// A row in the registers of G lanes: maximum first, then the sums of 2^x and 2^x x over the same registers, then the
// alternatives out of them.  One read of the logits bounds it without alternatives, the search for them with: 131,072 x
// 785 bf16 46 us (4.5 TB/s; 38 us where nothing has left the last-level cache dirty), with 5 alternatives 69, 20 105, 64
// 193; float 73 (5.7 TB/s), with 20 110; 20,480 rows bf16 9.6, behind a backward pass 11.5; 10,240 x 784 float with 20 13.1.
template <typename T, int G, int NE, bool TOP>
__global__ __launch_bounds__(kThreads) void logprobs_fwd_kernel(const T* __restrict__ logits, LogprobsArgs a) {
    typedef typename std::conditional<sizeof(T) == 2, ShortKey, LongKey>::type Keys;
    __shared__ typename Keys::type cand[TOP ? kThreads / G * candidates(G) : 1];
    const int lane = threadIdx.x & (G - 1), unit = threadIdx.x / G;
    const long long row = block_index() * (kThreads / G) + unit;
    if (row >= a.units) return;
    if (a.live && !a.live[row]) {
        dead_row<G>(a, row, lane);
        return;
    }
    const T* z = logits + row * a.row_stride;
    const Span<T, G, NE> span(z, 0, a.cols, lane);
    float v[NE];
    span.template load<true>(z, v);
    float m = v[0];
#pragma unroll
    for (int e = 1; e < NE; ++e) m = fmaxf(m, v[e]);
    Sums t{group_max<G>(m), 0.0f, 0.0f};
    const float mz = t.m == -INFINITY ? 0.0f : t.m;
#pragma unroll
    for (int e = 0; e < NE; ++e) add_power(v[e], mz, a.c, t.s, t.u);
    t.s = group_sum<G>(t.s), t.u = group_sum<G>(t.u);
    const RowStats r = row_stats(t, a.c_rel);
    if (lane == 0) row_outputs(a, z, row, r);
    if constexpr (TOP)
        select_lanes<G, NE, Keys>(
            v, a.top, cand + unit * candidates(G),
            [&](int e) {
                const int i = span.cls(e);
                return i < 0 ? 0ull : order_key(ld(z, i), i);
            },
            [&](int place, u64 k) { row_alternative(a, row, r, place, k); });
}

// What a workgroup has found of a part of a row's best classes so far: the k first are among them, in no order.
// `count` is the walk's alone: every wave reads it behind a barrier, and until the next barrier nothing but that same value
// is written to it.  `kept_count` is trim_list's: read between its barriers, set back behind its last one.  (As one counter
// a wave that ran ahead into trim_list set it back before the others had read it.)
struct TopList {
    u64 keys[kListMax];
    u64 kept[kListKeep];
    int count, kept_count;
};

// The largest 16-bit prefix that at least k of the n keys (n <= kListMax) reach; uniform, every wave for itself.
template <int Q>
__device__ __forceinline__ unsigned prefix_of(const u64* keys, int n, int k) {
    const int lane = threadIdx.x & 63;
    unsigned g[Q], bound = 0;
#pragma unroll
    for (int q = 0; q < Q; ++q) g[q] = q * 64 + lane < n ? (unsigned)(keys[q * 64 + lane] >> 48) : 0u;
    for (int bit = 15; bit >= 0; --bit) {
        const unsigned t = bound | (1u << bit);
        int c = 0;
#pragma unroll
        for (int q = 0; q < Q; ++q) c += __builtin_popcountll(__ballot(g[q] >= t));
        if (c >= k) bound = t;
    }
    return bound;
}

// Cuts the list back: what does not reach the prefix of its k-th key goes; where ties leave too much, all but the k
// first.  Returns the new count; `low` is a value that a class behind all of these has to exceed.
__device__ __forceinline__ int trim_list(TopList& list, int count, int k, float& low) {
    const unsigned bound = count <= 4 * 64 ? prefix_of<4>(list.keys, count, k)
                                           : (count <= 8 * 64 ? prefix_of<8>(list.keys, count, k)
                                                              : prefix_of<kListMax / 64>(list.keys, count, k));
    if (threadIdx.x == 0) list.kept_count = 0;
    __syncthreads();
    for (int r = threadIdx.x; r < count; r += kThreads) {
        const u64 own = list.keys[r];
        if ((unsigned)(own >> 48) >= bound) {
            const int at = atomicAdd(&list.kept_count, 1);
            if (at < kListKeep) list.kept[at] = own;
        }
    }
    __syncthreads();
    int n = list.kept_count;
    if (n > 2 * k) {
        rank_keys<kThreads>(list.keys, count, k, [&](int place, u64 key) { list.kept[place] = key; });
        __syncthreads();
        n = count < k ? count : k;
    }
    for (int r = threadIdx.x; r < n; r += kThreads) list.keys[r] = list.kept[r];
    __syncthreads();
    low = order_value(bound << 16);
    return n;
}

// A part of a longer row: a workgroup walks over it, kThreads * NE classes at a time, the next ones being loaded
// meanwhile.  Every wave keeps its own maximum and its lanes their own sums until the end.  The best classes gather in
// a list: of the first step all that reach the bound select_workgroup would take, of the later steps what exceeds
// the list's own bound, which rises whenever the list has grown to its limit and is cut back.  Steps that would overrun
// the list (rising rows, ties) or have no finite bound hand it their k first by select_workgroup instead.
//
// 2,048 x 131,071 bf16 with 64 alternatives: 125 us a call where calls follow each other, 4.3 TB/s (single launches 128 to
// 148), the vector units busy for four fifths of it (some 8 instructions a class for the sums, one of them an exponential
// that takes four times an addition; 9 for the alternatives); without alternatives 103 us, 5.2 TB/s.  2,048 x 65,537 float
// with 20: 103 us, 5.2 TB/s.
template <typename T, int NE, bool TOP>
__global__ __launch_bounds__(kThreads, sizeof(T) == 4 ? 5 : 8) void logprobs_stream_kernel(const T* __restrict__ logits,
                                                                                            LogprobsArgs a) {
    __shared__ float red[4][4];
    __shared__ typename std::conditional<TOP, TopShared, char>::type shared;
    __shared__ typename std::conditional<TOP, TopList, char>::type list;
    const int tid = threadIdx.x, lane = tid & 63;
    const long long unit = block_index();
    if (unit >= a.units) return;
    const long long row = a.splits == 1 ? unit : unit / a.splits;
    const int split = a.splits == 1 ? 0 : (int)(unit - row * a.splits);
    if (a.live && !a.live[row]) {
        if (a.splits == 1) dead_row<kThreads>(a, row, tid);
        return;
    }
    const T* z = logits + row * a.row_stride;
    using S = Span<T, kThreads, NE>;
    const int lo = split * a.per, hi = lo + a.per < a.cols ? lo + a.per : a.cols;
    S ahead(z, lo, hi, tid);
    unsigned raw[S::kWords];
    ahead.fetch(z, raw);
    Sums t{-INFINITY, 0.0f, 0.0f};  // (m of the wave; s, u of the lane)
    int count = 0;
    float low = -INFINITY;  // what a further class has to exceed ...
    bool bounded = false;   // ... once the list holds k classes above some finite value
    while (ahead.more()) {
        const S span = ahead;
        float v[NE];
        span.unpack(raw, v);
        ahead.next();
        if (ahead.more()) ahead.fetch(z, raw);
        float lane_max = v[0];
#pragma unroll
        for (int e = 1; e < NE; ++e) lane_max = fmaxf(lane_max, v[e]);
        if (__ballot(lane_max > t.m)) {
            const float m = group_max<64>(lane_max);
            if (t.m != -INFINITY) {
                const float d = (t.m - m) * a.c, f = __builtin_amdgcn_exp2f(d);
                t.u = f * (t.u + fmaxf(d, -1000.0f) * t.s);
                t.s *= f;
            }
            t.m = m;
        }
        const float mz = t.m == -INFINITY ? 0.0f : t.m;
#pragma unroll
        for (int e = 0; e < NE; ++e) add_power(v[e], mz, a.c, t.s, t.u);
        if constexpr (TOP) {
            const auto reload = [&](int e) {
                const int i = span.cls(e);
                return i < 0 ? 0ull : order_key(ld(z, i), i);
            };
            float reach = above(low);
            bool fits = true;
            if (!bounded) {
                const unsigned bound = group_bound(lane_max, a.top, shared);
                fits = bound > 0x7fu;
                low = order_value(bound << 16);
                reach = low;  // (classes of one step are not in order: those at the bound count as well)
            }
            if (tid == 0) list.count = count;
            __syncthreads();
            if (fits) {
                if (__ballot(lane_max >= reach)) {
                    unsigned hit = reach_mask<0, NE>(v, reach);
                    const int mine = __builtin_popcount(hit), upto = group_scan<64>(mine);
                    int at = wave_places(&list.count, upto) + upto - mine;
                    if (at + mine <= kListMax)
                        while (hit) {  // (a lane's only one is its largest)
                            const int e = __builtin_ctz(hit);
                            hit &= hit - 1;
                            const int i = span.inside(span.start(e / S::VE)) + e % S::VE;
                            list.keys[at++] = order_key(mine == 1 ? lane_max : ld(z, i), i);
                        }
                }
                __syncthreads();
                const int total = list.count;
                fits = total <= kListMax;
                if (fits) count = total, bounded = true;
            }
            if (!fits) {
                if (count > kListMax - kMaxTop) {
                    float unused;
                    count = trim_list(list, count, a.top, unused);
                }
                select_workgroup<NE>(v, a.top, shared, reload, [&](int place, u64 k) { list.keys[count + place] = k; });
                __syncthreads();
                count += a.top;
            }
            if (count > list_limit(a.top) || !fits) {
                count = trim_list(list, count, a.top, low);
                bounded = low > -INFINITY;  // (no bound from classes at -inf or NaN)
            }
        }
    }
    // the waves' sums
    t.s = group_sum<64>(t.s), t.u = group_sum<64>(t.u);
    if (lane == 0) red[tid >> 6][0] = t.m, red[tid >> 6][1] = t.s, red[tid >> 6][2] = t.u;
    __syncthreads();
    t = Sums{red[0][0], red[0][1], red[0][2]};
#pragma unroll
    for (int w = 1; w < 4; ++w) merge_sums(t, Sums{red[w][0], red[w][1], red[w][2]}, a.c);
    RowStats r;
    if (a.splits == 1) {
        r = row_stats(t, a.c_rel);
        if (tid == 0) row_outputs(a, z, row, r);
    } else if (tid == 0) {
        a.part[unit] = t;
    }
    if constexpr (TOP) {
        if (count > 2 * a.top) count = trim_list(list, count, a.top, low);
        rank_keys<kThreads>(list.keys, count, a.top, [&](int place, u64 key) {
            if (a.splits == 1) row_alternative(a, row, r, place, key);
            else a.part_keys[unit * a.top + place] = key;
        });
    }
}

// Joins the parts of a row: G threads, NE keys each.  Its latency is what it costs: 4 us for one row in 24 parts, 5 for
// 320 rows in 7.
template <typename T, int G, int NE>
__global__ __launch_bounds__(kThreads) void logprobs_join_kernel(const T* __restrict__ logits, LogprobsArgs a) {
    __shared__ typename std::conditional<G == 64, u64[4 * candidates(64)], TopShared>::type shared;
    const int lane = threadIdx.x & 63, tid = threadIdx.x & (G - 1);
    const long long row = block_index() * (kThreads / G) + threadIdx.x / G;
    if (row >= a.units) return;
    if (a.live && !a.live[row]) {
        dead_row<G>(a, row, tid);
        return;
    }
    // (every wave for itself)
    const Sums* part = a.part + row * a.splits;
    Sums t{-INFINITY, 0.0f, 0.0f};
    for (int i = lane; i < a.splits; i += 64) merge_sums(t, part[i], a.c);
    const float m = group_max<64>(t.m);
    merge_sums(t, Sums{m, 0.0f, 0.0f}, a.c);  // (to the common maximum)
    t.s = group_sum<64>(t.s), t.u = group_sum<64>(t.u);
    const RowStats r = row_stats(t, a.c_rel);
    if (tid == 0) row_outputs(a, logits + row * a.row_stride, row, r);
    if (a.top == 0) return;
    const int n = a.splits * a.top;
    const u64* keys = a.part_keys + row * n;
    // (A part's keys fall from place to place: where `top` divides 64 a thread would have the same place of every part, and
    // the bound from the threads' maxima would let half of all keys through.  The places move on from part to part then: 64
    // best of 300 x 20,011 float 22 us a call, without 34; 48 best, whose parts lie apart by themselves, 21 and 19.)
    const int step = 64 % a.top ? 0 : 64 / NE + 1;
    const auto key_of = [&](int e) { return e * G + ((tid + e * step) & (G - 1)); };
    float v[NE];
#pragma unroll
    for (int e = 0; e < NE; ++e) {
        const int i = key_of(e);
        const unsigned k = i < n ? (unsigned)(keys[i] >> 32) : 0u;
        v[e] = k ? order_value(k) : -INFINITY;
    }
    const auto reload = [&](int e) {
        const int i = key_of(e);
        return i < n ? keys[i] : 0ull;
    };
    const auto emit = [&](int place, u64 key) { row_alternative(a, row, r, place, key); };
    if constexpr (G == 64)
        select_lanes<G, NE, LongKey>(v, a.top, shared + (threadIdx.x / G) * candidates(G), reload, emit);
    else
        select_workgroup<NE>(v, a.top, shared, reload, emit);
}

// dlogits[c] = 1/T ([c = a] g_a + sum_j [c = i_j] g_j - p_c (g_a + sum_j g_j) - g_H p_c (log p_c + H)): the dense part
// is written first, the few classes with a gradient of their own are written again behind it by the same unit.
struct LogprobsBwdArgs {
    const void* tokens;
    const int* top_classes;
    const float* stats;
    const float* dlogprobs;
    const float* dentropy;
    const float* dtop;
    long long row_stride, units;
    int token_bytes, cols, splits, per, top, past;
    float c, c_lo, inv_t;
};

// A row, or a part of one, by G lanes:
//   dz_c = 1/T [ g_a [c = a] + sum_j g_j [c = i_j] - p_c (g_a + sum_j g_j + g_H (log p_c + H)) ],
// the dense part first, from the row's kept m, s and H, then the few classes with a gradient of their own over it.  Reads
// the logits, writes as much, and is bound by that: 131,072 x 785 bf16 84 us (4.9 TB/s read and written), float 145 us (5.7),
// 2,050 x 131,071 bf16 188 us (5.7), 2,048 x 65,537 float 196 us (5.5).
template <typename T, int G, int NE>
__global__ __launch_bounds__(kThreads) void logprobs_bwd_kernel(const T* __restrict__ logits, LogprobsBwdArgs a,
                                                               T* __restrict__ dlogits) {
    constexpr int L = G < 64 ? G : 64;  // (a workgroup: every wave for itself)
    const int lane = threadIdx.x & (L - 1), tid = threadIdx.x & (G - 1);
    // (from the last unit back: what the forward pass read last is still in the last-level cache)
    const long long unit = a.units - 1 - (block_index() * (kThreads / G) + threadIdx.x / G);
    if (unit < 0) return;
    const long long row = a.splits == 1 ? unit : unit / a.splits;
    const int split = a.splits == 1 ? 0 : (int)(unit - row * a.splits);
    using S = Span<T, G, NE>;
    const int lo = split * a.per, hi = lo + a.per < a.cols ? lo + a.per : a.cols;
    T* d = dlogits + row * a.cols;
    const S span(d, lo, hi, tid);  // (aligned as the gradient; dense logits lie the same way)
    const float4 stats = *reinterpret_cast<const float4*>(a.stats + 4 * row);
    const float m = stats.x, l2s = stats.y;
    const bool zero = l2s == INFINITY;  // a dead row, or no class has probability: nothing to move
    const T* z = logits + row * a.row_stride;
    float v[NE];
    if (!zero) span.template load<false>(z, v);
    const float ga = a.dlogprobs ? a.dlogprobs[row] : 0.0f, gh = a.dentropy ? a.dentropy[row] : 0.0f;
    const long long tok = a.dlogprobs ? class_at(a.tokens, a.token_bytes, row) : -1;
    float g = ga;
    bool both = false;  // the token is one of the alternatives
    if (a.dtop) {
        float gt = 0.0f;
        for (int j = lane; j < a.top; j += L) {
            gt += a.dtop[row * a.top + j];
            both |= a.top_classes[row * a.top + j] == tok;
        }
        g += group_sum<L>(gt);
        both = group_any<L>(both);
    }
    if (a.dlogprobs && ga != 0.0f && (tok < 0 || tok >= a.cols)) g = NAN;  // a class the row does not have
    // p (g + g_H (log p + H)) / T with p = 2^x / s and log p = ln 2 (x - log2 s): the row's constants put together
    const float k0 = -a.inv_t * stats.w * (g + gh * (stats.z - kLn2 * l2s)), k1 = -a.inv_t * stats.w * (gh * kLn2);
    const auto dense = [&](float zi) {
        const float x = (zi - m) * a.c;
        const float e = sizeof(T) == 4 ? power_exact(zi, m, a.c, a.c_lo) : __builtin_amdgcn_exp2f(x);
        return e * __builtin_fmaf(k1, fmaxf(x, -1000.0f), k0);
    };
#pragma unroll
    for (int t = 0; t < S::NV; ++t) {
        if (span.beyond(t)) break;
        float o[S::VE];
#pragma unroll
        for (int j = 0; j < S::VE; ++j) o[j] = zero ? 0.0f : dense(v[t * S::VE + j]);
        if constexpr (G >= 64 && S::VE * sizeof(T) == 16) {
            if (a.past) {
                span.store_past(d, t, o);
                continue;
            }
        }
        span.store(d, t, o);
    }
    if (zero) return;
    together<G>();
    if (tid >= L) return;
    if (a.dtop)
        for (int j = lane; j < a.top; j += L) {
            const int i = a.top_classes[row * a.top + j];
            if (i < lo || i >= hi) continue;
            const float o = __builtin_fmaf(a.inv_t, a.dtop[row * a.top + j] + (i == tok ? ga : 0.0f), dense(ld(z, i)));
            store_vector<1>(d + i, &o);
        }
    if (lane == 0 && !both && tok >= lo && tok < hi) {
        const float o = __builtin_fmaf(a.inv_t, ga, dense(ld(z, tok)));
        store_vector<1>(d + tok, &o);
    }
}

template <typename T, bool TOP>
struct LogprobsFwd {
    template <int G, int NE>
    static void run(const void* logits, const LogprobsArgs& a, hipStream_t s) {
        hipLaunchKernelGGL((logprobs_fwd_kernel<T, G, NE, TOP>), grid_of(a.units, G), dim3(kThreads), 0, s,
                           static_cast<const T*>(logits), a);
    }
    static void launch(const Cut& cut, const void* logits, const LogprobsArgs& a, hipStream_t s) {
        if (cut.lanes != kThreads)
            with_wave<LogprobsFwd, kNarrow>(cut, logits, a, s);
        else
            hipLaunchKernelGGL((logprobs_stream_kernel<T, 16, TOP>), grid_of(a.units, kThreads), dim3(kThreads), 0, s,
                               static_cast<const T*>(logits), a);
    }
};
template <typename T>
struct LogprobsBwd {
    template <int G, int NE>
    static void run(const void* logits, const LogprobsBwdArgs& a, void* dlogits, hipStream_t s) {
        hipLaunchKernelGGL((logprobs_bwd_kernel<T, G, NE>), grid_of(a.units, G), dim3(kThreads), 0, s,
                           static_cast<const T*>(logits), a, static_cast<T*>(dlogits));
    }
};
template <typename T, int G, int NE>
void launch_join(const void* logits, const LogprobsArgs& a, hipStream_t s) {
    hipLaunchKernelGGL((logprobs_join_kernel<T, G, NE>), grid_of(a.units, G), dim3(kThreads), 0, s,
                       static_cast<const T*>(logits), a);
}
// (n keys of a row's parts: a wave while they are few)
template <typename T>
void join_parts(int n, const void* logits, const LogprobsArgs& a, hipStream_t s) {
    if (n <= 64 * 4) launch_join<T, 64, 4>(logits, a, s);
    else if (n <= 64 * 8) launch_join<T, 64, 8>(logits, a, s);
    else if (n <= kThreads * 4) launch_join<T, kThreads, 4>(logits, a, s);
    else if (n <= kThreads * 8) launch_join<T, kThreads, 8>(logits, a, s);
    else launch_join<T, kThreads, 32>(logits, a, s);
}

int check_top(const char* who, int top, int cols) {
    ISG_REQUIRE(top >= 0 && top <= kMaxTop && top <= cols, ISG_EINVAL, "%s: top=%d of %d classes (at most %d)", who, top, cols,
                kMaxTop);
    return ISG_OK;
}

}  // namespace

extern "C" long long isg_token_logprobs_workspace_bytes(int rows, int cols, int top) {
    if (rows < 0 || cols < 1 || cols > kMaxCols || top < 0 || top > kMaxTop) return -1;
    const Cut cut = cut_forward(rows, cols, ISG_F32, 0, top);  // (rows of both types are in as many parts)
    return cut.splits == 1 ? 0 : (long long)rows * cut.splits * ((long long)sizeof(Sums) + 8 * top) + 8;
}

extern "C" int isg_token_logprobs_fwd(const void* logits, long long row_stride, const void* tokens, int token_bytes,
                                      const unsigned char* live, int rows, int cols, int dtype, float temperature,
                                      int top, float* logprobs, float* entropy, float* top_logprobs,
                                      int32_t* top_classes, float* stats, void* workspace, void* stream) {
    const char* who = "isg_token_logprobs_fwd";
    int rc = check_call(who, row_stride, rows, cols, dtype, temperature);
    if (rc != ISG_OK) return rc;
    rc = check_bytes(who, tokens, token_bytes);
    if (rc != ISG_OK) return rc;
    rc = check_top(who, top, cols);
    if (rc != ISG_OK) return rc;
    if (rows == 0) return ISG_OK;
    ISG_REQUIRE(logits && entropy && (!tokens || logprobs) && (top == 0 || (top_logprobs && top_classes)), ISG_EINVAL,
                "%s: null pointer", who);
    const Cut cut = cut_forward(rows, cols, dtype, 0, top);
    ISG_REQUIRE(cut.splits == 1 || workspace, ISG_EINVAL, "%s: %d x %d logits need a workspace", who, rows, cols);
    ISG_REQUIRE(((uintptr_t)workspace | (uintptr_t)stats) % 8 == 0 && (uintptr_t)stats % 16 == 0, ISG_EINVAL,
                "%s: workspace and stats must be aligned to 8 and 16 bytes", who);
    hipStream_t s = static_cast<hipStream_t>(stream);
    LogprobsArgs a{};
    a.tokens = tokens, a.live = live, a.logprobs = tokens ? logprobs : nullptr, a.entropy = entropy;
    a.top_logprobs = top_logprobs, a.top_classes = top_classes, a.stats = stats;
    a.row_stride = row_stride, a.units = (long long)rows * cut.splits;
    a.token_bytes = token_bytes, a.cols = cols, a.splits = cut.splits, a.per = cut.per, a.top = top;
    float c_lo;
    scale_of(temperature, a.c, c_lo, a.inv_t);
    a.c_rel = c_lo / a.c;
    if (cut.splits > 1) {
        a.part_keys = static_cast<u64*>(workspace);
        a.part = reinterpret_cast<Sums*>(a.part_keys + a.units * top);
    }
    if (dtype == ISG_F32)
        top > 0 ? LogprobsFwd<float, true>::launch(cut, logits, a, s) : LogprobsFwd<float, false>::launch(cut, logits, a, s);
    else
        top > 0 ? LogprobsFwd<__hip_bfloat16, true>::launch(cut, logits, a, s)
                : LogprobsFwd<__hip_bfloat16, false>::launch(cut, logits, a, s);
    rc = isg::check_launch("logprobs_fwd_kernel");
    if (rc != ISG_OK || cut.splits == 1) return rc;
    a.units = rows;
    if (dtype == ISG_F32) join_parts<float>(cut.splits * top, logits, a, s);
    else join_parts<__hip_bfloat16>(cut.splits * top, logits, a, s);
    return isg::check_launch("logprobs_join_kernel");
}

extern "C" int isg_token_logprobs_bwd(const void* logits, long long row_stride, const void* tokens, int token_bytes,
                                      const int32_t* top_classes, const float* stats, const float* dlogprobs,
                                      const float* dentropy, const float* dtop_logprobs, int rows, int cols, int dtype,
                                      float temperature, int top, void* dlogits, void* stream) {
    const char* who = "isg_token_logprobs_bwd";
    int rc = check_call(who, row_stride, rows, cols, dtype, temperature);
    if (rc != ISG_OK) return rc;
    rc = check_bytes(who, tokens, token_bytes);
    if (rc != ISG_OK) return rc;
    rc = check_top(who, top, cols);
    if (rc != ISG_OK) return rc;
    if (rows == 0) return ISG_OK;
    ISG_REQUIRE(logits && stats && dlogits && (!dlogprobs || tokens) && (!dtop_logprobs || (top > 0 && top_classes)),
                ISG_EINVAL, "%s: null pointer", who);
    ISG_REQUIRE((uintptr_t)stats % 16 == 0, ISG_EINVAL, "%s: stats must be aligned to 16 bytes", who);
    ISG_REQUIRE(dlogits != logits, ISG_EINVAL, "%s: dlogits must not alias the logits", who);
    const Cut cut = cut_backward(rows, cols, dtype, 0);
    hipStream_t s = static_cast<hipStream_t>(stream);
    LogprobsBwdArgs a{};
    a.tokens = tokens, a.top_classes = top_classes, a.stats = stats;
    a.dlogprobs = dlogprobs, a.dentropy = dentropy, a.dtop = dtop_logprobs;
    a.row_stride = row_stride, a.units = (long long)rows * cut.splits;
    a.token_bytes = token_bytes, a.cols = cols, a.splits = cut.splits, a.per = cut.per, a.top = top;
    a.past = beyond_cache(rows, cols, dtype);
    scale_of(temperature, a.c, a.c_lo, a.inv_t);
    if (dtype == ISG_F32) launch_backward<LogprobsBwd<float>, narrow_backward(ISG_F32, false)>(cut, logits, a, dlogits, s);
    else launch_backward<LogprobsBwd<__hip_bfloat16>, narrow_backward(ISG_BF16, false)>(cut, logits, a, dlogits, s);
    return isg::check_launch("logprobs_bwd_kernel");
}
