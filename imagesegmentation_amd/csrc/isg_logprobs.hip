// Log-probabilities of given classes with the row's entropy and its most probable classes, and the divergence of a
// row from a teacher's most probable classes - forward and backward over the class axis.
//
// A row z of n logits at temperature T has, with m = max z and x_c = (z_c - m) log2(e) / T,
//   log p_c = ln 2 (x_c - log2 s),   s = sum 2^x_c,   H = -sum p_c log p_c = ln 2 (log2 s - (sum 2^x_c x_c) / s);
// every term of H has one sign, so a confident row loses nothing to cancellation, and z_c - m comes first, so that
// rows of the type's lowest value are uniform rows and not overflows.  A class at -inf has no probability and adds
// nothing (its x is kept from meeting 0 * inf by a lower bound far below the smallest float).  All sums are float.
//
// Layout.  A row is read once, into registers: up to 2,048 classes by one wave (four rows to a workgroup, no barrier),
// longer ones by workgroups that walk over equal parts of it, whose results (maximum, sums, best classes) a second
// launch joins.
#include <hip/hip_bf16.h>

#include <math.h>

#include <type_traits>

#include "isg_common.h"

namespace {

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLog2eLo = (float)(1.44269504088896340736 - (double)kLog2e);  // (positive)
constexpr float kLn2 = 0.69314718055994530942f;
constexpr int kThreads = 256;
constexpr int kMaxTop = ISG_TOP_MAX;          // classes kept per row
constexpr int kMaxEntries = ISG_DISTILL_MAX;  // a teacher's classes per row
constexpr int kMaxCols = ISG_CLASSES_MAX;     // class axis
constexpr int kWaveCols = 2048;               // classes one wave holds at most (32 registers a lane)
constexpr int kCandidates = 256;              // alternatives in question per wave; a workgroup holds four times as many
constexpr int kListMax = 1024;                // alternatives a workgroup collects along its part of a row
constexpr int kListTrim = 256;                // ... before it goes back to the best, of which it may keep
constexpr int kListKeep = 128;                // this many

typedef unsigned long long u64;

// ---- across the lanes of a wave --------------------------------------------------------------------------------------
// Data-parallel moves as part of the operation itself: six instructions and no LDS.  A lane without a source keeps its
// value, lane 63 ends up with the whole wave's.  (Written out: as compiler builtins every step becomes a move, a
// quieting maximum and the operation.)  The s_nop are the two states such a read has to stay behind the write.
#define ISG_WAVE_STEPS(op)                                                 \
    "s_nop 1\n\t" op " %0, %0, %0 row_shr:1 row_mask:0xf bank_mask:0xf\n\t"  \
    "s_nop 1\n\t" op " %0, %0, %0 row_shr:2 row_mask:0xf bank_mask:0xf\n\t"  \
    "s_nop 1\n\t" op " %0, %0, %0 row_shr:4 row_mask:0xf bank_mask:0xf\n\t"  \
    "s_nop 1\n\t" op " %0, %0, %0 row_shr:8 row_mask:0xf bank_mask:0xf\n\t"  \
    "s_nop 1\n\t" op " %0, %0, %0 row_bcast:15 row_mask:0xa bank_mask:0xf\n\t" \
    "s_nop 1\n\t" op " %0, %0, %0 row_bcast:31 row_mask:0xc bank_mask:0xf\n\t" \
    "s_nop 1"
__device__ __forceinline__ float last_lane(float v) {
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}
__device__ __forceinline__ float wave_max(float v) {
    asm volatile(ISG_WAVE_STEPS("v_max_f32_dpp") : "+v"(v));
    return last_lane(v);
}
__device__ __forceinline__ float wave_sum(float v) {
    asm volatile(ISG_WAVE_STEPS("v_add_f32_dpp") : "+v"(v));
    return last_lane(v);
}
// sum of the lanes up to and including this one
__device__ __forceinline__ int wave_scan(int v) {
    asm volatile(ISG_WAVE_STEPS("v_add_u32_dpp") : "+v"(v));
    return v;
}
__device__ __forceinline__ u64 wave_max_key(u64 k) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const u64 other = __shfl_xor(k, o);
        k = other > k ? other : k;
    }
    return k;
}

// W waves that share a row: LDS written by one lane is there for the others
template <int W>
__device__ __forceinline__ void together() {
    if constexpr (W == 1) {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    } else {
        __syncthreads();
    }
}

__device__ __forceinline__ float ld(const float* p, long long i) { return p[i]; }
__device__ __forceinline__ float ld(const __hip_bfloat16* p, long long i) { return (float)p[i]; }

// N logits from any address, as floats (N sizeof(T) is 2 to 16 bytes: one load)
template <int N>
__device__ __forceinline__ void load_vector(const float* p, float* v) {
    __builtin_memcpy(v, p, N * 4);
}
template <int N>
__device__ __forceinline__ void load_vector(const __hip_bfloat16* p, float* v) {
    if constexpr (N == 1) {
        v[0] = (float)p[0];
    } else {
        unsigned w[N / 2];
        __builtin_memcpy(w, p, N * 2);
#pragma unroll
        for (int i = 0; i < N / 2; ++i) v[2 * i] = __uint_as_float(w[i] << 16), v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}
// (floats to bf16 round to nearest even, by the chip's own conversion)
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
template <int N>
__device__ __forceinline__ void store_vector(float* p, const float* v) {
    __builtin_memcpy(p, v, N * 4);
}
template <int N>
__device__ __forceinline__ void store_vector(__hip_bfloat16* p, const float* v) {
    if constexpr (N == 1) {
        const __bf16 b = (__bf16)v[0];
        __builtin_memcpy(p, &b, 2);
    } else {
        bf16x2 w[N / 2];
#pragma unroll
        for (int i = 0; i < N / 2; ++i) w[i] = __builtin_convertvector(f32x2{v[2 * i], v[2 * i + 1]}, bf16x2);
        __builtin_memcpy(p, w, N * 2);
    }
}

// Where the elements of a thread lie in its unit's part [lo, hi) of a row: NE of them in vectors of VE (16 bytes), the
// vectors of a slot side by side over the unit's W * 64 threads, on 16-byte boundaries of memory from `first` <= lo on.
// (Rows of 131,071 bf16 logits start on any even address, where a 16-byte load takes three cache accesses instead of one:
// the walk over 2,048 of them took 156 us instead of 141.  Boundaries of 128 bytes gained nothing more.)  The part's
// outer vectors may reach outside; they are read from lo and up to hi instead, and `start` tells which of their elements
// are this thread's own.
template <typename T, int W, int NE>
struct Span {
    static constexpr int VE = NE < 16 / (int)sizeof(T) ? NE : 16 / (int)sizeof(T);
    static constexpr int NV = NE / VE;
    static constexpr int kCols = W * 64 * NE;
    int lo, hi, first, lane;  // lane: of the unit's W * 64

    // z: the row, whose memory the vectors are aligned in
    __device__ __forceinline__ Span(const T* z, int lo_, int hi_, int lane_) : lo(lo_), hi(hi_), lane(lane_) {
        first = lo - (int)(((uintptr_t)z / sizeof(T) + (unsigned)lo) % VE);
    }
    __device__ __forceinline__ void next() { first += kCols; }  // to the following kCols classes
    __device__ __forceinline__ bool more() const { return first < hi; }
    __device__ __forceinline__ bool whole() const { return first >= lo && first + kCols <= hi; }  // (uniform)
    __device__ __forceinline__ bool empty(int slot) const { return first + slot * W * 64 * VE >= hi; }  // (uniform)
    __device__ __forceinline__ int start(int slot) const { return first + (slot * W * 64 + lane) * VE; }
    __device__ __forceinline__ int inside(int s) const {
        s = s < hi - VE ? s : hi - VE;
        return s > lo ? s : lo;
    }
    // the class of element e, or -1 where it is another thread's (or none)
    __device__ __forceinline__ int cls(int e) const {
        const int s = start(e / VE), i = inside(s) + e % VE;
        return i >= s && i < s + VE ? i : -1;
    }
    // thread and element of a class of the unit
    __device__ __forceinline__ void locate(int c, int& thread, int& e) const {
        const int vec = (c - first) / VE;
        thread = vec % (W * 64);
        e = vec / (W * 64) * VE + c - inside(first + vec * VE);
    }
    // the elements; those that are not this thread's as -inf (BLANK) or as whatever class lies there
    template <bool BLANK>
    __device__ __forceinline__ void load(const T* z, float (&v)[NE]) const {
#pragma unroll
        for (int t = 0; t < NV; ++t) {
            if (!empty(t)) {
                load_vector<VE>(z + inside(start(t)), v + t * VE);
            } else {
#pragma unroll
                for (int j = 0; j < VE; ++j) v[t * VE + j] = -INFINITY;
            }
        }
        if constexpr (BLANK) blank(v);
    }
    __device__ __forceinline__ void blank(float (&v)[NE]) const {
#pragma unroll
        for (int t = 0; t < NV; ++t) {
            const int f = first + t * W * 64 * VE;
            if (f >= lo && f + W * 64 * VE <= hi) continue;  // (uniform)
            const int s = start(t), from = s - inside(s);    // own: from <= j < from + VE
#pragma unroll
            for (int j = 0; j < VE; ++j) v[t * VE + j] = j >= from && j < from + VE ? v[t * VE + j] : -INFINITY;
        }
    }
    // the same in two halves, for loads that are on their way while other elements are worked on
    static constexpr int kWords = NE * (int)sizeof(T) / 4;
    __device__ __forceinline__ void fetch(const T* z, unsigned (&raw)[kWords]) const {
#pragma unroll
        for (int t = 0; t < NV; ++t) __builtin_memcpy(raw + t * (kWords / NV), z + inside(start(t)), 16);
    }
    __device__ __forceinline__ void unpack(const unsigned (&raw)[kWords], float (&v)[NE]) const {
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
            if constexpr (sizeof(T) == 4) v[i] = __uint_as_float(raw[i]);
            else v[2 * i] = __uint_as_float(raw[i] << 16), v[2 * i + 1] = __uint_as_float(raw[i] & 0xffff0000u);
        }
        if (!whole()) blank(v);
    }
    // a slot's gradients (what the outer vectors repeat of their neighbours they repeat with the same values)
    __device__ __forceinline__ void store(T* d, int t, const float* o) const {
        const int s = start(t);
        if (s < hi && s + VE > lo) store_vector<VE>(d + inside(s), o);
    }
};

// a class index stored as 4 or 8 bytes
__device__ __forceinline__ long long class_at(const void* p, int bytes, long long i) {
    return bytes == 8 ? static_cast<const long long*>(p)[i] : (long long)static_cast<const int*>(p)[i];
}

// Order of the alternatives as one integer: larger logits first (-0 equals 0, NaN below -inf), equal ones by class;
// 0 is no class.
__device__ __forceinline__ unsigned order_bits(float v) {
    const unsigned b = __float_as_uint(v + 0.0f);
    if (v != v) return 1u;
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float order_value(unsigned k) {
    return k == 1u ? NAN : __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}
// the next float in that order: v > x where v >= above(x)
__device__ __forceinline__ float above(float x) { return order_value(order_bits(x) + 1u); }
__device__ __forceinline__ u64 order_key(float v, int c) { return ((u64)order_bits(v) << 32) | (unsigned)~c; }

// one bit an element (bit e: element e) where v[e] >= low: a comparison and an addition with carry each
template <int NE>
__device__ __forceinline__ unsigned reach_mask(const float (&v)[NE], float low) {
    unsigned hit = 0;
    if constexpr (NE % 8 == 0) {
#pragma unroll
        for (int e = NE - 4; e >= 0; e -= 4) {
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
        for (int e = NE - 1; e >= 0; --e) hit = hit + hit + (v[e] >= low ? 1u : 0u);
    }
    return hit;
}

// log p of a logit; a row without any probability (log2 s = +inf) gives -inf.  In nats throughout: at T = 1 the
// type's lowest value has a finite logarithm, its binary one would overflow.
__device__ __forceinline__ float log_prob(float z, float m, float inv_t, float l2s) {
    return (z - m) * inv_t - kLn2 * l2s;
}

// 2^((z - m) (c + c_lo)) with the exponent's whole part taken off before anything is rounded: an exponent of -8 as one
// float is off by 5e-7 of the power already.  For float gradients and for differences of probabilities.
__device__ __forceinline__ float power_exact(float z, float m, float c, float c_lo) {
    const float d = z - m, n = rintf(fmaxf(d * c, -300.0f));
    return ldexpf(__builtin_amdgcn_exp2f(__builtin_fmaf(d, c_lo, __builtin_fmaf(d, c, -n))), (int)n);
}

// ---- the `top` first keys of a unit ----------------------------------------------------------------------------------
// The k-th largest of the threads' group maxima is a lower bound of the k-th largest element (k groups hold one at
// least as large), so the elements not below it are few more than k: k + k^2 / (2 groups) for values in any order.
// The bound is found to 16 bits by bisection - one comparison a group and a count of the wave's mask per bit, the
// scalar unit's work -, the elements above it are put side by side in LDS, and each one's place is the number of keys
// above its own.  Bounds that no finite logit supports and more ties than fit go one class at a time instead.
template <int W>
struct TopShared {
    u64 cand[4 * kCandidates];   // W = 1: a quarter for each wave
    unsigned group[W == 1 ? 1 : kThreads];
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

__device__ __forceinline__ unsigned group_bound(float lane_max, int k, TopShared<4>& sh) {
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

template <int W, int NE, typename Reload, typename Emit>
__device__ __forceinline__ void select_top(const float (&v)[NE], int k, TopShared<W>& sh, Reload reload, Emit emit) {
    constexpr int Q = W == 1 ? (NE < 4 ? NE : 4) : 1;
    constexpr int kCap = W == 1 ? kCandidates : 4 * kCandidates;
    const int lane = threadIdx.x & 63, tid = W == 1 ? lane : threadIdx.x;
    u64* cand = sh.cand + (W == 1 ? (threadIdx.x >> 6) * kCandidates : 0);
    float gm[Q];
#pragma unroll
    for (int q = 0; q < Q; ++q) {
        gm[q] = v[q];
#pragma unroll
        for (int e = q + Q; e < NE; e += Q) gm[q] = fmaxf(gm[q], v[e]);
    }
    unsigned bound = 0;
    if constexpr (W == 1) {
        if (k > 16) {  // (several groups a lane: fewer elements to each)
            unsigned g[Q];
#pragma unroll
            for (int q = 0; q < Q; ++q) g[q] = order_bits(gm[q]) >> 16;
            for (int bit = 15; bit >= 0; --bit) {
                const unsigned t = bound | (1u << bit);
                int n = 0;
#pragma unroll
                for (int q = 0; q < Q; ++q) n += __builtin_popcountll(__ballot(g[q] >= t));
                if (n >= k) bound = t;
            }
        } else {
            float lm = gm[0];
#pragma unroll
            for (int q = 1; q < Q; ++q) lm = fmaxf(lm, gm[q]);
            const unsigned g = order_bits(lm) >> 16;
            for (int bit = 15; bit >= 0; --bit) {
                const unsigned t = bound | (1u << bit);
                if (__builtin_popcountll(__ballot(g >= t)) >= k) bound = t;
            }
        }
    } else {
        if (tid == 0) sh.count = 0;
        bound = group_bound(gm[0], k, sh);
    }
    int total = kCap + 1;
    if (bound > 0x7fu) {  // (0x7f begins the key of -inf)
        const float low = order_value(bound << 16);
        unsigned hit = reach_mask(v, low);
        const int mine = __builtin_popcount(hit), upto = wave_scan(mine);
        int at = upto - mine;
        if constexpr (W == 1) {
            total = __builtin_amdgcn_readlane(upto, 63);
        } else {
            at += wave_places(&sh.count, upto);
            together<W>();
            total = sh.count;
        }
        if (total <= kCap) {
            while (hit) {
                const int e = __builtin_ctz(hit);
                hit &= hit - 1;
                cand[at++] = reload(e);
            }
            together<W>();
            for (int r = tid; r < total; r += W * 64) {
                const u64 own = cand[r];
                int place = 0;
                for (int o = 0; o < total; ++o) place += cand[o] > own ? 1 : 0;
                if (place < k) emit(place, own);
            }
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
            best = wave_max_key(best);
            if constexpr (W > 1) {
                together<W>();
                if (lane == 0) sh.best[tid >> 6] = best;
                together<W>();
#pragma unroll
                for (int w = 0; w < W; ++w) best = sh.best[w] > best ? sh.best[w] : best;
            }
            last = best;
            if (tid == 0) emit(j, best);
            if (best == 0) {  // (fewer classes than are asked for: the last part of a split row)
                for (int o = j + 1 + tid; o < k; o += W * 64) emit(o, 0ull);
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

// A part without any probability has m = -inf and s = 0.
template <int NE>
__device__ __forceinline__ Sums wave_sums(const float (&v)[NE], float c) {
    float m = v[0];
#pragma unroll
    for (int e = 1; e < NE; ++e) m = fmaxf(m, v[e]);
    m = wave_max(m);
    const float mz = m == -INFINITY ? 0.0f : m;
    float s = 0.0f, u = 0.0f;
#pragma unroll
    for (int e = 0; e < NE; ++e) add_power(v[e], mz, c, s, u);
    return Sums{m, wave_sum(s), wave_sum(u)};
}

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

// a dead row's outputs
template <int W>
__device__ __forceinline__ void dead_row(const LogprobsArgs& a, long long row, int tid) {
    if (tid == 0) {
        if (a.logprobs) a.logprobs[row] = 0.0f;
        a.entropy[row] = 0.0f;
        if (a.stats) *reinterpret_cast<float4*>(a.stats + 4 * row) = make_float4(0.0f, INFINITY, 0.0f, 0.0f);
    }
    for (int j = tid; j < a.top; j += W * 64) a.top_logprobs[row * a.top + j] = 0.0f, a.top_classes[row * a.top + j] = -1;
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

__device__ __forceinline__ long long block_index() { return (long long)blockIdx.y * gridDim.x + blockIdx.x; }

// ---- token_logprobs ------------------------------------------------------------------------------------------------
// A row of up to kWaveCols classes: one wave.
template <typename T, int NE, bool TOP>
__global__ __launch_bounds__(kThreads) void logprobs_fwd_kernel(const T* __restrict__ logits, LogprobsArgs a) {
    __shared__ typename std::conditional<TOP, TopShared<1>, char>::type shared;
    const int lane = threadIdx.x & 63;
    const long long row = block_index() * 4 + (threadIdx.x >> 6);
    if (row >= a.units) return;
    if (a.live && !a.live[row]) {
        dead_row<1>(a, row, lane);
        return;
    }
    const T* z = logits + row * a.row_stride;
    const Span<T, 1, NE> span(z, 0, a.cols, lane);
    float v[NE];
    span.template load<true>(z, v);
    const RowStats r = row_stats(wave_sums(v, a.c), a.c_rel);
    if (lane == 0) row_outputs(a, z, row, r);
    if constexpr (TOP)
        select_top<1, NE>(
            v, a.top, shared,
            [&](int e) {
                const int i = span.cls(e);
                return i < 0 ? 0ull : order_key(ld(z, i), i);
            },
            [&](int place, u64 k) { row_alternative(a, row, r, place, k); });
}

// What a workgroup has found of a part of a row's best classes so far: the k first are among them, in no order.
struct TopList {
    u64 keys[kListMax];
    u64 kept[kListKeep];
    int count;
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

// The k first keys of the list in order, through emit(place, key): the place of a key is the number of keys above it.
template <typename Emit>
__device__ __forceinline__ void rank_list(const TopList& list, int count, int k, Emit emit) {
    for (int r = threadIdx.x; r < count; r += kThreads) {
        const u64 own = list.keys[r];
        int place = 0;
#pragma unroll 4
        for (int o = 0; o < count; ++o) place += list.keys[o] > own ? 1 : 0;
        if (place < k) emit(place, own);
    }
}

// Cuts the list back: what does not reach the prefix of its k-th key goes; where ties leave too much, all but the k
// first.  Returns the new count; `low` is a value that a class behind all of these has to exceed.
__device__ __forceinline__ int trim_list(TopList& list, int count, int k, float& low) {
    const unsigned bound = count <= 4 * 64 ? prefix_of<4>(list.keys, count, k)
                                           : (count <= 8 * 64 ? prefix_of<8>(list.keys, count, k)
                                                              : prefix_of<kListMax / 64>(list.keys, count, k));
    if (threadIdx.x == 0) list.count = 0;
    __syncthreads();
    for (int r = threadIdx.x; r < count; r += kThreads) {
        const u64 own = list.keys[r];
        if ((unsigned)(own >> 48) >= bound) {
            const int at = atomicAdd(&list.count, 1);
            if (at < kListKeep) list.kept[at] = own;
        }
    }
    __syncthreads();
    int n = list.count;
    if (n > kListKeep) {
        rank_list(list, count, k, [&](int place, u64 key) { list.kept[place] = key; });
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
// a list: of the first step all that reach the bound select_top would take (see there), of the later steps what exceeds
// the list's own bound, which rises whenever the list has grown to kListTrim and is cut back.  Steps that would overrun
// the list (rising rows, ties) or have no finite bound hand it their k first by select_top instead.
template <typename T, int NE, bool TOP>
__global__ __launch_bounds__(kThreads, sizeof(T) == 4 ? 5 : 6) void logprobs_stream_kernel(const T* __restrict__ logits, LogprobsArgs a) {
    __shared__ float red[4][4];
    __shared__ typename std::conditional<TOP, TopShared<4>, char>::type shared;
    __shared__ typename std::conditional<TOP, TopList, char>::type list;
    const int tid = threadIdx.x, lane = tid & 63;
    const long long unit = block_index();
    if (unit >= a.units) return;
    const long long row = a.splits == 1 ? unit : unit / a.splits;
    const int split = a.splits == 1 ? 0 : (int)(unit - row * a.splits);
    if (a.live && !a.live[row]) {
        if (a.splits == 1) dead_row<4>(a, row, tid);
        return;
    }
    const T* z = logits + row * a.row_stride;
    using S = Span<T, 4, NE>;
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
            const float m = wave_max(lane_max);
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
                    unsigned hit = reach_mask(v, reach);
                    const int mine = __builtin_popcount(hit), upto = wave_scan(mine);
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
                select_top<4, NE>(v, a.top, shared, reload, [&](int place, u64 k) { list.keys[count + place] = k; });
                __syncthreads();
                count += a.top;
            }
            if (count > kListTrim || !fits) {
                count = trim_list(list, count, a.top, low);
                bounded = low > -INFINITY;  // (no bound from classes at -inf or NaN)
            }
        }
    }
    // the waves' sums
    t.s = wave_sum(t.s), t.u = wave_sum(t.u);
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
        rank_list(list, count, a.top, [&](int place, u64 key) {
            if (a.splits == 1) row_alternative(a, row, r, place, key);
            else a.part_keys[unit * a.top + place] = key;
        });
    }
}

// Joins the parts of a row: one unit of W waves, NE keys a thread.
template <typename T, int W, int NE>
__global__ __launch_bounds__(kThreads) void logprobs_join_kernel(const T* __restrict__ logits, LogprobsArgs a) {
    __shared__ TopShared<W> shared;
    const int lane = threadIdx.x & 63, tid = W == 1 ? lane : threadIdx.x;
    const long long row = W == 1 ? block_index() * 4 + (threadIdx.x >> 6) : block_index();
    if (row >= a.units) return;
    if (a.live && !a.live[row]) {
        dead_row<W>(a, row, tid);
        return;
    }
    // (every wave for itself)
    const Sums* part = a.part + row * a.splits;
    Sums t{-INFINITY, 0.0f, 0.0f};
    for (int i = lane; i < a.splits; i += 64) merge_sums(t, part[i], a.c);
    const float m = wave_max(t.m);
    merge_sums(t, Sums{m, 0.0f, 0.0f}, a.c);  // (to the common maximum)
    t.s = wave_sum(t.s), t.u = wave_sum(t.u);
    const RowStats r = row_stats(t, a.c_rel);
    if (tid == 0) row_outputs(a, logits + row * a.row_stride, row, r);
    if (a.top == 0) return;
    const int n = a.splits * a.top;
    const u64* keys = a.part_keys + row * n;
    float v[NE];
#pragma unroll
    for (int e = 0; e < NE; ++e) {
        const int i = e * W * 64 + tid;
        const unsigned k = i < n ? (unsigned)(keys[i] >> 32) : 0u;
        v[e] = k ? order_value(k) : -INFINITY;
    }
    select_top<W, NE>(
        v, a.top, shared,
        [&](int e) {
            const int i = e * W * 64 + tid;
            return i < n ? keys[i] : 0ull;
        },
        [&](int place, u64 key) { row_alternative(a, row, r, place, key); });
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
    int token_bytes, cols, splits, per, top;
    float c, c_lo, inv_t;
};

template <typename T, int W, int NE>
__global__ __launch_bounds__(kThreads) void logprobs_bwd_kernel(const T* __restrict__ logits, LogprobsBwdArgs a,
                                                               T* __restrict__ dlogits) {
    const int lane = threadIdx.x & 63, tid = W == 1 ? lane : threadIdx.x;
    // (from the last unit back: what the forward pass read last is still in the last-level cache)
    const long long unit = a.units - 1 - (W == 1 ? block_index() * 4 + (threadIdx.x >> 6) : block_index());
    if (unit < 0) return;
    const long long row = a.splits == 1 ? unit : unit / a.splits;
    const int split = a.splits == 1 ? 0 : (int)(unit - row * a.splits);
    using S = Span<T, W, NE>;
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
    // (every wave for itself; top <= 64: one alternative a lane)
    float gt = 0.0f;
    int ti = -1;
    if (a.dtop && lane < a.top) gt = a.dtop[row * a.top + lane], ti = a.top_classes[row * a.top + lane];
    float g = a.dtop ? wave_sum(gt) + ga : ga;
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
        if (span.empty(t)) break;
        float o[S::VE];
#pragma unroll
        for (int j = 0; j < S::VE; ++j) o[j] = zero ? 0.0f : dense(v[t * S::VE + j]);
        span.store(d, t, o);
    }
    if (zero) return;
    together<W>();
    if (tid >= 64) return;
    const bool both = __ballot(ti >= 0 && ti == tok) != 0;
    if (ti >= lo && ti < hi) {
        const float o = __builtin_fmaf(a.inv_t, gt + (ti == tok ? ga : 0.0f), dense(ld(z, ti)));
        store_vector<1>(d + ti, &o);
    }
    if (lane == 0 && !both && tok >= lo && tok < hi) {
        const float o = __builtin_fmaf(a.inv_t, ga, dense(ld(z, tok)));
        store_vector<1>(d + tok, &o);
    }
}

// ---- distill_rows --------------------------------------------------------------------------------------------------
// What the backward pass keeps of a row: the dense part of its gradient is coef * ib * 2^((z - mb) c); at the teacher's
// classes it is total * is * 2^((z - m) c) - q, and q of entry j is iv * 2^((v_j - mv) cv).  is = 0: a row without
// gradient.
struct DistillStats {
    float mb, ib, coef, total, m, is, mv, iv;
};

// maximum and sum of powers of a row's classes outside the teacher's entries, and of the entries' own classes
struct DistillPart {
    float m, s, me, se;
};

struct DistillArgs {
    const float* values;
    const void* classes;
    const unsigned char* live;
    float* loss;
    DistillStats* stats;
    DistillPart* part;  // [rows][splits]
    long long row_stride, units;
    int class_bytes, cols, splits, per, k, tail;
    float c, c_lo, c_near, inv_t;
};

// 2^((z - m) (c + c_lo)): log2(e) / T to twice a float's digits, as a rounded c shifts every exponent the same way
__device__ __forceinline__ float power(float z, float m, float c, float c_lo) {
    const float d = z - m;
    return __builtin_amdgcn_exp2f(__builtin_fmaf(d, c_lo, d * c));
}

// ... of the many classes of a row: of bf16 logits by the nearest float alone (x is off by 2^-25 of itself at most)
template <typename T>
__device__ __forceinline__ float power_of(const DistillArgs& a, float z, float m) {
    return sizeof(T) == 4 ? power(z, m, a.c, a.c_lo) : __builtin_amdgcn_exp2f((z - m) * a.c_near);
}

// A remaining mass that rounding alone can leave of the entries' log-probabilities (k of them, each good to 2^-24 of
// its size): where the student has no class outside the entries it is no mass, anything above it has nowhere to go.
constexpr float kNoMass = 1e-5f;

constexpr int kMarkCols = 131072;  // classes a workgroup's part may have: one bit each (16 KB)

// (m, s) of two disjoint parts
__device__ __forceinline__ void merge(float& m, float& s, float m2, float s2, float c, float c_lo) {
    const float n = fmaxf(m, m2);
    const float a = s == 0.0f ? 0.0f : s * power(m, n, c, c_lo), b = s2 == 0.0f ? 0.0f : s2 * power(m2, n, c, c_lo);
    m = n, s = a + b;
}

__device__ __forceinline__ void distill_dead(const DistillArgs& a, long long row) {
    a.loss[row] = 0.0f;
    if (a.stats) a.stats[row] = DistillStats{0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
}

// whether an earlier entry names the class as well
__device__ bool named_before(const DistillArgs& a, long long row, int j, long long cls) {
    for (int o = 0; o < j; ++o)
        if (class_at(a.classes, a.class_bytes, row * a.k + o) == cls) return true;
    return false;
}

// log(1 + x): the logarithm of the rounded sum, corrected for what the rounding took
__device__ __forceinline__ float log1p_of(float x) {
    const float u = 1.0f + x;
    return u == 1.0f ? x : kLn2 * __builtin_amdgcn_logf(u) * (x / (u - 1.0f));
}

// The loss of a row from its sums, by one wave.
template <typename T>
__device__ __forceinline__ void distill_finish(const DistillArgs& a, const T* z, long long row, const DistillPart& t) {
    const int lane = threadIdx.x & 63;
    const float* v = a.values + row * a.k;
    float m = t.m, s = t.s;
    if (a.tail) merge(m, s, t.me, t.se, a.c, a.c_lo);
    m = m == -INFINITY ? 0.0f : m;
    const float l2s = s == 0.0f ? INFINITY : __builtin_amdgcn_logf(s);
    // (log s as a whole number of ln 2 and the logarithm of a fraction: added one after the other to a difference of the
    // same size it loses a rounding of that difference, not one of its own that every entry of the row would share)
    const float s_exp = (float)__builtin_amdgcn_frexp_expf(s), s_log = kLn2 * __builtin_amdgcn_logf(__builtin_amdgcn_frexp_mantf(s));
    // the teacher's distribution over its entries
    const float cv = a.tail ? kLog2e : a.c, cv_lo = a.tail ? kLog2eLo : a.c_lo;
    float mv = 0.0f, lv = 0.0f, sv = 0.0f;
    bool bad = false;
    if (!a.tail) {
        mv = -INFINITY;
        for (int j = lane; j < a.k; j += 64)
            if (class_at(a.classes, a.class_bytes, row * a.k + j) >= 0) mv = fmaxf(mv, v[j]);
        mv = wave_max(mv);
        if (mv == -INFINITY) mv = 0.0f;
    }
    for (int j = lane; j < a.k; j += 64) {
        const long long i = class_at(a.classes, a.class_bytes, row * a.k + j);
        if (i >= 0) sv += power(v[j], mv, cv, cv_lo);
        bad |= i >= a.cols;
    }
    sv = wave_sum(sv);
    if (!a.tail) lv = sv == 0.0f ? INFINITY : __builtin_amdgcn_logf(sv);
    const float qsum = a.tail ? sv : (sv == 0.0f ? 0.0f : 1.0f);
    float qr = a.tail ? fmaxf(1.0f - sv, 0.0f) : 0.0f;
    float l = 0.0f;
    for (int j = lane; j < a.k; j += 64) {
        const long long i = class_at(a.classes, a.class_bytes, row * a.k + j);
        if (i < 0 || i >= a.cols) continue;
        const float q = power(v[j], mv, cv, cv_lo) * __builtin_amdgcn_exp2f(-lv);
        const float lq = (v[j] - mv) * (a.tail ? 1.0f : a.inv_t) - kLn2 * lv;
        const float d = lq - (ld(z, i) - m) * a.inv_t;  // log q - log p - log s
        if (q != 0.0f) l += s == 0.0f ? INFINITY : q * (__builtin_fmaf(s_exp, kLn2, d) + s_log);
    }
    l = wave_sum(l);
    bad = __ballot(bad) != 0;
    if (lane == 0) {
        float coef = qsum, mb = m, ib = 1.0f / s;
        if (a.tail) {
            const bool none = t.s == 0.0f;
            const float mr = t.m == -INFINITY ? 0.0f : t.m, lr = none ? INFINITY : __builtin_amdgcn_logf(t.s);
            if (none && qr <= kNoMass) qr = 0.0f;
            // The student's mass outside, and the logarithm of the masses' ratio: from the logarithms where it is no
            // normal float; where the entries have less than half of it from their masses, as 1 - (a few) per cent on
            // both sides would cancel.
            const float pr = t.s * power(mr, m, a.c, a.c_lo) / s, pe = t.se * power(t.me, m, a.c, a.c_lo) / s;
            float ratio;
            coef = none ? 0.0f : (qsum + qr) * pr - qr;
            if (pe < 0.5f && sv < 1.0f) {
                coef = sv - pe;
                ratio = log1p_of((pe - sv) / pr);
            } else {
                const float lpr = pr > 1e-30f ? __builtin_amdgcn_logf(pr) : (mr - m) * a.c + (lr - l2s);
                ratio = kLn2 * (__builtin_amdgcn_logf(qr) - lpr);
            }
            if (qr > 0.0f) l += none ? INFINITY : qr * ratio;
            mb = mr, ib = none ? 0.0f : 1.0f / t.s;
        }
        if (bad) l = NAN, coef = NAN;
        a.loss[row] = l;
        if (a.stats)
            a.stats[row] = DistillStats{mb, ib, coef, qsum + qr, m, s == 0.0f ? 0.0f : 1.0f / s, mv,
                                        a.tail ? 1.0f : (sv == 0.0f ? 0.0f : 1.0f / sv)};
    }
}

// loss = sum_j q_j (log q_j - log p_(i_j)), and with TAIL the mass outside the entries as one more class:
// + q_r (log q_r - log p_r), where p_r is summed over those classes themselves (1 - sum would cancel).  For that every
// class an entry names is marked in LDS and blanked when its thread comes to it; the entries' own classes are summed
// from a second look at them.

// The sums (me, se) over the classes the entries name in [lo, hi), each once; mark(class) says whether it was marked
// before.  W waves share the entries; the result is the wave's.
template <int W, typename T, typename Mark>
__device__ __forceinline__ void mark_entries(const DistillArgs& a, const T* z, long long row, int lo, int hi, unsigned* repeated,
                                             DistillPart& t, Mark mark) {
    const int tid = W == 1 ? (threadIdx.x & 63) : threadIdx.x;
    bool twice = false;
    for (int j = tid; j < a.k; j += W * 64) {
        const long long i = class_at(a.classes, a.class_bytes, row * a.k + j);
        if (i >= lo && i < hi) twice |= mark((int)i);
    }
    if constexpr (W == 1) {
        twice = __ballot(twice) != 0;
        together<W>();
    } else {
        if (twice) *repeated = 1u;
        together<W>();
        twice = *repeated != 0;
    }
    for (int j = tid; j < a.k; j += W * 64) {
        const long long i = class_at(a.classes, a.class_bytes, row * a.k + j);
        if (i < lo || i >= hi) continue;
        if (twice && named_before(a, row, j, i)) continue;
        const float zi = ld(z, i);
        merge(t.me, t.se, zi, zi == -INFINITY ? 0.0f : 1.0f, a.c, a.c_lo);
    }
    const float m = wave_max(t.me);
    t.se = wave_sum(t.se == 0.0f ? 0.0f : t.se * power(t.me, m, a.c, a.c_lo));
    t.me = m;
}

// A row of up to kWaveCols classes: one wave.
template <typename T, int NE, bool TAIL>
__global__ __launch_bounds__(kThreads) void distill_fwd_kernel(const T* __restrict__ logits, DistillArgs a) {
    __shared__ unsigned marks[TAIL ? kThreads : 1];
    const int lane = threadIdx.x & 63;
    const long long row = block_index() * 4 + (threadIdx.x >> 6);
    if (row >= a.units) return;
    if (a.live && !a.live[row]) {
        if (lane == 0) distill_dead(a, row);
        return;
    }
    const T* z = logits + row * a.row_stride;
    using S = Span<T, 1, NE>;
    const S span(z, 0, a.cols, lane);
    float v[NE];
    span.template load<true>(z, v);
    DistillPart t{-INFINITY, 0.0f, -INFINITY, 0.0f};
    if constexpr (TAIL) {
        unsigned* mine = marks + (threadIdx.x - lane);
        mine[lane] = 0u;
        together<1>();
        mark_entries<1>(a, z, row, 0, a.cols, nullptr, t, [&](int i) {
            int thread, e;
            span.locate(i, thread, e);
            return (atomicOr(&mine[thread], 1u << e) >> e & 1u) != 0;
        });
        const unsigned hit = mine[lane];
#pragma unroll
        for (int e = 0; e < NE; ++e) v[e] = hit >> e & 1u ? -INFINITY : v[e];
    }
    float m = v[0];
#pragma unroll
    for (int e = 1; e < NE; ++e) m = fmaxf(m, v[e]);
    t.m = wave_max(m);
    const float mz = t.m == -INFINITY ? 0.0f : t.m;
    float s = 0.0f;
#pragma unroll
    for (int e = 0; e < NE; ++e) s += power_of<T>(a, v[e], mz);
    t.s = wave_sum(s);
    distill_finish(a, z, row, t);
}

// A part of a longer row, walked over as in logprobs_stream_kernel.  The marks are one bit a class of the part.
template <typename T, int NE, bool TAIL>
__global__ __launch_bounds__(kThreads) void distill_stream_kernel(const T* __restrict__ logits, DistillArgs a) {
    __shared__ DistillPart red[4];
    __shared__ unsigned char marks[TAIL ? kMarkCols / 8 + 16 : 16] __attribute__((aligned(16)));
    __shared__ unsigned repeated;
    const int tid = threadIdx.x, lane = tid & 63;
    const long long unit = block_index();
    if (unit >= a.units) return;
    const long long row = a.splits == 1 ? unit : unit / a.splits;
    const int split = a.splits == 1 ? 0 : (int)(unit - row * a.splits);
    if (a.live && !a.live[row]) {
        if (tid == 0 && a.splits == 1) distill_dead(a, row);
        return;
    }
    const T* z = logits + row * a.row_stride;
    using S = Span<T, 4, NE>;
    const int lo = split * a.per, hi = lo + a.per < a.cols ? lo + a.per : a.cols;
    unsigned raw[S::kWords];
    S ahead(z, lo, hi, tid);
    const int zero = ahead.first;  // the class of the first mark
    ahead.fetch(z, raw);
    DistillPart t{-INFINITY, 0.0f, -INFINITY, 0.0f};
    if constexpr (TAIL) {
        unsigned* words = reinterpret_cast<unsigned*>(marks);
        for (int i = tid; i < (hi - zero + 31) / 32; i += kThreads) words[i] = 0u;
        if (tid == 0) repeated = 0u;
        __syncthreads();
        mark_entries<4>(a, z, row, lo, hi, &repeated, t, [&](int i) {
            const int b = i - zero;
            return (atomicOr(&words[b >> 5], 1u << (b & 31)) >> (b & 31) & 1u) != 0;
        });
    }
    float s = 0.0f;
    while (ahead.more()) {
        const S span = ahead;
        float v[NE];
        span.unpack(raw, v);
        ahead.next();
        if (ahead.more()) ahead.fetch(z, raw);
        if constexpr (TAIL) {
#pragma unroll
            for (int q = 0; q < S::NV; ++q) {
                const int first = span.start(q), b = first - zero;
                unsigned bits = 0;
                if (first < hi) bits = (unsigned)marks[b >> 3] >> (b & 7) & ((1u << S::VE) - 1u);
                if (__ballot(bits != 0)) {
                    const int from = first - span.inside(first);  // (an outer vector is read from further in)
                    bits = from >= 0 ? bits << from : bits >> -from;
#pragma unroll
                    for (int j = 0; j < S::VE; ++j) v[q * S::VE + j] = bits >> j & 1u ? -INFINITY : v[q * S::VE + j];
                }
            }
        }
        float lane_max = v[0];
#pragma unroll
        for (int e = 1; e < NE; ++e) lane_max = fmaxf(lane_max, v[e]);
        if (__ballot(lane_max > t.m)) {
            const float m = wave_max(lane_max);
            if (t.m != -INFINITY) s *= power(t.m, m, a.c, a.c_lo);
            t.m = m;
        }
        const float mz = t.m == -INFINITY ? 0.0f : t.m;
#pragma unroll
        for (int e = 0; e < NE; ++e) s += power_of<T>(a, v[e], mz);
    }
    t.s = wave_sum(s);
    if (lane == 0) red[tid >> 6] = t;
    __syncthreads();
    if (tid >= 64) return;
    t = red[0];
#pragma unroll
    for (int w = 1; w < 4; ++w) {
        merge(t.m, t.s, red[w].m, red[w].s, a.c, a.c_lo);
        if constexpr (TAIL) merge(t.me, t.se, red[w].me, red[w].se, a.c, a.c_lo);
    }
    if (a.splits == 1)
        distill_finish(a, z, row, t);
    else if (lane == 0)
        a.part[unit] = t;
}

// Joins the parts of a row: one wave.
template <typename T>
__global__ __launch_bounds__(kThreads) void distill_join_kernel(const T* __restrict__ logits, DistillArgs a) {
    const int lane = threadIdx.x & 63;
    const long long row = block_index() * 4 + (threadIdx.x >> 6);
    if (row >= a.units) return;
    if (a.live && !a.live[row]) {
        if (lane == 0) distill_dead(a, row);
        return;
    }
    DistillPart t{-INFINITY, 0.0f, -INFINITY, 0.0f};
    for (int i = lane; i < a.splits; i += 64) {
        const DistillPart p = a.part[row * a.splits + i];
        merge(t.m, t.s, p.m, p.s, a.c, a.c_lo);
        merge(t.me, t.se, p.me, p.se, a.c, a.c_lo);
    }
    const float m = wave_max(t.m), me = wave_max(t.me);
    t.s = wave_sum(t.s == 0.0f ? 0.0f : t.s * power(t.m, m, a.c, a.c_lo));
    t.se = wave_sum(t.se == 0.0f ? 0.0f : t.se * power(t.me, me, a.c, a.c_lo));
    t.m = m, t.me = me;
    distill_finish(a, logits + row * a.row_stride, row, t);
}

struct DistillBwdArgs {
    const float* values;
    const void* classes;
    const DistillStats* stats;
    const float* dloss;
    long long row_stride, units;
    int class_bytes, cols, splits, per, k, tail;
    float c, c_lo, inv_t;
};

template <typename T, int W, int NE>
__global__ __launch_bounds__(kThreads) void distill_bwd_kernel(const T* __restrict__ logits, DistillBwdArgs a,
                                                              T* __restrict__ dlogits) {
    __shared__ unsigned marks[kThreads];
    __shared__ unsigned repeated;
    const int lane = threadIdx.x & 63, tid = W == 1 ? lane : threadIdx.x;
    const long long unit = a.units - 1 - (W == 1 ? block_index() * 4 + (threadIdx.x >> 6) : block_index());
    if (unit < 0) return;
    const long long row = a.splits == 1 ? unit : unit / a.splits;
    const int split = a.splits == 1 ? 0 : (int)(unit - row * a.splits);
    using S = Span<T, W, NE>;
    const int lo = split * a.per, hi = lo + a.per < a.cols ? lo + a.per : a.cols;
    T* d = dlogits + row * a.cols;
    const S span(d, lo, hi, tid);  // (aligned as the gradient; dense logits lie the same way)
    const DistillStats st = a.stats[row];
    const bool zero = st.is == 0.0f;  // a dead row, or no class has probability
    const T* z = logits + row * a.row_stride;
    float v[NE];
    if (!zero) span.template load<false>(z, v);
    const float g = a.dloss[row] * a.inv_t;
    const float gc = g * st.coef * st.ib;
#pragma unroll
    for (int t = 0; t < S::NV; ++t) {
        if (span.empty(t)) break;
        float o[S::VE];
#pragma unroll
        for (int j = 0; j < S::VE; ++j) {
            const float zi = v[t * S::VE + j];
            const float e = sizeof(T) == 4 ? power_exact(zi, st.mb, a.c, a.c_lo) : __builtin_amdgcn_exp2f((zi - st.mb) * a.c);
            o[j] = zero ? 0.0f : gc * e;
        }
        span.store(d, t, o);
    }
    if (zero || st.coef != st.coef) return;  // (NaN: an entry the row does not have; the whole row is)
    // the entries' classes once more, behind the dense part
    unsigned* mine = marks + (W == 1 ? threadIdx.x - lane : 0);
    mine[tid] = 0u;
    if (W > 1 && tid == 0) repeated = 0u;
    together<W>();
    bool twice = false;
    for (int j = tid; j < a.k; j += W * 64) {
        const long long i = class_at(a.classes, a.class_bytes, row * a.k + j);
        if (i < lo || i >= hi) continue;
        int thread, e;
        span.locate((int)i, thread, e);
        twice |= (atomicOr(&mine[thread], 1u << e) >> e & 1u) != 0;
    }
    if constexpr (W == 1) {
        twice = __ballot(twice) != 0;
    } else {
        if (twice) repeated = 1u;
        together<W>();
        twice = repeated != 0;
    }
    const float cv = a.tail ? kLog2e : a.c, cv_lo = a.tail ? kLog2eLo : a.c_lo;
    for (int j = tid; j < a.k; j += W * 64) {
        const long long i = class_at(a.classes, a.class_bytes, row * a.k + j);
        if (i < lo || i >= hi) continue;
        float q = st.iv * power_exact(a.values[row * a.k + j], st.mv, cv, cv_lo);
        if (twice) {  // (every place of the class writes the same sum)
            q = 0.0f;
            for (int o = 0; o < a.k; ++o)
                if (class_at(a.classes, a.class_bytes, row * a.k + o) == i)
                    q += st.iv * power_exact(a.values[row * a.k + o], st.mv, cv, cv_lo);
        }
        const float p = st.is * power_exact(ld(z, i), st.m, a.c, a.c_lo);
        const float o = g * (st.total * p - q);
        store_vector<1>(d + i, &o);
    }
}

// ---- launches ------------------------------------------------------------------------------------------------------
// How a row is cut: one wave for what its registers hold.  Beyond, the forward passes walk over parts of a row, as many
// as give kUnits workgroups but of at least kWaveCols classes; the backward passes have nothing to join and take
// workgroups of at most 32 classes a thread.  Parts are equal but for the rounding to 8 classes; there is room for those
// that start between two boundaries (Span).
constexpr long long kUnits = 4096;
constexpr int kMaxSplits = 128;
struct Cut {
    int waves, ne, splits, per;
};
int equal_part(int cols, int splits) { return ((cols + splits - 1) / splits + 7) / 8 * 8; }
// 0: too long for a wave
int wave_elements(int cols, int dtype) {
    const int sizes[] = {1, 2, 4, 8, 16, 24, 32}, most = dtype == ISG_F32 ? 4 : 8;
    for (int ne : sizes)
        if (cols + (ne < most ? ne : most) - 1 <= 64 * ne) return ne;
    return 0;
}
Cut cut_forward(long long rows, int cols, int dtype) {
    if (const int ne = wave_elements(cols, dtype)) return Cut{1, ne, 1, cols};
    long long splits = (kUnits + rows - 1) / (rows > 0 ? rows : 1);
    const int most = cols / kWaveCols < kMaxSplits ? cols / kWaveCols : kMaxSplits, least = (cols + kMarkCols - 1) / kMarkCols;
    splits = splits > most ? most : splits;
    splits = splits < least ? least : splits;
    const int per = equal_part(cols, (int)splits);
    return Cut{4, 16, (cols + per - 1) / per, per};
}
Cut cut_backward(long long rows, int cols, int dtype) {
    if (const int ne = wave_elements(cols, dtype)) return Cut{1, ne, 1, cols};
    const auto parts = [&](int ne) { return (cols + kThreads * ne - 8 - 1) / (kThreads * ne - 8); };
    for (int ne = 8;; ne *= 2) {
        if (ne < 32 && rows * parts(2 * ne) >= 1024) continue;  // (still four workgroups for each of the 256 CUs)
        const int per = equal_part(cols, parts(ne));
        return Cut{4, ne, (cols + per - 1) / per, per};
    }
}

dim3 grid_of(long long units, int waves) {
    const long long blocks = waves == 1 ? (units + 3) / 4 : units;
    const long long x = blocks < (1 << 20) ? blocks : (1 << 20);
    return dim3((unsigned)x, (unsigned)((blocks + x - 1) / x));
}

// F::template run<NE>(...) for a wave's cut
template <typename F, typename... A>
void with_wave(int ne, A&&... args) {
    switch (ne) {
        case 1: F::template run<1>(args...); break;
        case 2: F::template run<2>(args...); break;
        case 4: F::template run<4>(args...); break;
        case 8: F::template run<8>(args...); break;
        case 16: F::template run<16>(args...); break;
        case 24: F::template run<24>(args...); break;
        default: F::template run<32>(args...);
    }
}

template <typename T, bool TOP>
struct LogprobsFwd {
    template <int NE>
    static void run(const void* logits, const LogprobsArgs& a, hipStream_t s) {
        hipLaunchKernelGGL((logprobs_fwd_kernel<T, NE, TOP>), grid_of(a.units, 1), dim3(kThreads), 0, s,
                           static_cast<const T*>(logits), a);
    }
    static void launch(const Cut& cut, const void* logits, const LogprobsArgs& a, hipStream_t s) {
        if (cut.waves == 1)
            with_wave<LogprobsFwd>(cut.ne, logits, a, s);
        else
            hipLaunchKernelGGL((logprobs_stream_kernel<T, 16, TOP>), grid_of(a.units, 4), dim3(kThreads), 0, s,
                               static_cast<const T*>(logits), a);
    }
};
template <typename T, int W, int NE>
void launch_join(const void* logits, const LogprobsArgs& a, hipStream_t s) {
    hipLaunchKernelGGL((logprobs_join_kernel<T, W, NE>), grid_of(a.units, W), dim3(kThreads), 0, s,
                       static_cast<const T*>(logits), a);
}
template <typename T>
struct LogprobsBwd {
    template <int NE, int W = 1>
    static void run(const void* logits, const LogprobsBwdArgs& a, void* dlogits, hipStream_t s) {
        hipLaunchKernelGGL((logprobs_bwd_kernel<T, W, NE>), grid_of(a.units, W), dim3(kThreads), 0, s,
                           static_cast<const T*>(logits), a, static_cast<T*>(dlogits));
    }
};
template <typename T, bool TAIL>
struct DistillFwd {
    template <int NE>
    static void run(const void* logits, const DistillArgs& a, hipStream_t s) {
        hipLaunchKernelGGL((distill_fwd_kernel<T, NE, TAIL>), grid_of(a.units, 1), dim3(kThreads), 0, s,
                           static_cast<const T*>(logits), a);
    }
    static void launch(const Cut& cut, const void* logits, const DistillArgs& a, hipStream_t s) {
        if (cut.waves == 1)
            with_wave<DistillFwd>(cut.ne, logits, a, s);
        else
            hipLaunchKernelGGL((distill_stream_kernel<T, 16, TAIL>), grid_of(a.units, 4), dim3(kThreads), 0, s,
                               static_cast<const T*>(logits), a);
    }
};
template <typename T>
struct DistillBwd {
    template <int NE, int W = 1>
    static void run(const void* logits, const DistillBwdArgs& a, void* dlogits, hipStream_t s) {
        hipLaunchKernelGGL((distill_bwd_kernel<T, W, NE>), grid_of(a.units, W), dim3(kThreads), 0, s,
                           static_cast<const T*>(logits), a, static_cast<T*>(dlogits));
    }
};
template <typename F, typename... A>
void launch_backward(const Cut& cut, A&&... args) {
    if (cut.waves == 1) with_wave<F>(cut.ne, args...);
    else if (cut.ne == 8) F::template run<8, 4>(args...);
    else if (cut.ne == 16) F::template run<16, 4>(args...);
    else F::template run<32, 4>(args...);
}

// The keys of a row's parts: one wave while they fit its registers.
template <typename T>
void join_parts(int n, const void* logits, const LogprobsArgs& a, hipStream_t s) {
    if (n <= 64 * 4) launch_join<T, 1, 4>(logits, a, s);
    else if (n <= 64 * 8) launch_join<T, 1, 8>(logits, a, s);
    else if (n <= kThreads * 4) launch_join<T, 4, 4>(logits, a, s);
    else if (n <= kThreads * 8) launch_join<T, 4, 8>(logits, a, s);
    else launch_join<T, 4, 32>(logits, a, s);
}

int check_call(const char* who, long long row_stride, int rows, int cols, int dtype, float temperature) {
    ISG_REQUIRE(rows >= 0 && cols >= 1 && cols <= kMaxCols, ISG_EINVAL, "%s: bad shape rows=%d cols=%d (at most %d classes)",
                who, rows, cols, kMaxCols);
    ISG_REQUIRE(dtype == ISG_F32 || dtype == ISG_BF16, ISG_EDTYPE, "%s: dtype %d", who, dtype);
    ISG_REQUIRE(row_stride >= cols, ISG_EINVAL, "%s: rows of %d classes %lld elements apart", who, cols, row_stride);
    ISG_REQUIRE(temperature >= 1e-30f && temperature <= 1e30f, ISG_EINVAL, "%s: temperature %g", who, (double)temperature);
    return ISG_OK;
}

int check_bytes(const char* who, const void* classes, int bytes) {
    ISG_REQUIRE(!classes || bytes == 4 || bytes == 8, ISG_EINVAL, "%s: classes of %d bytes (4 or 8)", who, bytes);
    return ISG_OK;
}

int check_top(const char* who, int top, int cols) {
    ISG_REQUIRE(top >= 0 && top <= kMaxTop && top <= cols, ISG_EINVAL, "%s: top=%d of %d classes (at most %d)", who, top, cols,
                kMaxTop);
    return ISG_OK;
}

int check_entries(const char* who, int k, int tail) {
    ISG_REQUIRE(k >= 1 && k <= kMaxEntries, ISG_EINVAL, "%s: k=%d classes of the teacher (1 to %d)", who, k, kMaxEntries);
    ISG_REQUIRE(tail == 0 || tail == 1, ISG_EINVAL, "%s: tail=%d", who, tail);
    return ISG_OK;
}

// log2(e) / T as the float below it and what is missing, which is positive (an infinite distance times both parts is an
// infinity of one sign)
void scale_of(float temperature, float& c, float& c_lo, float& inv_t) {
    const double exact = 1.4426950408889634074 / (double)temperature;
    c = (float)exact;
    if ((double)c >= exact) c = nextafterf(c, 0.0f);
    c_lo = (float)(exact - (double)c);
    inv_t = (float)(1.0 / (double)temperature);
}

}  // namespace

extern "C" long long isg_token_logprobs_workspace_bytes(int rows, int cols, int top) {
    if (rows < 0 || cols < 1 || cols > kMaxCols || top < 0 || top > kMaxTop) return -1;
    const Cut cut = cut_forward(rows, cols, ISG_BF16);  // (the same for float: types differ in rows of one part)
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
    const Cut cut = cut_forward(rows, cols, dtype);
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
    ISG_REQUIRE(dlogits != logits, ISG_EINVAL, "%s: dlogits must not alias the logits", who);
    const Cut cut = cut_backward(rows, cols, dtype);
    hipStream_t s = static_cast<hipStream_t>(stream);
    LogprobsBwdArgs a{};
    a.tokens = tokens, a.top_classes = top_classes, a.stats = stats;
    a.dlogprobs = dlogprobs, a.dentropy = dentropy, a.dtop = dtop_logprobs;
    a.row_stride = row_stride, a.units = (long long)rows * cut.splits;
    a.token_bytes = token_bytes, a.cols = cols, a.splits = cut.splits, a.per = cut.per, a.top = top;
    scale_of(temperature, a.c, a.c_lo, a.inv_t);
    if (dtype == ISG_F32) launch_backward<LogprobsBwd<float>>(cut, logits, a, dlogits, s);
    else launch_backward<LogprobsBwd<__hip_bfloat16>>(cut, logits, a, dlogits, s);
    return isg::check_launch("logprobs_bwd_kernel");
}

extern "C" long long isg_distill_workspace_bytes(int rows, int cols) {
    if (rows < 0 || cols < 1 || cols > kMaxCols) return -1;
    const Cut cut = cut_forward(rows, cols, ISG_BF16);  // (the same for float: types differ in rows of one part)
    return cut.splits == 1 ? 0 : (long long)rows * cut.splits * (long long)sizeof(DistillPart);
}

extern "C" int isg_distill_fwd(const void* logits, long long row_stride, const float* values, const void* classes,
                               int class_bytes, const unsigned char* live, int rows, int cols, int k, int dtype,
                               float temperature, int tail, float* loss, float* stats, void* workspace, void* stream) {
    const char* who = "isg_distill_fwd";
    int rc = check_call(who, row_stride, rows, cols, dtype, temperature);
    if (rc != ISG_OK) return rc;
    rc = check_entries(who, k, tail);
    if (rc != ISG_OK) return rc;
    rc = check_bytes(who, classes, class_bytes);
    if (rc != ISG_OK) return rc;
    if (rows == 0) return ISG_OK;
    ISG_REQUIRE(logits && values && classes && loss, ISG_EINVAL, "%s: null pointer", who);
    const Cut cut = cut_forward(rows, cols, dtype);
    ISG_REQUIRE(cut.splits == 1 || workspace, ISG_EINVAL, "%s: %d x %d logits need a workspace", who, rows, cols);
    hipStream_t s = static_cast<hipStream_t>(stream);
    DistillArgs a{};
    a.values = values, a.classes = classes, a.live = live, a.loss = loss;
    a.stats = reinterpret_cast<DistillStats*>(stats), a.part = static_cast<DistillPart*>(workspace);
    a.row_stride = row_stride, a.units = (long long)rows * cut.splits;
    a.class_bytes = class_bytes, a.cols = cols, a.splits = cut.splits, a.per = cut.per, a.k = k, a.tail = tail;
    scale_of(temperature, a.c, a.c_lo, a.inv_t);
    a.c_near = (float)(1.4426950408889634074 / (double)temperature);
    if (dtype == ISG_F32)
        tail ? DistillFwd<float, true>::launch(cut, logits, a, s) : DistillFwd<float, false>::launch(cut, logits, a, s);
    else
        tail ? DistillFwd<__hip_bfloat16, true>::launch(cut, logits, a, s)
             : DistillFwd<__hip_bfloat16, false>::launch(cut, logits, a, s);
    rc = isg::check_launch("distill_fwd_kernel");
    if (rc != ISG_OK || cut.splits == 1) return rc;
    a.units = rows;
    if (dtype == ISG_F32)
        hipLaunchKernelGGL(distill_join_kernel<float>, grid_of(rows, 1), dim3(kThreads), 0, s,
                           static_cast<const float*>(logits), a);
    else
        hipLaunchKernelGGL(distill_join_kernel<__hip_bfloat16>, grid_of(rows, 1), dim3(kThreads), 0, s,
                           static_cast<const __hip_bfloat16*>(logits), a);
    return isg::check_launch("distill_join_kernel");
}

extern "C" int isg_distill_bwd(const void* logits, long long row_stride, const float* values, const void* classes,
                               int class_bytes, const float* stats, const float* dloss, int rows, int cols, int k,
                               int dtype, float temperature, int tail, void* dlogits, void* stream) {
    const char* who = "isg_distill_bwd";
    int rc = check_call(who, row_stride, rows, cols, dtype, temperature);
    if (rc != ISG_OK) return rc;
    rc = check_entries(who, k, tail);
    if (rc != ISG_OK) return rc;
    rc = check_bytes(who, classes, class_bytes);
    if (rc != ISG_OK) return rc;
    if (rows == 0) return ISG_OK;
    ISG_REQUIRE(logits && values && classes && stats && dloss && dlogits, ISG_EINVAL, "%s: null pointer", who);
    ISG_REQUIRE(dlogits != logits, ISG_EINVAL, "%s: dlogits must not alias the logits", who);
    const Cut cut = cut_backward(rows, cols, dtype);
    hipStream_t s = static_cast<hipStream_t>(stream);
    DistillBwdArgs a{};
    a.values = values, a.classes = classes, a.stats = reinterpret_cast<const DistillStats*>(stats), a.dloss = dloss;
    a.row_stride = row_stride, a.units = (long long)rows * cut.splits;
    a.class_bytes = class_bytes, a.cols = cols, a.splits = cut.splits, a.per = cut.per, a.k = k, a.tail = tail;
    scale_of(temperature, a.c, a.c_lo, a.inv_t);
    if (dtype == ISG_F32) launch_backward<DistillBwd<float>>(cut, logits, a, dlogits, s);
    else launch_backward<DistillBwd<__hip_bfloat16>>(cut, logits, a, dlogits, s);
    return isg::check_launch("distill_bwd_kernel");
}
