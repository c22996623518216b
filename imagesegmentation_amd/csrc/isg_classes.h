// What the kernels over the class axis share (isg_logprobs.hip, isg_distill.hip): how a row lies over the lanes, sums and
// maxima across them, exponents, the order of the classes, and how launches cut them.
//
// A row z of n logits at temperature T has, with m = max z and x_c = (z_c - m) log2(e) / T,
//   log p_c = ln 2 (x_c - log2 s),   s = sum 2^x_c,   H = -sum p_c log p_c = ln 2 (log2 s - (sum 2^x_c x_c) / s);
// both terms of H have one sign, and z_c - m comes first, so that rows of the type's lowest value are uniform rows and not
// overflows.  A class at -inf has no probability and adds nothing (its x is kept from meeting 0 * inf by a lower bound far
// below the smallest float).  All sums are float.  s is 1 + e in a row whose other classes have e of the mass together, and
// is rounded before its logarithm: log p and H are good to some 1e-7 absolutely, not relatively.  Of an e below 6e-8 nothing
// is left in log p of the row's class (0 for -e), and H = e (1 - log e) lacks its first e, a twentieth or so.  (A sum
// without the maximum would keep it, at an operation more a class.)
//
// Layout.  A row is read once, into registers: up to about 1,000 classes by 16 lanes (four rows a wave: what a row costs
// once - reductions, logarithms, outputs - is paid for four rows in the same instructions), up to about 2,000 by 32
// lanes, or by a whole wave where there are few rows or much to do for each class that counts (cut_forward, cut_backward).
// Longer rows are walked over by workgroups, a part of the row each, whose results a second launch joins.
#pragma once
#include <hip/hip_bf16.h>

#include <math.h>

#include <type_traits>

#include "isg_common.h"

namespace {

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLog2eLo = (float)(1.44269504088896340736 - (double)kLog2e);  // (positive)
constexpr float kLn2 = 0.69314718055994530942f;
constexpr int kThreads = 256;
constexpr int kMaxCols = ISG_CLASSES_MAX;

typedef unsigned long long u64;

// ---- across lanes: G of them (16, 32 or 64 side by side) share a row ---------------------------------------------------
// Data-parallel moves as part of the operation itself: four instructions for 16 lanes, six for a wave, and no LDS.
// (Written out: as compiler builtins every step becomes a move, a quieting maximum and the operation.)  The s_nop are
// the two states such a read has to stay behind the write.
#define ISG_ROTATIONS(op)                                                  \
    "s_nop 1\n\t" op " %0, %0, %0 row_ror:8 row_mask:0xf bank_mask:0xf\n\t"  \
    "s_nop 1\n\t" op " %0, %0, %0 row_ror:4 row_mask:0xf bank_mask:0xf\n\t"  \
    "s_nop 1\n\t" op " %0, %0, %0 row_ror:2 row_mask:0xf bank_mask:0xf\n\t"  \
    "s_nop 1\n\t" op " %0, %0, %0 row_ror:1 row_mask:0xf bank_mask:0xf\n\t"  \
    "s_nop 1"
// (a lane without a source keeps its value; the last lane ends up with everything)
#define ISG_SHIFTS(op)                                                     \
    "s_nop 1\n\t" op " %0, %0, %0 row_shr:1 row_mask:0xf bank_mask:0xf\n\t"  \
    "s_nop 1\n\t" op " %0, %0, %0 row_shr:2 row_mask:0xf bank_mask:0xf\n\t"  \
    "s_nop 1\n\t" op " %0, %0, %0 row_shr:4 row_mask:0xf bank_mask:0xf\n\t"  \
    "s_nop 1\n\t" op " %0, %0, %0 row_shr:8 row_mask:0xf bank_mask:0xf\n\t"
#define ISG_BCAST15(op) "s_nop 1\n\t" op " %0, %0, %0 row_bcast:15 row_mask:0xa bank_mask:0xf\n\t"
#define ISG_BCAST31(op) "s_nop 1\n\t" op " %0, %0, %0 row_bcast:31 row_mask:0xc bank_mask:0xf\n\t"

__device__ __forceinline__ float last_lane(float v) {
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}
// the value of the 16 lanes beside: rows 0 and 1 of a wave (2 and 3) exchanged
__device__ __forceinline__ unsigned other_row(unsigned v, unsigned& own) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    own = r[0];
    return r[1];
}
template <int G>
__device__ __forceinline__ float group_max(float v) {
    if constexpr (G == 64) {
        asm volatile(ISG_SHIFTS("v_max_f32_dpp") ISG_BCAST15("v_max_f32_dpp") ISG_BCAST31("v_max_f32_dpp") "s_nop 1" : "+v"(v));
        return last_lane(v);
    }
    asm volatile(ISG_ROTATIONS("v_max_f32_dpp") : "+v"(v));
    if constexpr (G == 32) {
        unsigned own;
        const unsigned o = other_row(__float_as_uint(v), own);
        v = fmaxf(__uint_as_float(own), __uint_as_float(o));
    }
    return v;
}
template <int G>
__device__ __forceinline__ float group_sum(float v) {
    if constexpr (G == 64) {
        asm volatile(ISG_SHIFTS("v_add_f32_dpp") ISG_BCAST15("v_add_f32_dpp") ISG_BCAST31("v_add_f32_dpp") "s_nop 1" : "+v"(v));
        return last_lane(v);
    }
    asm volatile(ISG_ROTATIONS("v_add_f32_dpp") : "+v"(v));
    if constexpr (G == 32) {
        unsigned own;
        const unsigned o = other_row(__float_as_uint(v), own);
        v = __uint_as_float(own) + __uint_as_float(o);
    }
    return v;
}
template <int G>
__device__ __forceinline__ int group_sum(int v) {
    if constexpr (G == 64) {
        asm volatile(ISG_SHIFTS("v_add_u32_dpp") ISG_BCAST15("v_add_u32_dpp") ISG_BCAST31("v_add_u32_dpp") "s_nop 1" : "+v"(v));
        return __builtin_amdgcn_readlane(v, 63);
    }
    asm volatile(ISG_ROTATIONS("v_add_u32_dpp") : "+v"(v));
    if constexpr (G == 32) {
        unsigned own;
        const unsigned o = other_row((unsigned)v, own);
        v = (int)(own + o);
    }
    return v;
}
// sum of the group's lanes up to and including this one
template <int G>
__device__ __forceinline__ int group_scan(int v) {
    if constexpr (G == 16) asm volatile(ISG_SHIFTS("v_add_u32_dpp") "s_nop 1" : "+v"(v));
    if constexpr (G == 32) asm volatile(ISG_SHIFTS("v_add_u32_dpp") ISG_BCAST15("v_add_u32_dpp") "s_nop 1" : "+v"(v));
    if constexpr (G == 64)
        asm volatile(ISG_SHIFTS("v_add_u32_dpp") ISG_BCAST15("v_add_u32_dpp") ISG_BCAST31("v_add_u32_dpp") "s_nop 1" : "+v"(v));
    return v;
}
template <int G>
__device__ __forceinline__ bool group_any(bool b) {
    const u64 mask = __ballot(b);
    if constexpr (G == 64) {
        return mask != 0;
    } else {
        const unsigned lane = threadIdx.x & 63;
        return (unsigned)(mask >> (lane & ~(unsigned)(G - 1)) & ((1ull << G) - 1ull)) != 0u;
    }
}
template <int G>
__device__ __forceinline__ u64 group_max_key(u64 k) {
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) {
        const u64 other = __shfl_xor(k, o);
        k = other > k ? other : k;
    }
    return k;
}
// LDS written by one of the G threads of a unit is there for the others
template <int G>
__device__ __forceinline__ void together() {
    if constexpr (G <= 64) {
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
// vectors of a slot side by side over the unit's G threads, on 16-byte boundaries of memory from `first` <= lo on.
// (Rows of 131,071 bf16 logits start on any even address, where a 16-byte load takes three cache accesses instead of one:
// the walk over 2,048 of them took 156 us instead of 141.  Boundaries of 128 bytes gained nothing more.)  The part's
// outer vectors may reach outside; they are read from lo and up to hi instead, and `start` tells which of their elements
// are this thread's own.  hi - lo is at least VE.
template <typename T, int G, int NE>
struct Span {
    static constexpr int VE = NE < 16 / (int)sizeof(T) ? NE : 16 / (int)sizeof(T);
    static constexpr int NV = NE / VE;
    static constexpr int kCols = G * NE;
    int lo, hi, first, lane;  // lane: of the unit's G

    // z: the row, whose memory the vectors are aligned in
    __device__ __forceinline__ Span(const T* z, int lo_, int hi_, int lane_) : lo(lo_), hi(hi_), lane(lane_) {
        first = lo - (int)(((uintptr_t)z / sizeof(T) + (unsigned)lo) % VE);
    }
    __device__ __forceinline__ void next() { first += kCols; }  // to the following kCols classes
    __device__ __forceinline__ bool more() const { return first < hi; }
    __device__ __forceinline__ int start(int slot) const { return first + (slot * G + lane) * VE; }
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
        thread = vec % G;
        e = vec / G * VE + c - inside(first + vec * VE);
    }
    // (both the same for every row of a launch: `first` is less than VE classes in front of lo)
    __device__ __forceinline__ bool beyond(int slot) const { return lo - (VE - 1) + slot * G * VE >= hi; }
    __device__ __forceinline__ bool whole(int slot) const { return slot > 0 && lo + (slot + 1) * G * VE <= hi; }
    // the elements of a unit's only step; those that are not this thread's as -inf (BLANK) or as whatever class lies there
    template <bool BLANK>
    __device__ __forceinline__ void load(const T* z, float (&v)[NE]) const {
#pragma unroll
        for (int t = 0; t < NV; ++t) {
            if (!beyond(t)) {
                load_vector<VE>(z + inside(start(t)), v + t * VE);
            } else {
#pragma unroll
                for (int j = 0; j < VE; ++j) v[t * VE + j] = -INFINITY;
            }
        }
        if constexpr (BLANK) {
#pragma unroll
            for (int t = 0; t < NV; ++t)
                if (!whole(t)) blank(t, v);
        }
    }
    __device__ __forceinline__ void blank(int t, float (&v)[NE]) const {
        const int s = start(t), from = s - inside(s);  // own: from <= j < from + VE
#pragma unroll
        for (int j = 0; j < VE; ++j) v[t * VE + j] = j >= from && j < from + VE ? v[t * VE + j] : -INFINITY;
    }
    // the same in two halves, for a step's loads that are on their way while the step before is worked on
    static constexpr int kWords = NE * (int)sizeof(T) / 4;
    __device__ __forceinline__ void fetch(const T* z, unsigned (&raw)[kWords < 1 ? 1 : kWords]) const {
#pragma unroll
        for (int t = 0; t < NV; ++t) __builtin_memcpy(raw + t * (kWords / NV), z + inside(start(t)), 16);
    }
    __device__ __forceinline__ void unpack(const unsigned (&raw)[kWords < 1 ? 1 : kWords], float (&v)[NE]) const {
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
            if constexpr (sizeof(T) == 4) v[i] = __uint_as_float(raw[i]);
            else v[2 * i] = __uint_as_float(raw[i] << 16), v[2 * i + 1] = __uint_as_float(raw[i] & 0xffff0000u);
        }
        if (first >= lo && first + kCols <= hi) return;
#pragma unroll
        for (int t = 0; t < NV; ++t) blank(t, v);
    }
    // a slot's gradients (what the outer vectors repeat of their neighbours they repeat with the same values)
    __device__ __forceinline__ void store(T* d, int t, const float* o) const {
        const int s = start(t);
        if (s < hi && s + VE > lo) store_vector<VE>(d + inside(s), o);
    }
    // ... that are not to stay in the caches (beyond_cache)
    __device__ __forceinline__ void store_past(T* d, int t, const float* o) const {
        static_assert(VE * sizeof(T) == 16);
        typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
        typedef u32x4 u32x4_any __attribute__((aligned(2)));
        const int s = start(t);
        if (s >= hi || s + VE <= lo) return;
        T w[VE];
        store_vector<VE>(w, o);
        u32x4 x;
        __builtin_memcpy(&x, w, 16);
        __builtin_nontemporal_store(x, reinterpret_cast<u32x4_any*>(d + inside(s)));
    }
    // the same without what they repeat (where a thread's values are its own alone)
    __device__ __forceinline__ void store_own(T* d, int t, const T* o) const {
        const int s = start(t);
        if (s >= lo && s + VE <= hi) {
            __builtin_memcpy(d + s, o, VE * sizeof(T));
        } else if (s < hi && s + VE > lo) {
            const int at = inside(s);
#pragma unroll
            for (int j = 0; j < VE; ++j)
                if (at + j >= s && at + j < s + VE) d[at + j] = o[j];
        }
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

__device__ __forceinline__ long long block_index() { return (long long)blockIdx.y * gridDim.x + blockIdx.x; }

// ---- launches ------------------------------------------------------------------------------------------------------
// How a row is cut: `lanes` lanes of a wave for what their registers hold.  Beyond, the forward passes walk over parts of
// a row, as many as give about kUnits workgroups but of at least kPartCols classes; the backward passes have nothing
// to join and take workgroups of at most 32 classes a thread.  Parts are equal but for the rounding to 8 classes; there is
// room for those that start between two boundaries (Span).
//
// About 2,048 workgroups are on the chip at once, eight to a CU for bf16 (64 registers a thread), five to seven for float.
// Twice as many (more parts a row) measured the same without alternatives beyond 100,000 classes (2,048 x 131,071 bf16 98
// and 101 us, float 182 and 180), and slower where a part costs something of its own: 2,048 x 9,001 float 15 and 19, with 20
// alternatives 25 and 32; 2,048 x 50,177 float with 20 82 and 88; 2,048 x 131,071 bf16 with 64 128 and 148.  (They gain
// where 2,048 leave an uneven rest: 1,300 x 131,071 float with 20 131 for 137, 1,500 x 9,001 without 14.5 for 16.)
constexpr long long kUnits = 2048;
constexpr int kPartCols = 2048;
constexpr int kMaxSplits = 128;
constexpr int kMarkCols = 131072;  // classes a part may have (one mark each in LDS, 16 KB)
struct Cut {
    int lanes, ne, splits, per;  // lanes = kThreads: workgroups
};
// (The rounding must not use up the last part, where the others are hundreds: a vector has to fit into it.)
inline int equal_part(int cols, int splits) {
    const int even = (cols + splits - 1) / splits, per = (even + 7) / 8 * 8, last = (cols - 1) % per + 1;
    return splits > 1 && last < 64 ? even : per;
}
// A row by 16 lanes of a wave where `narrow` classes a lane hold it (beyond 64: also by 32 lanes), else by a whole wave;
// lanes = 0: too long for that.  `entries`: places a row needs in its threads' registers, four a thread (sixteen in rows of
// 64 classes).
inline Cut cut_wave(int cols, int dtype, int entries, int narrow) {
    const int most = dtype == ISG_F32 ? 4 : 8;
    for (int ne : {1, 4, 8, 16, 24, 32, 40, 48, 56, 64})
        if (ne <= narrow && cols + (ne < most ? ne : most) - 1 <= 16 * ne) return Cut{16, ne, 1, cols};
    if (narrow > 64)
        for (int ne : {48, 64})
            if (cols + most - 1 <= 32 * ne) return Cut{32, ne, 1, cols};
    for (int ne : {1, 4, 8, 16, 24, 32})
        if ((ne == 1 || entries <= 256) && cols + (ne < most ? ne : most) - 1 <= 64 * ne) return Cut{64, ne, 1, cols};
    return Cut{0, 0, 1, cols};
}
// Few rows take a wave each (5,000 x 785 bf16 5.0 us, by 16 lanes 5.8; 20 best 8.4 and 12.5).  Many take 16 lanes each: what
// a row costs once is paid for four of them in the same instructions (131,072 x 785 bf16 47 us, by waves 63; 5 best 70 and
// 91; distilled with 16 entries and a tail 61 and 97).  What grows with the best classes or the entries is paid by fewer
// lanes so: many of those in long rows are a whole wave's again (20 best of 10,240 x 785 bf16 12.7 us, by 16 lanes 14.7, of
// 66,000 x 1,000 57 and 66; 64 entries of 131,072 x 785 74 and 86, of 66,000 x 380 28 and 24).
// From some 380 to 640 classes it depends on the rows, as 16 lanes first fill the chip's waves at many of them: 20 best of
// 505 bf16 by a wave and by 16 lanes 15.2 and 16.1 us at 20,480 rows, 32.2 and 31.5 at 49,152, 78 and 69 at 131,072; float
// 16.8 and 17.8, 33.6 and 34.4, 89 and 83; 64 best bf16 28.5 and 35.2, 60.8 and 65.6, 152 and 147; beyond 512 classes 20 best
// of bf16 would cross earlier (570: 18.5 and 17.2 at 20,480 rows) and 64 of float later (182 and 197 at 131,072 x 633).
constexpr int kNarrow = 65, kNarrowMany = 40;  // (kNarrowMany: more than 16 entries or best classes)
inline Cut cut_forward(long long rows, int cols, int dtype, int entries, int best) {
    int narrow = rows > 8192 && entries <= 64 ? kNarrow : 0;
    if (narrow && (entries > 16 || best > 16)) narrow = best > 16 && rows <= 49152 ? 24 : kNarrowMany;
    const Cut wave = cut_wave(cols, dtype, entries, narrow);
    if (wave.lanes) return wave;
    long long splits = (kUnits + rows - 1) / (rows > 0 ? rows : 1);
    const int most = cols / kPartCols < kMaxSplits ? cols / kPartCols : kMaxSplits, least = (cols + kMarkCols - 1) / kMarkCols;
    splits = splits > most ? most : splits;
    splits = splits < least ? least : splits;
    const int per = equal_part(cols, (int)splits);
    return Cut{kThreads, 16, (cols + per - 1) / per, per};
}
// The backward passes have less to pay once a row, and longer runs of memory by a whole wave: 131,072 x 785 bf16 84 us, by
// 16 lanes 88; float 138 and 150; 64 entries bf16 100 and 142; 66,000 x 380 bf16 22.9 and 22.4, float 32.6 and 33.8; x 120
// 20 and 9.5; x 250 with 64 entries 29 and 33.
constexpr int narrow_backward(int dtype, bool many) { return many ? 8 : (dtype == ISG_F32 ? 24 : 32); }
inline Cut cut_backward(long long rows, int cols, int dtype, int entries) {
    const int narrow = rows <= 8192 || entries > 64 ? 0 : narrow_backward(dtype, entries > 16);
    const Cut wave = cut_wave(cols, dtype, entries, narrow);
    if (wave.lanes) return wave;
    const auto parts = [&](int ne) { return (cols + kThreads * ne - 8 - 1) / (kThreads * ne - 8); };
    for (int ne = 8;; ne *= 2) {
        if (ne < 32 && rows * parts(2 * ne) >= 1024) continue;  // (still four workgroups for each of the 256 CUs)
        const int per = equal_part(cols, parts(ne));
        return Cut{kThreads, ne, (cols + per - 1) / per, per};
    }
}

// Whether a gradient is more than the last-level cache holds (256 MB).  What reads it next does not find it there either,
// and left in the cache it has to be written back under the next kernel's reads.  Both ways in one run each: 2,048 x 131,071
// bf16 distilled (two parts a row then), forward and backward 118 + 185 us, written past the cache 95 + 191; 8,192 x 12,545
// float 105 + 140 and 77 + 157; log-probabilities of 131,072 x 785 float 100 + 136 and 74 + 148.  (Not by 16 lanes, whose
// vectors are 256 bytes of a row: 103 + 150 and 73 + 190; and not of short rows distilled, whose forward pass waits for less:
// nothing gained.)
inline bool beyond_cache(long long rows, int cols, int dtype) {
    return rows * cols * (dtype == ISG_F32 ? 4 : 2) > (256ll << 20);
}

// `units` of `threads` threads each in workgroups of kThreads, over two grid axes
inline dim3 grid_of(long long units, int threads) {
    const long long blocks = (units * threads + kThreads - 1) / kThreads;
    const long long x = blocks < (1 << 20) ? blocks : (1 << 20);
    return dim3((unsigned)x, (unsigned)((blocks + x - 1) / x));
}

// F::template run<G, NE>(...) for a wave's cut, up to NARROW classes a lane by 16 lanes (beyond 64: also by 32 lanes)
template <typename F, int NARROW, typename... A>
void with_wave(const Cut& cut, A&&... args) {
    if constexpr (NARROW > 64)
        if (cut.lanes == 32) {
            if (cut.ne == 48) F::template run<32, 48>(args...);
            else F::template run<32, 64>(args...);
            return;
        }
    if (cut.lanes == 64) {
        switch (cut.ne) {
            case 1: F::template run<64, 1>(args...); break;
            case 4: F::template run<64, 4>(args...); break;
            case 8: F::template run<64, 8>(args...); break;
            case 16: F::template run<64, 16>(args...); break;
            case 24: F::template run<64, 24>(args...); break;
            default: F::template run<64, 32>(args...);
        }
        return;
    }
    switch (cut.ne) {
        case 1: F::template run<16, 1>(args...); break;
        case 4: F::template run<16, 4>(args...); break;
        case 8: F::template run<16, 8>(args...); break;
    }
    if constexpr (NARROW >= 24) switch (cut.ne) {
        case 16: F::template run<16, 16>(args...); break;
        case 24: F::template run<16, 24>(args...); break;
    }
    if constexpr (NARROW >= 32)
        if (cut.ne == 32) F::template run<16, 32>(args...);
    if constexpr (NARROW >= 40)
        if (cut.ne == 40) F::template run<16, 40>(args...);
    if constexpr (NARROW >= 64) switch (cut.ne) {
        case 48: F::template run<16, 48>(args...); break;
        case 56: F::template run<16, 56>(args...); break;
        case 64: F::template run<16, 64>(args...); break;
    }
}
template <typename F, int NARROW, typename... A>
void launch_backward(const Cut& cut, A&&... args) {
    if (cut.lanes != kThreads) with_wave<F, NARROW>(cut, args...);
    else if (cut.ne == 8) F::template run<kThreads, 8>(args...);
    else if (cut.ne == 16) F::template run<kThreads, 16>(args...);
    else F::template run<kThreads, 32>(args...);
}

inline int check_call(const char* who, long long row_stride, int rows, int cols, int dtype, float temperature) {
    ISG_REQUIRE(rows >= 0 && cols >= 1 && cols <= kMaxCols, ISG_EINVAL, "%s: bad shape rows=%d cols=%d (at most %d classes)",
                who, rows, cols, kMaxCols);
    ISG_REQUIRE(dtype == ISG_F32 || dtype == ISG_BF16, ISG_EDTYPE, "%s: dtype %d", who, dtype);
    ISG_REQUIRE(row_stride >= cols, ISG_EINVAL, "%s: rows of %d classes %lld elements apart", who, cols, row_stride);
    ISG_REQUIRE(temperature >= 1e-30f && temperature <= 1e30f, ISG_EINVAL, "%s: temperature %g", who, (double)temperature);
    return ISG_OK;
}

inline int check_bytes(const char* who, const void* classes, int bytes) {
    ISG_REQUIRE(!classes || bytes == 4 || bytes == 8, ISG_EINVAL, "%s: classes of %d bytes (4 or 8)", who, bytes);
    return ISG_OK;
}

// log2(e) / T as the float below it and what is missing, which is positive (an infinite distance times both parts is an
// infinity of one sign)
inline void scale_of(float temperature, float& c, float& c_lo, float& inv_t) {
    const double exact = 1.4426950408889634074 / (double)temperature;
    c = (float)exact;
    if ((double)c >= exact) c = nextafterf(c, 0.0f);
    c_lo = (float)(exact - (double)c);
    inv_t = (float)(1.0 / (double)temperature);
}

}  // namespace
