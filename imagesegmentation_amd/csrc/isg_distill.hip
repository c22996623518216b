// The divergence of a row from a teacher's most probable classes, forward and backward (layout: isg_classes.h).
//   loss = sum_j q_j (log q_j - log p_{i_j})  (+ q_r (log q_r - log p_r), p_r = sum over the classes outside the entries)
// with q = softmax(v / T), or with a tail q = exp(v) and q_r = max(0, 1 - sum q).  Q = sum q + q_r; the gradient is
//   dz_c = g/T (Q p_c - q_c) for an entry,  g/T Q p_c for the others,  with a tail g/T (Q p_r - q_r) p_c / p_r for them.
// p_r is summed over its own classes, not taken as 1 - the rest, which a confident student would leave no digits of.
#include "isg_classes.h"

namespace {

constexpr int kMaxEntries = ISG_DISTILL_MAX;  // a teacher's classes per row

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

// A row's entries in the registers of its G threads: entry i * G + thread in place i < N.  (One place where
// that holds a row's k, else four; sixteen, for every k there can be, where a wave closes a row of any length and for rows
// too short for a workgroup.)
constexpr int places(int lanes, int ne, int n) { return lanes == 64 && ne == 1 ? 16 : n; }
template <int G, int N>
struct Entries {
    int cls[N];    // -1: none, cols: a class the row does not have
    float val[N];

    __device__ __forceinline__ void load(const float* values, const void* classes, int bytes, long long row, int k, int cols) {
        const int thread = threadIdx.x & (G - 1);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            cls[i] = -1, val[i] = 0.0f;
            const int j = i * G + thread;
            if (i * G < k && j < k) {
                const long long c = class_at(classes, bytes, row * k + j);
                cls[i] = c < 0 ? -1 : (c < cols ? (int)c : cols);
                val[i] = values[row * k + j];
            }
        }
    }
    // the logits of the classes in [lo, hi), -inf for the others
    template <typename T>
    __device__ __forceinline__ void gather(const T* z, int lo, int hi, float (&ze)[N]) const {
#pragma unroll
        for (int i = 0; i < N; ++i) ze[i] = cls[i] >= lo && cls[i] < hi ? ld(z, cls[i]) : -INFINITY;
    }
};

// whether an earlier entry names the class as well
__device__ __noinline__ bool named_before(const void* classes, int bytes, long long row, int k, int j, int cls) {
    for (int o = 0; o < j; ++o)
        if (class_at(classes, bytes, row * k + o) == cls) return true;
    return false;
}

// log(1 + x): the logarithm of the rounded sum, corrected for what the rounding took
__device__ __forceinline__ float log1p_of(float x) {
    const float u = 1.0f + x;
    return u == 1.0f ? x : kLn2 * __builtin_amdgcn_logf(u) * (x / (u - 1.0f));
}

// The loss of a row from its sums, by G lanes of a wave.
template <int G, int N>
__device__ __forceinline__ void distill_finish(const DistillArgs& a, const Entries<G, N>& en, const float (&ze)[N],
                                               long long row, const DistillPart& t) {
    const int lane = threadIdx.x & (G - 1);
    float m = t.m, s = t.s;
    if (a.tail) merge(m, s, t.me, t.se, a.c, a.c_lo);
    m = m == -INFINITY ? 0.0f : m;
    const float l2s = s == 0.0f ? INFINITY : __builtin_amdgcn_logf(s);
    // (log s as a whole number of ln 2 and the logarithm of a fraction: added one after the other to a difference of the
    // same size it loses a rounding of that difference, not one of its own that every entry of the row would share)
    const float s_exp = (float)__builtin_amdgcn_frexp_expf(s), s_log = kLn2 * __builtin_amdgcn_logf(__builtin_amdgcn_frexp_mantf(s));
    // the teacher's distribution over its entries
    const float cv = a.tail ? kLog2e : a.c, cv_lo = a.tail ? kLog2eLo : a.c_lo;
    float mv = 0.0f, lv = 0.0f, sv = 0.0f, q[N];
    bool bad = false;
    if (!a.tail) {
        mv = -INFINITY;
#pragma unroll
        for (int i = 0; i < N; ++i) mv = en.cls[i] >= 0 ? fmaxf(mv, en.val[i]) : mv;
        mv = group_max<G>(mv);
        if (mv == -INFINITY) mv = 0.0f;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
        q[i] = 0.0f;
        if (i * G < a.k) {
            q[i] = en.cls[i] >= 0 ? power(en.val[i], mv, cv, cv_lo) : 0.0f;
            sv += q[i];
            bad |= en.cls[i] >= a.cols;
        }
    }
    sv = group_sum<G>(sv);
    if (!a.tail) lv = sv == 0.0f ? INFINITY : __builtin_amdgcn_logf(sv);
    const float qsum = a.tail ? sv : (sv == 0.0f ? 0.0f : 1.0f);
    float qr = a.tail ? fmaxf(1.0f - sv, 0.0f) : 0.0f;
    float l = 0.0f;
    const float iv = a.tail ? 1.0f : (sv == 0.0f ? 0.0f : 1.0f / sv);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if (i * G < a.k) {
            const float qi = q[i] * iv;
            const float lq = (en.val[i] - mv) * (a.tail ? 1.0f : a.inv_t) - kLn2 * lv;
            const float d = lq - (ze[i] - m) * a.inv_t;  // log q - log p - log s
            const float term = s == 0.0f ? INFINITY : qi * (__builtin_fmaf(s_exp, kLn2, d) + s_log);
            if (qi != 0.0f && en.cls[i] < a.cols) l += term;
        }
    }
    l = group_sum<G>(l);
    bad = group_any<G>(bad);
    if (lane == 0) {
        float coef = qsum, mb = m, ib = 1.0f / s;
        if (a.tail) {
            const bool none = t.s == 0.0f;
            const float mr = t.m == -INFINITY ? 0.0f : t.m, lr = none ? INFINITY : __builtin_amdgcn_logf(t.s);
            if (none && qr <= kNoMass) qr = 0.0f;
            // The student's mass outside, and the logarithm of the masses' ratio: from the logarithms where it is no
            // normal float; where the entries have less than half of it on both sides from their masses, as 1 - (a
            // few per cent) over the same would lose them.
            const float pr = t.s * power(mr, m, a.c, a.c_lo) / s, pe = t.se * power(t.me, m, a.c, a.c_lo) / s;
            float ratio;
            coef = none ? 0.0f : (qsum + qr) * pr - qr;
            if (pe < 0.5f && sv < 1.0f) coef = sv - pe;
            if (pe < 0.5f && sv < 0.5f) {
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
            a.stats[row] = DistillStats{mb, ib, coef, qsum + qr, m, s == 0.0f ? 0.0f : 1.0f / s, mv, iv};
    }
}

// loss = sum_j q_j (log q_j - log p_(i_j)), and with TAIL the mass outside the entries as one more class:
// + q_r (log q_r - log p_r), where p_r is summed over those classes themselves (1 - sum would cancel).  For that every
// class an entry names is marked in LDS and blanked when its thread comes to it; the entries' own classes are summed
// from a second look at them.

// The sums (me, se) over the classes the entries name in [lo, hi), each once; mark(class) says whether it was marked
// before.  The G threads of the unit share the entries; the result is the wave's (or its group's).
template <int G, int N, typename Mark>
__device__ __forceinline__ void mark_entries(const DistillArgs& a, const Entries<G, N>& en, const float (&ze)[N],
                                             long long row, int lo, int hi, unsigned* repeated, DistillPart& t, Mark mark) {
    constexpr int L = G < 64 ? G : 64;
    bool twice = false;
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if (i * G < a.k) {
            if (en.cls[i] >= lo && en.cls[i] < hi) twice |= mark(en.cls[i]);
            m = fmaxf(m, ze[i]);
        }
    }
    t.me = group_max<L>(m);
    if constexpr (G <= 64) {
        twice = group_any<G>(twice);
        together<G>();
    } else {
        if (twice) *repeated = 1u;
        together<G>();
        twice = *repeated != 0;
    }
    const float mz = t.me == -INFINITY ? 0.0f : t.me;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if (i * G < a.k) {
            bool first = en.cls[i] >= lo && en.cls[i] < hi;
            if (twice && first)
                first = !named_before(a.classes, a.class_bytes, row, a.k, i * G + (int)(threadIdx.x & (G - 1)), en.cls[i]);
            if (first) t.se += power(ze[i], mz, a.c, a.c_lo);
        }
    }
    t.se = group_sum<L>(t.se);
}

// A row in the registers of G lanes, its entries beside them; with a tail the entries' classes are marked in LDS (a bit
// each), taken out of the registers and summed apart.  131,072 x 785 bf16 with 16 entries and a tail 59 us (3.5 TB/s;
// sums, marks and the closing logarithms weigh as much as the read), with 64 entries without 76; float, 64 and a tail,
// 113 (3.6 TB/s); 20,480 rows bf16 13.5.  (Behind backward passes, whose gradients have left the cache dirty.)
template <typename T, int G, int NE, int N, bool TAIL>
__global__ __launch_bounds__(kThreads) void distill_fwd_kernel(const T* __restrict__ logits, DistillArgs a) {
    __shared__ u64 marks[TAIL ? kThreads : 1];  // a thread's elements that an entry names, one bit each
    const int lane = threadIdx.x & (G - 1);
    const long long row = block_index() * (kThreads / G) + threadIdx.x / G;
    if (row >= a.units) return;
    if (a.live && !a.live[row]) {
        if (lane == 0) distill_dead(a, row);
        return;
    }
    const T* z = logits + row * a.row_stride;
    using S = Span<T, G, NE>;
    const S span(z, 0, a.cols, lane);
    Entries<G, N> en;
    en.load(a.values, a.classes, a.class_bytes, row, a.k, a.cols);
    float v[NE], ze[N];
    span.template load<true>(z, v);
    en.gather(z, 0, a.cols, ze);
    DistillPart t{-INFINITY, 0.0f, -INFINITY, 0.0f};
    if constexpr (TAIL) {
        u64* mine = marks + (threadIdx.x - lane);
        mine[lane] = 0ull;
        together<G>();
        mark_entries(a, en, ze, row, 0, a.cols, nullptr, t, [&](int i) {
            int thread, e;
            span.locate(i, thread, e);
            return (atomicOr(&mine[thread], 1ull << e) >> e & 1ull) != 0;
        });
        const unsigned hit[2] = {(unsigned)mine[lane], (unsigned)(mine[lane] >> 32)};
#pragma unroll
        for (int e = 0; e < NE; ++e) v[e] = hit[e / 32] >> (e % 32) & 1u ? -INFINITY : v[e];
    }
    float m = v[0];
#pragma unroll
    for (int e = 1; e < NE; ++e) m = fmaxf(m, v[e]);
    t.m = group_max<G>(m);
    const float mz = t.m == -INFINITY ? 0.0f : t.m;
    float s = 0.0f;
#pragma unroll
    for (int e = 0; e < NE; ++e) s += power_of<T>(a, v[e], mz);
    t.s = group_sum<G>(s);
    distill_finish(a, en, ze, row, t);
}

// The loss of a longer row, by one wave.
template <typename T>
__device__ __forceinline__ void finish_row(const DistillArgs& a, const T* z, long long row, const DistillPart& t) {
    Entries<64, 16> en;
    en.load(a.values, a.classes, a.class_bytes, row, a.k, a.cols);
    float ze[16];
    en.gather(z, 0, a.cols, ze);
    distill_finish(a, en, ze, row, t);
}

// A part of a longer row: a workgroup walks over it, kThreads * NE classes at a time, the next ones being loaded
// meanwhile.  Every wave keeps its own maximum and its lanes their own sums until the end.  The marks are one bit a class
// of the part.  Bound by the read: 2,048 x 131,071 bf16 with 64 entries 104 us (5.2 TB/s), 8,192 x 12,545 float with 32
// 76 us (5.4 TB/s); with a tail the marks add to it, 1,500 x 65,537 float with 64 72 us (5.4), 1,002 x 100,003 bf16 with
// 256 44 us (4.6).
template <typename T, int NE, bool TAIL>
__global__ __launch_bounds__(kThreads, sizeof(T) == 4 ? 7 : 8) void distill_stream_kernel(const T* __restrict__ logits,
                                                                                           DistillArgs a) {
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
    using S = Span<T, kThreads, NE>;
    const int lo = split * a.per, hi = lo + a.per < a.cols ? lo + a.per : a.cols;
    unsigned raw[S::kWords];
    S ahead(z, lo, hi, tid);
    const int zero = ahead.first;  // the class of the first mark
    ahead.fetch(z, raw);
    DistillPart t{-INFINITY, 0.0f, -INFINITY, 0.0f};
    if constexpr (TAIL) {
        Entries<kThreads, 4> en;
        en.load(a.values, a.classes, a.class_bytes, row, a.k, a.cols);
        float ze[4];
        en.gather(z, lo, hi, ze);
        unsigned* words = reinterpret_cast<unsigned*>(marks);
        for (int i = tid; i < (hi - zero + 31) / 32; i += kThreads) words[i] = 0u;
        if (tid == 0) repeated = 0u;
        __syncthreads();
        mark_entries(a, en, ze, row, lo, hi, &repeated, t, [&](int i) {
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
            const float m = group_max<64>(lane_max);
            if (t.m != -INFINITY) s *= power(t.m, m, a.c, a.c_lo);
            t.m = m;
        }
        const float mz = t.m == -INFINITY ? 0.0f : t.m;
#pragma unroll
        for (int e = 0; e < NE; ++e) s += power_of<T>(a, v[e], mz);
    }
    t.s = group_sum<64>(s);
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
        finish_row(a, z, row, t);
    else if (lane == 0)
        a.part[unit] = t;
}

// Joins the parts of a row: one wave.  Latency: 5.4 us for 640 rows in 4 parts, 10 for 1,002 rows of 256 entries.
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
    const float m = group_max<64>(t.m), me = group_max<64>(t.me);
    t.s = group_sum<64>(t.s == 0.0f ? 0.0f : t.s * power(t.m, m, a.c, a.c_lo));
    t.se = group_sum<64>(t.se == 0.0f ? 0.0f : t.se * power(t.me, me, a.c, a.c_lo));
    t.m = m, t.me = me;
    finish_row(a, logits + row * a.row_stride, row, t);
}

struct DistillBwdArgs {
    const float* values;
    const void* classes;
    const DistillStats* stats;
    const float* dloss;
    long long row_stride, units;
    int class_bytes, cols, splits, per, k, tail;
    float c, c_lo, inv_t;
    int past;
};

// A row, or a part of one, by G lanes: the dense part from the row's kept constants, the entries' own values over it.  Reads
// the logits and writes as much: 2,048 x 131,071 bf16 190 us (5.6 TB/s read and written), 8,192 x 12,545 float 155 us
// (5.3), 131,072 x 785 bf16 with 16 entries 101 us (4.1), float with 64 152 us (5.4).
template <typename T, int G, int NE, int N>
__global__ __launch_bounds__(kThreads) void distill_bwd_kernel(const T* __restrict__ logits, DistillBwdArgs a,
                                                              T* __restrict__ dlogits) {
    __shared__ u64 marks[kThreads];
    __shared__ unsigned repeated;
    __shared__ __attribute__((aligned(16))) T image[G <= 64 ? kThreads * Span<T, G, NE>::VE : 1];
    const int tid = threadIdx.x & (G - 1);
    // (from the last unit back: what the forward pass read last is still in the last-level cache)
    const long long unit = a.units - 1 - (block_index() * (kThreads / G) + threadIdx.x / G);
    if (unit < 0) return;
    const long long row = a.splits == 1 ? unit : unit / a.splits;
    const int split = a.splits == 1 ? 0 : (int)(unit - row * a.splits);
    using S = Span<T, G, NE>;
    const int lo = split * a.per, hi = lo + a.per < a.cols ? lo + a.per : a.cols;
    T* d = dlogits + row * a.cols;
    const S span(d, lo, hi, tid);  // (aligned as the gradient; dense logits lie the same way)
    const DistillStats st = a.stats[row];
    const bool zero = st.is == 0.0f;  // a dead row, or no class has probability
    const T* z = logits + row * a.row_stride;
    const float g = a.dloss[row] * a.inv_t, gc = g * st.coef * st.ib;
    const bool plain = zero || st.coef != st.coef;  // (NaN: an entry the row does not have; the whole row is)
    Entries<G, N> en;
    float v[NE], ze[N], own[N];
    const auto fetch_entries = [&] {
        en.load(a.values, a.classes, a.class_bytes, row, a.k, a.cols);
        en.gather(z, lo, hi, ze);
    };
    const auto dense = [&](int t, float(&o)[S::VE]) {
#pragma unroll
        for (int j = 0; j < S::VE; ++j) {
            const float zi = v[t * S::VE + j];
            const float e = sizeof(T) == 4 ? power_exact(zi, st.mb, a.c, a.c_lo) : __builtin_amdgcn_exp2f((zi - st.mb) * a.c);
            o[j] = zero ? 0.0f : gc * e;
        }
    };
    // the entries' own gradients
    const auto own_gradients = [&] {
        u64* mine = marks + (threadIdx.x - tid);
        mine[tid] = 0ull;
        if (G > 64 && tid == 0) repeated = 0u;
        together<G>();
        bool twice = false;
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (i * G < a.k && en.cls[i] >= lo && en.cls[i] < hi) {
                int thread, e;
                span.locate(en.cls[i], thread, e);
                twice |= (atomicOr(&mine[thread], 1ull << e) >> e & 1ull) != 0;
            }
        if constexpr (G <= 64) {
            twice = group_any<G>(twice);
        } else {
            if (twice) repeated = 1u;
            together<G>();
            twice = repeated != 0;
        }
        const float cv = a.tail ? kLog2e : a.c, cv_lo = a.tail ? kLog2eLo : a.c_lo;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int c = en.cls[i];
            own[i] = 0.0f;
            if (i * G >= a.k || c < lo || c >= hi) continue;
            float q = st.iv * power_exact(en.val[i], st.mv, cv, cv_lo);
            if (twice) {  // (every place of the class writes the same sum)
                q = 0.0f;
                for (int o = 0; o < a.k; ++o)
                    if (class_at(a.classes, a.class_bytes, row * a.k + o) == c)
                        q += st.iv * power_exact(a.values[row * a.k + o], st.mv, cv, cv_lo);
            }
            own[i] = g * (st.total * (st.is * power_exact(ze[i], st.m, a.c, a.c_lo)) - q);
        }
    };
    if constexpr (G <= 64) {
        // A slot's vectors go through LDS, where the entries' values take their places: stored one by one behind the row
        // they cost a write of 64 bytes each (131,072 x 785 float with 64 entries, by 16 lanes: 230 us for 179; bf16 144 for 142).
        if (!zero) {
            fetch_entries();
            span.template load<false>(z, v);
            own_gradients();
        }
        int slot[N], place[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            slot[i] = -1, place[i] = 0;
            if (i * G < a.k && !plain && en.cls[i] >= lo && en.cls[i] < hi) {
                int thread, e;
                span.locate(en.cls[i], thread, e);
                slot[i] = e / S::VE, place[i] = (threadIdx.x - tid + thread) * S::VE + e % S::VE;
            }
        }
        T* mine = image + threadIdx.x * S::VE;
#pragma unroll
        for (int t = 0; t < S::NV; ++t) {
            if (span.beyond(t)) break;
            float o[S::VE];
            dense(t, o);
            store_vector<S::VE>(mine, o);
            together<G>();
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (slot[i] == t) store_vector<1>(image + place[i], own + i);
            together<G>();
            T out[S::VE];
            __builtin_memcpy(out, mine, S::VE * sizeof(T));
            span.store_own(d, t, out);
        }
    } else {
        // (A row in parts: the entries' work waits until the dense part has been stored, for more waves and an earlier
        // start of the stores.  Before it: 204 us for 188 at 2,048 x 131,071 bf16 in 17 parts, 134 for 141 at 8,192 x
        // 12,545 float in 2.)
        if (!zero) {
            fetch_entries();
            span.template load<false>(z, v);
        }
#pragma unroll
        for (int t = 0; t < S::NV; ++t) {
            if (span.beyond(t)) break;
            float o[S::VE];
            dense(t, o);
            if (a.past) span.store_past(d, t, o);
            else span.store(d, t, o);
        }
        if (plain) return;
        own_gradients();  // (with the barrier between the dense stores and the entries')
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (i * G < a.k && en.cls[i] >= lo && en.cls[i] < hi) store_vector<1>(d + en.cls[i], own + i);
    }
}

template <typename T, bool TAIL, int PLACES>
struct DistillFwd {
    template <int G, int NE>
    static void run(const void* logits, const DistillArgs& a, hipStream_t s) {
        hipLaunchKernelGGL((distill_fwd_kernel<T, G, NE, places(G, NE, PLACES), TAIL>), grid_of(a.units, G), dim3(kThreads), 0, s,
                           static_cast<const T*>(logits), a);
    }
};
template <typename T, bool TAIL>
void launch_forward(const Cut& cut, const void* logits, const DistillArgs& a, hipStream_t s) {
    if (cut.lanes == kThreads)
        hipLaunchKernelGGL((distill_stream_kernel<T, 16, TAIL>), grid_of(a.units, kThreads), dim3(kThreads), 0, s,
                           static_cast<const T*>(logits), a);
    else if (a.k <= cut.lanes)
        with_wave<DistillFwd<T, TAIL, 1>, kNarrow>(cut, logits, a, s);
    else
        with_wave<DistillFwd<T, TAIL, 4>, kNarrowMany>(cut, logits, a, s);
}
template <typename T, int PLACES>
struct DistillBwd {
    template <int G, int NE>
    static void run(const void* logits, const DistillBwdArgs& a, void* dlogits, hipStream_t s) {
        hipLaunchKernelGGL((distill_bwd_kernel<T, G, NE, places(G, NE, PLACES)>), grid_of(a.units, G), dim3(kThreads), 0, s,
                           static_cast<const T*>(logits), a, static_cast<T*>(dlogits));
    }
};
template <typename T>
void launch_gradient(const Cut& cut, const void* logits, const DistillBwdArgs& a, void* dlogits, hipStream_t s) {
    constexpr int dtype = std::is_same<T, float>::value ? ISG_F32 : ISG_BF16;
    // (16 lanes hold 16 entries in one place each: more of them are cut_backward's `many`)
    if (a.k <= cut.lanes) launch_backward<DistillBwd<T, 1>, narrow_backward(dtype, false)>(cut, logits, a, dlogits, s);
    else launch_backward<DistillBwd<T, 4>, narrow_backward(dtype, true)>(cut, logits, a, dlogits, s);
}

int check_entries(const char* who, int k, int tail) {
    ISG_REQUIRE(k >= 1 && k <= kMaxEntries, ISG_EINVAL, "%s: k=%d classes of the teacher (1 to %d)", who, k, kMaxEntries);
    ISG_REQUIRE(tail == 0 || tail == 1, ISG_EINVAL, "%s: tail=%d", who, tail);
    return ISG_OK;
}

}  // namespace

extern "C" long long isg_distill_workspace_bytes(int rows, int cols) {
    if (rows < 0 || cols < 1 || cols > kMaxCols) return -1;
    const Cut cut = cut_forward(rows, cols, ISG_F32, 0, 0);  // (rows of both types are in as many parts)
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
    const Cut cut = cut_forward(rows, cols, dtype, k, 0);
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
        tail ? launch_forward<float, true>(cut, logits, a, s) : launch_forward<float, false>(cut, logits, a, s);
    else
        tail ? launch_forward<__hip_bfloat16, true>(cut, logits, a, s)
             : launch_forward<__hip_bfloat16, false>(cut, logits, a, s);
    rc = isg::check_launch("distill_fwd_kernel");
    if (rc != ISG_OK || cut.splits == 1) return rc;
    a.units = rows;
    if (dtype == ISG_F32)
        hipLaunchKernelGGL(distill_join_kernel<float>, grid_of(rows, 64), dim3(kThreads), 0, s,
                           static_cast<const float*>(logits), a);
    else
        hipLaunchKernelGGL(distill_join_kernel<__hip_bfloat16>, grid_of(rows, 64), dim3(kThreads), 0, s,
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
    const Cut cut = cut_backward(rows, cols, dtype, k);
    hipStream_t s = static_cast<hipStream_t>(stream);
    DistillBwdArgs a{};
    a.values = values, a.classes = classes, a.stats = reinterpret_cast<const DistillStats*>(stats), a.dloss = dloss;
    a.row_stride = row_stride, a.units = (long long)rows * cut.splits;
    a.class_bytes = class_bytes, a.cols = cols, a.splits = cut.splits, a.per = cut.per, a.k = k, a.tail = tail;
    a.past = beyond_cache(rows, cols, dtype);
    scale_of(temperature, a.c, a.c_lo, a.inv_t);
    if (dtype == ISG_F32) launch_gradient<float>(cut, logits, a, dlogits, s);
    else launch_gradient<__hip_bfloat16>(cut, logits, a, dlogits, s);
    return isg::check_launch("distill_bwd_kernel");
}
