// Log-probabilities of given classes with the row's entropy and its most probable classes, and the divergence of a
// row from a teacher's most probable classes - forward and backward over the class axis.
//
// A row z of n logits at temperature T has, with m = max z and x_c = (z_c - m) log2(e) / T,
//   log p_c = ln 2 (x_c - log2 s),   s = sum 2^x_c,   H = -sum p_c log p_c = ln 2 (log2 s - (sum 2^x_c x_c) / s);
// every term of H has one sign, so a confident row loses nothing to cancellation, and z_c - m comes first, so that
// rows of the type's lowest value are uniform rows and not overflows.  A class at -inf has no probability and adds
// nothing (its x is kept from meeting 0 * inf by a lower bound far below the smallest float).  All sums are float.
#include <hip/hip_bf16.h>

#include "isg_common.h"

namespace {

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;
constexpr int kThreads = 256;
constexpr int kMaxTop = ISG_TOP_MAX;          // classes kept per row
constexpr int kMaxEntries = ISG_DISTILL_MAX;  // a teacher's classes per row
constexpr int kMaxCols = ISG_CLASSES_MAX;     // class axis

template <typename T>
__device__ __forceinline__ float ld(const T* p, long long i) {
    return (float)p[i];
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
    return v;
}
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

// the value over a workgroup of kThreads, in a fixed order; `red` is kThreads / 64 floats of LDS
__device__ float block_max(float v, float* red) {
    v = wave_max(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[0];
    for (int w = 1; w < kThreads / 64; ++w) v = fmaxf(v, red[w]);
    return v;
}
__device__ float block_sum(float v, float* red) {
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[0];
    for (int w = 1; w < kThreads / 64; ++w) v += red[w];
    return v;
}

// a class index stored as 4 or 8 bytes
__device__ __forceinline__ long long class_at(const void* p, int bytes, long long i) {
    return bytes == 8 ? static_cast<const long long*>(p)[i] : (long long)static_cast<const int*>(p)[i];
}

// Order of the alternatives as one integer: larger logits first (-0 equals 0, NaN last), equal ones by class.
__device__ __forceinline__ unsigned order_bits(float v) {
    const unsigned b = __float_as_uint(v + 0.0f);
    if (v != v) return 0u;
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ unsigned long long order_key(float v, int c) {
    return ((unsigned long long)order_bits(v) << 32) | (unsigned)~c;
}
__device__ __forceinline__ unsigned long long wave_max_key(unsigned long long k) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const unsigned long long other = __shfl_xor(k, o);
        k = other > k ? other : k;
    }
    return k;
}

// x = (z - m) log2(e) / T and its power; u_term is 2^x x with 0 for a class without probability
__device__ __forceinline__ void power(float z, float m, float c, float& e, float& u_term) {
    const float x = (z - m) * c;
    e = exp2f(x);
    u_term = e * fmaxf(x, -1000.0f);
}

// log p of a logit; a row without any probability (log2 s = +inf) gives -inf.  In nats throughout: at T = 1 the
// type's lowest value has a finite logarithm, its binary one would overflow.
__device__ __forceinline__ float log_prob(float z, float m, float inv_t, float l2s) {
    return (z - m) * inv_t - kLn2 * l2s;
}

// ---- token_logprobs ------------------------------------------------------------------------------------------------
// One workgroup per row: a pass for the maximum, one for the sums, one per kept class.
template <typename T>
__global__ __launch_bounds__(kThreads) void logprobs_fwd_kernel(
    const T* __restrict__ logits, long long row_stride, const void* __restrict__ tokens, int token_bytes,
    const unsigned char* __restrict__ live, int cols, float c, float inv_t, int top, float* __restrict__ logprobs,
    float* __restrict__ entropy, float* __restrict__ top_logprobs, int* __restrict__ top_classes,
    float* __restrict__ stats) {
    __shared__ float red[kThreads / 64];
    __shared__ unsigned long long redk[kThreads / 64];
    const long long row = blockIdx.x;
    const int tid = threadIdx.x;
    if (live && !live[row]) {
        if (tid == 0) {
            if (logprobs) logprobs[row] = 0.0f;
            entropy[row] = 0.0f;
            if (stats) stats[4 * row] = 0.0f, stats[4 * row + 1] = 0.0f, stats[4 * row + 2] = 0.0f, stats[4 * row + 3] = 0.0f;
        }
        for (int j = tid; j < top; j += kThreads) top_logprobs[row * top + j] = 0.0f, top_classes[row * top + j] = -1;
        return;
    }
    const T* z = logits + row * row_stride;
    float m = -INFINITY;
    for (int i = tid; i < cols; i += kThreads) m = fmaxf(m, ld(z, i));
    m = block_max(m, red);
    if (m == -INFINITY) m = 0.0f;  // no class has probability (or all are NaN): 2^-inf sums to nothing
    float s = 0.0f, u = 0.0f;
    for (int i = tid; i < cols; i += kThreads) {
        float e, ut;
        power(ld(z, i), m, c, e, ut);
        s += e, u += ut;
    }
    s = block_sum(s, red);
    u = block_sum(u, red);
    const float l2s = s == 0.0f ? INFINITY : log2f(s);
    const float H = s == 0.0f ? 0.0f : kLn2 * (l2s - u / s);
    if (tid == 0) {
        if (tokens) {
            const long long a = class_at(tokens, token_bytes, row);
            logprobs[row] = a >= 0 && a < cols ? log_prob(ld(z, a), m, inv_t, l2s) : NAN;
        }
        entropy[row] = H;
        if (stats) stats[4 * row] = m, stats[4 * row + 1] = l2s, stats[4 * row + 2] = H, stats[4 * row + 3] = 0.0f;
    }
    unsigned long long last = ~0ull;
    for (int j = 0; j < top; ++j) {
        unsigned long long best = 0;
        for (int i = tid; i < cols; i += kThreads) {
            const unsigned long long k = order_key(ld(z, i), i);
            if (k < last && k > best) best = k;
        }
        best = wave_max_key(best);
        __syncthreads();
        if ((tid & 63) == 0) redk[tid >> 6] = best;
        __syncthreads();
        for (int w = 0; w < kThreads / 64; ++w) best = redk[w] > best ? redk[w] : best;
        last = best;
        if (tid == 0) {
            const int cls = (int)~(unsigned)best;
            top_logprobs[row * top + j] = log_prob(ld(z, cls), m, inv_t, l2s);
            top_classes[row * top + j] = cls;
        }
    }
}

// dlogits[c] = 1/T ([c = a] g_a + sum_j [c = i_j] g_j - p_c (g_a + sum_j g_j) - g_H p_c (log p_c + H)): the dense part
// is written first, the few classes with a gradient of their own are written again behind it.
template <typename T>
__global__ __launch_bounds__(kThreads) void logprobs_bwd_kernel(
    const T* __restrict__ logits, long long row_stride, const void* __restrict__ tokens, int token_bytes,
    const unsigned char* __restrict__ live, const int* __restrict__ top_classes, const float* __restrict__ stats,
    const float* __restrict__ dlogprobs, const float* __restrict__ dentropy, const float* __restrict__ dtop, int cols,
    float c, float inv_t, int top, T* __restrict__ dlogits) {
    __shared__ float red[kThreads / 64];
    const long long row = blockIdx.x;
    const int tid = threadIdx.x;
    T* d = dlogits + row * cols;
    const float m = stats[4 * row], l2s = stats[4 * row + 1], H = stats[4 * row + 2];
    if ((live && !live[row]) || l2s == INFINITY) {  // dead, or no class has probability: nothing to move
        for (int i = tid; i < cols; i += kThreads) d[i] = (T)0.0f;
        return;
    }
    const T* z = logits + row * row_stride;
    const float ga = dlogprobs ? dlogprobs[row] : 0.0f, gh = dentropy ? dentropy[row] : 0.0f;
    const long long a = dlogprobs ? class_at(tokens, token_bytes, row) : -1;
    float g = 0.0f;
    if (dtop)
        for (int j = tid; j < top; j += kThreads) g += dtop[row * top + j];
    g = dtop ? block_sum(g, red) : 0.0f;
    g += ga;
    if (dlogprobs && ga != 0.0f && (a < 0 || a >= cols)) g = NAN;  // a class the row does not have
    auto dense = [&](int i, float& p) {
        const float x = (ld(z, i) - m) * c - l2s;
        p = exp2f(x);
        return -p * (g + gh * (kLn2 * fmaxf(x, -1000.0f) + H));
    };
    for (int i = tid; i < cols; i += kThreads) {
        float p;
        d[i] = (T)(inv_t * dense(i, p));
    }
    __syncthreads();
    const int entries = (dtop ? top : 0) + 1;
    for (int j = tid; j < entries; j += kThreads) {
        const long long i = j + 1 < entries ? (long long)top_classes[row * top + j] : a;
        if (i < 0 || i >= cols) continue;
        float own = i == a ? ga : 0.0f, p;
        for (int k = 0; k + 1 < entries; ++k) own += top_classes[row * top + k] == i ? dtop[row * top + k] : 0.0f;
        d[i] = (T)(inv_t * (dense((int)i, p) + own));
    }
}

// ---- distill_rows --------------------------------------------------------------------------------------------------
// What the backward pass keeps of a row: the dense part of its gradient is coef * 2^((z - mb) c - lb); at the
// teacher's classes it is total * 2^((z - m) c - l2s) - q.  q of entry j is 2^((v_j - mv) cv - lv).
struct DistillStats {
    float mb, lb, coef, total, m, l2s, mv, lv;
};

// A remaining mass that rounding alone can leave of the entries' log-probabilities (k of them, each good to 2^-24 of
// its size): where the student has no class outside the entries it is no mass, anything above it has nowhere to go.
constexpr float kNoMass = 1e-5f;

constexpr int kMarkCols = 32768;  // columns marked at a time (4 KB of bits)

// One workgroup per row.  loss = sum_j q_j (log q_j - log p_(i_j)), and with `tail` the mass outside the entries as one
// more class: + q_r (log q_r - log p_r), where p_r is summed over those classes themselves (1 - sum would cancel).
template <typename T>
__global__ __launch_bounds__(kThreads) void distill_fwd_kernel(
    const T* __restrict__ logits, long long row_stride, const float* __restrict__ values,
    const void* __restrict__ classes, int class_bytes, const unsigned char* __restrict__ live, int cols, int k, float c,
    float inv_t, int tail, float* __restrict__ loss, DistillStats* __restrict__ stats) {
    __shared__ float red[kThreads / 64];
    __shared__ unsigned marks[kMarkCols / 32];
    const long long row = blockIdx.x;
    const int tid = threadIdx.x;
    if (live && !live[row]) {
        if (tid == 0) {
            loss[row] = 0.0f;
            if (stats) stats[row] = DistillStats{0.0f, 0.0f, 0.0f, 0.0f, 0.0f, INFINITY, 0.0f, 0.0f};
        }
        return;
    }
    const T* z = logits + row * row_stride;
    const float* v = values + row * k;
    float m = -INFINITY;
    for (int i = tid; i < cols; i += kThreads) m = fmaxf(m, ld(z, i));
    m = block_max(m, red);
    if (m == -INFINITY) m = 0.0f;
    // the teacher's distribution over its entries
    float mv = 0.0f, lv = 0.0f, bad = 0.0f;
    const float cv = tail ? kLog2e : c;
    if (!tail) {
        mv = -INFINITY;
        for (int j = tid; j < k; j += kThreads)
            if (class_at(classes, class_bytes, row * k + j) >= 0) mv = fmaxf(mv, v[j]);
        mv = block_max(mv, red);
        if (mv == -INFINITY) mv = 0.0f;
    }
    float sv = 0.0f;
    for (int j = tid; j < k; j += kThreads) {
        const long long i = class_at(classes, class_bytes, row * k + j);
        if (i >= 0) sv += exp2f((v[j] - mv) * cv);
        if (i >= cols) bad = 1.0f;
    }
    sv = block_sum(sv, red);
    bad = block_max(bad, red);
    if (!tail) lv = sv == 0.0f ? INFINITY : log2f(sv);
    const float qsum = tail ? sv : (sv == 0.0f ? 0.0f : 1.0f);
    float qr = tail ? fmaxf(1.0f - sv, 0.0f) : 0.0f;
    // the student's sums: over every class, and over the classes outside the entries
    float s = 0.0f, mr = -INFINITY, sr = 0.0f;
    for (int base = 0; base < cols; base += kMarkCols) {
        const int end = base + kMarkCols < cols ? base + kMarkCols : cols;
        if (tail) {
            __syncthreads();
            for (int i = tid; i < kMarkCols / 32; i += kThreads) marks[i] = 0u;
            __syncthreads();
            for (int j = tid; j < k; j += kThreads) {
                const long long i = class_at(classes, class_bytes, row * k + j);
                if (i >= base && i < end) atomicOr(&marks[(i - base) >> 5], 1u << ((i - base) & 31));
            }
            __syncthreads();
        }
        for (int i = base + tid; i < end; i += kThreads) {
            const float zi = ld(z, i);
            s += exp2f((zi - m) * c);
            if (tail && !(marks[(i - base) >> 5] >> ((i - base) & 31) & 1u)) {
                if (zi > mr) sr = sr * exp2f((mr - zi) * c) + 1.0f, mr = zi;
                else if (zi != -INFINITY) sr += exp2f((zi - mr) * c);
            }
        }
    }
    s = block_sum(s, red);
    const float l2s = s == 0.0f ? INFINITY : log2f(s);
    float lr = INFINITY;
    if (tail) {
        const float gm = block_max(mr, red);
        const float scale = mr == -INFINITY ? 0.0f : exp2f((mr - gm) * c);
        sr = block_sum(sr * scale, red);
        mr = gm == -INFINITY ? 0.0f : gm;
        lr = sr == 0.0f ? INFINITY : log2f(sr);
    }
    float l = 0.0f;
    for (int j = tid; j < k; j += kThreads) {
        const long long i = class_at(classes, class_bytes, row * k + j);
        if (i < 0 || i >= cols) continue;
        const float q = exp2f((v[j] - mv) * cv - lv);
        const float lq = (v[j] - mv) * (tail ? 1.0f : inv_t) - kLn2 * lv;
        if (q != 0.0f) l += q * (lq - log_prob(ld(z, i), m, inv_t, l2s));
    }
    l = block_sum(l, red);
    if (tid == 0) {
        float coef = qsum, mb = m, lb = l2s;
        if (tail) {
            const float lpr = (mr - m) * c + lr - l2s;  // log2 of the student's mass outside
            const bool none = lr == INFINITY;
            if (none && qr <= kNoMass) qr = 0.0f;
            if (qr > 0.0f) l += none ? INFINITY : qr * kLn2 * (log2f(qr) - lpr);
            coef = none ? 0.0f : (qsum + qr) * exp2f(lpr) - qr;
            mb = mr, lb = lr;
        }
        if (bad != 0.0f) l = NAN, coef = NAN;
        loss[row] = l;
        if (stats) stats[row] = DistillStats{mb, lb, coef, qsum + qr, m, l2s, mv, lv};
    }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void distill_bwd_kernel(
    const T* __restrict__ logits, long long row_stride, const float* __restrict__ values,
    const void* __restrict__ classes, int class_bytes, const DistillStats* __restrict__ stats,
    const float* __restrict__ dloss, int cols, int k, float c, float inv_t, int tail, T* __restrict__ dlogits) {
    const long long row = blockIdx.x;
    const int tid = threadIdx.x;
    T* d = dlogits + row * cols;
    const DistillStats st = stats[row];
    if (st.l2s == INFINITY) {  // dead, or no class has probability
        for (int i = tid; i < cols; i += kThreads) d[i] = (T)0.0f;
        return;
    }
    const T* z = logits + row * row_stride;
    const float g = dloss[row] * inv_t;
    for (int i = tid; i < cols; i += kThreads) {
        // (no class outside the entries has probability: lb = +inf and the product is 0)
        const float p = st.lb == INFINITY ? 0.0f : exp2f((ld(z, i) - st.mb) * c - st.lb);
        d[i] = (T)(g * (st.coef * p));
    }
    __syncthreads();
    const float cv = tail ? kLog2e : c;
    if (st.coef != st.coef) return;  // an entry the row does not have: the row is NaN
    for (int j = tid; j < k; j += kThreads) {
        const long long i = class_at(classes, class_bytes, row * k + j);
        if (i < 0 || i >= cols) continue;
        float q = 0.0f;
        for (int o = 0; o < k; ++o)
            if (class_at(classes, class_bytes, row * k + o) == i) q += exp2f((values[row * k + o] - st.mv) * cv - st.lv);
        const float p = exp2f((ld(z, i) - st.m) * c - st.l2s);
        d[i] = (T)(g * (st.total * p - q));
    }
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

}  // namespace

extern "C" int isg_token_logprobs_fwd(const void* logits, long long row_stride, const void* tokens, int token_bytes,
                                      const unsigned char* live, int rows, int cols, int dtype, float temperature,
                                      int top, float* logprobs, float* entropy, float* top_logprobs,
                                      int32_t* top_classes, float* stats, void* stream) {
    const char* who = "isg_token_logprobs_fwd";
    int rc = check_call(who, row_stride, rows, cols, dtype, temperature);
    if (rc != ISG_OK) return rc;
    rc = check_bytes(who, tokens, token_bytes);
    if (rc != ISG_OK) return rc;
    ISG_REQUIRE(top >= 0 && top <= kMaxTop && top <= cols, ISG_EINVAL, "%s: top=%d of %d classes (at most %d)", who, top, cols,
                kMaxTop);
    if (rows == 0) return ISG_OK;
    ISG_REQUIRE(logits && entropy && (!tokens || logprobs) && (top == 0 || (top_logprobs && top_classes)), ISG_EINVAL,
                "%s: null pointer", who);
    hipStream_t s = static_cast<hipStream_t>(stream);
    const float c = kLog2e / temperature, inv_t = 1.0f / temperature;
    if (dtype == ISG_F32)
        hipLaunchKernelGGL(logprobs_fwd_kernel<float>, dim3(rows), dim3(kThreads), 0, s, static_cast<const float*>(logits),
                           row_stride, tokens, token_bytes, live, cols, c, inv_t, top, logprobs, entropy, top_logprobs, top_classes,
                           stats);
    else
        hipLaunchKernelGGL(logprobs_fwd_kernel<__hip_bfloat16>, dim3(rows), dim3(kThreads), 0, s,
                           static_cast<const __hip_bfloat16*>(logits), row_stride, tokens, token_bytes, live, cols, c, inv_t, top,
                           logprobs, entropy, top_logprobs, top_classes, stats);
    return isg::check_launch("logprobs_fwd_kernel");
}

extern "C" int isg_token_logprobs_bwd(const void* logits, long long row_stride, const void* tokens, int token_bytes,
                                      const unsigned char* live, const int32_t* top_classes, const float* stats,
                                      const float* dlogprobs, const float* dentropy, const float* dtop_logprobs, int rows,
                                      int cols, int dtype, float temperature, int top, void* dlogits, void* stream) {
    const char* who = "isg_token_logprobs_bwd";
    int rc = check_call(who, row_stride, rows, cols, dtype, temperature);
    if (rc != ISG_OK) return rc;
    rc = check_bytes(who, tokens, token_bytes);
    if (rc != ISG_OK) return rc;
    ISG_REQUIRE(top >= 0 && top <= kMaxTop && top <= cols, ISG_EINVAL, "%s: top=%d of %d classes (at most %d)", who, top, cols,
                kMaxTop);
    if (rows == 0) return ISG_OK;
    ISG_REQUIRE(logits && stats && dlogits && (!dlogprobs || tokens) && (!dtop_logprobs || (top > 0 && top_classes)),
                ISG_EINVAL, "%s: null pointer", who);
    ISG_REQUIRE(dlogits != logits, ISG_EINVAL, "%s: dlogits must not alias the logits", who);
    hipStream_t s = static_cast<hipStream_t>(stream);
    const float c = kLog2e / temperature, inv_t = 1.0f / temperature;
    if (dtype == ISG_F32)
        hipLaunchKernelGGL(logprobs_bwd_kernel<float>, dim3(rows), dim3(kThreads), 0, s, static_cast<const float*>(logits),
                           row_stride, tokens, token_bytes, live, top_classes, stats, dlogprobs, dentropy, dtop_logprobs,
                           cols, c, inv_t, top, static_cast<float*>(dlogits));
    else
        hipLaunchKernelGGL(logprobs_bwd_kernel<__hip_bfloat16>, dim3(rows), dim3(kThreads), 0, s,
                           static_cast<const __hip_bfloat16*>(logits), row_stride, tokens, token_bytes, live, top_classes,
                           stats, dlogprobs, dentropy, dtop_logprobs, cols, c, inv_t, top,
                           static_cast<__hip_bfloat16*>(dlogits));
    return isg::check_launch("logprobs_bwd_kernel");
}

namespace {
int check_entries(const char* who, int k, int tail) {
    ISG_REQUIRE(k >= 1 && k <= kMaxEntries, ISG_EINVAL, "%s: k=%d classes of the teacher (1 to %d)", who, k, kMaxEntries);
    ISG_REQUIRE(tail == 0 || tail == 1, ISG_EINVAL, "%s: tail=%d", who, tail);
    return ISG_OK;
}
}  // namespace

extern "C" int isg_distill_fwd(const void* logits, long long row_stride, const float* values, const void* classes,
                               int class_bytes, const unsigned char* live, int rows, int cols, int k, int dtype,
                               float temperature, int tail, float* loss, float* stats, void* stream) {
    const char* who = "isg_distill_fwd";
    int rc = check_call(who, row_stride, rows, cols, dtype, temperature);
    if (rc != ISG_OK) return rc;
    rc = check_entries(who, k, tail);
    if (rc != ISG_OK) return rc;
    rc = check_bytes(who, classes, class_bytes);
    if (rc != ISG_OK) return rc;
    if (rows == 0) return ISG_OK;
    ISG_REQUIRE(logits && values && classes && loss, ISG_EINVAL, "%s: null pointer", who);
    hipStream_t s = static_cast<hipStream_t>(stream);
    const float c = kLog2e / temperature, inv_t = 1.0f / temperature;
    DistillStats* st = reinterpret_cast<DistillStats*>(stats);
    if (dtype == ISG_F32)
        hipLaunchKernelGGL(distill_fwd_kernel<float>, dim3(rows), dim3(kThreads), 0, s, static_cast<const float*>(logits),
                           row_stride, values, classes, class_bytes, live, cols, k, c, inv_t, tail, loss, st);
    else
        hipLaunchKernelGGL(distill_fwd_kernel<__hip_bfloat16>, dim3(rows), dim3(kThreads), 0, s,
                           static_cast<const __hip_bfloat16*>(logits), row_stride, values, classes, class_bytes, live, cols,
                           k, c, inv_t, tail, loss, st);
    return isg::check_launch("distill_fwd_kernel");
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
    hipStream_t s = static_cast<hipStream_t>(stream);
    const float c = kLog2e / temperature, inv_t = 1.0f / temperature;
    const DistillStats* st = reinterpret_cast<const DistillStats*>(stats);
    if (dtype == ISG_F32)
        hipLaunchKernelGGL(distill_bwd_kernel<float>, dim3(rows), dim3(kThreads), 0, s, static_cast<const float*>(logits),
                           row_stride, values, classes, class_bytes, st, dloss, cols, k, c, inv_t, tail,
                           static_cast<float*>(dlogits));
    else
        hipLaunchKernelGGL(distill_bwd_kernel<__hip_bfloat16>, dim3(rows), dim3(kThreads), 0, s,
                           static_cast<const __hip_bfloat16*>(logits), row_stride, values, classes, class_bytes, st, dloss,
                           cols, k, c, inv_t, tail, static_cast<__hip_bfloat16*>(dlogits));
    return isg::check_launch("distill_bwd_kernel");
}
