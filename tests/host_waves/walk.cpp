// logprobs_stream_kernel on the host (built with this folder first on the include path and KERNELS naming the kernel's
// source, cut off before its launches).
#include "isg_classes.h"

// what the sources write as instructions of a wave
namespace {
template <>
float group_max<64>(float v) {
    return waves::fold(v, 63, __LINE__, [](float a, float b) { return fmaxf(a, b); });
}
template <>
float group_sum<64>(float v) {
    return waves::fold(v, 63, __LINE__, [](float a, float b) { return a + b; });
}
template <>
int group_sum<64>(int v) {
    return waves::fold(v, 63, __LINE__, [](int a, int b) { return a + b; });
}
template <>
int group_scan<64>(int v) {
    return waves::fold(v, waves::lane(), __LINE__, [](int a, int b) { return a + b; });
}
}  // namespace
// (the four comparisons of reach_mask)
#define asm(...)                                  \
    a = b = c = d = 0;                            \
    for (int q_ = 3; q_ >= 0; --q_) hit = hit + hit + (v[e + q_] >= low)
#include KERNELS
#undef asm

namespace {
struct Call {
    const float* row;
    LogprobsArgs args;
};
void thread_body(void* p) {
    const Call& c = *static_cast<const Call*>(p);
    logprobs_stream_kernel<float, 16, true>(c.row, c.args);
}
}  // namespace

// One row in one part: its `top` best classes, their log-probabilities and the entropy; `order`: of the four waves.
extern "C" int walk(const float* row, int cols, int top, const int* order, float* entropy, float* top_logprobs,
                    int32_t* top_classes) {
    Call c{};
    c.row = row;
    LogprobsArgs& a = c.args;
    a.entropy = entropy, a.top_logprobs = top_logprobs, a.top_classes = top_classes;
    a.row_stride = cols, a.units = 1, a.token_bytes = 4, a.cols = cols, a.splits = 1, a.per = cols, a.top = top;
    float c_lo;
    scale_of(1.0f, a.c, c_lo, a.inv_t);
    a.c_rel = c_lo / a.c;
    waves::grid_dim = Uint3{1, 1, 1};
    return waves::run_block(kThreads, order, thread_body, &c);
}
