// What the kernels of the linear cross entropy share.
#pragma once
#include <stdint.h>

#include "common.h"

namespace lb {

// Each row's class, as the caller holds it: int32 or int64, `step` elements apart. A row whose class is `ignored` does not count; classes outside the
// vocabulary are clamped into it.
struct Targets {
    const void* at;
    long long step, ignored;
    int wide, classes;
#ifdef __CUDACC__
    __device__ __forceinline__ int of(long long row) const {  // -1: does not count
        const long long t = wide ? ((const long long*)at)[row * step] : (long long)((const int*)at)[row * step];
        return t == ignored ? -1 : (int)(t < 0 ? 0 : t >= classes ? classes - 1 : t);
    }
#endif
};

// One row's logits over a span of the vocabulary: their largest and the sum of exp(logit - largest), of exp(logit) where the largest is infinite.
struct SpanSum {
    float most, sum;
};

#ifdef __CUDACC__
constexpr float kLog2e = 1.4426950408889634f;
__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// What is taken away from logits whose largest is `most`, before their exponentials are. Where that is infinite they stay as they are: sums of them are then zero, or infinite,
// as the log-sum-exp is.
__device__ __forceinline__ float base_of(float most) { return fabsf(most) == INFINITY ? 0.0f : most; }
// The sum of two spans.
__device__ __forceinline__ SpanSum join(SpanSum a, SpanSum b) {
    const float most = fmaxf(a.most, b.most), base = base_of(most);
    return {most, a.sum * exp2_approx((a.most - base) * kLog2e) + b.sum * exp2_approx((b.most - base) * kLog2e)};
}
#endif

}  // namespace lb
