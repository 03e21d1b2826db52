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

// One row's logits over a span of the vocabulary: their largest and the sum of exp(logit - largest).
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
// The sum of two spans. Where nothing is above -inf the sum stays what it is, zero.
__device__ __forceinline__ SpanSum join(SpanSum a, SpanSum b) {
    const float most = fmaxf(a.most, b.most), base = most == -INFINITY ? 0.0f : most;
    return {most, a.sum * exp2_approx((a.most - base) * kLog2e) + b.sum * exp2_approx((b.most - base) * kLog2e)};
}
#endif

}  // namespace lb
