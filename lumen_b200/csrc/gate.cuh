// The activations of the gated feed-forward block and their slopes.
//
// Silu is a s(a) and the tanh form of gelu is a s(2 t), t = sqrt(2 / pi) (a + 0.044715 a^3), since (1 + tanh(t)) / 2 = s(2 t): one sigmoid each, as the
// traced functions spell them (-inf gives NaN there and here). Relu is max(a, 0); NaN stays NaN. Slopes: s + a s (1 - s) t', with t' = 1 or
// 2 sqrt(2 / pi) (1 + 3 x 0.044715 a^2); relu's is 1 where a > 0 and 0 elsewhere.
#pragma once
#include <stdint.h>

#include "pair.cuh"

namespace lb {

enum Activation : int { ACT_SILU = 0, ACT_GELU = 1, ACT_RELU = 2 };

// 1 / (1 + exp(-t)). FAST: the hardware's exponential and reciprocal, whose few units in the last place of float32 (of exp, as many as |t|) vanish
// in a rounding to 16 bits; it gives 0 where exp(-t) is above 2^126, and a s is at most 1e-36 there.
template <bool FAST>
__device__ __forceinline__ float sigmoid(float t) {
    return FAST ? __fdividef(1.0f, 1.0f + __expf(-t)) : 1.0f / (1.0f + expf(-t));
}
template <int ACT>
__device__ __forceinline__ float sigmoid_argument(float a) {
    return ACT == ACT_SILU ? a : 1.5957691216057308f * (a + 0.044715f * a * a * a);
}

template <int ACT, bool FAST>
__device__ __forceinline__ float activation(float a) {
    if (ACT == ACT_RELU) return a <= 0.0f ? 0.0f : a;
    return a * sigmoid<FAST>(sigmoid_argument<ACT>(a));
}
// The activation, and its slope in `slope`.
template <int ACT, bool FAST>
__device__ __forceinline__ float activation_slope(float a, float& slope) {
    if (ACT == ACT_RELU) {
        slope = a > 0.0f ? 1.0f : 0.0f;
        return a <= 0.0f ? 0.0f : a;
    }
    const float s = sigmoid<FAST>(sigmoid_argument<ACT>(a));
    const float turn = ACT == ACT_SILU ? 1.0f : 1.5957691216057308f * (1.0f + 0.134145f * a * a);
    slope = s == 0.0f || s == 1.0f ? s : s + a * s * (1.0f - s) * turn;  // (far out the last product would be infinity times zero)
    return a * s;
}

// The same for two at a time, with the hardware's exponential and reciprocal.
__device__ __forceinline__ Pair sigmoid(Pair t) {
    const float2 x = apart(t * both(-1.4426950408889634f, -1.4426950408889634f));
    float2 e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.x) : "f"(x.x));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.y) : "f"(x.y));
    e = apart(both(e.x, e.y) + both(1.0f, 1.0f));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.x) : "f"(e.x));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.y) : "f"(e.y));
    return both(r.x, r.y);
}
template <int ACT>
__device__ __forceinline__ Pair activation(Pair a) {
    if (ACT == ACT_RELU) {
        const float2 x = apart(a);
        return both(x.x <= 0.0f ? 0.0f : x.x, x.y <= 0.0f ? 0.0f : x.y);
    }
    if (ACT == ACT_SILU) return a * sigmoid(a);
    const Pair k = both(0.07135481627260025f, 0.07135481627260025f), one = both(1.5957691216057308f, 1.5957691216057308f);
    return a * sigmoid(a * fma2(a * a, k, one));
}
// Beyond +-100 every sigmoid here is 0 or 1; a NaN stays.
__device__ __forceinline__ float within_100(float a) {
    asm("min.NaN.f32 %0, %0, 0f42C80000;" : "+f"(a));
    asm("max.NaN.f32 %0, %0, 0fC2C80000;" : "+f"(a));
    return a;
}
template <int ACT>
__device__ __forceinline__ Pair activation_slope(Pair a, Pair& slope) {
    const float2 x = apart(a);
    if (ACT == ACT_RELU) {
        slope = both(x.x > 0.0f ? 1.0f : 0.0f, x.y > 0.0f ? 1.0f : 0.0f);
        return both(x.x <= 0.0f ? 0.0f : x.x, x.y <= 0.0f ? 0.0f : x.y);
    }
    const Pair one = both(1.0f, 1.0f), in = both(within_100(x.x), within_100(x.y));
    Pair s, turn = in;  // in t'
    if (ACT == ACT_SILU) {
        s = sigmoid(in);
    } else {
        const Pair first = both(1.5957691216057308f, 1.5957691216057308f), square = in * in;
        s = sigmoid(in * fma2(square, both(0.07135481627260025f, 0.07135481627260025f), first));
        turn = in * fma2(square, both(0.21406444881780076f, 0.21406444881780076f), first);
    }
    slope = s * fma2(turn, fma2(s, both(-1.0f, -1.0f), one), one);  // s (1 + a t' (1 - s))
    return a * s;
}

}  // namespace lb
