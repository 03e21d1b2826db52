// The AdamW step over all of a model's tensors: g' = g c with c = min(1, max_norm / (norm + 1e-6)) or 1,
// m = b1 m + (1 - b1) g', v = b2 v + (1 - b2) g'^2, w = w (1 - lr decay) - lr (m / (1 - b1^t)) / (sqrt(v / (1 - b2^t)) + eps).
//
// All tensors' elements are cut into chunks; the blocks of a grid that fills the GPU once take chunks in turn, and a chunk's tensor is found by
// bisection in a table that travels as a kernel parameter. The products and sums of both moments are rounded one by one, as the traced program's
// step (nn.adamw_update) rounds them; w is computed in float32 and rounded once to its type.
//
// Bound by memory: all of a thread's loads are on their way at once, 16 elements of it in vectors of 32 bytes. 158 M bfloat16 weights with float32 moments 536 us, 6.45 TB/s (groups of eight
// elements in 16-byte vectors 605, two of them 613; three blocks an SM 560, four 567). 30 M values of three types with float32 gradients and copies, at odd places, 164.
//
// Moments in 8 bits: blocks of 256 elements share a float32 scale s = max / 448, and hold m / s and sqrt(v) / s as e4m3, to nearest. sqrt(v) needs half
// the exponents that v does, and what is not zero does not become zero (a weight whose denominator vanished would jump). The scale is the block's
// largest value itself, not a power of two: it moves a little in every step, and it is by that that the others' roundings do not repeat. Changes of v of a
// thousandth a step are far below half a step of e4m3 (a sixteenth); simulated over 3000 steps of normal gradients, the mean ratio of these
// denominators to exact ones is 1.04 (standard deviation 0.2) with b2 = 0.999 and 1.01 (0.08) with 0.95, where scales that are powers of two freeze at 0.4 and 2.1.
#include <cmath>
#include <type_traits>

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "convert.cuh"
#include "dense_lists.h"
#include "launch.cuh"
#include "pair.cuh"

namespace lb {
namespace {

constexpr int kThreads = 256, kMost = 240;
constexpr int kBlock = 256;  // elements that share a scale
constexpr int chunk_elements(int bits) { return bits == 8 ? 6144 : 4096; }
constexpr int blocks_per_sm(int bits) { return bits == 8 ? 3 : 2; }

struct AdamwTable {
    void *p[kMost], *m[kMost], *v[kMost];
    const void* g[kMost];
    float *master[kMost], *m_scale[kMost], *v_scale[kMost];
    long long n[kMost];
    int first[kMost + 1];   // first chunk of each tensor
    uint8_t dtype[kMost], grad[kMost];
    int8_t head[kMost];     // elements in front of the first one that vectors are aligned from; -1: they are nowhere
    int count;
    // the step
    float b1, b1_rest, b2, b2_rest, eps;
    double log_b1, log_b2, decay, lr, max_norm, step;
    const void* step_at;    // null: `step`
    int step_dtype;
    const float *lr_at, *norm_at;  // null: `lr`; no clipping
};
static_assert(sizeof(AdamwTable) <= 32000, "kernel parameters");

// What every element's step needs.
struct Step {
    float b1, b1_rest, b2, b2_rest, eps, factor, keep, rate, root_c2;  // keep: 1 - lr decay; rate: lr / (1 - b1^t); root_c2: 1 / sqrt(1 - b2^t)
};
__device__ Step this_step(const AdamwTable& t, Step* shared) {
    if (threadIdx.x == 0) {
        double step = t.step;
        if (t.step_at) step = t.step_dtype == LB_F32 ? (double)*(const float*)t.step_at : t.step_dtype == LB_I64 ? (double)*(const long long*)t.step_at : (double)*(const int*)t.step_at;
        const double lr = t.lr_at ? (double)*t.lr_at : t.lr;
        Step s{t.b1, t.b1_rest, t.b2, t.b2_rest, t.eps};
        s.keep = (float)(1.0 - lr * t.decay);
        s.rate = (float)(lr / -expm1(step * t.log_b1));
        s.root_c2 = (float)(1.0 / sqrt(-expm1(step * t.log_b2)));
        s.factor = 1.0f;
        if (t.norm_at) {
            const float quotient = __frcp_rn(*t.norm_at + 1e-6f) * (float)t.max_norm;
            s.factor = quotient >= 1.0f ? 1.0f : quotient;  // NaN stays
        }
        *shared = s;
    }
    __syncthreads();
    return *shared;
}
__device__ __forceinline__ void moments(const Step& s, float g, float& m, float& v) {
    g *= s.factor;
    m = __fadd_rn(__fmul_rn(m, s.b1), __fmul_rn(g, s.b1_rest));
    v = __fadd_rn(__fmul_rn(v, s.b2), __fmul_rn(__fmul_rn(g, g), s.b2_rest));
}
// w keep - m rate / (sqrt(v) sqrt(c2) + eps), with the hardware's root and quotient: a few units in the last place of float32 of a step that is small beside the weight.
__device__ __forceinline__ float moved(const Step& s, float w, float m, float root) { return w * s.keep - __fdividef(m * s.rate, fmaf(root, s.root_c2, s.eps)); }
__device__ __forceinline__ float root_of(float v) {
    float r;
    asm("sqrt.approx.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}

// 32 bytes, aligned to as many; moments and gradients are not read again before the next step.
template <class T>
__device__ __forceinline__ void load_wide(const T* p, uint32_t* w) {
    asm volatile("ld.global.L2::evict_first.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                 : "l"(__cvta_generic_to_global(p)) : "memory");
}
template <class T>
__device__ __forceinline__ void store_wide(T* p, const uint32_t* w) {
    asm volatile("st.global.L2::evict_first.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(__cvta_generic_to_global(p)), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]),
                 "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
}

// N elements as they lie in memory, on a boundary of N of them or 32 bytes.
template <class T, int N>
struct Some {
    static constexpr int words = N * (int)sizeof(T) / 4;
    static_assert(words == 4 || words % 8 == 0, "whole vectors");
    uint32_t w[words];
    __device__ __forceinline__ void load(const T* p) {
        if constexpr (words == 4) {
            const uint4 a = *(const uint4*)p;
            w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w;
        } else {
#pragma unroll
            for (int k = 0; k < words; k += 8) load_wide((const uint32_t*)p + k, w + k);
        }
    }
    __device__ __forceinline__ void store(T* p) const {
        if constexpr (words == 4) {
            *(uint4*)p = make_uint4(w[0], w[1], w[2], w[3]);
        } else {
#pragma unroll
            for (int k = 0; k < words; k += 8) store_wide((uint32_t*)p + k, w + k);
        }
    }
    __device__ __forceinline__ void widen(float* x) const {
#pragma unroll
        for (int k = 0; k < words; k++) {
            if constexpr (sizeof(T) == 4) {
                x[k] = __uint_as_float(w[k]);
            } else if constexpr (std::is_same_v<T, __half>) {
                const float2 f = __half22float2(*(const __half2*)&w[k]);
                x[2 * k] = f.x, x[2 * k + 1] = f.y;
            } else {
                x[2 * k] = __uint_as_float(w[k] << 16), x[2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
            }
        }
    }
    __device__ __forceinline__ void narrow(const float* x) {
#pragma unroll
        for (int k = 0; k < words; k++) {
            if constexpr (sizeof(T) == 4) {
                w[k] = __float_as_uint(x[k]);
            } else if constexpr (std::is_same_v<T, __half>) {
                const __half2 h = __floats2half2_rn(x[2 * k], x[2 * k + 1]);
                w[k] = *(const uint32_t*)&h;
            } else {
                const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * k], x[2 * k + 1]);
                w[k] = *(const uint32_t*)&h;
            }
        }
    }
};

constexpr int kEach = 16;  // elements of a thread
// All loads of a thread's elements are on their way at a time.
template <class P, class G, bool MASTER>
__device__ __forceinline__ void chunk_step(const AdamwTable& t, int k, long long at, int n, const Step& s) {
    P* p = (P*)t.p[k] + at;
    const G* g = (const G*)t.g[k] + at;
    float *m = (float*)t.m[k] + at, *v = (float*)t.v[k] + at, *master = MASTER ? t.master[k] + at : nullptr;
    const int head = t.head[k] < 0 ? n : min(n, (int)t.head[k]), groups = (n - head) / kEach;
    using W = std::conditional_t<MASTER, float, P>;
    W* from = MASTER ? (W*)master : (W*)p;
    static_assert(chunk_elements(32) == kThreads * kEach, "one group a thread");
    if ((int)threadIdx.x < groups) {
        const int e = head + kEach * threadIdx.x;
        Some<W, kEach> w;
        Some<G, kEach> gg;
        Some<float, kEach> mm, vv;
        gg.load(g + e), mm.load(m + e), vv.load(v + e), w.load(from + e);
        float x[kEach], y[kEach], m1[kEach], v1[kEach];
        w.widen(x), gg.widen(y), mm.widen(m1), vv.widen(v1);
#pragma unroll
        for (int j = 0; j < kEach; j++) moments(s, y[j], m1[j], v1[j]), x[j] = moved(s, x[j], m1[j], root_of(v1[j]));
        mm.narrow(m1), vv.narrow(v1), w.narrow(x);
        mm.store(m + e), vv.store(v + e), w.store(from + e);
        if constexpr (MASTER) {
            Some<P, kEach> out;
            out.narrow(x), out.store(p + e);
        }
    }
    for (int i = threadIdx.x; i < n - groups * kEach; i += kThreads) {
        const int e = i < head ? i : groups * kEach + i;
        float mm = m[e], vv = v[e];
        moments(s, to_float(g[e]), mm, vv);
        const float w = moved(s, MASTER ? master[e] : to_float(p[e]), mm, root_of(vv));
        p[e] = from_float<P>(w), m[e] = mm, v[e] = vv;
        if (MASTER) master[e] = w;
    }
}

// ---- moments in 8 bits: one warp's block of 256 elements, eight in a row to a lane ------------------------------------

// Codes of two elements and their values.
__device__ __forceinline__ Pair from_e4m3(uint32_t two) {
    const __half2 h = __half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)two, __NV_E4M3));
    const float2 f = __half22float2(h);
    return both(f.x, f.y);
}
__device__ __forceinline__ uint32_t to_e4m3(float2 x) { return (uint32_t)__nv_cvt_float2_to_fp8x2(x, __NV_SATFINITE, __NV_E4M3); }
// The largest magnitude of a warp's values; NaN is above all.
__device__ __forceinline__ float warp_most(float x) { return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(x) & 0x7fffffffu)); }
__device__ __forceinline__ float more(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float inverse(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float inverse_root(float x) {  // (of subnormal values too)
    float r;
    asm("rsqrt.approx.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// Codes `m` and `v`, weights and gradients of a lane's eight elements after a step; the block's scales in `sm` and `sv`.
//
// What is held is found by products and sums that are rounded one by one, as the 32-bit moments are, by roots with a step of Newton's iteration, which leaves them rounded but
// for a rare unit in the last place, and by a block's reciprocal, rounded: a code next to the middle of two is then the same whoever computes it, and one that is not
// makes the weight's next step another by a sixteenth. The weight's own step has the hardware's reciprocal.
//
// Bound by issued instructions (69 % of the slots) and memory: 158 M bfloat16 weights 303 - 317 us, 5.2 TB/s at best; 2 % less where v below 2^-126 has a wrong root; 62 instructions an
// element took 366, where root and quotient of each are the exact functions. Two blocks an SM with four blocks of 256 at once were slower by 5 %, four with two by 3 %.
__device__ __forceinline__ void eight_step(const Step& s, uint2& m, uint2& v, float& sm, float& sv, float* w, const float* g) {
    uint32_t cm[4] = {m.x & 0xffff, m.x >> 16, m.y & 0xffff, m.y >> 16}, cv[4] = {v.x & 0xffff, v.x >> 16, v.y & 0xffff, v.y >> 16};
    auto same = [](float x) { return both(x, x); };
    // (a packed product in front of a packed sum may become one instruction with it, whose product is not rounded: sums are scalar)
    auto sum = [](Pair a, Pair b) {
        const float2 x = apart(a), y = apart(b);
        return make_float2(__fadd_rn(x.x, y.x), __fadd_rn(x.y, y.y));
    };
    Pair root[4];
    float2 mm[4];
    float top_m = 0.0f, top_v = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const Pair gg = both(g[2 * j], g[2 * j + 1]) * same(s.factor), r = from_e4m3(cv[j]) * same(sv);
        mm[j] = sum(from_e4m3(cm[j]) * same(sm) * same(s.b1), gg * same(s.b1_rest));
        const float2 vv = sum(r * r * same(s.b2), gg * gg * same(s.b2_rest));
        const Pair v2 = both(vv.x, vv.y), y = both(inverse_root(fmaxf(vv.x, 0x1p-149f)), inverse_root(fmaxf(vv.y, 0x1p-149f))), near = v2 * y;
        root[j] = fma2(fma2(-near, near, v2), y * same(0.5f), near);
        const float2 den = apart(fma2(root[j], same(s.root_c2), same(s.eps)));
        const float2 moved = apart(fma2(both(mm[j].x, mm[j].y) * both(inverse(den.x), inverse(den.y)), same(-s.rate), both(w[2 * j], w[2 * j + 1]) * same(s.keep)));
        w[2 * j] = moved.x, w[2 * j + 1] = moved.y;
        const float2 b = apart(root[j]);
        top_m = more(more(top_m, fabsf(mm[j].x)), fabsf(mm[j].y)), top_v = more(more(top_v, b.x), b.y);
    }
    const float most_m = warp_most(top_m), most_v = warp_most(top_v);
    const bool no_m = most_m < 0x1p-100f, no_v = most_v < 0x1p-100f;
    // one reciprocal for both: odd lanes have the roots'
    const bool odd = threadIdx.x & 1;
    const float mine = __frcp_rn(odd ? most_v : most_m) * 448.0f, other = __shfl_xor_sync(0xffffffffu, mine, 1);
    const float inv_m = no_m ? 0.0f : odd ? other : mine, inv_v = no_v ? 0.0f : odd ? mine : other;
    sm = no_m ? 0.0f : most_m * (1.0f / 448.0f), sv = no_v ? 0.0f : most_v * (1.0f / 448.0f);
#pragma unroll
    for (int j = 0; j < 4; j++) {
        float2 x = apart(root[j] * same(inv_v));
        const float2 some = apart(root[j] * same(0x1p100f));  // a root is zero or more than 2^-75
        x.x = fmaxf(x.x, fminf(some.x, 0x1p-9f)), x.y = fmaxf(x.y, fminf(some.y, 0x1p-9f));
        cv[j] = to_e4m3(x), cm[j] = to_e4m3(apart(both(mm[j].x, mm[j].y) * same(inv_m)));
    }
    m = make_uint2(cm[0] | cm[1] << 16, cm[2] | cm[3] << 16), v = make_uint2(cv[0] | cv[1] << 16, cv[2] | cv[3] << 16);
}

// A block that is short, or whose memory vectors do not fit.
template <class P, class G, bool MASTER>
__device__ __forceinline__ void odd_block(P* p, const G* g, uint8_t* m, uint8_t* v, float* master, float* m_scale, float* v_scale, int n, const Step& s) {
    const int lane = threadIdx.x & 31, e = lane * 8, count = max(0, min(8, n - e));
    float sm = *m_scale, sv = *v_scale, w[8], gg[8];
    union {
        uint2 all;
        uint8_t one[8];
    } cm, cv;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const bool in = j < count;
        cm.one[j] = in ? m[e + j] : 0, cv.one[j] = in ? v[e + j] : 0, gg[j] = in ? to_float(g[e + j]) : 0.0f;
        w[j] = !in ? 0.0f : MASTER ? master[e + j] : to_float(p[e + j]);
    }
    eight_step(s, cm.all, cv.all, sm, sv, w, gg);
    __syncwarp();  // every lane has read the scales
    if (lane == 0) *m_scale = sm, *v_scale = sv;
#pragma unroll
    for (int j = 0; j < 8; j++)
        if (j < count) {
            m[e + j] = cm.one[j], v[e + j] = cv.one[j], p[e + j] = from_float<P>(w[j]);
            if (MASTER) master[e + j] = w[j];
        }
}
// A warp has the loads of U blocks on their way at a time.
template <class P, class G, bool MASTER>
__device__ __forceinline__ void chunk_step_8bit(const AdamwTable& t, int k, long long at, int n, const Step& s) {
    P* p = (P*)t.p[k] + at;
    const G* g = (const G*)t.g[k] + at;
    uint8_t *m = (uint8_t*)t.m[k] + at, *v = (uint8_t*)t.v[k] + at;
    float *master = MASTER ? t.master[k] + at : nullptr, *m_scale = t.m_scale[k] + at / kBlock, *v_scale = t.v_scale[k] + at / kBlock;
    using W = std::conditional_t<MASTER, float, P>;
    W* from = MASTER ? (W*)master : (W*)p;
    constexpr int warps = kThreads / 32, U = sizeof(W) + sizeof(G) <= 4 ? 3 : 2;
    const int lane = threadIdx.x & 31, warp = threadIdx.x / 32, whole = t.head[k] == 0 ? n / kBlock : 0;
    struct Held {
        Some<W, 8> w;
        Some<G, 8> g;
        uint2 m, v;
        float sm, sv;
    };
    for (int first = warp; first < whole; first += U * warps) {
        Held held[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int b = first + u * warps < whole ? first + u * warps : first, e = b * kBlock + lane * 8;
            held[u].w.load(from + e), held[u].g.load(g + e);
            held[u].m = *(const uint2*)(m + e), held[u].v = *(const uint2*)(v + e), held[u].sm = m_scale[b], held[u].sv = v_scale[b];
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int b = first + u * warps, e = b * kBlock + lane * 8;
            if (b < whole) {
                Held& now = held[u];
                float w[8], gg[8];
                now.w.widen(w), now.g.widen(gg);
                eight_step(s, now.m, now.v, now.sm, now.sv, w, gg);
                now.w.narrow(w), now.w.store(from + e);
                *(uint2*)(m + e) = now.m, *(uint2*)(v + e) = now.v;
                if (lane == 0) m_scale[b] = now.sm, v_scale[b] = now.sv;
                if constexpr (MASTER) {
                    Some<P, 8> out;
                    out.narrow(w), out.store(p + e);
                }
            }
        }
    }
    for (int b = whole + warp; b * kBlock < n; b += warps) {
        const int e = b * kBlock;
        odd_block<P, G, MASTER>(p + e, g + e, m + e, v + e, MASTER ? master + e : nullptr, m_scale + b, v_scale + b, min(kBlock, n - e), s);
    }
}

template <int BITS, class P, class G, bool MASTER>
__device__ __forceinline__ void chunk_of(const AdamwTable& t, int k, long long at, int n, const Step& s) {
    if constexpr (BITS == 8) chunk_step_8bit<P, G, MASTER>(t, k, at, n, s);
    else chunk_step<P, G, MASTER>(t, k, at, n, s);
}
template <int BITS, class P>
__device__ __forceinline__ void chunk_of(const AdamwTable& t, int k, long long at, int n, const Step& s) {
    const bool wide = t.grad[k] == LB_F32;
    if (t.master[k]) {
        if (wide) chunk_of<BITS, P, float, true>(t, k, at, n, s);
        else chunk_of<BITS, P, P, true>(t, k, at, n, s);
    } else {
        if (wide) chunk_of<BITS, P, float, false>(t, k, at, n, s);
        else chunk_of<BITS, P, P, false>(t, k, at, n, s);
    }
}
template <int BITS>
__global__ void __launch_bounds__(kThreads, blocks_per_sm(BITS)) adamw_kernel(const __grid_constant__ AdamwTable t) {
    __shared__ Step shared;
    grid_wait();
    const Step s = this_step(t, &shared);
    int k = tensor_of(t, blockIdx.x);
    for (int c = blockIdx.x; c < t.first[t.count]; c += gridDim.x) {
        while (t.first[k + 1] <= c) k++;
        const long long at = (long long)(c - t.first[k]) * chunk_elements(BITS);
        const int n = (int)min((long long)chunk_elements(BITS), t.n[k] - at);
        if (t.dtype[k] == LB_F32) chunk_of<BITS, float, float, false>(t, k, at, n, s);
        else if (t.dtype[k] == LB_BF16) chunk_of<BITS, __nv_bfloat16>(t, k, at, n, s);
        else chunk_of<BITS, __half>(t, k, at, n, s);
    }
}

// ---- host side ------------------------------------------------------------------------------------------------------

[[noreturn]] void refuse(const std::string& why) { fail(LB_ERR_INVALID, "adamw: " + why); }

void scalar(const lb_tensor* t, std::initializer_list<int> dtypes, const char* what) {
    if (!t) return;
    bool fits = t->ptr && t->rank >= 0 && t->rank <= LB_MAX_RANK && std::find(dtypes.begin(), dtypes.end(), t->dtype) != dtypes.end();
    for (int d = 0; fits && d < t->rank; d++) fits = t->shape[d] == 1;
    if (!fits || (uintptr_t)t->ptr % dtype_size(t->dtype)) refuse(format("%s is one value on the GPU", what));
}

void run_adamw(const lb_adamw_desc* desc, const lb_tensor* params, const lb_tensor* grads, const lb_tensor* ms, const lb_tensor* vs, const lb_tensor* m_scales,
               const lb_tensor* v_scales, const lb_tensor* masters, int n, const lb_tensor* step, const lb_tensor* lr, const lb_tensor* norm, void* stream) {
    if (!desc || n < 0 || (n && (!params || !grads || !ms || !vs))) refuse("null argument");
    if (!m_scales != !v_scales) refuse("both moments have scales, or neither");
    const int bits = m_scales ? 8 : 32;
    auto number = [](double x, const char* what) {
        if (!std::isfinite(x)) refuse(format("%s must be finite", what));
    };
    if (!lr) number(desc->lr, "lr");
    number(desc->eps, "eps"), number(desc->weight_decay, "weight_decay");
    if (desc->eps < 0.0) refuse("eps must not be negative");
    for (const double b : {desc->beta1, desc->beta2})
        if (!(b >= 0.0 && b < 1.0)) refuse("betas must be in [0, 1)");
    if (!step && !(desc->step >= 1)) refuse("steps are counted from 1");
    if (norm && (!(desc->max_norm >= 0.0) || std::isinf(desc->max_norm))) refuse("max_norm must be finite and not negative");
    scalar(step, {LB_F32, LB_I32, LB_I64}, "the step count (float32, int32 or int64)");
    scalar(lr, {LB_F32}, "the learning rate (float32)"), scalar(norm, {LB_F32}, "the norm (float32)");

    static const char* const names[] = {"parameter", "gradient", "first moment", "second moment", "float32 copy", "scales", "step count", "learning rate", "norm"};
    if (n >= 1 << 24) fail(LB_ERR_UNSUPPORTED, "adamw: too many tensors");
    std::vector<Place> places;
    places.reserve((size_t)n * 7 + 3);
    std::vector<long long> count((size_t)n);
    auto look = [&](const lb_tensor& t, const lb_tensor& like, int dtype, uint32_t what, int k, bool written) {
        if (t.rank < 0 || t.rank > LB_MAX_RANK) refuse(format("%s %d has rank %d", names[what], k, t.rank));
        if (t.dtype != dtype) refuse(format("%s %d is %s, not %s", names[what], k, dtype_name(t.dtype), dtype_name(dtype)));
        if (!same_order(t, like)) refuse(format("%s %d must have its parameter's shape and strides", names[what], k));
        if (count[k] && (!t.ptr || (uintptr_t)t.ptr % dtype_size(dtype))) refuse(format("%s %d has no memory or is not aligned to its elements", names[what], k));
        places.push_back({(uintptr_t)t.ptr, (uintptr_t)t.ptr + (size_t)count[k] * dtype_size(dtype), (uint32_t)k, what, written});
    };
    for (int k = 0; k < n; k++) {
        const lb_tensor& p = params[k];
        if (p.rank < 0 || p.rank > LB_MAX_RANK) refuse(format("parameter %d has rank %d", k, p.rank));
        if (p.dtype != LB_F32 && p.dtype != LB_BF16 && p.dtype != LB_F16) refuse(format("parameter %d is %s: float16, bfloat16 or float32", k, dtype_name(p.dtype)));
        count[k] = dense_elements(p);
        if (count[k] < 0) refuse(format("parameter %d is not dense", k));
        if (count[k] / chunk_elements(32) >= INT32_MAX / kMost) fail(LB_ERR_UNSUPPORTED, format("adamw: parameter %d has too many elements", k));
        look(p, p, p.dtype, 0, k, true);
        look(grads[k], p, grads[k].dtype == LB_F32 ? LB_F32 : p.dtype, 1, k, false);
        look(ms[k], p, bits == 8 ? LB_U8 : LB_F32, 2, k, true), look(vs[k], p, bits == 8 ? LB_U8 : LB_F32, 3, k, true);
        if (masters && masters[k].ptr && count[k]) {
            if (p.dtype == LB_F32) refuse(format("parameter %d is float32 itself: it has no float32 copy", k));
            look(masters[k], p, LB_F32, 4, k, true);
        }
        for (const lb_tensor* scales : {m_scales, v_scales}) {
            if (!scales) continue;
            const lb_tensor& t = scales[k];
            const long long blocks = (count[k] + kBlock - 1) / kBlock;
            if (t.dtype != LB_F32 || t.rank != 1 || t.shape[0] != blocks || (blocks > 1 && t.stride[0] != 1))
                refuse(format("the scales of parameter %d must be dense float32 [%lld], one for %d elements", k, blocks, kBlock));
            if (blocks && (!t.ptr || (uintptr_t)t.ptr % 4)) refuse(format("the scales of parameter %d have no memory or are not aligned", k));
            places.push_back({(uintptr_t)t.ptr, (uintptr_t)t.ptr + (size_t)blocks * 4, (uint32_t)k, 5, true});
        }
    }
    for (const lb_tensor* t : {step, lr, norm})
        if (t) places.push_back({(uintptr_t)t->ptr, (uintptr_t)t->ptr + dtype_size(t->dtype), 0, t == step ? 6u : t == lr ? 7u : 8u, false});
    const Place *a, *b;
    if (meeting(places, a, b)) refuse(format("%s %d and %s %d share memory", names[a->what], (int)a->index, names[b->what], (int)b->index));
    driver();

    const int grid = device_info().sms * blocks_per_sm(bits);
    for (int k = 0; k < n;) {
        AdamwTable t;
        t.b1 = (float)desc->beta1, t.b1_rest = (float)(1.0 - desc->beta1), t.b2 = (float)desc->beta2, t.b2_rest = (float)(1.0 - desc->beta2), t.eps = (float)desc->eps;
        t.log_b1 = std::log(desc->beta1), t.log_b2 = std::log(desc->beta2), t.decay = desc->weight_decay, t.lr = desc->lr, t.max_norm = desc->max_norm;
        t.step = (double)desc->step, t.step_at = step ? step->ptr : nullptr, t.step_dtype = step ? step->dtype : 0;
        t.lr_at = lr ? (const float*)lr->ptr : nullptr, t.norm_at = norm ? (const float*)norm->ptr : nullptr;
        t.count = 0;
        long long first = 0;
        for (; k < n && t.count < kMost; k++) {
            if (!count[k]) continue;
            const int i = t.count++;
            t.p[i] = params[k].ptr, t.g[i] = grads[k].ptr, t.m[i] = ms[k].ptr, t.v[i] = vs[k].ptr, t.n[i] = count[k];
            t.master[i] = masters ? (float*)masters[k].ptr : nullptr;
            t.m_scale[i] = m_scales ? (float*)m_scales[k].ptr : nullptr, t.v_scale[i] = v_scales ? (float*)v_scales[k].ptr : nullptr;
            t.dtype[i] = (uint8_t)params[k].dtype, t.grad[i] = (uint8_t)grads[k].dtype;
            // vectors are 32 bytes, but for moments in 8 bits, whose eight elements are 8 bytes of codes and 16 of 16-bit values
            int head = -1;
            for (int h = 0; h < 16 && head < 0; h++) {
                auto fits = [&](const void* ptr, int dtype) { return !ptr || ((uintptr_t)ptr + (size_t)h * dtype_size(dtype)) % (bits == 8 ? 8 * dtype_size(dtype) : 32) == 0; };
                if (fits(t.p[i], params[k].dtype) && fits(t.g[i], grads[k].dtype) && fits(t.m[i], ms[k].dtype) && fits(t.v[i], vs[k].dtype) && fits(t.master[i], LB_F32)) head = h;
            }
            t.head[i] = (int8_t)head, t.first[i] = (int)first;
            first += (count[k] + chunk_elements(bits) - 1) / chunk_elements(bits);
        }
        t.first[t.count] = (int)first;
        if (!first) continue;
        auto kernel = bits == 8 ? adamw_kernel<8> : adamw_kernel<32>;
        launch_overlapped(kernel, dim3((unsigned)std::min<long long>(first, grid)), dim3(kThreads), 0, (cudaStream_t)stream, 0, t);
    }
}

}  // namespace
}  // namespace lb

extern "C" {

int lb_adamw_step(const lb_adamw_desc* desc, const lb_tensor* params, const lb_tensor* grads, const lb_tensor* exp_avg, const lb_tensor* exp_avg_sq,
                  const lb_tensor* exp_avg_scale, const lb_tensor* exp_avg_sq_scale, const lb_tensor* masters, int n_tensors, const lb_tensor* step, const lb_tensor* lr,
                  const lb_tensor* norm, void* stream) {
    return lb::guarded([&] { lb::run_adamw(desc, params, grads, exp_avg, exp_avg_sq, exp_avg_scale, exp_avg_sq_scale, masters, n_tensors, step, lr, norm, stream); });
}
}
