// The AdamW step over all of a model's tensors: g' = g c with c = min(1, max_norm / (norm + 1e-6)) or 1,
// m = b1 m + (1 - b1) g', v = b2 v + (1 - b2) g'^2, w = w (1 - lr decay) - lr (m / (1 - b1^t)) / (sqrt(v / (1 - b2^t)) + eps).
//
// All tensors' elements are cut into chunks; the blocks of a grid that fills the GPU once take chunks in turn, and a chunk's tensor is found by
// bisection in a table that travels as a kernel parameter. The products and sums of both moments are rounded one by one, as the traced program's
// step (nn.adamw_update) rounds them; w is computed in float32 and rounded once to its type.
//
// Moments in 8 bits: blocks of 256 elements share a float32 scale s = max / 448, and hold m / s and sqrt(v) / s as e4m3, to nearest. sqrt(v) needs half
// the exponents that v does, and what is not zero does not become zero (a weight whose denominator vanished would jump). The scale is the block's
// largest value itself, not a power of two: it moves a little in every step, and it is by that that the others' roundings do not repeat. Changes of v of a
// thousandth a step are far below half a step of e4m3 (a sixteenth); simulated over 3000 steps of normal gradients, the mean ratio of these
// denominators to exact ones is 1.04 (standard deviation 0.2) with b2 = 0.999 and 1.01 (0.08) with 0.95, where scales that are powers of two freeze at 0.4 and 2.1.
#include <cmath>

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "convert.cuh"
#include "dense_lists.h"
#include "launch.cuh"

namespace lb {
namespace {

constexpr int kThreads = 256, kMost = 240;
constexpr int kBlock = 256;  // elements that share a scale
constexpr int chunk_elements(int bits) { return bits == 8 ? 8192 : 4096; }

struct AdamwTable {
    void *p[kMost], *m[kMost], *v[kMost];
    const void* g[kMost];
    float *master[kMost], *m_scale[kMost], *v_scale[kMost];
    long long n[kMost];
    int first[kMost + 1];   // first chunk of each tensor
    uint8_t dtype[kMost], grad[kMost];
    int8_t head[kMost];     // elements in front of the first one that groups of eight are aligned from; -1: they are nowhere
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
    float b1, b1_rest, b2, b2_rest, eps, factor, keep, rate, c2;  // keep: 1 - lr decay; rate: lr / (1 - b1^t); c2: 1 / (1 - b2^t)
};
__device__ Step this_step(const AdamwTable& t, Step* shared) {
    if (threadIdx.x == 0) {
        double step = t.step;
        if (t.step_at) step = t.step_dtype == LB_F32 ? (double)*(const float*)t.step_at : t.step_dtype == LB_I64 ? (double)*(const long long*)t.step_at : (double)*(const int*)t.step_at;
        const double lr = t.lr_at ? (double)*t.lr_at : t.lr;
        Step s{t.b1, t.b1_rest, t.b2, t.b2_rest, t.eps};
        s.keep = (float)(1.0 - lr * t.decay);
        s.rate = (float)(lr / -expm1(step * t.log_b1));
        s.c2 = (float)(1.0 / -expm1(step * t.log_b2));
        s.factor = 1.0f;
        if (t.norm_at) {
            const double quotient = t.max_norm / ((double)*t.norm_at + 1e-6);
            s.factor = quotient >= 1.0 ? 1.0f : (float)quotient;  // NaN stays
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
__device__ __forceinline__ float moved(const Step& s, float w, float m, float v) { return w * s.keep - m * s.rate / (__fsqrt_rn(v * s.c2) + s.eps); }

// Eight elements, aligned to as many.
__device__ __forceinline__ void load8(const float* p, float* x) {
    const float4 a = ((const float4*)p)[0], b = ((const float4*)p)[1];
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
}
__device__ __forceinline__ void store8(float* p, const float* x) {
    ((float4*)p)[0] = make_float4(x[0], x[1], x[2], x[3]), ((float4*)p)[1] = make_float4(x[4], x[5], x[6], x[7]);
}
template <class T>
__device__ __forceinline__ void load8(const T* p, float* x) {
    const uint4 w = *(const uint4*)p;
    const T* e = (const T*)&w;
#pragma unroll
    for (int k = 0; k < 8; k++) x[k] = to_float(e[k]);
}
template <class T>
__device__ __forceinline__ void store8(T* p, const float* x) {
    uint4 w;
    T* e = (T*)&w;
#pragma unroll
    for (int k = 0; k < 8; k++) e[k] = from_float<T>(x[k]);
    *(uint4*)p = w;
}

template <class P, class G, bool MASTER>
__device__ __forceinline__ void chunk_step(const AdamwTable& t, int k, long long at, int n, const Step& s) {
    P* p = (P*)t.p[k] + at;
    const G* g = (const G*)t.g[k] + at;
    float *m = (float*)t.m[k] + at, *v = (float*)t.v[k] + at, *master = MASTER ? t.master[k] + at : nullptr;
    const int head = t.head[k] < 0 ? n : min(n, (int)t.head[k]), eights = (n - head) / 8;
    for (int i = threadIdx.x; i < eights; i += kThreads) {
        const int e = head + 8 * i;
        float w[8], gg[8], mm[8], vv[8];
        load8(g + e, gg), load8(m + e, mm), load8(v + e, vv);
        if (MASTER) load8(master + e, w);
        else load8(p + e, w);
#pragma unroll
        for (int j = 0; j < 8; j++) moments(s, gg[j], mm[j], vv[j]), w[j] = moved(s, w[j], mm[j], vv[j]);
        store8(p + e, w), store8(m + e, mm), store8(v + e, vv);
        if (MASTER) store8(master + e, w);
    }
    for (int i = threadIdx.x; i < n - eights * 8; i += kThreads) {
        const int e = i < head ? i : eights * 8 + i;
        float mm = m[e], vv = v[e];
        moments(s, to_float(g[e]), mm, vv);
        const float w = moved(s, MASTER ? master[e] : to_float(p[e]), mm, vv);
        p[e] = from_float<P>(w), m[e] = mm, v[e] = vv;
        if (MASTER) master[e] = w;
    }
}

__device__ __forceinline__ float from_e4m3(uint8_t c) { return __half2float(__half(__nv_cvt_fp8_to_halfraw(c, __NV_E4M3))); }

// One warp's block of 256 elements, eight in a row to a lane.
template <class P, class G, bool MASTER>
__device__ __forceinline__ void block_step(P* p, const G* g, uint8_t* m, uint8_t* v, float* master, float* m_scale, float* v_scale, int n, bool whole, const Step& s) {
    const int lane = threadIdx.x & 31, e = lane * 8, count = max(0, min(8, n - e));
    const float sm = *m_scale, sv = *v_scale;
    float w[8], gg[8], mm[8], vv[8];
    uint8_t cm[8], cv[8];
    if (whole) {
        *(uint2*)cm = *(const uint2*)(m + e), *(uint2*)cv = *(const uint2*)(v + e);
        load8(g + e, gg);
        if (MASTER) load8(master + e, w);
        else load8(p + e, w);
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const bool in = j < count;
            cm[j] = in ? m[e + j] : 0, cv[j] = in ? v[e + j] : 0, gg[j] = in ? to_float(g[e + j]) : 0.0f;
            w[j] = !in ? 0.0f : MASTER ? master[e + j] : to_float(p[e + j]);
        }
    }
    uint32_t top_m = 0, top_v = 0;  // as bits: what is not negative is ordered alike, NaN above all
#pragma unroll
    for (int j = 0; j < 8; j++) {
        mm[j] = __fmul_rn(from_e4m3(cm[j]), sm);
        const float root = __fmul_rn(from_e4m3(cv[j]), sv);
        vv[j] = __fmul_rn(root, root);
        moments(s, gg[j], mm[j], vv[j]);
        w[j] = moved(s, w[j], mm[j], vv[j]);
        vv[j] = __fsqrt_rn(vv[j]);
        top_m = max(top_m, __float_as_uint(mm[j]) & 0x7fffffffu), top_v = max(top_v, __float_as_uint(vv[j]) & 0x7fffffffu);
    }
    const float most_m = __uint_as_float(__reduce_max_sync(0xffffffffu, top_m)), most_v = __uint_as_float(__reduce_max_sync(0xffffffffu, top_v));
    const bool no_m = most_m < 0x1p-100f, no_v = most_v < 0x1p-100f;
    const float inv_m = no_m ? 0.0f : __fdiv_rn(448.0f, most_m), inv_v = no_v ? 0.0f : __fdiv_rn(448.0f, most_v);
#pragma unroll
    for (int j = 0; j < 8; j++) {
        float x = __fmul_rn(vv[j], inv_v);
        if (x < 0x1p-9f && vv[j] > 0.0f) x = 0x1p-9f;
        cm[j] = __nv_cvt_float_to_fp8(__fmul_rn(mm[j], inv_m), __NV_SATFINITE, __NV_E4M3), cv[j] = __nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3);
    }
    __syncwarp();  // every lane has read the scales
    if (lane == 0) *m_scale = no_m ? 0.0f : __fdiv_rn(most_m, 448.0f), *v_scale = no_v ? 0.0f : __fdiv_rn(most_v, 448.0f);
    if (whole) {
        *(uint2*)(m + e) = *(uint2*)cm, *(uint2*)(v + e) = *(uint2*)cv;
        store8(p + e, w);
        if (MASTER) store8(master + e, w);
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (j < count) {
                m[e + j] = cm[j], v[e + j] = cv[j], p[e + j] = from_float<P>(w[j]);
                if (MASTER) master[e + j] = w[j];
            }
    }
}
template <class P, class G, bool MASTER>
__device__ __forceinline__ void chunk_step_8bit(const AdamwTable& t, int k, long long at, int n, const Step& s) {
    for (int b = threadIdx.x / 32; b * kBlock < n; b += kThreads / 32) {
        const long long e = at + (long long)b * kBlock, i = e / kBlock;
        const int count = min(kBlock, n - b * kBlock);
        block_step<P, G, MASTER>((P*)t.p[k] + e, (const G*)t.g[k] + e, (uint8_t*)t.m[k] + e, (uint8_t*)t.v[k] + e, MASTER ? t.master[k] + e : nullptr, t.m_scale[k] + i,
                                 t.v_scale[k] + i, count, count == kBlock && t.head[k] == 0, s);
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
__global__ void __launch_bounds__(kThreads, 2) adamw_kernel(const __grid_constant__ AdamwTable t) {
    __shared__ Step shared;
    grid_wait();
    const Step s = this_step(t, &shared);
    for (int c = blockIdx.x; c < t.first[t.count]; c += gridDim.x) {
        const int k = tensor_of(t, c);
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

    std::vector<Place> places;
    places.reserve((size_t)n * 7 + 3);
    std::vector<long long> count((size_t)n);
    auto look = [&](const lb_tensor& t, const lb_tensor& like, int dtype, const char* what, int k, bool written) {
        if (t.rank < 0 || t.rank > LB_MAX_RANK) refuse(format("%s %d has rank %d", what, k, t.rank));
        if (t.dtype != dtype) refuse(format("%s %d is %s, not %s", what, k, dtype_name(t.dtype), dtype_name(dtype)));
        if (!same_order(t, like)) refuse(format("%s %d must have its parameter's shape and strides", what, k));
        if (count[k] && (!t.ptr || (uintptr_t)t.ptr % dtype_size(dtype))) refuse(format("%s %d has no memory or is not aligned to its elements", what, k));
        places.push_back({(uintptr_t)t.ptr, (uintptr_t)t.ptr + (size_t)count[k] * dtype_size(dtype), what, k, written});
    };
    for (int k = 0; k < n; k++) {
        const lb_tensor& p = params[k];
        if (p.rank < 0 || p.rank > LB_MAX_RANK) refuse(format("parameter %d has rank %d", k, p.rank));
        if (p.dtype != LB_F32 && p.dtype != LB_BF16 && p.dtype != LB_F16) refuse(format("parameter %d is %s: float16, bfloat16 or float32", k, dtype_name(p.dtype)));
        count[k] = dense_elements(p);
        if (count[k] < 0) refuse(format("parameter %d is not dense", k));
        if (count[k] / chunk_elements(32) >= INT32_MAX / kMost) fail(LB_ERR_UNSUPPORTED, format("adamw: parameter %d has too many elements", k));
        look(p, p, p.dtype, "parameter", k, true);
        look(grads[k], p, grads[k].dtype == LB_F32 ? LB_F32 : p.dtype, "gradient", k, false);
        look(ms[k], p, bits == 8 ? LB_U8 : LB_F32, "first moment", k, true), look(vs[k], p, bits == 8 ? LB_U8 : LB_F32, "second moment", k, true);
        if (masters && masters[k].ptr && count[k]) {
            if (p.dtype == LB_F32) refuse(format("parameter %d is float32 itself: it has no float32 copy", k));
            look(masters[k], p, LB_F32, "float32 copy", k, true);
        }
        for (const lb_tensor* scales : {m_scales, v_scales}) {
            if (!scales) continue;
            const lb_tensor& t = scales[k];
            const long long blocks = (count[k] + kBlock - 1) / kBlock;
            if (t.dtype != LB_F32 || t.rank != 1 || t.shape[0] != blocks || (blocks > 1 && t.stride[0] != 1))
                refuse(format("the scales of parameter %d must be dense float32 [%lld], one for %d elements", k, blocks, kBlock));
            if (blocks && (!t.ptr || (uintptr_t)t.ptr % 4)) refuse(format("the scales of parameter %d have no memory or are not aligned", k));
            places.push_back({(uintptr_t)t.ptr, (uintptr_t)t.ptr + (size_t)blocks * 4, "scales", k, true});
        }
    }
    for (const lb_tensor* t : {step, lr, norm})
        if (t) places.push_back({(uintptr_t)t->ptr, (uintptr_t)t->ptr + dtype_size(t->dtype), t == step ? "step count" : t == lr ? "learning rate" : "norm", 0, false});
    const Place *a, *b;
    if (meeting(places, a, b)) refuse(format("%s %d and %s %d share memory", a->what, a->index, b->what, b->index));
    driver();

    const int grid = device_info().sms * 2;
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
            // vectors are 16 bytes of all tensors' types but codes, which take 8
            int head = -1;
            for (int h = 0; h < 8 && head < 0; h++) {
                auto fits = [&](const void* ptr, int dtype) { return !ptr || ((uintptr_t)ptr + (size_t)h * dtype_size(dtype)) % std::min(16, 8 * dtype_size(dtype)) == 0; };
                if (fits(t.p[i], params[k].dtype) && fits(t.g[i], grads[k].dtype) && fits(t.m[i], ms[k].dtype) && fits(t.v[i], vs[k].dtype) && fits(t.master[i], LB_F32)) head = h;
            }
            t.head[i] = (int8_t)head, t.first[i] = (int)first;
            first += (count[k] + chunk_elements(bits) - 1) / chunk_elements(bits);
        }
        t.first[t.count] = (int)first;
        if (!first) continue;
        launch_overlapped(bits == 8 ? adamw_kernel<8> : adamw_kernel<32>, dim3((unsigned)std::min<long long>(first, grid)), dim3(kThreads), 0, (cudaStream_t)stream, 0, t);
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
