// The global norm over many tensors, and clipping by it: n = sqrt(sum over all tensors of x^2), c = min(1, max_norm / (n + 1e-6)), out = c x.
//
// All tensors' elements are cut into chunks of kChunkBytes; the blocks of a grid that fills the GPU once take chunks in turn, and a chunk's tensor is
// found by bisection in a table that travels as a kernel parameter. Each block leaves the sum of its chunks' squares; what follows adds
// the blocks' sums up, every block for itself and in the same order: no atomics, the same bits every time (on GPUs with the same number of SMs).
//
// Squares are taken in float32 and added up four or eight at a time; a group whose sum leaves float32's normal range is squared again
// in 64 bits, and groups are added up in 64 bits: the norm is right for all that float32 holds. A norm that is infinite or NaN gives
// c = 0 or NaN, as the quotient says.
//
// Bound by memory: the norm reads every tensor once. Clipping reads it a second time and writes it; where c is 1 and the result's place is
// the operand's, nothing is left to do. The second pass walks the chunks backwards, and the last 64 MB that the first one reads stay in the L2 for it
// (evict-last; all else goes first). 158 M bfloat16 values (317 MB): the squares take 47.6 us alone, 6.66 TB/s, clipping into other memory 147.5
// us in all, 951 MB at 6.45 TB/s (nothing kept 152.2, 96 MB 148.5); loads of 16 bytes and four a thread in flight 159, 16-byte stores past the L2 no
// gain, eight blocks to an SM 220; in place over the bound 157.6 in a graph (into other memory 149.5). Tables of one call share the 64 MB, the last ones first
// (grad_norm.h): 300 tensors of 600 MB 291 us, 700 of 560 MB 279, with as much for every table 297 and 291. In place within the bound nothing reads what is kept: a
// pass over the gradients behind the call is faster by it (158 M values from the end 216 -> 198 us), six passes over other data that just fits the L2 take 4 to 8 us longer
// (80 MB 100 -> 108), and data that is smaller or larger than that no longer than before. The norm of 60 M values of three types, 160 MB, 30 us with both launches, 5.3 TB/s.
#include <algorithm>
#include <cmath>
#include <vector>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "grad_norm.h"
#include "launch.cuh"

namespace lb {
namespace {

constexpr int kThreads = 256, kBlocksPerSm = 3;
constexpr int kReads = 4, kScales = 2;                      // 32-byte loads of a thread in flight: squares, scaling (which holds its results too)
constexpr int kChunkBytes = kThreads * 32 * kReads;         // 32 KB of the operand
constexpr int kKeep = (64 << 20) / kChunkBytes;              // chunks whose second reading finds them in the L2
constexpr int kMost = 240;                                  // tensors of one launch (a table for 32 is handed over 0.1 us faster, and is not worth its kernels)

struct NormTable {
    const void* x[kMost];
    void* out[kMost];
    long long n[kMost];
    int first[kMost + 1];  // first chunk of each tensor
    uint8_t dtype[kMost];
    int count;
};
static_assert(sizeof(NormTable) <= 32000, "kernel parameters");

template <class T> struct Of;
template <> struct Of<float> {
    static constexpr int per = 4;
    __device__ static void widen(const uint4& v, float* x) { x[0] = __uint_as_float(v.x), x[1] = __uint_as_float(v.y), x[2] = __uint_as_float(v.z), x[3] = __uint_as_float(v.w); }
    __device__ static uint4 narrow(const float* x) { return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3])); }
    __device__ static float get(const float* p) { return *p; }
    __device__ static void put(float* p, float x) { *p = x; }
};
template <> struct Of<__nv_bfloat16> {
    static constexpr int per = 8;
    __device__ static void widen(const uint4& v, float* x) {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int k = 0; k < 4; k++) x[2 * k] = __uint_as_float(w[k] << 16), x[2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
    }
    __device__ static uint4 narrow(const float* x) {
        uint32_t w[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * k], x[2 * k + 1]);
            w[k] = *(const uint32_t*)&h;
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
    __device__ static float get(const __nv_bfloat16* p) { return __bfloat162float(*p); }
    __device__ static void put(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }
};
template <> struct Of<__half> {
    static constexpr int per = 8;
    __device__ static void widen(const uint4& v, float* x) {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const float2 f = __half22float2(*(const __half2*)&w[k]);
            x[2 * k] = f.x, x[2 * k + 1] = f.y;
        }
    }
    __device__ static uint4 narrow(const float* x) {
        uint32_t w[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const __half2 h = __floats2half2_rn(x[2 * k], x[2 * k + 1]);
            w[k] = *(const uint32_t*)&h;
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
    __device__ static float get(const __half* p) { return __half2float(*p); }
    __device__ static void put(__half* p, float x) { *p = __float2half_rn(x); }
};

// 32 bytes, aligned to as many, and what becomes of their place in the L2: KEEP what will be read again, let go first what will not.
struct Wide {
    uint4 lo, hi;
};
template <bool KEEP>
__device__ __forceinline__ Wide load_wide(const Wide* p) {
    Wide w;
    if (KEEP)
        asm volatile("ld.global.L2::evict_last.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=r"(w.lo.x), "=r"(w.lo.y), "=r"(w.lo.z), "=r"(w.lo.w), "=r"(w.hi.x), "=r"(w.hi.y), "=r"(w.hi.z), "=r"(w.hi.w)
                     : "l"(__cvta_generic_to_global(p)) : "memory");
    else
        asm volatile("ld.global.L2::evict_first.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=r"(w.lo.x), "=r"(w.lo.y), "=r"(w.lo.z), "=r"(w.lo.w), "=r"(w.hi.x), "=r"(w.hi.y), "=r"(w.hi.z), "=r"(w.hi.w)
                     : "l"(__cvta_generic_to_global(p)) : "memory");
    return w;
}
__device__ __forceinline__ void store_wide(Wide* p, const Wide& w) {
    asm volatile("st.global.L2::evict_first.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(__cvta_generic_to_global(p)), "r"(w.lo.x), "r"(w.lo.y),
                 "r"(w.lo.z), "r"(w.lo.w), "r"(w.hi.x), "r"(w.hi.y), "r"(w.hi.z), "r"(w.hi.w)
                 : "memory");
}

// The sum of squares of a group, exact to float32's rounding whatever the values' size.
template <int N>
__device__ __forceinline__ double squares(const float* x) {
    float s = 0.0f;
#pragma unroll
    for (int k = 0; k < N; k++) s += x[k] * x[k];
    if (s >= 1e-30f && s <= 1e38f) return s;  // smaller: squares may have lost digits; larger, or NaN: they may have overflowed
    double t = 0.0;
#pragma unroll
    for (int k = 0; k < N; k++) t += (double)x[k] * x[k];
    return t;
}

__device__ __forceinline__ double block_sum(double v, double* held) {  // to all threads
    for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    if ((threadIdx.x & 31) == 0) held[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.0;
#pragma unroll
    for (int k = 0; k < kThreads / 32; k++) v += held[k];
    return v;
}

// The tensor that chunk `c` lies in: the last whose first chunk is not behind it (an empty tensor has none).
__device__ __forceinline__ int tensor_of(const NormTable& t, int c) {
    int lo = 0, hi = t.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (t.first[mid] <= c) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

template <class T, bool KEEP>
__device__ __forceinline__ double chunk_squares(const T* x, int n) {
    constexpr int per = Of<T>::per;
    const int head = min(n, (int)((32 - ((uintptr_t)x & 31)) & 31) / (int)sizeof(T)), wides = (n - head) / (2 * per);
    const Wide* v = (const Wide*)(x + head);
    double sum = 0.0;
    for (int i0 = threadIdx.x; i0 < wides; i0 += kThreads * kReads) {
        Wide w[kReads];
#pragma unroll
        for (int k = 0; k < kReads; k++) w[k] = i0 + k * kThreads < wides ? load_wide<KEEP>(v + i0 + k * kThreads) : Wide{};
#pragma unroll
        for (int k = 0; k < kReads; k++) {
            float f[2 * per];
            Of<T>::widen(w[k].lo, f), Of<T>::widen(w[k].hi, f + per);
            sum += squares<per>(f), sum += squares<per>(f + per);
        }
    }
    const int ends = n - wides * 2 * per;  // before and behind the vectors: less than two of them
    if ((int)threadIdx.x < ends) {
        const float f = Of<T>::get(x + ((int)threadIdx.x < head ? threadIdx.x : wides * 2 * per + threadIdx.x));
        sum += (double)f * f;
    }
    return sum;
}

template <class T>
__device__ __forceinline__ void chunk_scale(const T* x, T* out, int n, float c, float before) {
    constexpr int per = Of<T>::per;
    int head = n, wides = 0;  // operand and result aligned differently: by the element
    if ((((uintptr_t)x ^ (uintptr_t)out) & 31) == 0) head = min(n, (int)((32 - ((uintptr_t)x & 31)) & 31) / (int)sizeof(T)), wides = (n - head) / (2 * per);
    const Wide* v = (const Wide*)(x + head);
    Wide* o = (Wide*)(out + head);
    for (int i0 = threadIdx.x; i0 < wides; i0 += kThreads * kScales) {
        Wide w[kScales];
#pragma unroll
        for (int k = 0; k < kScales; k++)
            if (i0 + k * kThreads < wides) w[k] = load_wide<false>(v + i0 + k * kThreads);
#pragma unroll
        for (int k = 0; k < kScales; k++)
            if (i0 + k * kThreads < wides) {
                float f[2 * per];
                Of<T>::widen(w[k].lo, f), Of<T>::widen(w[k].hi, f + per);
#pragma unroll
                for (int j = 0; j < 2 * per; j++) f[j] = f[j] * before * c;
                store_wide(o + i0 + k * kThreads, Wide{Of<T>::narrow(f), Of<T>::narrow(f + per)});
            }
    }
    for (int i = threadIdx.x; i < n - wides * 2 * per; i += kThreads) {
        const int at = i < head ? i : wides * 2 * per + i;
        Of<T>::put(out + at, Of<T>::get(x + at) * before * c);
    }
}

__global__ void __launch_bounds__(kThreads, kBlocksPerSm) norm_squares_kernel(const __grid_constant__ NormTable t, double* partial, int keep) {
    __shared__ double held[kThreads / 32];
    grid_wait();
    double sum = 0.0;
    for (int c = blockIdx.x; c < t.first[t.count]; c += gridDim.x) {
        const int k = tensor_of(t, c), dtype = t.dtype[k];
        const int per = kChunkBytes / (dtype == LB_F32 ? 4 : 2);
        const long long at = (long long)(c - t.first[k]) * per;
        const int n = (int)min((long long)per, t.n[k] - at);
        if (t.first[t.count] - c <= keep) {
            if (dtype == LB_F32) sum += chunk_squares<float, true>((const float*)t.x[k] + at, n);
            else if (dtype == LB_BF16) sum += chunk_squares<__nv_bfloat16, true>((const __nv_bfloat16*)t.x[k] + at, n);
            else sum += chunk_squares<__half, true>((const __half*)t.x[k] + at, n);
        } else {
            if (dtype == LB_F32) sum += chunk_squares<float, false>((const float*)t.x[k] + at, n);
            else if (dtype == LB_BF16) sum += chunk_squares<__nv_bfloat16, false>((const __nv_bfloat16*)t.x[k] + at, n);
            else sum += chunk_squares<__half, false>((const __half*)t.x[k] + at, n);
        }
    }
    sum = block_sum(sum, held);
    if (threadIdx.x == 0) partial[blockIdx.x] = sum;
}

// The norm from the blocks' sums: every thread of every block that asks gets the same bits.
__device__ __forceinline__ double total_norm(const double* partial, int parts, double* held) {
    double sum = 0.0;
    for (int i = threadIdx.x; i < parts; i += kThreads) sum += partial[i];
    return sqrt(block_sum(sum, held));
}

__global__ void __launch_bounds__(kThreads) norm_kernel(const double* partial, int parts, float* norm) {
    __shared__ double held[kThreads / 32];
    grid_wait();
    const double n = total_norm(partial, parts, held);
    if (threadIdx.x == 0) *norm = (float)n;
}

__global__ void __launch_bounds__(kThreads, kBlocksPerSm) norm_scale_kernel(const __grid_constant__ NormTable t, const double* partial, int parts, double max_norm, float* norm) {
    __shared__ double held[kThreads / 32];
    grid_wait();
    const double n = total_norm(partial, parts, held);
    if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)n;
    const double quotient = max_norm / (n + 1e-6);
    const double factor = quotient >= 1.0 ? 1.0 : quotient;  // NaN stays
    const float before = factor < 1e-30 ? 5.421010862427522e-20f : 1.0f;  // 2^-64: a factor below float32's normal range is two
    const float c = (float)(factor / before);
    const int chunks = t.first[t.count];
    for (int i = blockIdx.x; i < chunks; i += gridDim.x) {
        const int chunk = chunks - 1 - i, k = tensor_of(t, chunk), dtype = t.dtype[k];
        if (factor == 1.0 && t.x[k] == t.out[k]) continue;
        const int per = kChunkBytes / (dtype == LB_F32 ? 4 : 2);
        const long long at = (long long)(chunk - t.first[k]) * per;
        const int m = (int)min((long long)per, t.n[k] - at);
        if (dtype == LB_F32) chunk_scale((const float*)t.x[k] + at, (float*)t.out[k] + at, m, c, before);
        else if (dtype == LB_BF16) chunk_scale((const __nv_bfloat16*)t.x[k] + at, (__nv_bfloat16*)t.out[k] + at, m, c, before);
        else chunk_scale((const __half*)t.x[k] + at, (__half*)t.out[k] + at, m, c, before);
    }
}

// ---- host side ------------------------------------------------------------------------------------------------------

[[noreturn]] void refuse(const std::string& why) { fail(LB_ERR_INVALID, "grad_norm: " + why); }

// The number of elements of a tensor that fills its memory without gaps, in any order of its dimensions; refuses others.
long long dense_elements(const lb_tensor& t, int index) {
    if (t.rank < 0 || t.rank > LB_MAX_RANK) refuse(format("tensor %d has rank %d", index, t.rank));
    if (t.dtype != LB_F32 && t.dtype != LB_BF16 && t.dtype != LB_F16) refuse(format("tensor %d is %s: float16, bfloat16 or float32", index, dtype_name(t.dtype)));
    long long n = 1;
    for (int d = 0; d < t.rank; d++) {
        if (t.shape[d] < 0) refuse(format("tensor %d has a negative size", index));
        n *= t.shape[d];
    }
    if (n && (!t.ptr || (uintptr_t)t.ptr % dtype_size(t.dtype))) refuse(format("tensor %d has no memory or is not aligned to its elements", index));
    if (n <= 1) return n;
    long long step = 1;
    bool used[LB_MAX_RANK] = {};
    for (int found = 0; step < n;) {  // the dimension that strides by what is filled so far
        int next = -1;
        for (int d = 0; d < t.rank && next < 0; d++)
            if (!used[d] && t.shape[d] > 1 && t.stride[d] == step) next = d;
        if (next < 0 || found++ > LB_MAX_RANK) refuse(format("tensor %d is not dense", index));
        used[next] = true, step *= t.shape[next];
    }
    return n;
}

struct Range {
    uintptr_t from, to;
    int index;
};

size_t scratch_bytes(int n) { return (size_t)((n + kMost - 1) / kMost) * sm_count_hint() * kBlocksPerSm * sizeof(double); }

// The launches for tensors that have been looked at, kMost of them (those with elements) a table.
void launch_norm(const lb_tensor* xs, const lb_tensor* outs, int n, const std::vector<long long>& count, double max_norm, float* norm, double* partial, cudaStream_t s) {
    const int grid = device_info().sms * kBlocksPerSm;
    std::vector<long long> chunks((size_t)n);
    for (int k = 0; k < n; k++) {
        const int per = kChunkBytes / dtype_size(xs[k].dtype);
        chunks[k] = (count[k] + per - 1) / per;
    }
    const std::vector<NormPass> passes = norm_passes(chunks, kMost, outs ? kKeep : 0);
    std::vector<NormTable> tables(passes.size());
    std::vector<int> blocks;
    int parts = 0;
    for (size_t at = 0; at < passes.size(); at++) {
        NormTable& t = tables[at];
        t.count = 0;
        int first = 0;
        for (int k = passes[at].from; k < passes[at].to; k++) {
            if (!count[k]) continue;
            const int i = t.count++;
            t.x[i] = xs[k].ptr, t.out[i] = outs ? outs[k].ptr : nullptr, t.n[i] = count[k], t.dtype[i] = (uint8_t)xs[k].dtype;
            t.first[i] = first, first += (int)chunks[k];
        }
        t.first[t.count] = first;
        blocks.push_back(std::min(first, grid));
        if (!first) continue;
        launch_overlapped(norm_squares_kernel, dim3((unsigned)blocks.back()), dim3(kThreads), 0, s, 0, t, partial + parts, passes[at].keep);
        parts += blocks.back();
    }
    if (!outs || !parts) {
        launch_overlapped(norm_kernel, dim3(1), dim3(kThreads), 0, s, 0, (const double*)partial, parts, norm);
        return;
    }
    bool first = true;
    for (size_t k = tables.size(); k-- > 0;) {
        if (!blocks[k]) continue;
        launch_overlapped(norm_scale_kernel, dim3((unsigned)blocks[k]), dim3(kThreads), 0, s, 0, tables[k], (const double*)partial, parts, max_norm, first ? norm : nullptr);
        first = false;
    }
}

// `outs` null: the norm alone.
void run_norm(const lb_tensor* xs, const lb_tensor* outs, int n, double max_norm, const lb_tensor* norm, void* scratch, size_t bytes, void* stream) {
    if (n < 0 || (n && !xs) || !norm) refuse("null argument");
    if (norm->dtype != LB_F32 || norm->rank > LB_MAX_RANK || !norm->ptr || (uintptr_t)norm->ptr % 4) refuse("the norm is one float32 value");
    for (int d = 0; d < norm->rank; d++)
        if (norm->shape[d] != 1) refuse("the norm is one float32 value");
    std::vector<long long> count((size_t)n);
    for (int k = 0; k < n; k++) {
        count[k] = dense_elements(xs[k], k);
        if (count[k] / (kChunkBytes / 4) >= INT32_MAX / kMost) fail(LB_ERR_UNSUPPORTED, format("grad_norm: tensor %d has too many elements", k));
        if (!outs) continue;
        bool same = outs[k].rank == xs[k].rank && outs[k].dtype == xs[k].dtype;
        for (int d = 0; same && d < xs[k].rank; d++) same = outs[k].shape[d] == xs[k].shape[d] && (outs[k].stride[d] == xs[k].stride[d] || xs[k].shape[d] == 1);
        if (count[k] && (!outs[k].ptr || (uintptr_t)outs[k].ptr % dtype_size(xs[k].dtype))) refuse(format("result %d has no memory or is not aligned to its elements", k));
        if (!same) refuse(format("result %d must have its operand's shape, strides and dtype", k));
    }
    if (outs) {  // what is written is written once, and read by nothing else; the norm among it
        for (int k = 0; k < n; k++) {
            const uintptr_t bytes = (uintptr_t)count[k] * dtype_size(xs[k].dtype), at = (uintptr_t)norm->ptr;
            for (const uintptr_t from : {(uintptr_t)xs[k].ptr, (uintptr_t)outs[k].ptr})
                if (bytes && at + 4 > from && at < from + bytes) refuse(format("the norm and %s %d share memory", from == (uintptr_t)xs[k].ptr ? "tensor" : "result", k));
        }
        std::vector<Range> out;
        for (int k = 0; k < n; k++)
            if (count[k]) out.push_back({(uintptr_t)outs[k].ptr, (uintptr_t)outs[k].ptr + (size_t)count[k] * dtype_size(outs[k].dtype), k});
        std::sort(out.begin(), out.end(), [](const Range& a, const Range& b) { return a.from < b.from; });
        for (size_t k = 1; k < out.size(); k++)
            if (out[k].from < out[k - 1].to) refuse(format("results %d and %d share memory", out[k - 1].index, out[k].index));
        for (int k = 0; k < n; k++) {
            if (!count[k] || xs[k].ptr == outs[k].ptr) continue;  // in place: disjoint from the others as its result is
            const uintptr_t from = (uintptr_t)xs[k].ptr, to = from + (size_t)count[k] * dtype_size(xs[k].dtype);
            auto at = std::upper_bound(out.begin(), out.end(), from, [](uintptr_t v, const Range& r) { return v < r.to; });
            if (at != out.end() && at->from < to) refuse(format("tensor %d and result %d share memory", k, at->index));
        }
    }
    const size_t need = scratch_bytes(n);
    if (n && (!scratch || bytes < need || (uintptr_t)scratch % 16)) refuse(format("%zu bytes of scratch are needed, 16-byte aligned", need));
    driver();
    launch_norm(xs, outs, n, count, max_norm, (float*)norm->ptr, (double*)scratch, (cudaStream_t)stream);
}

}  // namespace
}  // namespace lb

extern "C" {

size_t lb_grad_norm_scratch_bytes(int n_tensors) { return n_tensors > 0 ? lb::scratch_bytes(n_tensors) : 0; }

int lb_grad_norm(const lb_tensor* tensors, int n_tensors, const lb_tensor* norm, void* scratch, size_t scratch_bytes, void* stream) {
    return lb::guarded([&] { lb::run_norm(tensors, nullptr, n_tensors, 0.0, norm, scratch, scratch_bytes, stream); });
}

int lb_clip_grad_norm(const lb_tensor* tensors, const lb_tensor* outputs, int n_tensors, double max_norm, const lb_tensor* norm, void* scratch,
                      size_t scratch_bytes, void* stream) {
    return lb::guarded([&] {
        if (!(max_norm >= 0.0) || std::isinf(max_norm)) lb::refuse("max_norm must be finite and not negative");
        if (n_tensors && !outputs) lb::refuse("null argument");
        lb::run_norm(tensors, outputs, n_tensors, max_norm, norm, scratch, scratch_bytes, stream);
    });
}
}
