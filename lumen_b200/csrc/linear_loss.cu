// Softmax cross entropy of a projection to a vocabulary, straight from hidden states x [T, D] and weights W [V, D]: z = x W^T,
// lse_t = log sum_v exp(z_tv), loss_t = lse_t - z_t,target(t); backward with g_t the gradient of loss_t: dz_tv = (exp(z_tv - lse_t) - [v = target(t)]) g_t,
// dx = dz W, dW = dz^T x. Rows that do not count have loss and dz of zero. The logits are never kept: forward, each span of the vocabulary leaves
// its largest logit and the sum of exponentials below it, and what follows joins the spans' pairs; backward, they are computed anew for one piece of
// the vocabulary at a time, whose dz (rounded to the operands' type, as an operand of the tensor cores has to be) is what the two products read.
//
// The work is the products', in whose epilogues the rest is (gemm.cu, gemm_skinny.cu); kernels here prepare rows, join spans, and are the way of layouts and types that the tensor
// cores do not take. Bound by the tensor cores and, with few rows, by the weights' bytes. us, bfloat16: 16384 x 1024 x 32768 forward 697 (1.58 PFLOP/s; 804 under the power
// cap, where a library product of that many FLOPs takes 769), backward 2440 - 2800 there for 3.3 TFLOP of products; 4 tokens of it 12.6 in a graph (67 MB, 5.3 TB/s with both kernels), 61 x 4096 x 131072 180
// (1.07 GB, 6.0 TB/s). Pieces of 256 MB of dz: 64 MB, which would stay in the L2, 2700 us where these take 2460, 128 MB 2470, 512 MB 2320.
#include <algorithm>
#include <cmath>
#include <initializer_list>

#include "convert.cuh"
#include "gemm.h"
#include "launch.cuh"
#include "linear_loss.h"
#include "overlap.h"
#include "pair.cuh"
#include "parts.cuh"

namespace lb {
bool gemm(const lb_tensor& a, const lb_tensor& b, const lb_tensor& d, int epilogue, int kernel_choice, void* stream, void* scratch, size_t scratch_bytes,
          const lb_tensor* aux, const GemmTuning* tuning, SimtProblem* held = nullptr);

namespace {

[[noreturn]] void refuse(const std::string& why) { fail(LB_ERR_INVALID, "linear_cross_entropy: " + why); }

// ---- forward --------------------------------------------------------------------------------------------------------

constexpr int kRowThreads = 128;

// Sums over the threads of a block, to all of them.
__device__ __forceinline__ SpanSum block_join(SpanSum v, SpanSum* held) {
    for (int d = 16; d; d >>= 1) v = join(v, SpanSum{__shfl_xor_sync(0xffffffffu, v.most, d), __shfl_xor_sync(0xffffffffu, v.sum, d)});
    if ((threadIdx.x & 31) == 0) held[threadIdx.x >> 5] = v;
    __syncthreads();
    v = held[0];
    for (int k = 1; k < (int)blockDim.x / 32; k++) v = join(v, held[k]);
    __syncthreads();
    return v;
}

// The span sums of logits that lie in memory, float32 [rows, cols], columns `first` and on of the vocabulary, a span of kSpan columns a block; and the target's
// logit where it is among them.
constexpr int kEach = 16, kSpan = kRowThreads * kEach;
__global__ void __launch_bounds__(kRowThreads) span_kernel(const float* logits, long long ld, long long rows, int first, int cols, Targets targets, SpanSum* spans, float* hit) {
    __shared__ SpanSum held[kRowThreads / 32];
    grid_wait();
    const int from = blockIdx.x * kSpan;
    for (long long row = blockIdx.y; row < rows; row += gridDim.y) {
        const float* z = logits + row * ld;
        float v[kEach], most = -INFINITY;
#pragma unroll
        for (int k = 0; k < kEach; k++) {
            const int c = from + threadIdx.x + k * kRowThreads;
            v[k] = c < cols ? z[c] : -INFINITY, most = fmaxf(most, v[k]);
        }
        const float base = base_of(most);
        float sum = 0.0f;
#pragma unroll
        for (int k = 0; k < kEach; k++) sum += exp2_approx((v[k] - base) * kLog2e);
        const SpanSum all = block_join({most, sum}, held);
        if (threadIdx.x == 0) {
            spans[blockIdx.x * rows + row] = all;
            const int target = targets.of(row) - first;
            if (target >= from && target < min(cols, from + kSpan)) hit[row] = z[target];
        }
    }
}

// Few rows of float32, straight from the weights, which are read once: a warp takes four classes' rows at a time, its lanes a vector of K each, against all tokens (from
// the L1), and the lanes' sums are added at the end. A block's 32 classes are a span; with `logits` those are stored instead. Up to four tokens, and layouts without vectors up to 16.
// Bound by the time that a warp's four vectors take to arrive: weights of 1024 x 32768 1 token 31 us in a graph, 4.3 TB/s; of 200 x 93558 4 tokens 24.
constexpr int kFewWarps = 8, kFewRows = 4, kFewSpan = kFewWarps * kFewRows, kFewTokens = 16;
template <int TOKENS, int VEC>
__global__ void __launch_bounds__(kFewWarps * 32) few_kernel(const float* x, long long ld_x, const float* w, long long ld_w, int T, int D, int V, Targets targets, SpanSum* spans,
                                                             float* hit, float* logits, long long ld) {
    __shared__ float z[TOKENS][kFewSpan];
    grid_wait();
    typedef std::conditional_t<VEC == 4, float4, float> Vec;
    const int warp = threadIdx.x / 32, lane = threadIdx.x & 31, row0 = blockIdx.x * kFewSpan + warp * kFewRows;
    float acc[kFewRows][TOKENS] = {};
    const float* rows[kFewRows];
#pragma unroll
    for (int r = 0; r < kFewRows; r++) rows[r] = w + (long long)min(row0 + r, V - 1) * ld_w;
    for (int k = lane * VEC; k < D; k += 32 * VEC) {
        float a[kFewRows][VEC];
#pragma unroll
        for (int r = 0; r < kFewRows; r++) *(Vec*)a[r] = *(const Vec*)(rows[r] + k);
#pragma unroll
        for (int t = 0; t < TOKENS; t++) {
            float b[VEC];
            *(Vec*)b = *(const Vec*)(x + (long long)min(t, T - 1) * ld_x + k);
#pragma unroll
            for (int r = 0; r < kFewRows; r++)
#pragma unroll
                for (int j = 0; j < VEC; j++) acc[r][t] = fmaf(a[r][j], b[j], acc[r][t]);
        }
    }
    // the lanes' sums: at each step a lane hands the half of the values over that the other one keeps
    float* v = &acc[0][0];
    int first = 0;
    constexpr int ALL = kFewRows * TOKENS;
#pragma unroll
    for (int d = 16, n = ALL; d; d >>= 1) {
        if (n > 1) {
            n /= 2;
            const bool upper = lane & d;
#pragma unroll
            for (int i = 0; i < ALL / 2; i++) {
                if (i >= n) continue;
                const float give = upper ? v[i] : v[i + n], keep = upper ? v[i + n] : v[i];
                v[i] = keep + __shfl_xor_sync(0xffffffffu, give, d);
            }
            if (upper) first += n;
        } else {
            v[0] += __shfl_xor_sync(0xffffffffu, v[0], d);
        }
    }
#pragma unroll
    for (int i = 0; i < (ALL > 32 ? ALL / 32 : 1); i++) z[(first + i) % TOKENS][warp * kFewRows + (first + i) / TOKENS] = v[i];
    __syncthreads();
    const int at = blockIdx.x * kFewSpan + lane;
    for (int t = warp; t < T; t += kFewWarps) {
        const float v = z[t][lane];
        const bool in = at < V;
        if (logits) {
            if (in) logits[t * ld + at] = v;
            continue;
        }
        float most = in ? v : -INFINITY;
#pragma unroll
        for (int d = 16; d; d >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, d));
        const float base = base_of(most);
        float sum = in ? exp2_approx((v - base) * kLog2e) : 0.0f;
#pragma unroll
        for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        if (lane == 0) spans[(long long)blockIdx.x * T + t] = {most, sum};
        if (in && targets.of(t) == at) hit[t] = v;
    }
}

// Rows of 16-bit elements, 16-byte aligned, to where they begin on 128 bytes; a warp a row.
__global__ void __launch_bounds__(256) align_kernel(const uint4* x, long long ld_x, long long rows, int vectors, uint4* out, long long ld_out) {
    grid_wait();
    const int lane = threadIdx.x & 31;
    for (long long row = (long long)blockIdx.x * 8 + threadIdx.x / 32; row < rows; row += (long long)gridDim.x * 8)
#pragma unroll 4
        for (int c = lane; c < vectors; c += 32) out[row * ld_out + c] = x[row * ld_x + c];
}

// What a block of rows adds to the loss.
struct LossSum {
    double sum;
    long long counted;
};
__device__ __forceinline__ LossSum block_sum(LossSum v, LossSum* held) {
    for (int d = 16; d; d >>= 1) v.sum += __shfl_xor_sync(0xffffffffu, v.sum, d), v.counted += __shfl_xor_sync(0xffffffffu, v.counted, d);
    if ((threadIdx.x & 31) == 0) held[threadIdx.x >> 5] = v;
    __syncthreads();
    v = held[0];
    for (int k = 1; k < (int)blockDim.x / 32; k++) v.sum += held[k].sum, v.counted += held[k].counted;
    __syncthreads();
    return v;
}

// Joins the spans of each row ([span][row]), R rows a block and 256 / R threads a row, eight spans of a thread on their way at a time, in an order of their own: the same bits every
// time. With `value` the block is the only one, and leaves the sum or mean itself.
template <int R>
__global__ void __launch_bounds__(256) rows_kernel(const SpanSum* spans, int n_spans, long long rows, const float* hit, Targets targets, float* lse, float* losses, LossSum* sums,
                                                   float* value, bool mean) {
    __shared__ SpanSum held[256];
    __shared__ LossSum total[8];
    grid_wait();
    constexpr int G = 256 / R, AHEAD = 8;
    const int r = threadIdx.x % R, group = threadIdx.x / R;
    const long long row = (long long)blockIdx.x * R + r;
    SpanSum v{-INFINITY, 0.0f};
    if (row < rows)
        for (int k0 = group; k0 < n_spans; k0 += G * AHEAD) {
            SpanSum next[AHEAD];
#pragma unroll
            for (int k = 0; k < AHEAD; k++) next[k] = k0 + k * G < n_spans ? spans[(long long)(k0 + k * G) * rows + row] : SpanSum{-INFINITY, 0.0f};
            float most = v.most;
#pragma unroll
            for (int k = 0; k < AHEAD; k++) most = fmaxf(most, next[k].most);
            const float base = base_of(most);
            float sum = v.sum * exp2_approx((v.most - base) * kLog2e);
#pragma unroll
            for (int k = 0; k < AHEAD; k++) sum += next[k].sum * exp2_approx((next[k].most - base) * kLog2e);
            v = {most, sum};
        }
    held[threadIdx.x] = v;
    for (int half = G / 2; half; half /= 2) {
        __syncthreads();
        if (group < half) held[threadIdx.x] = join(held[threadIdx.x], held[threadIdx.x + half * R]);
    }
    LossSum mine{0.0, 0};
    if (group == 0 && row < rows) {
        v = held[threadIdx.x];
        const float all = v.most + logf(v.sum);
        lse[row] = all;
        const bool counts = targets.of(row) >= 0;
        const float loss = counts ? all - hit[row] : 0.0f;
        if (losses) losses[row] = loss;
        mine = {loss, counts};
    }
    if (!sums && !value) return;
    mine = block_sum(mine, total);
    if (threadIdx.x) return;
    if (value) *value = (float)(mean ? mine.sum / (double)max(mine.counted, 1LL) : mine.sum);
    else sums[blockIdx.x] = mine;
}
__global__ void __launch_bounds__(256) loss_kernel(const LossSum* sums, long long n, bool mean, float* loss) {
    __shared__ LossSum total[8];
    grid_wait();
    LossSum v{0.0, 0};
    for (long long k = threadIdx.x; k < n; k += 256) v.sum += sums[k].sum, v.counted += sums[k].counted;
    v = block_sum(v, total);
    if (threadIdx.x == 0) *loss = (float)(mean ? v.sum / (double)max(v.counted, 1LL) : v.sum);
}

// ---- backward -------------------------------------------------------------------------------------------------------

// Rows that count, and the largest |d_loss| of them.
struct RowCount {
    long long counted;
    float most;
};
__device__ __forceinline__ RowCount block_count(RowCount v, RowCount* held) {
    for (int d = 16; d; d >>= 1) v.counted += __shfl_xor_sync(0xffffffffu, v.counted, d), v.most = fmaxf(v.most, __shfl_xor_sync(0xffffffffu, v.most, d));
    if ((threadIdx.x & 31) == 0) held[threadIdx.x >> 5] = v;
    __syncthreads();
    v = held[0];
    for (int k = 1; k < (int)blockDim.x / 32; k++) v.counted += held[k].counted, v.most = fmaxf(v.most, held[k].most);
    __syncthreads();
    return v;
}
struct LossGrad {
    const float* at;  // null: one
    long long step;
    __device__ __forceinline__ float of(long long row) const { return at ? at[row * step] : 1.0f; }
};
__global__ void __launch_bounds__(256) count_kernel(Targets targets, LossGrad grad, long long rows, RowCount* counts) {
    __shared__ RowCount held[8];
    grid_wait();
    RowCount v{0, 0.0f};
    for (long long row = (long long)blockIdx.x * 256 + threadIdx.x; row < rows; row += (long long)gridDim.x * 256)
        if (targets.of(row) >= 0) v.counted++, v.most = fmaxf(v.most, fabsf(grad.of(row)));
    v = block_count(v, held);
    if (threadIdx.x == 0) counts[blockIdx.x] = v;
}

// Of each row: the gradient of its logits' scale g (zero where it does not count), its class, and a copy of x whose rows that do not count are zero, so that
// what stands there (padding may hold infinities or NaN) does not get into dW. 16 bits: g in units of the largest, so that of equal ones, as a mean's are, no rounding of dz is all rows' own,
// times 2^13 for float16, since most of dz is far below its smallest values; `undo` is what takes both away again. REST: as many rows of x again, for what dz's rounding leaves.
template <class T, bool REST>
__global__ void __launch_bounds__(256) row_grads_kernel(Targets targets, LossGrad grad, long long rows, const RowCount* counts, int n_counts, bool mean, const T* x, long long ld_x,
                                                        long long x_col, int D, T* x_out, long long ld_out, float* g, int* classes, float* undo) {
    __shared__ RowCount held[8];
    grid_wait();
    RowCount all{0, 0.0f};
    if (counts) {
        for (int k = threadIdx.x; k < n_counts; k += 256) all.counted += counts[k].counted, all.most = fmaxf(all.most, counts[k].most);
    } else {
        for (long long row = threadIdx.x; row < rows; row += 256)
            if (targets.of(row) >= 0) all.counted++, all.most = fmaxf(all.most, fabsf(grad.of(row)));
    }
    all = block_count(all, held);
    const float counted = mean ? (float)max(all.counted, 1LL) : 1.0f;
    const float top = std::is_same_v<T, __half> ? 8192.0f : 1.0f;
    const bool scaled = undo && all.most > 0.0f && all.most < INFINITY;
    if (undo && blockIdx.x == 0 && threadIdx.x == 0) *undo = scaled ? all.most / counted / top : 1.0f;
    constexpr int V = 16 / sizeof(T);
    const bool vectors = x_col == 1 && D % V == 0 && ld_x % V == 0 && (uintptr_t)x % 16 == 0;
    const int lane = threadIdx.x & 31;
    for (long long row = (long long)blockIdx.x * 8 + threadIdx.x / 32; row < rows; row += (long long)gridDim.x * 8) {  // a warp a row
        const int target = targets.of(row);
        if (lane == 0) g[row] = target < 0 ? 0.0f : scaled ? grad.of(row) / all.most * top : grad.of(row) / counted, classes[row] = target;
        const T* from = x + row * ld_x;
        T* to = x_out + row * ld_out;
        if (vectors) {
#pragma unroll 4
            for (int c = lane; c < D / V; c += 32) {
                const uint4 v = target < 0 ? make_uint4(0u, 0u, 0u, 0u) : ((const uint4*)from)[c];
                ((uint4*)to)[c] = v;
                if (REST) ((uint4*)(to + rows * ld_out))[c] = v;
            }
        } else {
            for (int c = lane; c < D; c += 32) {
                const T v = target < 0 ? from_float<T>(0.0f) : from[c * x_col];
                to[c] = v;
                if (REST) to[rows * ld_out + c] = v;
            }
        }
    }
}

// float32 values in three parts of bfloat16, [rows][3][part] with zeros behind the columns. Rows of class -1 are zero.
__global__ void __launch_bounds__(256) parts_kernel(const float* from, long long row_step, long long col_step, long long rows, int cols, int part, const int* classes,
                                                    __nv_bfloat16* to) {
    grid_wait();
    const bool vectors = col_step == 1 && row_step % 4 == 0 && cols % 4 == 0 && (uintptr_t)from % 16 == 0;
    for (long long row = blockIdx.y; row < rows; row += gridDim.y) {
        const bool there = !classes || classes[row] >= 0;
        const float* x = from + row * row_step;
        __nv_bfloat16* out = to + row * 3 * part;
        for (int c = (blockIdx.x * 256 + threadIdx.x) * 4; c < part; c += gridDim.x * 1024) {
            float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            if (there && c < cols) {
                if (vectors) {
                    const float4 w = *(const float4*)(x + c);
                    v[0] = w.x, v[1] = w.y, v[2] = w.z, v[3] = w.w;
                } else {
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        if (c + j < cols) v[j] = x[(c + j) * col_step];
                }
            }
            uint32_t parts[3][2];
            parts_of<true>(v, parts);
#pragma unroll
            for (int k = 0; k < 3; k++) *(uint2*)(out + (long long)k * part + c) = make_uint2(parts[k][0], parts[k][1]);
        }
    }
}

// dz of logits that lie in memory; may take their place. `rests`: what its rounding leaves, rounded, as many rows below.
template <class T>
__global__ void __launch_bounds__(kRowThreads) slope_kernel(const float* logits, long long ld, long long rows, int first, int cols, const float* lse, long long lse_step,
                                                            const float* g, const int* classes, T* out, long long ld_out, bool rests) {
    grid_wait();
    for (long long row = blockIdx.y; row < rows; row += gridDim.y) {
        const float all = lse[row * lse_step], scale = g[row];
        const int at = classes[row], target = at - first;
        for (int c = blockIdx.x * kRowThreads + threadIdx.x; c < cols; c += gridDim.x * kRowThreads) {
            const float d = at < 0 ? 0.0f : (expf(logits[row * ld + c] - all) - (c == target ? 1.0f : 0.0f)) * scale;
            const T rounded = from_float<T>(d);
            out[row * ld_out + c] = rounded;
            if (rests) {
                const float rest = d - to_float(rounded);
                out[(rows + row) * ld_out + c] = from_float<T>(fabsf(rest) < INFINITY ? rest : 0.0f);  // (infinity and NaN leave nothing)
            }
        }
    }
}

// sum = (first piece: 0, else sum) + product, which is `ranges` sums to add up in their order; the last piece's is rounded into `out` instead, times `undo` where there is one.
template <class T>
__global__ void __launch_bounds__(256) fold_kernel(const float* product, int ranges, long long rows, int D, float* sum, bool begins, T* out, long long ld_out, const float* undo) {
    grid_wait();
    const float scale = undo ? *undo : 1.0f;
    for (long long row = blockIdx.y; row < rows; row += gridDim.y)
        for (int c = blockIdx.x * 256 + threadIdx.x; c < D; c += gridDim.x * 256) {
            const long long i = row * D + c;
            float v = begins ? 0.0f : sum[i];
#pragma unroll 4
            for (int k = 0; k < ranges; k++) v += product[(long long)k * rows * D + i];
            if (out) out[row * ld_out + c] = from_float<T>(v * scale);
            else sum[i] = v;
        }
}

// Both gradients of a few rows in one pass over the weights: a thread has four columns of x and of dx's sums in registers, for every class it reads the weights' four, which the class's dz takes
// to dx, and writes dW's. A block's range of classes is a part of dx, to be added up. `rests`: dz's second parts are T rows below. Bound by the loads' way and, with more tokens, by the products. A
// backward pass in a graph, products by themselves -> this, us: float32 4 tokens of 1024 x 32768 197 -> 89 (the floor of one reading and one writing of the weights 41), 16 of it 241 -> 121, of
// 344 x 116036 504 -> 178; bfloat16, whose tensor cores take more tokens for the same time, 4 of 1024 x 32768 66 -> 58, but 5 67 -> 71.
constexpr int kGradThreads = 128, kGradClasses = 64;
constexpr int grad_tokens(int item) { return item == 4 ? 16 : 4; }
constexpr int grad_blocks(int tokens) { return tokens == 16 ? 3 : 4; }  // on an SM
template <class E>
__device__ __forceinline__ void load4(const E* at, Pair* v) {
    if constexpr (sizeof(E) == 4) {
        const float4 f = *(const float4*)at;
        v[0] = both(f.x, f.y), v[1] = both(f.z, f.w);
    } else {
        const uint2 raw = *(const uint2*)at;
        const E* e = (const E*)&raw;
        v[0] = both(to_float(e[0]), to_float(e[1])), v[1] = both(to_float(e[2]), to_float(e[3]));
    }
}
template <class E, int TOKENS>
__global__ void __launch_bounds__(kGradThreads, grad_blocks(TOKENS)) few_grads_kernel(const E* x, long long ld_x, const E* w, long long ld_w, const E* dz, long long ld, bool rests, int T, int D,
                                                                                      int classes, int each, E* dw, long long ld_dw, float* dx, const float* undo) {
    __shared__ float4 z4[kGradClasses][TOKENS / 4];
    constexpr int AHEAD = TOKENS <= 8 ? 8 : 4;
    grid_wait();
    const int c = (blockIdx.x * kGradThreads + threadIdx.x) * 4, first = blockIdx.y * each, last = min(classes, first + each);
    const bool in = c < D;
    const float scale = undo ? *undo : 1.0f;
    Pair xs[TOKENS][2], sums[TOKENS][2];
#pragma unroll
    for (int t = 0; t < TOKENS; t++) {
        xs[t][0] = xs[t][1] = sums[t][0] = sums[t][1] = both(0.0f, 0.0f);
        if (in && t < T) load4(x + t * ld_x + c, xs[t]);
    }
    for (int v0 = first; v0 < last; v0 += kGradClasses) {
        const int n = min(kGradClasses, last - v0);
        __syncthreads();
        for (int i = threadIdx.x; i < kGradClasses * TOKENS; i += kGradThreads) {
            const int v = i % kGradClasses, t = i / kGradClasses;
            float d = 0.0f;
            if (t < T && v < n) {
                d = to_float(dz[t * ld + v0 + v]);
                if (rests) d += to_float(dz[(T + t) * ld + v0 + v]);
            }
            ((float*)z4[v])[t] = d;
        }
        __syncthreads();
        if (!in) continue;
        const E* from = w + (long long)v0 * ld_w + c;
        E* to = dw + (long long)v0 * ld_dw + c;
        for (int v1 = 0; v1 < n; v1 += AHEAD) {
            Pair ws[AHEAD][2];
#pragma unroll
            for (int u = 0; u < AHEAD; u++) load4(from + (long long)min(v1 + u, n - 1) * ld_w, ws[u]);
#pragma unroll
            for (int u = 0; u < AHEAD; u++) {
                if (v1 + u >= n) break;
                Pair d[2] = {both(0.0f, 0.0f), both(0.0f, 0.0f)};
#pragma unroll
                for (int q = 0; q < TOKENS / 4; q++) {
                    const float4 z = z4[v1 + u][q];
                    const float zs[4] = {z.x, z.y, z.z, z.w};
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const Pair zz = both(zs[j], zs[j]);
                        const int t = 4 * q + j;
                        d[0] = fma2(xs[t][0], zz, d[0]), d[1] = fma2(xs[t][1], zz, d[1]);
                        sums[t][0] = fma2(ws[u][0], zz, sums[t][0]), sums[t][1] = fma2(ws[u][1], zz, sums[t][1]);
                    }
                }
                const float2 lo = apart(d[0]), hi = apart(d[1]);
                E* row = to + (long long)(v1 + u) * ld_dw;
                if constexpr (sizeof(E) == 4) {
                    *(float4*)row = make_float4(lo.x, lo.y, hi.x, hi.y);
                } else {
                    const E e[4] = {from_float<E>(lo.x * scale), from_float<E>(lo.y * scale), from_float<E>(hi.x * scale), from_float<E>(hi.y * scale)};
                    uint2 raw;
                    memcpy(&raw, e, 8);
                    *(uint2*)row = raw;
                }
            }
        }
    }
    if (!in) return;
#pragma unroll
    for (int t = 0; t < TOKENS; t++) {
        const float2 lo = apart(sums[t][0]), hi = apart(sums[t][1]);
        if (t < T) *(float4*)(dx + ((long long)blockIdx.y * T + t) * D + c) = make_float4(lo.x, lo.y, hi.x, hi.y);
    }
}

// fold_kernel for many sums: eight threads take every eighth of a value's.
template <class T>
__global__ void __launch_bounds__(256) fold_many_kernel(const float* product, int ranges, long long rows, int D, float* sum, bool begins, T* out, long long ld_out, const float* undo) {
    __shared__ float held[8][32];
    grid_wait();
    const float scale = undo ? *undo : 1.0f;
    const int group = threadIdx.x / 32, lane = threadIdx.x & 31, c = blockIdx.x * 32 + lane;
    for (long long row = blockIdx.y; row < rows; row += gridDim.y) {
        const long long i = row * D + c;
        float v = 0.0f;
        if (c < D) {
#pragma unroll 8
            for (int k = group; k < ranges; k += 8) v += product[(long long)k * rows * D + i];
        }
        __syncthreads();
        held[group][lane] = v;
        __syncthreads();
        if (group || c >= D) continue;
        v = begins ? 0.0f : sum[i];
#pragma unroll
        for (int k = 0; k < 8; k++) v += held[k][lane];
        if (out) out[row * ld_out + c] = from_float<T>(v * scale);
        else sum[i] = v;
    }
}

// ---- host side ------------------------------------------------------------------------------------------------------

lb_tensor matrix(void* ptr, int dtype, long long rows, long long cols, long long ld) {
    lb_tensor t{};
    t.ptr = ptr, t.dtype = dtype, t.rank = 2, t.shape[0] = rows, t.shape[1] = cols, t.stride[0] = ld, t.stride[1] = 1;
    return t;
}
lb_tensor transposed(const lb_tensor& t) {
    lb_tensor u = t;
    std::swap(u.shape[0], u.shape[1]), std::swap(u.stride[0], u.stride[1]);
    return u;
}
// The dimensions of a tensor but the last `keep` as one, which have to be evenly spaced: [rows, last] or [rows].
lb_tensor as_rows(const lb_tensor* t, int keep, const char* what) {
    if (!t) refuse(format("%s is missing", what));
    if (t->rank < keep || t->rank > LB_MAX_RANK) refuse(format("%s must have rank %d or more", what, keep));
    for (int d = 0; d < t->rank; d++)
        if (t->shape[d] < 0) refuse(format("%s has a negative size", what));
    const int lead = t->rank - keep;
    long long rows = 1, step = 0;
    for (int d = 0; d < lead; d++)
        if (t->shape[d] == 0) rows = 0;  // no rows: nothing about their spacing
    for (int d = lead - 1; d >= 0 && rows; d--) {
        if (t->shape[d] == 1) continue;
        if (rows != 1 && t->stride[d] != step * rows) fail(LB_ERR_UNSUPPORTED, format("linear_cross_entropy: the rows of %s are not evenly spaced", what));
        if (rows == 1) step = t->stride[d];
        rows *= t->shape[d];
    }
    lb_tensor m{};
    m.ptr = t->ptr, m.dtype = t->dtype, m.rank = 1 + keep, m.shape[0] = rows, m.stride[0] = step;
    if (keep) {
        m.shape[1] = t->shape[lead], m.stride[1] = t->stride[lead];
        if (rows <= 1) m.stride[0] = m.stride[1] == 1 ? m.shape[1] : 1;
    }
    return m;
}
void in_memory(const lb_tensor& t, const char* what) {
    long long n = 1;
    for (int d = 0; d < t.rank; d++) n *= t.shape[d];
    if (n && (!t.ptr || (uintptr_t)t.ptr % dtype_size(t.dtype))) refuse(format("%s has no memory or is not aligned to its elements", what));
}
void written(const lb_tensor& t, const char* what) {
    if (t.shape[1] > 1 && t.stride[1] != 1) fail(LB_ERR_UNSUPPORTED, format("linear_cross_entropy: %s must be row-major", what));
    if (t.shape[0] > 1 && t.stride[0] < t.shape[1]) refuse(format("the rows of %s overlap", what));
}
// What is written shares no memory with what is read, or written.
void keep_apart(std::initializer_list<const lb_tensor*> results, std::initializer_list<const lb_tensor*> operands) {
    for (auto out = results.begin(); out != results.end(); ++out) {
        for (const lb_tensor* o : operands)
            if (share_memory(**out, *o)) refuse("a result shares memory with an operand");
        for (auto other = results.begin(); other != out; ++other)
            if (share_memory(**out, **other)) refuse("two results share memory");
    }
}

size_t up(size_t bytes) { return (bytes + 255) / 256 * 256; }
long long up(long long n, long long to) { return (n + to - 1) / to * to; }

constexpr long long kPieceBytes = 256LL << 20;  // of a piece's logits or their gradients

struct Loss {
    int reduction, dtype;
    long long T, D, V;
    lb_tensor x, w, t;
    Targets targets;
    char* scratch = nullptr;
    size_t held = 0;  // bytes of scratch given out

    Loss(const lb_loss_desc* desc, const lb_tensor* x_t, const lb_tensor* w_t, const lb_tensor* targets_t) {
        if (!desc) refuse("null argument");
        reduction = desc->reduction;
        if (reduction < LB_REDUCTION_NONE || reduction > LB_REDUCTION_MEAN) refuse("unknown reduction");
        x = as_rows(x_t, 1, "x");
        if (!w_t || w_t->rank != 2) refuse("the weights must be [classes, width]");
        w = as_rows(w_t, 1, "weight"), t = as_rows(targets_t, 0, "targets");
        dtype = x.dtype;
        if (dtype != LB_F32 && dtype != LB_BF16 && dtype != LB_F16) refuse("float16, bfloat16 or float32 operands");
        T = x.shape[0], D = x.shape[1], V = w.shape[0];
        if (w.dtype != dtype || w.shape[1] != D) refuse(format("weight must be [classes, %lld] of x's dtype, got %s[%lld, %lld]", D, dtype_name(w.dtype), V, (long long)w.shape[1]));
        if (targets_t->rank != x_t->rank - 1) refuse("targets must have the shape of x without its last dimension");
        for (int d = 0; d < targets_t->rank; d++)
            if (targets_t->shape[d] != x_t->shape[d]) refuse("targets must have the shape of x without its last dimension");
        if (t.dtype != LB_I32 && t.dtype != LB_I64) refuse("targets must be int32 or int64");
        if (D < 1 || V < 1) refuse("a width or vocabulary of zero");
        if (T > INT32_MAX || D > INT32_MAX || V > INT32_MAX) fail(LB_ERR_UNSUPPORTED, "linear_cross_entropy: sizes of at most 2^31 - 1");
        in_memory(x, "x"), in_memory(w, "weight"), in_memory(t, "targets");
        targets = {t.ptr, t.stride[0], desc->ignore_index, t.dtype == LB_I64, (int)V};
    }
    template <class U>
    U* take(size_t count) {  // memory of the call's scratch; counted alone where there is none
        U* at = (U*)(scratch + held);
        held += up(count * sizeof(U));
        return scratch ? at : nullptr;
    }
    // A row value of each row: float32, [rows] in any even spacing.
    lb_tensor row_values(const lb_tensor* v, const lb_tensor* like, const char* what) const {
        lb_tensor r = as_rows(v, 0, what);
        if (r.dtype != LB_F32 || v->rank != like->rank) refuse(format("%s must be float32 of the targets' shape", what));
        for (int d = 0; d < v->rank; d++)
            if (v->shape[d] != like->shape[d]) refuse(format("%s must be float32 of the targets' shape", what));
        in_memory(r, what);
        return r;
    }
    // Whether float32 operands go to the tensor cores in parts of 16 bits: from 3e7 products on. Six products of parts take less than one of float32 on the CUDA cores; making the
    // parts moves ten bytes an element of the weights, and each product fetches the part that it takes, which are twelve more, from memory where K is long (1024 and more: a pass over K of the
    // tiles under way does not stay in the L2). us of the loss and of both gradients in a graph, CUDA cores -> parts: 64 x 2048 x 32768 392 -> 298 and 1248 -> 529; 300 x 64 x 5000
    // 20.6 -> 18.6 and 59.7 -> 53.6; 1000 x 128 x 2000 36 -> 19 and 107 -> 53; 2000 x 1024 x 8000 1300 -> 156 and 4055 -> 493. Where the loss does not gain by it: 33 x 344 x 116035 248 -> 236
    // (both eager, gradients 763 -> 445), 64 x 3296 x 84985 1382 -> 1460 (5450 -> 2510), which elementary operations do in 790 (100 rows of it 2735 -> 1484, those 1441). Up to 32 rows' losses,
    // and the logits of 16 rows' gradients, come straight from the weights.
    bool in_parts() const { return dtype == LB_F32 && T > kFewTokens && (double)T * (double)V * (double)D >= 3e7; }
    // The vocabulary in pieces whose [width, piece] of `item` bytes an element takes about kPieceBytes.
    long long piece_of(int item, long long width) const {
        const long long most = std::max(256LL, kPieceBytes / item / std::max(1LL, width) / 256 * 256);
        return std::min(V, most);
    }
};

size_t product_scratch(const lb_tensor& a, const lb_tensor& b) { return lb_gemm_operands_scratch_bytes(&a, &b); }
lb_tensor rows_of(const lb_tensor& m, long long first, long long count) {
    lb_tensor r = m;
    r.ptr = (char*)m.ptr + first * m.stride[0] * dtype_size(m.dtype), r.shape[0] = count;
    return r;
}
// Rows that a float32 result of the tensor-core kernels is stored to in vectors.
bool in_vectors(const lb_tensor& t) { return (uintptr_t)t.ptr % 16 == 0 && t.stride[1] == 1 && (t.shape[0] <= 1 || (t.stride[0] % 8 == 0 && t.stride[0] >= t.shape[1])); }
// float32 values in parts, as a tensor of the first of them.
lb_tensor parted(void* ptr, long long rows, long long cols, long long part) { return matrix(ptr, LB_BF16, rows, cols, 3 * part); }
void split(const lb_tensor& t, const int* classes, const lb_tensor& to, cudaStream_t s);

template <class F>
void by_type(int dtype, F f) {
    if (dtype == LB_F32) f((float*)nullptr);
    else if (dtype == LB_BF16) f((__nv_bfloat16*)nullptr);
    else f((__half*)nullptr);
}
// A grid of rows by columns (`across` a block): whole columns first, rows in turn beyond 16 blocks an SM.
dim3 by_rows(long long rows, long long cols, int across) {
    const long long x = std::max(1LL, (cols + across - 1) / across);
    return dim3((unsigned)x, (unsigned)std::min<long long>(std::max(1LL, rows), std::max(1LL, sm_count_hint() * 16 / x)));
}
unsigned row_blocks(long long rows) { return (unsigned)std::min<long long>(std::max(1LL, rows), (long long)sm_count_hint() * 16); }

void split(const lb_tensor& t, const int* classes, const lb_tensor& to, cudaStream_t s) {
    const long long part = to.stride[0] / 3;
    launch_overlapped(parts_kernel, by_rows(t.shape[0], part, 1024), dim3(256), 0, s, 0, (const float*)t.ptr, (long long)t.stride[0], (long long)t.stride[1], (long long)t.shape[0],
                      (int)t.shape[1], (int)part, classes, (__nv_bfloat16*)to.ptr);
}

// Whether few_kernel takes the products of x and w; the vectors that both can be read in.
bool few_float32(const lb_tensor& x, const lb_tensor& w) { return x.dtype == LB_F32 && x.shape[0] <= kFewTokens && x.stride[1] == 1 && w.stride[1] == 1; }
void run_few(const lb_tensor& x, const lb_tensor& w, const Targets& targets, SpanSum* spans, float* hit, float* logits, long long ld, cudaStream_t s) {
    auto vectors = [](const lb_tensor& t) { return (uintptr_t)t.ptr % 16 == 0 && (t.shape[0] <= 1 || t.stride[0] % 4 == 0); };
    const int T = (int)x.shape[0], D = (int)x.shape[1], V = (int)w.shape[0];
    const bool vec = D % 4 == 0 && vectors(x) && vectors(w);
    auto go = [&](auto kernel) {
        launch_overlapped(kernel, dim3((unsigned)((V + kFewSpan - 1) / kFewSpan)), dim3(kFewWarps * 32), 0, s, 0, (const float*)x.ptr, (long long)x.stride[0], (const float*)w.ptr,
                          (long long)w.stride[0], T, D, V, targets, spans, hit, logits, ld);
    };
    if (T <= 4) vec ? go(few_kernel<4, 4>) : go(few_kernel<4, 1>);
    else T <= 8 ? go(few_kernel<8, 1>) : go(few_kernel<16, 1>);  // (those of whole vectors are skinny_float_loss's)
}

struct Forward : Loss {
    using Loss::Loss;
    lb_tensor loss, lse;

    void results(const lb_tensor* loss_t, const lb_tensor* lse_t, const lb_tensor* targets_t) {
        lse = row_values(lse_t, targets_t, "lse");
        if (T > 1 && lse.stride[0] != 1) refuse("lse must be dense");
        if (reduction == LB_REDUCTION_NONE) {
            loss = row_values(loss_t, targets_t, "loss");
            if (T > 1 && loss.stride[0] != 1) refuse("loss must be dense");
            return;
        }
        loss = as_rows(loss_t, 0, "loss");
        if (loss.dtype != LB_F32 || loss.shape[0] != 1) refuse("the loss is one float32 value");
        in_memory(loss, "loss");
    }
    void run(cudaStream_t s, bool only_count) {
        held = 0;
        const bool few16 = T && skinny_takes(x, w), float_tiles = T && skinny_float_takes(x, w), few32 = T && !float_tiles && few_float32(x, w), few = few16 || few32 || float_tiles, parts = !few && in_parts(), fused = few || (T && gemm_loss_takes(x, w));
        // some rows at a time, whose spans (or copies) stay small whatever the number of rows
        const long long part = up(D, 64), at_once = few ? T : std::min(T, fused ? std::max(4096LL, kPieceBytes / 8 / gemm_spans(V) / 1024 * 1024) : 65536LL);
        const long long piece = parts ? piece_of(6, std::max(at_once, part)) : piece_of(4, at_once), pieces = (V + piece - 1) / piece, last = V - (pieces - 1) * piece;
        auto spans_of = [&](long long cols) { return parts ? (long long)gemm_spans(cols) : (cols + kSpan - 1) / kSpan; };
        const long long n_spans = float_tiles ? skinny_float_spans(T, V) : few32 ? (V + kFewSpan - 1) / kFewSpan : few ? skinny_spans(V) : fused ? gemm_spans(V) : (pieces - 1) * spans_of(piece) + spans_of(last);
        // rows of a block: enough for every SM, or all of a few, whose sum is then theirs
        const int R = T >= 32LL * sm_count_hint() ? 32 : T >= 512 || (T <= 8 && reduction != LB_REDUCTION_NONE) ? 8 : 1;
        const long long blocks = (at_once + R - 1) / R, rounds = T ? (T + at_once - 1) / at_once : 0, all_blocks = rounds ? (rounds - 1) * blocks + (T - (rounds - 1) * at_once + R - 1) / R : 0;
        // Rows that begin within a sector, of both operands, slow the product down (8192 x 840 x 20000 279 us, 208 where they do in one of them only; 2600 x 840 x 10007 46.8 and 38.6): then x
        // is copied first, which with the copy takes 215 us and 40.8; 500 x 840 x 20000 takes 36.5 instead of 44.0.
        auto within = [](const lb_tensor& t) { return t.stride[0] % 16 != 0; };
        const bool aligns = fused && !few && at_once > 128 && D % 8 == 0 && x.stride[1] == 1 && w.stride[1] == 1 && within(x) && within(w);
        char* x_copy = take<char>(aligns ? at_once * part * 2 : 0);
        SpanSum* spans = take<SpanSum>(n_spans * at_once);
        float* hit = take<float>(at_once);
        const bool alone = all_blocks == 1, mean = reduction == LB_REDUCTION_MEAN;
        LossSum* sums = reduction == LB_REDUCTION_NONE || alone ? nullptr : take<LossSum>(all_blocks);
        const long long ld = up(piece, 8);
        float* logits = take<float>(fused || parts ? 0 : at_once * ld);
        char *x_parts = take<char>(parts ? at_once * 6 * part : 0), *w_parts = take<char>(parts ? piece * 6 * part : 0);
        const size_t more = T && !fused && !parts ? product_scratch(rows_of(x, 0, at_once), transposed(rows_of(w, 0, piece))) : 0;
        void* product = take<char>(more);
        if (only_count) return;
        for (long long round = 0; round < rounds; round++) {
            const long long t0 = round * at_once, n = std::min(at_once, T - t0);
            const lb_tensor rows = rows_of(x, t0, n), copies = parted(x_parts, n, D, part);
            Targets classes = targets;
            classes.at = (const char*)targets.at + t0 * targets.step * (targets.wide ? 8 : 4);
            if (float_tiles) skinny_float_loss(rows, w, classes, spans, hit, nullptr, 0, s);
            else if (few32) run_few(rows, w, classes, spans, hit, nullptr, 0, s);
            else if (few16) skinny_loss(rows, w, classes, spans, hit, s);
            else if (fused) {
                lb_tensor operand = rows;
                if (aligns) {
                    operand.ptr = x_copy, operand.stride[0] = part;
                    launch_overlapped(align_kernel, dim3(row_blocks((n + 7) / 8)), dim3(256), 0, s, 0, (const uint4*)rows.ptr, (long long)x.stride[0] / 8, n, (int)(D / 8), (uint4*)x_copy, part / 8);
                }
                gemm_loss(operand, w, classes, 0, spans, hit, s);
            }
            if (parts) split(rows, nullptr, copies, s);
            for (long long k = 0; k < pieces && !fused; k++) {
                const long long first = k * piece, cols = std::min(piece, V - first);
                SpanSum* to = spans + k * spans_of(piece) * n;
                if (parts) {
                    const lb_tensor weights = parted(w_parts, cols, D, part);
                    if (pieces > 1 || round == 0) split(rows_of(w, first, cols), nullptr, weights, s);
                    gemm_loss(copies, weights, classes, (int)first, to, hit, s, {part, part});
                } else {
                    gemm(rows, transposed(rows_of(w, first, cols)), matrix(logits, LB_F32, n, cols, ld), EPI_NONE, 0, s, product, more, nullptr, nullptr);
                    launch_overlapped(span_kernel, by_rows(n, cols, kSpan), dim3(kRowThreads), 0, s, 0, (const float*)logits, ld, n, (int)first, (int)cols, classes, to, hit);
                }
            }
            auto join_rows = [&](auto kernel) {
                launch_overlapped(kernel, dim3((unsigned)((n + R - 1) / R)), dim3(256), 0, s, 0, (const SpanSum*)spans, (int)n_spans, n, (const float*)hit, classes, (float*)lse.ptr + t0,
                                  reduction == LB_REDUCTION_NONE ? (float*)loss.ptr + t0 : nullptr, sums ? sums + round * blocks : nullptr,
                                  reduction != LB_REDUCTION_NONE && alone ? (float*)loss.ptr : nullptr, mean);
            };
            R == 32 ? join_rows(rows_kernel<32>) : R == 8 ? join_rows(rows_kernel<8>) : join_rows(rows_kernel<1>);
        }
        if (reduction != LB_REDUCTION_NONE && !alone) launch_overlapped(loss_kernel, dim3(1), dim3(256), 0, s, 0, (const LossSum*)sums, all_blocks, mean, (float*)loss.ptr);
    }
};

struct Backward : Loss {
    using Loss::Loss;
    lb_tensor grad{}, lse, dx, dw;

    // Ranges of K, the vocabulary, that d_x of up to 128 rows of 16 bits is cut into on the one-CTA tiles: an SM each, from 384 blocks of K on and where there are more than 16
    // (the eight that lb_gemm's narrow tiles are cut into at most would walk 48 blocks and more). 0: lb_gemm's own choice. us of the backward pass in a graph, that -> these:
    //   16 x 1024 x 32768 72.7 -> 61.2, 33 of it 75.1 -> 62.8, 128 of it 76.0 -> 66.2
    //   not taken: 5 x 496 x 18250 38 -> 40, 16 x 512 x 8000 24.3 -> 26.3, 128 x 4096 x 32768 (nine ranges) 179 -> 182
    int few_ranges(long long K) const {
        const long long blocks = (K + 63) / 64, tiles = (D + 255) / 256, ranges = sm_count_hint() / tiles;
        return dtype == LB_F32 || T > 128 || blocks < 384 || ranges <= 16 ? 0 : (int)std::min(ranges, blocks / 8);
    }
    // Ranges of a long K that d_x is cut into on the CUDA cores, where a sum is one chain: until every SM has four of the blocks of 128 threads that a product of so few rows has.
    int core_ranges(long long K) const {
        const long long tiles = (T + 15) / 16 * ((D + 31) / 32);
        return (int)std::max(1LL, std::min({4LL * sm_count_hint() / tiles, K / 256, 64LL}));
    }

    long long few_grad_slots() const { return (long long)sm_count_hint() * grad_blocks(T <= 8 ? 8 : 16); }

    void results(const lb_tensor* dx_t, const lb_tensor* dw_t) {
        dx = as_rows(dx_t, 1, "d_x"), dw = as_rows(dw_t, 1, "d_weight");
        if (dx.dtype != dtype || dx.shape[0] != T || dx.shape[1] != D) refuse("d_x must have the shape and dtype of x");
        if (dw.dtype != dtype || dw_t->rank != 2 || dw.shape[0] != V || dw.shape[1] != D) refuse("d_weight must have the shape and dtype of the weights");
        in_memory(dx, "d_x"), in_memory(dw, "d_weight"), written(dx, "d_x"), written(dw, "d_weight");
    }
    void operands(const lb_tensor* grad_t, const lb_tensor* lse_t, const lb_tensor* targets_t) {
        lse = row_values(lse_t, targets_t, "lse");
        if (!grad_t) return;
        if (reduction == LB_REDUCTION_NONE) {
            grad = row_values(grad_t, targets_t, "d_loss");
            return;
        }
        grad = as_rows(grad_t, 0, "d_loss");
        if (grad.dtype != LB_F32 || grad.shape[0] != 1) refuse("the gradient of the loss is one float32 value");
        grad.stride[0] = 0;
        in_memory(grad, "d_loss");
    }
    void run(cudaStream_t s, bool only_count) {
        held = 0;
        const int item = dtype_size(dtype);
        if (T == 0) {  // no scratch
            if (!only_count) LB_CUDA(cudaMemset2DAsync(dw.ptr, (size_t)(V > 1 ? dw.stride[0] : D) * item, 0, (size_t)D * item, (size_t)V, s));
            return;
        }
        const bool scaled = item == 2;  // `undo` is what the products' results are to be multiplied by
        // dz of few rows is held in two parts, the second what the rounding of the first leaves, as rows of their own (of x too): with as few terms a sum's error would be that of one rounding, and
        // the products' tiles have the room
        const bool rests = item == 2 && T <= 64;
        const long long R = rests ? 2 * T : T;
        const bool fused = gemm_loss_takes(x, w), parts = in_parts() && D % 8 == 0 && in_vectors(dx) && in_vectors(dw);
        auto in_fours = [&](const lb_tensor& t) { return (uintptr_t)t.ptr % (4 * item) == 0 && t.stride[1] == 1 && (t.shape[0] <= 1 || t.stride[0] % 4 == 0); };
        const bool one_pass = T <= grad_tokens(item) && D % 4 == 0 && in_fours(w) && in_fours(dw);
        // d_weight in 16 bits that no tiles can store is rounded from float32 sums of a piece, which are bounded as dz is
        const bool dw_sums = scaled && !one_pass && !(D % 8 == 0 && in_vectors(dw));
        const long long part = up(D, 64), piece = parts ? piece_of(6, std::max(T, part)) : std::min(piece_of(fused ? 2 : 4, R), dw_sums ? piece_of(4, D) : V), pieces = (V + piece - 1) / piece,
                        ld = up(piece, 64), ld_kept = up(D, 64);  // rows of whole 128 bytes
        const long long slices = (D / 4 + kGradThreads - 1) / kGradThreads, each = std::max(16LL, one_pass ? (piece * slices + few_grad_slots() - 1) / few_grad_slots() : 1);
        const int n_counts = (int)std::min<long long>(64, (T + 255) / 256);
        RowCount* counts = take<RowCount>(n_counts);
        float *g = take<float>(T), *undo = take<float>(1);
        int* classes = take<int>(T);
        char *x_kept = take<char>(parts ? T * 6 * part : R * ld_kept * item), *w_parts = take<char>(parts ? piece * 6 * part : 0);
        float* logits = take<float>(fused || parts ? 0 : T * ld);
        char* slopes = parts ? take<char>(T * 6 * ld) : dtype == LB_F32 ? (char*)logits : take<char>(R * ld * item);
        const lb_tensor kept = matrix(x_kept, dtype, T, D, ld_kept), kept_all = matrix(x_kept, dtype, R, D, ld_kept), dz = matrix(slopes, dtype, R, piece, ld);
        // sums over pieces, and what takes the scale away: in the products' epilogue where they run on whole tiles or narrow ones, else behind them
        // (both in one launch where that fills the GPU better)
        const lb_tensor sums_a[] = {transposed(dz), dz}, sums_b[] = {kept_all, rows_of(w, 0, piece)}, sums_out[] = {dw, dx};
        const bool folds = pieces > 1 || scaled, tiles = !one_pass, both = tiles && !parts && !rests && gemm_sums_pay(sums_a, sums_b, sums_out),
                   dx_tiles = both || (tiles && folds && !rests && gemm_sum_takes(sums_a[1], sums_b[1], dx)), dw_tiles = both || (tiles && scaled && gemm_sum_takes(sums_a[0], sums_b[0], dw)),
                   dw_narrow = tiles && scaled && pieces == 1 && !dw_tiles && gemm_narrow_ranges(sums_a[0], sums_b[0]),
                   dx_narrow = tiles && scaled && !rests && pieces == 1 && !dx_tiles && gemm_narrow_ranges(sums_a[1], sums_b[1]);
        const int ranges = dtype != LB_F32 || one_pass ? 1 : parts ? gemm_part_ranges(T, D, piece) : core_ranges(piece), dw_ranges = parts ? gemm_part_ranges(piece, D, T) : 1;
        float *dx_piece = ranges > 1 || (tiles && folds && !dx_tiles && !dx_narrow && !parts) ? take<float>((ranges + 1) * T * D) : nullptr, *dx_sum = pieces > 1 ? take<float>(T * D) : nullptr;
        float* dw_piece = (tiles && scaled && !dw_tiles && !dw_narrow) || dw_ranges > 1 ? take<float>(dw_ranges * piece * D) : nullptr;
        float* dx_ranges = one_pass ? take<float>((piece + each - 1) / each * T * D) : nullptr;
        size_t more = 0;
        if (!parts && !fused) more = product_scratch(x, transposed(rows_of(w, 0, piece)));
        if (!parts && tiles) more = std::max({more, product_scratch(dz, rows_of(w, 0, piece)), product_scratch(transposed(dz), kept_all)});
        const GemmTuning few{tiles ? few_ranges(piece) : 0, 0};
        if (few.splits > 1) more = std::max<size_t>(more, (size_t)few.splits * R * D * 4);
        void* product = take<char>(more);
        if (only_count) return;
        const LossGrad d_loss{(const float*)grad.ptr, grad.stride[0]};
        const bool counts_itself = T <= 1024;  // every block: a launch (2 us) costs more than that
        if (!counts_itself) launch_overlapped(count_kernel, dim3((unsigned)n_counts), dim3(256), 0, s, 0, targets, d_loss, T, counts);
        by_type(dtype, [&](auto* type) {
            using E = std::remove_pointer_t<decltype(type)>;
            auto go = [&](auto kernel) {
                launch_overlapped(kernel, dim3(row_blocks((T + 7) / 8)), dim3(256), 0, s, 0, targets, d_loss, T, counts_itself ? (const RowCount*)nullptr : (const RowCount*)counts, n_counts,
                                  reduction == LB_REDUCTION_MEAN, (const E*)x.ptr, (long long)x.stride[0], (long long)x.stride[1], parts ? 0 : (int)D, (E*)x_kept, ld_kept, g, classes, scaled ? undo : nullptr);
            };
            if constexpr (sizeof(E) == 2) rests ? go(row_grads_kernel<E, true>) : go(row_grads_kernel<E, false>);
            else go(row_grads_kernel<E, false>);
        });
        if (parts) split(x, classes, parted(x_kept, T, D, part), s);
        for (long long k = 0; k < pieces; k++) {
            const long long first = k * piece, cols = std::min(piece, V - first);
            const lb_tensor rows = rows_of(w, first, cols);
            auto fold = [&](const float* from, int ranges, const lb_tensor& to, float* sum, bool begins, bool ends) {
                by_type(dtype, [&](auto* type) {
                    using E = std::remove_pointer_t<decltype(type)>;
                    launch_overlapped(fold_kernel<E>, by_rows(to.shape[0], D, 256), dim3(256), 0, s, 0, from, ranges, (long long)to.shape[0], (int)D,
                                      sum, begins, ends ? (E*)to.ptr : (E*)nullptr, (long long)to.stride[0], scaled ? (const float*)undo : (const float*)nullptr);
                });
            };
            if (parts) {
                const lb_tensor xp = parted(x_kept, T, D, part), wp = parted(w_parts, cols, D, part), dp = parted(slopes, T, cols, ld), dw_rows = rows_of(dw, first, cols);
                split(rows, nullptr, wp, s);
                gemm_loss_slopes(xp, wp, (const float*)lse.ptr, lse.stride[0], g, classes, (int)first, dp, s, {part, part}, ld);
                const lb_tensor a[] = {transposed(dp), dp}, b[] = {xp, wp};
                float* const sum[] = {nullptr, dx_sum};
                const bool begins[] = {true, k == 0};
                const lb_tensor* const out[] = {&dw_rows, k == pieces - 1 ? &dx : nullptr};
                const Parts apart[] = {{ld, part}, {ld, part}};
                if (ranges == 1 && dw_ranges == 1 && gemm_sums_fit(a, b)) {
                    gemm_sums(a, b, sum, begins, out, nullptr, s, apart);
                    continue;
                }
                for (int i = 0; i < 2; i++) {
                    const int n = i ? gemm_part_ranges(T, D, cols) : gemm_part_ranges(cols, D, T);
                    float* partial = i ? dx_piece : dw_piece;
                    if (n == 1 || n > (i ? ranges : dw_ranges)) {  // (a shorter piece may want more than there is memory for)
                        gemm_sum(a[i], b[i], sum[i], begins[i], out[i], nullptr, s, apart[i]);
                    } else {
                        gemm_part_sums(a[i], b[i], n, partial, s, apart[i]);
                        fold(partial, n, i ? dx : dw_rows, i ? dx_sum : nullptr, begins[i], out[i] != nullptr);
                    }
                }
                continue;
            }
            lb_tensor z = matrix(logits, LB_F32, T, cols, ld), d = dz, dw_rows = rows_of(dw, first, cols);
            d.shape[1] = cols;
            if (fused) gemm_loss_slopes(kept, rows, (const float*)lse.ptr, lse.stride[0], g, classes, (int)first, d, s);
            else if (skinny_float_takes(x, rows)) skinny_float_loss(x, rows, targets, nullptr, nullptr, logits, ld, s);
            else if (few_float32(x, rows)) run_few(x, rows, targets, nullptr, nullptr, logits, ld, s);
            else gemm(x, transposed(rows), z, EPI_NONE, 0, s, product, more, nullptr, nullptr);
            if (!fused) by_type(dtype, [&](auto* type) {
                using E = std::remove_pointer_t<decltype(type)>;
                launch_overlapped(slope_kernel<E>, by_rows(T, cols, 4 * kRowThreads), dim3(kRowThreads), 0, s, 0, (const float*)logits, ld, T, (int)first, (int)cols, (const float*)lse.ptr,
                                  (long long)lse.stride[0], (const float*)g, (const int*)classes, (E*)slopes, ld, rests);
            });
            const bool begins = k == 0, ends = k == pieces - 1;
            if (one_pass) {
                const long long n_ranges = (cols + each - 1) / each;
                const float* times = scaled ? undo : nullptr;
                by_type(dtype, [&](auto* type) {
                    using E = std::remove_pointer_t<decltype(type)>;
                    auto go = [&](auto kernel) {
                        launch_overlapped(kernel, dim3((unsigned)slices, (unsigned)n_ranges), dim3(kGradThreads), 0, s, 0, (const E*)x_kept, ld_kept, (const E*)rows.ptr, (long long)w.stride[0],
                                          (const E*)slopes, ld, rests, (int)T, (int)D, (int)cols, (int)each, (E*)dw_rows.ptr, (long long)dw.stride[0], dx_ranges, times);
                    };
                    if constexpr (grad_tokens(sizeof(E)) == 4) go(few_grads_kernel<E, 4>);
                    else T <= 4 ? go(few_grads_kernel<E, 4>) : T <= 8 ? go(few_grads_kernel<E, 8>) : go(few_grads_kernel<E, 16>);
                    launch_overlapped(fold_many_kernel<E>, by_rows(T, D, 32), dim3(256), 0, s, 0, (const float*)dx_ranges, (int)n_ranges, T, (int)D, dx_sum, begins,
                                      ends ? (E*)dx.ptr : (E*)nullptr, (long long)dx.stride[0], times);
                });
                continue;
            }
            if (both) {
                const lb_tensor a[] = {transposed(d), d}, b[] = {kept, rows};
                float* const sum[] = {nullptr, dx_sum};
                const bool first_of[] = {true, begins};
                const lb_tensor* const out[] = {&dw_rows, ends ? &dx : nullptr};
                gemm_sums(a, b, sum, first_of, out, scaled ? undo : nullptr, s);
                continue;
            }
            if (dtype == LB_F32) {  // what leaves SMs idle by itself shares a launch
                SimtProblem q[2];
                gemm(transposed(d), kept, dw_rows, EPI_NONE, 0, s, nullptr, 0, nullptr, nullptr, &q[0]);
                if (ranges > 1) {  // as many products of a batch
                    const long long whole = std::min<long long>(ranges, cols), each = cols / whole;
                    lb_tensor a = d, b = rows, out = matrix(dx_piece, LB_F32, T, D, D);
                    a.rank = b.rank = out.rank = 3;
                    a.shape[0] = b.shape[0] = out.shape[0] = whole, a.shape[1] = T, a.shape[2] = b.shape[1] = each, b.shape[2] = out.shape[2] = D, out.shape[1] = T;
                    a.stride[0] = each, a.stride[1] = ld, a.stride[2] = 1, b.stride[0] = each * rows.stride[0], b.stride[1] = rows.stride[0], b.stride[2] = rows.stride[1];
                    out.stride[0] = T * D, out.stride[1] = D, out.stride[2] = 1;
                    gemm(a, b, out, EPI_NONE, 0, s, nullptr, 0, nullptr, nullptr, nullptr);
                    const long long at = whole * each;
                    int count = (int)whole;
                    if (at < cols) {  // what is left, fewer than there are ranges
                        lb_tensor a_end = d, b_end = rows_of(rows, at, cols - at);
                        a_end.ptr = (float*)d.ptr + at, a_end.shape[1] = cols - at;
                        gemm(a_end, b_end, matrix(dx_piece + whole * T * D, LB_F32, T, D, D), EPI_NONE, 0, s, nullptr, 0, nullptr, nullptr, nullptr);
                        count++;
                    }
                    gemm_simt_many(q, 1, device_info().sms, true, s);
                    fold(dx_piece, count, dx, dx_sum, begins, ends);
                    continue;
                }
                gemm(d, rows, folds ? matrix(dx_piece, LB_F32, T, D, D) : dx, EPI_NONE, 0, s, nullptr, 0, nullptr, nullptr, &q[1]);
                gemm_simt_many(q, 2, device_info().sms, true, s);
                if (folds) fold(dx_piece, 1, dx, dx_sum, begins, ends);
                continue;
            }
            if (dw_tiles) {
                gemm_sum(transposed(d), kept_all, nullptr, true, &dw_rows, undo, s);
            } else if (dw_narrow) {
                gemm_narrow(transposed(d), kept_all, dw_rows, undo, s);
            } else {
                gemm(transposed(d), kept_all, matrix(dw_piece, LB_F32, cols, D, D), EPI_NONE, 0, s, product, more, nullptr, nullptr);
                fold(dw_piece, 1, dw_rows, nullptr, true, true);
            }
            if (dx_tiles) {
                gemm_sum(d, rows, dx_sum, begins, ends ? &dx : nullptr, undo, s);
            } else if (dx_narrow) {
                gemm_narrow(d, rows, dx, undo, s);
            } else {
                const GemmTuning ranges_of{few_ranges(cols), 0};
                const bool cut = ranges_of.splits > 1;
                gemm(d, rows, matrix(dx_piece, LB_F32, R, D, D), EPI_NONE, cut ? 3 : 0, s, product, more, nullptr, cut ? &ranges_of : nullptr);
                fold(dx_piece, rests ? 2 : 1, dx, dx_sum, begins, ends);
            }
        }
    }
};

void give_scratch(Loss& l, size_t need, void* scratch, size_t bytes) {
    if (need && (!scratch || bytes < need || (uintptr_t)scratch % 16)) refuse(format("%zu bytes of scratch are needed, 16-byte aligned", need));
    l.scratch = (char*)scratch;
}

}  // namespace
}  // namespace lb

extern "C" {

int lb_linear_cross_entropy_scratch_bytes(const lb_loss_desc* desc, const lb_tensor* x, const lb_tensor* weight, const lb_tensor* targets, size_t* bytes) {
    return lb::guarded([&] {
        if (!bytes) lb::refuse("null argument");
        lb::Forward f(desc, x, weight, targets);
        f.run(nullptr, true);
        *bytes = f.held;
    });
}

int lb_linear_cross_entropy(const lb_loss_desc* desc, const lb_tensor* x, const lb_tensor* weight, const lb_tensor* targets, const lb_tensor* loss, const lb_tensor* lse,
                            void* scratch, size_t scratch_bytes, void* stream) {
    return lb::guarded([&] {
        lb::Forward f(desc, x, weight, targets);
        f.results(loss, lse, targets);
        lb::keep_apart({&f.loss, &f.lse}, {&f.x, &f.w, &f.t});
        f.run(nullptr, true);
        lb::give_scratch(f, f.held, scratch, scratch_bytes);
        lb::driver();
        f.run((cudaStream_t)stream, false);
    });
}

int lb_linear_cross_entropy_bwd_scratch_bytes(const lb_loss_desc* desc, const lb_tensor* x, const lb_tensor* weight, const lb_tensor* targets, const lb_tensor* d_x,
                                              const lb_tensor* d_weight, size_t* bytes) {
    return lb::guarded([&] {
        if (!bytes) lb::refuse("null argument");
        lb::Backward b(desc, x, weight, targets);
        b.results(d_x, d_weight);
        b.run(nullptr, true);
        *bytes = b.held;
    });
}

int lb_linear_cross_entropy_bwd(const lb_loss_desc* desc, const lb_tensor* d_loss, const lb_tensor* x, const lb_tensor* weight, const lb_tensor* targets, const lb_tensor* lse,
                                const lb_tensor* d_x, const lb_tensor* d_weight, void* scratch, size_t scratch_bytes, void* stream) {
    return lb::guarded([&] {
        lb::Backward b(desc, x, weight, targets);
        b.results(d_x, d_weight), b.operands(d_loss, lse, targets);
        const lb_tensor& g = d_loss ? b.grad : b.lse;
        lb::keep_apart({&b.dx, &b.dw}, {&b.x, &b.w, &b.t, &b.lse, &g});
        b.run(nullptr, true);
        lb::give_scratch(b, b.held, scratch, scratch_bytes);
        lb::driver();
        b.run((cudaStream_t)stream, false);
    });
}
}
