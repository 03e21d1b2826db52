// Norms of queries and keys for each head and the position rotation, in one pass over both, forward and backward.
//
// A row x is one head's H elements at one position. With r = 1 / sqrt(mean(x^2) + eps) and z = x r w, the pairs (a, b) of the first R
// elements - (i, i + R/2), or neighbours (2i, 2i + 1) - turn by the angle of their token: y_a = z_a c - z_b s, y_b = z_b c + z_a s, where c and s
// are row `position` of two float32 tables; the rest is y = z. Backward: dz by the transposed turn (dz_a = dy_a c + dy_b s,
// dz_b = dy_b c - dy_a s), dw = sum over rows of dz x r, and with u = dz w: dx = r (u - x r^2 mean(u x)). Statistics, products and
// sums are float32; each result is rounded once. Nothing is kept between the passes: r is found again from the row, which the backward
// pass reads anyway.
//
// The weight gradients add up in registers over the rows of a thread, over a block's threads in shared memory, and over the blocks
// in a second kernel: always in the same order, so that results repeat bit for bit.
//
// Bound by memory with many rows, and before that by instructions: the arithmetic is packed, and what a row costs beside it (addresses, its sums' shuffles,
// the root) is shared by as many elements a thread as registers hold. us of the backward of 32768 tokens x 40 heads x 128, bfloat16, 1.0 GB: a warp a
// row, by the element 2227; rows in registers, eight elements a thread 304; the next rows on their way into shared memory 258; packed arithmetic and a hardware
// root 217; sixteen elements a thread 191 (165 in a graph, 6.09 TB/s of 6.53; under the power cap 194). Forward in a graph 109 us, 6.16 TB/s; 3062 x 40 x 128
// forward 13.6 us, 4.6 TB/s (weights read behind the first rows, in vectors: before that 14.9); 512 tokens x 40 x 128 4.9 us.
#include <algorithm>

#include "convert.cuh"
#include "divide.cuh"
#include "launch.cuh"
#include "overlap.h"
#include "pair.cuh"

namespace lb {
namespace {

constexpr int kMaxDim = 256;

// One of the two operands: queries or keys.
struct RopeSide {
    const void* x;
    const void* dy;  // backward
    void* out;       // y, or dx
    const void* w;   // null: all ones
    void* dw;
    float* partial;  // [blocks][H]: the blocks' sums of dw
    long long x_b, x_s, x_n, x_h, dy_b, dy_s, dy_n, dy_h, out_b, out_s, out_n, out_h;
    int heads, blocks;
    Divisor by_chunks;  // of a token's heads
    int w_f32;       // w and dw are float32, whatever the rows' type
    int w_vec;       // w is 16-byte aligned
};
struct RopeArgs {
    RopeSide side[2];
    const float *cos, *sin;
    long long ld_cos, ld_sin, cos_i, sin_i;
    const void* positions;  // null: 0, 1, 2 ...
    int positions_64;
    long long pos_b, pos_s;
    int table, batch, seq, H, R, interleaved, lanes;
    float eps;
    Divisor by_seq;
};

// The row of the tables that a token turns by: its position, clamped into them.
__device__ __forceinline__ int table_row(const RopeArgs& p, int b, int s) {
    if (!p.positions) return s;
    const long long at = b * p.pos_b + s * p.pos_s;
    const long long pos = p.positions_64 ? ((const long long*)p.positions)[at] : (long long)((const int*)p.positions)[at];
    return (int)(pos < 0 ? 0 : (pos >= p.table ? p.table - 1 : pos));
}

template <class T>
__device__ __forceinline__ float weight(const RopeSide& q, int i) {
    return !q.w ? 1.0f : q.w_f32 ? ((const float*)q.w)[i] : to_float(((const T*)q.w)[i]);
}

// Any head dim, strides and alignment, for the rows that the kernels below cannot take: right, not fast (32768 tokens x 40 heads x 128, bfloat16, rows that begin on 2
// bytes: 1490 us forward, 2077 backward, of 103 and 154; it stays for odd head dims, element strides and tables that are not dense). A warp a row, its elements lane by lane; the row waits in shared memory, so that a pair's
// members find one another and results may go where the operand was.
constexpr int kRowWarps = 8;
template <class T, bool BWD>
__global__ void __launch_bounds__(kRowWarps * 32) rope_rows_kernel(const RopeArgs p) {
    __shared__ float held[kRowWarps][2][kMaxDim];
    grid_wait();
    const int side = blockIdx.x < p.side[0].blocks ? 0 : 1;
    const RopeSide& q = p.side[side];
    const int block = side ? blockIdx.x - p.side[0].blocks : blockIdx.x;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, H = p.H, R = p.R;
    float *x = held[warp][0], *dy = held[warp][1];
    float sum[kMaxDim / 32] = {};
    const long long rows = (long long)p.batch * p.seq * q.heads;
    for (long long row = (long long)block * kRowWarps + warp; row < rows; row += (long long)q.blocks * kRowWarps) {
        const long long token = row / q.heads;
        const int n = (int)(row - token * q.heads), b = (int)(token / p.seq), s = (int)(token - (long long)b * p.seq);
        const T* from = (const T*)q.x + b * q.x_b + s * q.x_s + n * q.x_n;
        float ss = 0.0f;
        __syncwarp();
        for (int i = lane; i < H; i += 32) {
            const float v = to_float(from[i * q.x_h]);
            x[i] = v, ss += v * v;
        }
        if (BWD) {
            const T* g = (const T*)q.dy + b * q.dy_b + s * q.dy_s + n * q.dy_n;
            for (int i = lane; i < H; i += 32) dy[i] = to_float(g[i * q.dy_h]);
        }
        __syncwarp();
        for (int d = 16; d; d >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, d);
        const float r = 1.0f / sqrtf(ss / H + p.eps);
        const int at = table_row(p, b, s);
        const float *cos = p.cos + at * p.ld_cos, *sin = p.sin + at * p.ld_sin;
        T* to = (T*)q.out + b * q.out_b + s * q.out_s + n * q.out_n;
        float u[kMaxDim / 32], mean = 0.0f;
#pragma unroll
        for (int j = 0; j < kMaxDim / 32; j++) {
            const int i = lane + 32 * j;
            if (i >= H) break;
            float c = 1.0f, sn = 0.0f;  // y_i = z_i c + z_other sn
            int other = i;
            if (i < R) {
                const int pair = p.interleaved ? i / 2 : (i < R / 2 ? i : i - R / 2);
                const bool first = p.interleaved ? i % 2 == 0 : i < R / 2;
                other = p.interleaved ? i ^ 1 : (first ? i + R / 2 : i - R / 2);
                c = cos[pair * p.cos_i], sn = sin[pair * p.sin_i];
                if (first != BWD) sn = -sn;
            }
            if (!BWD) {
                const float turned = i < R ? x[other] * r * weight<T>(q, other) * sn : 0.0f;
                to[i * q.out_h] = from_float<T>(x[i] * r * weight<T>(q, i) * c + turned);
            } else {
                const float dz = i < R ? dy[i] * c + dy[other] * sn : dy[i];
                sum[j] += dz * (x[i] * r);
                u[j] = dz * weight<T>(q, i);
                mean += u[j] * (x[i] * r);
            }
        }
        if (BWD) {
            for (int d = 16; d; d >>= 1) mean += __shfl_xor_sync(0xffffffffu, mean, d);
            mean /= H;
#pragma unroll
            for (int j = 0; j < kMaxDim / 32; j++)
                if (lane + 32 * j < H) to[(lane + 32 * j) * q.out_h] = from_float<T>(r * (u[j] - x[lane + 32 * j] * r * mean));
        }
    }
    if (BWD && q.w) {
        __syncthreads();
        float* sums = &held[0][0][0];  // [warp][H]
#pragma unroll
        for (int j = 0; j < kMaxDim / 32; j++)
            if (lane + 32 * j < H) sums[warp * kMaxDim + lane + 32 * j] = sum[j];
        __syncthreads();
        for (int i = threadIdx.x; i < H; i += blockDim.x) {
            float t = 0.0f;
            for (int k = 0; k < kRowWarps; k++) t += sums[k * kMaxDim + i];
            q.partial[(long long)block * H + i] = t;
        }
    }
}

// Four elements of a row, as two pairs of float32 and back; the address is a multiple of their size.
template <class T> struct Four;
template <> struct Four<float> {
    float4 v;
    __device__ __forceinline__ void load(const float* p) { v = *(const float4*)p; }
    __device__ __forceinline__ void widen(Pair* x) const { x[0] = both(v.x, v.y), x[1] = both(v.z, v.w); }
    __device__ __forceinline__ static void store(float* p, const Pair* x) {
        const float2 lo = apart(x[0]), hi = apart(x[1]);
        *(float4*)p = make_float4(lo.x, lo.y, hi.x, hi.y);
    }
};
template <> struct Four<__nv_bfloat16> {
    uint2 v;
    __device__ __forceinline__ void load(const __nv_bfloat16* p) { v = *(const uint2*)p; }
    __device__ __forceinline__ void widen(Pair* x) const {
        x[0] = both(__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xffff0000u)), x[1] = both(__uint_as_float(v.y << 16), __uint_as_float(v.y & 0xffff0000u));
    }
    __device__ __forceinline__ static void store(__nv_bfloat16* p, const Pair* x) {
        const __nv_bfloat162 lo = __float22bfloat162_rn(apart(x[0])), hi = __float22bfloat162_rn(apart(x[1]));
        *(uint2*)p = make_uint2(*(const uint32_t*)&lo, *(const uint32_t*)&hi);
    }
};
template <> struct Four<__half> {
    uint2 v;
    __device__ __forceinline__ void load(const __half* p) { v = *(const uint2*)p; }
    __device__ __forceinline__ void widen(Pair* x) const {
        const float2 lo = __half22float2(*(const __half2*)&v.x), hi = __half22float2(*(const __half2*)&v.y);
        x[0] = both(lo.x, lo.y), x[1] = both(hi.x, hi.y);
    }
    __device__ __forceinline__ static void store(__half* p, const Pair* x) {
        const __half2 lo = __float22half2_rn(apart(x[0])), hi = __float22half2_rn(apart(x[1]));
        *(uint2*)p = make_uint2(*(const uint32_t*)&lo, *(const uint32_t*)&hi);
    }
};

// N elements of a row, four or (16-bit types) eight.
template <class T, int N> struct Run;
template <class T> struct Run<T, 4> : Four<T> {};
template <class T> struct Run<T, 8> {
    uint4 v;
    __device__ __forceinline__ void load(const T* p) { v = *(const uint4*)p; }
    __device__ __forceinline__ void widen(Pair* x) const { Four<T>{make_uint2(v.x, v.y)}.widen(x), Four<T>{make_uint2(v.z, v.w)}.widen(x + 2); }
    __device__ __forceinline__ static void store(T* p, const Pair* x) {
        uint2 h[2];
        Four<T>::store((T*)&h[0], x), Four<T>::store((T*)&h[1], x + 2);
        *(uint4*)p = make_uint4(h[0].x, h[0].y, h[1].x, h[1].y);
    }
};

// A thread's N pairs turned: the first members in the first half of v, the second ones in the other, or neighbours in one register pair each; BACK: the
// other way.
template <bool BACK, int N>
__device__ __forceinline__ void turn(Pair* v, const Pair* c, const Pair* s, bool neighbours) {
    if (neighbours) {
#pragma unroll
        for (int j = 0; j < N; j++) {
            const float2 x = apart(v[j]), cc = apart(c[j / 2]), ss = apart(s[j / 2]);
            const float cj = j % 2 ? cc.y : cc.x, sj = BACK ? -(j % 2 ? ss.y : ss.x) : (j % 2 ? ss.y : ss.x);
            v[j] = fma2(both(x.y, x.x), both(-sj, sj), v[j] * both(cj, cj));
        }
    } else {
#pragma unroll
        for (int j = 0; j < N / 2; j++) {
            const Pair a = v[j], b = v[N / 2 + j], n = BACK ? -s[j] : s[j];
            v[j] = fma2(-n, b, a * c[j]), v[N / 2 + j] = fma2(n, a, b * c[j]);
        }
    }
}

// Head dims and rotated parts that are multiples of 2 N (N: 4 or 8), rows of aligned pieces of N elements: `p.lanes` lanes of a warp a row (a power of two), 2 N
// elements each, both members of N pairs among them, so that a row is in registers once and its elements meet only in the sums of its statistics.
constexpr int kGroupThreads = 256;

// What a thread keeps for all its rows.
template <class T, bool BWD, int N>
struct Lane {
    int c, e0, e1;  // its place in the row, its two runs of N elements
    bool live, turns;
    Pair w[N], sum[BWD ? N : 1];

    __device__ __forceinline__ explicit Lane(const RopeArgs& p) {
        c = threadIdx.x & (p.lanes - 1), live = c * 2 * N < p.H, turns = c < p.R / (2 * N);
        const bool beside = p.interleaved || !turns;
        e0 = beside ? 2 * N * c : N * c, e1 = beside ? e0 + N : p.R / 2 + N * c;
        if (BWD) {
#pragma unroll
            for (int j = 0; j < N; j++) sum[j] = both(0.0f, 0.0f);
        }
    }
    __device__ __forceinline__ void weights(const RopeSide& q) {
        if (q.w && q.w_vec && live) {
            if (q.w_f32) {
#pragma unroll
                for (int j = 0; j < N / 4; j++) {
                    Four<float> lo, hi;
                    lo.load((const float*)q.w + e0 + 4 * j), hi.load((const float*)q.w + e1 + 4 * j);
                    lo.widen(w + 2 * j), hi.widen(w + N / 2 + 2 * j);
                }
            } else {
                Run<T, N> lo, hi;
                lo.load((const T*)q.w + e0), hi.load((const T*)q.w + e1);
                lo.widen(w), hi.widen(w + N / 2);
            }
            return;
        }
#pragma unroll
        for (int j = 0; j < N; j++) {
            const int i = j < N / 2 ? e0 + 2 * j : e1 + 2 * j - N;
            w[j] = live ? both(weight<T>(q, i), weight<T>(q, i + 1)) : both(0.0f, 0.0f);
        }
    }
    // One row, executed by the whole warp: x and, backward, y = dy go in, y = the result comes out. Zeros go in where a lane has no part of its row;
    // where there is no row (`there`), whatever goes in stays among the lanes that would have it. 1 / sqrt by the hardware's 2^-22 and a Newton step.
    __device__ __forceinline__ void row(const RopeArgs& p, float per, bool there, const Pair* x, Pair* y, const Pair* cs, const Pair* sn) {
        Pair squares = x[0] * x[0], products;
#pragma unroll
        for (int j = 1; j < N; j++) squares = fma2(x[j], x[j], squares);
        if (BWD) {
            if (turns) turn<true, N>(y, cs, sn, p.interleaved);  // dz
            products = y[0] * w[0] * x[0];
#pragma unroll
            for (int j = 1; j < N; j++) products = fma2(y[j] * w[j], x[j], products);
        }
        const float2 s2 = apart(squares), d2 = BWD ? apart(products) : make_float2(0.0f, 0.0f);
        float ss = s2.x + s2.y, dot = d2.x + d2.y;
#pragma unroll
        for (int d = 16; d; d >>= 1) {
            if (d >= p.lanes) continue;
            ss += __shfl_xor_sync(0xffffffffu, ss, d);
            if (BWD) dot += __shfl_xor_sync(0xffffffffu, dot, d);
        }
        const float v = ss * per + p.eps;
        float r = rsqrtf(v);
        if (v > 1e-30f && v < 1e30f) r *= 1.5f - 0.5f * v * r * r;
        const Pair rr = both(r, r);
        if (!BWD) {
#pragma unroll
            for (int j = 0; j < N; j++) y[j] = x[j] * rr * w[j];
            if (turns) turn<false, N>(y, cs, sn, p.interleaved);
        } else {
            const float mean = -dot * r * per * r;
            const Pair mm = both(mean, mean);
#pragma unroll
            for (int j = 0; j < N; j++) {
                const Pair unit = x[j] * rr;
                if (there) sum[j] = fma2(y[j], unit, sum[j]);
                y[j] = fma2(unit, mm, y[j] * w[j] * rr);
            }
        }
    }
    // A block's sums of dw, all threads: [group][H] in shared memory, its rows added up.
    __device__ __forceinline__ void leave(const RopeArgs& p, const RopeSide& q, int block, float* held) {
        __syncthreads();
        const int groups = kGroupThreads / p.lanes, g = threadIdx.x / p.lanes;
        if (live) {
#pragma unroll
            for (int j = 0; j < N; j++) *(float2*)(held + g * p.H + (j < N / 2 ? e0 + 2 * j : e1 + 2 * j - N)) = apart(sum[j]);
        }
        __syncthreads();
        for (int i = threadIdx.x; i < p.H; i += kGroupThreads) {
            float t = 0.0f;
            for (int k = 0; k < groups; k++) t += held[k * p.H + i];
            q.partial[(long long)block * p.H + i] = t;
        }
    }
};

// Few rows: one a group of lanes at a time, its loads straight into registers.
template <class T, bool BWD>
__global__ void __launch_bounds__(kGroupThreads, 3) rope_few_kernel(const RopeArgs p) {
    __shared__ float held[BWD ? kGroupThreads * 8 : 1];
    grid_wait();
    const int side = blockIdx.x < p.side[0].blocks ? 0 : 1;
    const RopeSide& q = p.side[side];
    const int block = side ? blockIdx.x - p.side[0].blocks : blockIdx.x, groups = kGroupThreads / p.lanes;
    Lane<T, BWD, 4> lane(p);
    lane.weights(q);
    const float per = 1.0f / (float)p.H;
    const long long rows = (long long)p.batch * p.seq * q.heads;
    for (long long base = (long long)block * groups; base < rows; base += (long long)q.blocks * groups) {
        const long long mine = base + threadIdx.x / p.lanes;
        const bool there = mine < rows && lane.live;
        const unsigned row = (unsigned)(mine < rows ? mine : rows - 1), token = row / q.heads;
        const int n = (int)(row - token * q.heads), b = (int)(token / p.seq), s = (int)(token - (unsigned)b * p.seq);
        Pair x[4] = {}, y[4] = {}, cs[2] = {}, sn[2] = {};
        Four<T> in[2], grad[2];
        Four<float> turned[2];
        if (there) {
            const T* from = (const T*)q.x + b * q.x_b + s * q.x_s + n * q.x_n;
            in[0].load(from + lane.e0), in[1].load(from + lane.e1);
            if (BWD) {
                const T* g = (const T*)q.dy + b * q.dy_b + s * q.dy_s + n * q.dy_n;
                grad[0].load(g + lane.e0), grad[1].load(g + lane.e1);
            }
            if (lane.turns) {
                const long long at = table_row(p, b, s);
                turned[0].load(p.cos + at * p.ld_cos + 4 * lane.c), turned[1].load(p.sin + at * p.ld_sin + 4 * lane.c);
            }
            in[0].widen(x), in[1].widen(x + 2);
            if (BWD) grad[0].widen(y), grad[1].widen(y + 2);
            if (lane.turns) turned[0].widen(cs), turned[1].widen(sn);
        }
        lane.row(p, per, there, x, y, cs, sn);
        if (there) {
            T* to = (T*)q.out + b * q.out_b + s * q.out_s + n * q.out_n;
            Four<T>::store(to + lane.e0, y), Four<T>::store(to + lane.e1, y + 2);
        }
    }
    if (BWD && q.w) lane.leave(p, q, block, held);
}

// Many rows: a group of lanes takes HEADS heads of a token at a time, which turn by the same angles, and has the next token's (or the next
// heads') rows on their way into shared memory meanwhile: every thread copies what it reads itself, so that it waits for nobody else. Elements a thread, heads at a
// time and blocks to an SM, us of that backward / forward: 8, 4, 3 217 / 144; 8, 4, 2 222; 8, 2, 3 243; 8, 2, 4 285; 16, 2, 2 191 / 111; 16, 4, 2 - / 131;
// 16, 1, 2 - / 144. At two blocks to an SM a thread has 128 registers, and the backward's sixteen elements spill 68 bytes (36 of loads); at
// three, 80 registers, float32's eight spill 12 (16).
__device__ __forceinline__ void copy_async(void* to, const void* from, int bytes) {
    const uint32_t at = (uint32_t)__cvta_generic_to_shared(to);
    const size_t src = __cvta_generic_to_global(from);
    if (bytes == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at), "l"(src) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(at), "l"(src) : "memory");
}
// Heads of a group at a time, blocks of an SM, bytes of its ring.
template <class T, bool BWD, int N>
constexpr int many_heads() { return sizeof(T) == 4 || N == 8 ? 2 : 4; }
template <int N>
constexpr int many_per_sm() { return N == 8 ? 2 : 3; }
template <class T, bool BWD, int N>
constexpr int many_smem() { return 2 * many_heads<T, BWD, N>() * (BWD ? 4 : 2) * kGroupThreads * (int)sizeof(Run<T, N>); }
template <class T, bool BWD, int N>
__global__ void __launch_bounds__(kGroupThreads, many_per_sm<N>()) rope_many_kernel(const RopeArgs p) {
    constexpr int HEADS = many_heads<T, BWD, N>(), RUNS = BWD ? 4 : 2, STAGE = HEADS * RUNS * kGroupThreads;
    extern __shared__ __align__(16) uint8_t smem[];
    Run<T, N>* ring = (Run<T, N>*)smem + threadIdx.x;  // [stage][head][run][thread]
    grid_wait();
    const int side = blockIdx.x < p.side[0].blocks ? 0 : 1;
    const RopeSide& q = p.side[side];
    const int block = side ? blockIdx.x - p.side[0].blocks : blockIdx.x, groups = kGroupThreads / p.lanes;
    Lane<T, BWD, N> lane(p);
    const float per = 1.0f / (float)p.H;
    const unsigned chunks = q.by_chunks.d, tasks = (unsigned)(p.batch * p.seq) * chunks, step = (unsigned)(q.blocks * groups);
    unsigned task = (unsigned)(block * groups + threadIdx.x / p.lanes);
    const unsigned rounds = (tasks - min(tasks, (unsigned)(block * groups)) + step - 1) / step;  // the same for the whole block

    struct Place {
        int b, s, n0;
    };
    auto place = [&](unsigned t) {
        const unsigned token = q.by_chunks.div(t), b = p.by_seq.div(token);
        return Place{(int)b, (int)(token - b * p.seq), (int)(t - token * chunks) * HEADS};
    };
    auto fetch = [&](const Place& at, int stage) {
        const T* from = (const T*)q.x + at.b * q.x_b + at.s * q.x_s + at.n0 * q.x_n;
        const T* grad = BWD ? (const T*)q.dy + at.b * q.dy_b + at.s * q.dy_s + at.n0 * q.dy_n : nullptr;
        Run<T, N>* to = ring + stage * STAGE;
#pragma unroll
        for (int k = 0; k < HEADS; k++)
            if (lane.live && at.n0 + k < q.heads) {
                copy_async(to + (k * RUNS + 0) * kGroupThreads, from + k * q.x_n + lane.e0, sizeof(Run<T, N>));
                copy_async(to + (k * RUNS + 1) * kGroupThreads, from + k * q.x_n + lane.e1, sizeof(Run<T, N>));
                if (BWD) {
                    copy_async(to + (k * RUNS + RUNS - 2) * kGroupThreads, grad + k * q.dy_n + lane.e0, sizeof(Run<T, N>));
                    copy_async(to + (k * RUNS + RUNS - 1) * kGroupThreads, grad + k * q.dy_n + lane.e1, sizeof(Run<T, N>));
                }
            }
    };
    // angles one task ahead, the position that they are found by two
    Four<float> cs_next[N / 4] = {}, sn_next[N / 4] = {};
    auto angles = [&](int at) {
        if (!lane.turns) return;
#pragma unroll
        for (int j = 0; j < N / 4; j++)
            cs_next[j].load(p.cos + at * p.ld_cos + N * lane.c + 4 * j), sn_next[j].load(p.sin + at * p.ld_sin + N * lane.c + 4 * j);
    };
    auto position = [&](unsigned t) {
        const Place at = place(t);
        return table_row(p, at.b, at.s);
    };
    if (!lane.live)  // nothing is copied for lanes behind the row's end
        for (int k = 0; k < 2 * HEADS * RUNS; k++) ring[k * kGroupThreads] = Run<T, N>{};
    Place here = {}, next = {};
    int after = 0;
    if (task < tasks) next = place(task), fetch(next, 0), angles(position(task));
    if (task < tasks && tasks - task > step) after = position(task + step);
    asm volatile("cp.async.commit_group;" ::: "memory");
    lane.weights(q);  // (behind the first rows, which are longer on their way)
    for (unsigned round = 0; round < rounds; round++, task += step) {
        const bool there = task < tasks && lane.live;
        here = next;
        Pair cs[N / 2], sn[N / 2];
#pragma unroll
        for (int j = 0; j < N / 4; j++) cs_next[j].widen(cs + 2 * j), sn_next[j].widen(sn + 2 * j);
        if (task < tasks && tasks - task > step) {
            next = place(task + step);
            fetch(next, (round + 1) & 1);
            angles(after);
            if (tasks - task - step > step) after = position(task + 2 * step);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        asm volatile("cp.async.wait_group 1;" ::: "memory");
        T* to = (T*)q.out + here.b * q.out_b + here.s * q.out_s + here.n0 * q.out_n;
        const Run<T, N>* held = ring + (round & 1) * STAGE;
#pragma unroll
        for (int k = 0; k < HEADS; k++) {
            const bool row = there && here.n0 + k < q.heads;
            if (!__any_sync(0xffffffffu, row)) break;
            Pair x[N], y[N];
            held[(k * RUNS + 0) * kGroupThreads].widen(x), held[(k * RUNS + 1) * kGroupThreads].widen(x + N / 2);
            if (BWD) held[(k * RUNS + RUNS - 2) * kGroupThreads].widen(y), held[(k * RUNS + RUNS - 1) * kGroupThreads].widen(y + N / 2);
            lane.row(p, per, row, x, y, cs, sn);
            if (row) Run<T, N>::store(to + k * q.out_n + lane.e0, y), Run<T, N>::store(to + k * q.out_n + lane.e1, y + N / 2);
        }
    }
    if (BWD && q.w) {
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        lane.leave(p, q, block, (float*)smem);
    }
}

// dw: the blocks' sums, 32 columns a block, 32 of its rows beside one another, sixteen loads of a thread in flight.
template <class T>
__global__ void __launch_bounds__(1024) rope_weights_kernel(const RopeArgs p) {
    __shared__ float held[32][33];
    grid_wait();
    const RopeSide& q = p.side[blockIdx.y];
    if (!q.w) return;
    const int lane = threadIdx.x & 31, part = threadIdx.x >> 5, i = blockIdx.x * 32 + lane;
    float sum = 0.0f;
    if (i < p.H) {
        for (int k0 = part; k0 < q.blocks; k0 += 32 * 16) {
            float v[16];
#pragma unroll
            for (int k = 0; k < 16; k++) v[k] = k0 + 32 * k < q.blocks ? q.partial[(long long)(k0 + 32 * k) * p.H + i] : 0.0f;
#pragma unroll
            for (int k = 0; k < 16; k++) sum += v[k];
        }
    }
    held[part][lane] = sum;
    __syncthreads();
    if (part == 0 && i < p.H) {
#pragma unroll
        for (int k = 1; k < 32; k++) sum += held[k][lane];
        if (q.w_f32) ((float*)q.dw)[i] = sum;
        else ((T*)q.dw)[i] = from_float<T>(sum);
    }
}

// ---- host side ------------------------------------------------------------------------------------------------------

[[noreturn]] void refuse(const std::string& why) { fail(LB_ERR_INVALID, "qk_norm_rope: " + why); }

long long elements(const lb_tensor& t) {
    long long n = 1;
    for (int d = 0; d < t.rank; d++) n *= t.shape[d];
    return n;
}
void in_memory(const lb_tensor* t, const char* what) {
    if (t && elements(*t) && (!t->ptr || (uintptr_t)t->ptr % dtype_size(t->dtype))) refuse(format("%s has no memory or is not aligned to its elements", what));
}
void same_shape(const lb_tensor& a, const lb_tensor& b, const char* what) {
    bool same = a.rank == b.rank && a.dtype == b.dtype;
    for (int d = 0; same && d < a.rank; d++) same = a.shape[d] == b.shape[d];
    if (!same) refuse(format("%s must have its operand's shape and dtype", what));
    in_memory(&b, what);
}
// A result, and the operands whose memory it may be, row for row: every row is read by the threads that write it, before they do. Rows of other blocks are read
// and written at any time, so all else that a call is given lies apart from it, and its elements from one another.
struct Result {
    const lb_tensor* t;
    const char* what;
    int own[2];  // numbers of operands
};
struct Operand {
    const lb_tensor* t;
    const char* what;
};
void keep_apart(const Result* results, int n_results, const Operand* operands, int n_operands) {
    Extent written[4], read[9];
    for (int k = 0; k < n_operands; k++)
        if (operands[k].t) read[k] = extent(*operands[k].t);
    for (int r = 0; r < n_results; r++) {
        const Result& out = results[r];
        if (!out.t) continue;
        if (overlaps_itself(*out.t)) refuse(format("elements of %s share GPU memory with one another", out.what));
        written[r] = extent(*out.t);
        for (int k = 0; k < n_operands; k++) {
            const lb_tensor* t = operands[k].t;
            if (!t || !written[r].meets(read[k]) || ((k == out.own[0] || k == out.own[1]) && same_places(*out.t, *t))) continue;
            if (share_memory(*out.t, *t)) refuse(format("%s shares GPU memory with %s", out.what, operands[k].what));
        }
        for (int k = 0; k < r; k++)
            if (results[k].t && written[r].meets(written[k]) && share_memory(*out.t, *results[k].t)) refuse(format("%s shares GPU memory with %s", out.what, results[k].what));
    }
}
// No dimension of a result is repeated.
void written(const lb_tensor& t, const char* what) {
    for (int d = 0; d < t.rank; d++)
        if (t.shape[d] > 1 && t.stride[d] == 0) refuse(format("%s is written and cannot be a broadcast view", what));
}
void weights(RopeSide& side, const lb_tensor* w, int H, int dtype, const char* what) {
    if (!w) return;
    if (w->rank != 1 || w->shape[0] != H || (w->dtype != dtype && w->dtype != LB_F32)) refuse(format("%s must be [%d] of the rows' dtype or float32", what, H));
    if (H > 1 && w->stride[0] != 1) refuse(format("%s must be dense", what));
    in_memory(w, what);
    side.w = w->ptr, side.w_f32 = w->dtype == LB_F32, side.w_vec = (uintptr_t)w->ptr % 16 == 0;
}

// Both sides' blocks, in proportion to their rows: at most what fills the GPU once, at least one where a side has rows.
constexpr int kBlocksPerSm = 4;  // at most; the scratch holds a sum for each
void share_blocks(RopeArgs& p, int groups, int heads, int sms, int per_sm) {
    const long long tokens = (long long)p.batch * p.seq, most = (long long)sms * per_sm;
    long long need[2];
    for (int k = 0; k < 2; k++) need[k] = (tokens * ((p.side[k].heads + heads - 1) / heads) + groups - 1) / groups;
    const long long all = need[0] + need[1];
    for (int k = 0; k < 2; k++) p.side[k].blocks = (int)(all <= most ? need[k] : need[k] ? std::max(1LL, most * need[k] / all) : 0);
}

// Whether rows can be taken in pieces of `run` elements by groups of lanes.
bool in_pieces(const RopeArgs& p, int dtype, bool bwd, int run) {
    if (p.H % (2 * run) || p.R % (2 * run) || p.cos_i != 1 || p.sin_i != 1 || p.ld_cos % 4 || p.ld_sin % 4 || (uintptr_t)p.cos % 16 || (uintptr_t)p.sin % 16) return false;
    const int per = run, bytes = run * dtype_size(dtype);
    auto fits = [&](const void* ptr, long long b, long long s, long long n, long long h, int heads) {
        return (uintptr_t)ptr % bytes == 0 && (b % per == 0 || p.batch == 1) && (s % per == 0 || p.seq == 1) && (n % per == 0 || heads <= 1) && h == 1;
    };
    for (const RopeSide& q : p.side)
        if (q.heads && (!fits(q.x, q.x_b, q.x_s, q.x_n, q.x_h, q.heads) || !fits(q.out, q.out_b, q.out_s, q.out_n, q.out_h, q.heads) ||
                        (bwd && !fits(q.dy, q.dy_b, q.dy_s, q.dy_n, q.dy_h, q.heads))))
            return false;
    return true;
}

struct RopeCall {
    RopeArgs p{};
    int dtype = 0;
    long long rows = 0;
};

RopeCall check_rope(const lb_rope_desc* desc, const lb_tensor* q, const lb_tensor* k, const lb_tensor* cos, const lb_tensor* sin, const lb_tensor* positions,
                    const lb_tensor* wq, const lb_tensor* wk) {
    if (!desc || !q || !k || !cos || !sin) refuse("null argument");
    RopeCall c;
    RopeArgs& p = c.p;
    if (q->rank != 4 || k->rank != 4) refuse("queries and keys must be [batch, sequence, heads, head dim]");
    if (q->dtype != k->dtype || (q->dtype != LB_F32 && q->dtype != LB_BF16 && q->dtype != LB_F16)) refuse("queries and keys must share a dtype: float16, bfloat16 or float32");
    if (q->shape[0] != k->shape[0] || q->shape[1] != k->shape[1] || q->shape[3] != k->shape[3]) refuse("queries and keys must share batch, sequence and head dim");
    for (int d = 0; d < 4; d++)
        if (q->shape[d] < 0 || k->shape[d] < 0) refuse("negative size");
    if (q->shape[3] < 1 || q->shape[3] > kMaxDim) refuse(format("head dims of 1 to %d", kMaxDim));
    if (elements(*q) / q->shape[3] > INT32_MAX || elements(*k) / k->shape[3] > INT32_MAX || q->shape[0] * q->shape[1] > INT32_MAX)
        fail(LB_ERR_UNSUPPORTED, "qk_norm_rope: more than 2^31 - 1 rows in one call");
    c.dtype = q->dtype;
    p.batch = (int)q->shape[0], p.seq = (int)q->shape[1], p.H = (int)q->shape[3];
    if (cos->rank != 2 || sin->rank != 2 || cos->dtype != LB_F32 || sin->dtype != LB_F32 || cos->shape[0] != sin->shape[0] || cos->shape[1] != sin->shape[1])
        refuse("cos and sin must be float32 tables of one shape [positions, rotated pairs]");
    if (cos->shape[1] < 1 || 2 * cos->shape[1] > p.H) refuse(format("the tables' %lld pairs must be 1 to %d for a head dim of %d", (long long)cos->shape[1], p.H / 2, p.H));
    if (cos->shape[0] > INT32_MAX) refuse("tables of at most 2^31 - 1 positions");
    p.table = (int)cos->shape[0], p.R = (int)(2 * cos->shape[1]);
    p.cos = (const float*)cos->ptr, p.sin = (const float*)sin->ptr;
    p.ld_cos = cos->stride[0], p.cos_i = cos->stride[1], p.ld_sin = sin->stride[0], p.sin_i = sin->stride[1];
    if (cos->shape[1] == 1) p.cos_i = p.sin_i = 1;
    const long long tokens = (long long)p.batch * p.seq;
    if (tokens && p.table < 1) refuse("the tables have no position");
    if (positions) {
        if (positions->dtype != LB_I32 && positions->dtype != LB_I64) refuse("positions must be int32 or int64");
        const bool flat = positions->rank == 1;
        if ((!flat && positions->rank != 2) || positions->shape[positions->rank - 1] != p.seq || (!flat && positions->shape[0] != p.batch))
            refuse("positions must be [sequence] or [batch, sequence]");
        p.positions = positions->ptr, p.positions_64 = positions->dtype == LB_I64;
        p.pos_b = flat ? 0 : positions->stride[0], p.pos_s = positions->stride[flat ? 0 : 1];
    } else if (p.table < p.seq) {
        refuse(format("the tables hold %d positions, the sequence has %d", p.table, p.seq));
    }
    if (!(desc->eps >= 0.0f)) refuse("eps must not be negative");
    in_memory(q, "queries"), in_memory(k, "keys"), in_memory(cos, "cos"), in_memory(sin, "sin"), in_memory(positions, "positions");
    p.eps = desc->eps, p.interleaved = desc->interleaved != 0;
    const lb_tensor* x[2] = {q, k};
    for (int s = 0; s < 2; s++) {
        RopeSide& side = p.side[s];
        side.x = x[s]->ptr, side.heads = (int)x[s]->shape[2];
        side.x_b = x[s]->stride[0], side.x_s = x[s]->stride[1], side.x_n = x[s]->stride[2], side.x_h = x[s]->stride[3];
    }
    weights(p.side[0], wq, p.H, c.dtype, "the queries' weight");
    weights(p.side[1], wk, p.H, c.dtype, "the keys' weight");
    c.rows = elements(*q) / p.H + elements(*k) / p.H;
    return c;
}

template <class T, bool BWD, int N>
void launch_many(RopeArgs& p, int sms, cudaStream_t stream) {
    constexpr int kHeads = many_heads<T, BWD, N>();
    p.lanes = 1;
    while (p.lanes * 2 * N < p.H) p.lanes *= 2;
    first_use_on_device((const void*)rope_many_kernel<T, BWD, N>, [] {
        LB_CUDA(cudaFuncSetAttribute(rope_many_kernel<T, BWD, N>, cudaFuncAttributeMaxDynamicSharedMemorySize, many_smem<T, BWD, N>()));
    });
    share_blocks(p, kGroupThreads / p.lanes, kHeads, sms, many_per_sm<N>());
    p.by_seq.set((uint32_t)std::max(p.seq, 1));
    for (RopeSide& q : p.side) q.by_chunks.set((uint32_t)std::max((q.heads + kHeads - 1) / kHeads, 1));
    launch_overlapped(rope_many_kernel<T, BWD, N>, dim3((unsigned)(p.side[0].blocks + p.side[1].blocks)), dim3(kGroupThreads), (many_smem<T, BWD, N>()), stream, 0, p);
}
template <class T, bool BWD>
void launch_rope(RopeCall& c, cudaStream_t stream) {
    RopeArgs& p = c.p;
    const int sms = device_info().sms;
    auto blocks = [&] { return dim3((unsigned)(p.side[0].blocks + p.side[1].blocks)); };
    if (c.rows && in_pieces(p, c.dtype, BWD, 4)) {
        p.lanes = 1;
        while (p.lanes * 8 < p.H) p.lanes *= 2;
        const int groups = kGroupThreads / p.lanes;
        // below four rows a group of the kernel for few, a second and third round of which cost less than the other kernel's start (512 tokens x 40
        // heads x 128, forward: 20480 rows 4.9 us; 1024 tokens on the other 5.8)
        if (c.rows < (long long)sms * 3 * groups * 4) {
            share_blocks(p, groups, 1, sms, 3);
            launch_overlapped(rope_few_kernel<T, BWD>, blocks(), dim3(kGroupThreads), 0, stream, 0, p);
        } else if (sizeof(T) == 2 && in_pieces(p, c.dtype, BWD, 8)) {
            if constexpr (sizeof(T) == 2) launch_many<T, BWD, 8>(p, sms, stream);
        } else {
            launch_many<T, BWD, 4>(p, sms, stream);
        }
    } else if (c.rows) {
        share_blocks(p, kRowWarps, 1, sms, kBlocksPerSm);
        launch_overlapped(rope_rows_kernel<T, BWD>, blocks(), dim3(kRowWarps * 32), 0, stream, 0, p);
    }
    if (BWD && (p.side[0].w || p.side[1].w)) launch_overlapped(rope_weights_kernel<T>, dim3((unsigned)((p.H + 31) / 32), 2), dim3(1024), 0, stream, 0, p);
}
template <bool BWD>
void run_rope(RopeCall& c, void* stream) {
    driver();
    cudaStream_t s = (cudaStream_t)stream;
    if (c.dtype == LB_F32) launch_rope<float, BWD>(c, s);
    else if (c.dtype == LB_BF16) launch_rope<__nv_bfloat16, BWD>(c, s);
    else launch_rope<__half, BWD>(c, s);
}

size_t scratch_bytes(int H) { return (size_t)sm_count_hint() * kBlocksPerSm * H * sizeof(float) * 2; }

}  // namespace
}  // namespace lb

extern "C" {

int lb_qk_norm_rope(const lb_rope_desc* desc, const lb_tensor* q, const lb_tensor* k, const lb_tensor* cos, const lb_tensor* sin, const lb_tensor* positions,
                    const lb_tensor* q_weight, const lb_tensor* k_weight, const lb_tensor* q_out, const lb_tensor* k_out, void* stream) {
    return lb::guarded([&] {
        lb::RopeCall c = lb::check_rope(desc, q, k, cos, sin, positions, q_weight, k_weight);
        if (!q_out || !k_out) lb::refuse("null argument");
        const lb_tensor *in[2] = {q, k}, *out[2] = {q_out, k_out};
        for (int s = 0; s < 2; s++) {
            lb::same_shape(*in[s], *out[s], "a result");
            lb::written(*out[s], "a result");
            lb::RopeSide& side = c.p.side[s];
            side.out = out[s]->ptr, side.out_b = out[s]->stride[0], side.out_s = out[s]->stride[1], side.out_n = out[s]->stride[2], side.out_h = out[s]->stride[3];
        }
        const lb::Result results[] = {{q_out, "the queries' result", {0, 0}}, {k_out, "the keys' result", {1, 1}}};
        const lb::Operand operands[] = {{q, "the queries"}, {k, "the keys"}, {cos, "cos"}, {sin, "sin"}, {positions, "positions"}, {q_weight, "the queries' weight"}, {k_weight, "the keys' weight"}};
        lb::keep_apart(results, 2, operands, 7);
        if (c.rows) lb::run_rope<false>(c, stream);
    });
}

size_t lb_qk_norm_rope_bwd_scratch_bytes(int head_dim) { return head_dim > 0 ? lb::scratch_bytes(head_dim) : 0; }

int lb_qk_norm_rope_bwd(const lb_rope_desc* desc, const lb_tensor* d_q_out, const lb_tensor* d_k_out, const lb_tensor* q, const lb_tensor* k,
                        const lb_tensor* cos, const lb_tensor* sin, const lb_tensor* positions, const lb_tensor* q_weight, const lb_tensor* k_weight,
                        const lb_tensor* d_q, const lb_tensor* d_k, const lb_tensor* d_q_weight, const lb_tensor* d_k_weight, void* scratch,
                        size_t scratch_bytes, void* stream) {
    return lb::guarded([&] {
        lb::RopeCall c = lb::check_rope(desc, q, k, cos, sin, positions, q_weight, k_weight);
        if (!d_q_out || !d_k_out || !d_q || !d_k) lb::refuse("null argument");
        const lb_tensor *in[2] = {q, k}, *dy[2] = {d_q_out, d_k_out}, *dx[2] = {d_q, d_k}, *w[2] = {q_weight, k_weight}, *dw[2] = {d_q_weight, d_k_weight};
        for (int s = 0; s < 2; s++) {
            lb::same_shape(*in[s], *dy[s], "a gradient");
            lb::same_shape(*in[s], *dx[s], "a gradient");
            lb::written(*dx[s], "a gradient");
            lb::RopeSide& side = c.p.side[s];
            side.dy = dy[s]->ptr, side.dy_b = dy[s]->stride[0], side.dy_s = dy[s]->stride[1], side.dy_n = dy[s]->stride[2], side.dy_h = dy[s]->stride[3];
            side.out = dx[s]->ptr, side.out_b = dx[s]->stride[0], side.out_s = dx[s]->stride[1], side.out_n = dx[s]->stride[2], side.out_h = dx[s]->stride[3];
            if (!w[s] != !dw[s]) lb::refuse("a weight has a gradient, and no weight has none");
            if (dw[s]) {
                lb::same_shape(*w[s], *dw[s], "a weight's gradient");
                if (c.p.H > 1 && dw[s]->stride[0] != 1) lb::refuse("a weight's gradient must be dense");
                side.dw = dw[s]->ptr;
            }
        }
        if (c.p.side[0].w || c.p.side[1].w) {
            const size_t need = lb::scratch_bytes(c.p.H);
            if (!scratch || scratch_bytes < need || (uintptr_t)scratch % 16) lb::refuse(lb::format("the weights' gradients need %zu bytes of scratch, 16-byte aligned", need));
            c.p.side[0].partial = (float*)scratch;
            c.p.side[1].partial = (float*)((char*)scratch + need / 2);
        }
        const lb::Result results[] = {{d_q, "the queries' gradient", {0, 2}}, {d_k, "the keys' gradient", {1, 3}}, {d_q_weight, "the queries' weight's gradient", {7, 7}},
                                      {d_k_weight, "the keys' weight's gradient", {8, 8}}};  // (the weights' are written by a second kernel)
        const lb::Operand operands[] = {{q, "the queries"}, {k, "the keys"}, {d_q_out, "the gradient of the queries' result"}, {d_k_out, "the gradient of the keys' result"}, {cos, "cos"},
                                        {sin, "sin"}, {positions, "positions"}, {q_weight, "the queries' weight"}, {k_weight, "the keys' weight"}};
        lb::keep_apart(results, 4, operands, 9);
        if (c.rows || c.p.side[0].w || c.p.side[1].w) lb::run_rope<true>(c, stream);
    });
}
}
