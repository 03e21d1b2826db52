// Products of a few tokens (up to 32) with a weight matrix, and the gated block's: the weights are read once, and that is what a call costs.
//
// out [M, N] = x [M, K] w^T with w [N, K], rows along K. A block takes 16 rows of w (of the gated block eight of each weight) or, where that leaves SMs
// without a block, eight, its warps a range of K each; partial sums meet in shared memory and are added in the warps' order. The rows go from
// global memory into registers in the layout of mma.sync's first operand and the tokens into that of its second (16 x 8 tiles: tokens are the
// short side, and no tile of a tcgen05 product is shorter than 128 rows): which eight elements along K a lane holds is free as long as both sides
// agree, so that each of its loads is 16 contiguous bytes. Up to 24 loads of a lane are in flight.
//
// Bound by the bytes of w, the time a load takes to arrive and, with more tokens, by reading those from the L2: 4 tokens with weights of 1024 x 4096 take 5.7 us
// for both halves of the gated block where the weights' 25 MB are in the L2, 4.5 TB/s.
#include <algorithm>

#include "gate.cuh"
#include "gemm.h"
#include "launch.cuh"

namespace lb {
namespace {

constexpr int kMaxWarps = 16, kMaxTokens = 32;
// 32-wide blocks of K a warp has in flight: 96 registers of each lane, 64 and 96
constexpr int ahead(int tokens) { return tokens == 8 ? 8 : 4; }

// 16 bytes, or zeros; in the order that these are written in, ahead of the products. STREAM: not to be read again soon.
template <bool STREAM>
__device__ __forceinline__ uint4 load_if(const void* at, bool there) {
    uint4 v;
    if (STREAM)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %5, 0;\n\tmov.b32 %0, 0;\n\tmov.b32 %1, 0;\n\tmov.b32 %2, 0;\n\tmov.b32 %3, 0;\n\t"
                     "@p ld.global.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];\n\t}"
                     : "=&r"(v.x), "=&r"(v.y), "=&r"(v.z), "=&r"(v.w)
                     : "l"(__cvta_generic_to_global(at)), "r"((int)there));
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %5, 0;\n\tmov.b32 %0, 0;\n\tmov.b32 %1, 0;\n\tmov.b32 %2, 0;\n\tmov.b32 %3, 0;\n\t"
                     "@p ld.global.v4.b32 {%0, %1, %2, %3}, [%4];\n\t}"
                     : "=&r"(v.x), "=&r"(v.y), "=&r"(v.z), "=&r"(v.w)
                     : "l"(__cvta_generic_to_global(at)), "r"((int)there));
    return v;
}

struct SkinnyArgs {
    const void *x, *w;
    long long ld_x, ld_w;
    void* out;        // h or y
    void* kept;       // gated: both projections side by side; null: not kept
    const void* add;  // plain: a residual, added to the rounded sum
    long long ld_out, ld_kept, ld_add;
    int M, N, K;      // N: columns of `out`
    int warps, per_warp;  // 32-wide blocks of K a warp takes
    int act;
};

template <bool F16>
__device__ __forceinline__ void mma_16x8(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if (F16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <bool F16>
__device__ __forceinline__ uint16_t round16(float x) {
    return F16 ? __half_as_ushort(__float2half_rn(x)) : __bfloat16_as_ushort(__float2bfloat16_rn(x));
}
template <bool F16>
__device__ __forceinline__ float widen16(uint16_t x) {
    return F16 ? __half2float(__ushort_as_half(x)) : __uint_as_float((uint32_t)x << 16);
}

struct SkinnyLossArgs : SkinnyArgs {
    Targets targets;
    SpanSum* spans;  // [block][M]
    float* hit;
};

// PLAIN, GATED, LOSS: a product; the gated block's; the linear cross entropy's span sums, of which a block's classes are one: 4 tokens of 1024 x 32768 take 10.1 us, 6.6 TB/s.
enum SkinnyKind : int { SKINNY_PLAIN, SKINNY_GATED, SKINNY_LOSS };

// GATED: rows 0..7 of a tile are the gate's, 8..15 the other projection's. ROWS: 16, or 8 with the tile's second half empty. TOKENS: 8, 16 or 32.
template <SkinnyKind KIND, bool F16, int ROWS, int TOKENS, class Args>
__global__ void __launch_bounds__(kMaxWarps * 32, 1) skinny_kernel(const Args p) {
    constexpr bool GATED = KIND == SKINNY_GATED;
    __shared__ float sums[kMaxWarps][16][TOKENS + 1];
    grid_wait();
    constexpr int TILES = TOKENS / 8;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int row0 = blockIdx.x * (GATED ? 8 : ROWS);
    // the lane's rows of w, its tokens
    const bool low = row0 + g < p.N, high = ROWS == 16 && (GATED ? low : row0 + 8 + g < p.N);
    const uint16_t* w_low = (const uint16_t*)p.w + (long long)(low ? row0 + g : 0) * p.ld_w + 8 * t;
    const uint16_t* w_high = (const uint16_t*)p.w + (high ? (long long)row0 + g + (GATED ? p.N : 8) : 0) * p.ld_w + 8 * t;
    const uint16_t* token[TILES];
    bool there[TILES];
#pragma unroll
    for (int n = 0; n < TILES; n++) there[n] = 8 * n + g < p.M, token[n] = (const uint16_t*)p.x + (long long)(there[n] ? 8 * n + g : 0) * p.ld_x + 8 * t;
    float acc[TILES][4] = {};
    constexpr int AHEAD = ahead(TOKENS);
    const int blocks = (p.K + 31) / 32, first = warp * p.per_warp, last = min(blocks, first + p.per_warp);
    for (int k0 = first; k0 < last; k0 += AHEAD) {
        uint4 a[AHEAD], b[AHEAD], x[AHEAD][TILES];
#pragma unroll
        for (int i = 0; i < AHEAD; i++) {
            const int k = (k0 + i) * 32;
            const bool in = k0 + i < last && k + 8 * t < p.K;
            a[i] = load_if<true>(w_low + k, in && low);
            b[i] = ROWS == 16 ? load_if<true>(w_high + k, in && high) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
            for (int n = 0; n < TILES; n++) x[i][n] = load_if<false>(token[n] + k, in && there[n]);
        }
#pragma unroll
        for (int i = 0; i < AHEAD; i++) {
#pragma unroll
            for (int n = 0; n < TILES; n++) {
                mma_16x8<F16>(acc[n], a[i].x, b[i].x, a[i].y, b[i].y, x[i][n].x, x[i][n].y);
                mma_16x8<F16>(acc[n], a[i].z, b[i].z, a[i].w, b[i].w, x[i][n].z, x[i][n].w);
            }
        }
    }
#pragma unroll
    for (int n = 0; n < TILES; n++) {
        sums[warp][g][8 * n + 2 * t] = acc[n][0], sums[warp][g][8 * n + 2 * t + 1] = acc[n][1];
        if (ROWS == 16) sums[warp][8 + g][8 * n + 2 * t] = acc[n][2], sums[warp][8 + g][8 * n + 2 * t + 1] = acc[n][3];
    }
    __syncthreads();
    constexpr int COLS = GATED ? 8 : ROWS;
    for (int i = threadIdx.x; i < COLS * TOKENS; i += blockDim.x) {
        const int c = i % COLS, m = i / COLS;
        if constexpr (KIND == SKINNY_LOSS) {  // COLS lanes a token
            float z = 0.0f;
            for (int k = 0; k < p.warps; k++) z += sums[k][c][m];
            const bool in = row0 + c < p.N;
            float most = in ? z : -INFINITY;
#pragma unroll
            for (int d = COLS / 2; d; d >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, d));
            const float base = most == -INFINITY ? 0.0f : most;
            float sum = in ? exp2_approx((z - base) * kLog2e) : 0.0f;
#pragma unroll
            for (int d = COLS / 2; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
            if (m < p.M) {
                if (c == 0) p.spans[(long long)blockIdx.x * p.M + m] = SpanSum{most, sum};
                if (in && p.targets.of(m) == row0 + c) p.hit[m] = z;
            }
            continue;
        }
        if (m >= p.M || row0 + c >= p.N) continue;
        float a = 0.0f, b = 0.0f;
        for (int k = 0; k < p.warps; k++) {
            a += sums[k][c][m];
            if (GATED) b += sums[k][8 + c][m];
        }
        uint16_t* out = (uint16_t*)p.out + m * p.ld_out + row0 + c;
        if (GATED) {
            const float h = (p.act == ACT_SILU ? activation<ACT_SILU, true>(a) : p.act == ACT_GELU ? activation<ACT_GELU, true>(a) : activation<ACT_RELU, true>(a)) * b;
            *out = round16<F16>(h);
            if (p.kept) {
                uint16_t* kept = (uint16_t*)p.kept + m * p.ld_kept + row0 + c;
                kept[0] = round16<F16>(a), kept[p.N] = round16<F16>(b);
            }
        } else {
            uint16_t y = round16<F16>(a);
            if (p.add) y = round16<F16>(__fadd_rn(widen16<F16>(((const uint16_t*)p.add)[m * p.ld_add + row0 + c]), widen16<F16>(y)));
            *out = y;
        }
    }
}

// Rows of a block's tile: 16 where three quarters of the SMs get one, else 8. us of a gated block of 1 and 8 tokens in a graph, 8 -> 16: 512 columns 3.7, 4.1 -> 4.1,
// 4.5; 1024 5.2, 6.2 -> 5.8, 6.9; 2048 21.6, 23.1 -> 20.0, 21.1; 2400 26.2, 25.3 -> 25.8, 24.5; 4096 72.2, 74.2 -> 67.3, 66.7
int skinny_rows(long long N, int sms) { return (N + 15) / 16 * 4 >= 3 * sms ? 16 : 8; }

template <SkinnyKind KIND, bool F16, class Args>
void launch_skinny(Args& p, int sms, cudaStream_t s) {
    constexpr bool GATED = KIND == SKINNY_GATED;
    const int blocks = (p.K + 31) / 32;
    // a warp takes some blocks of K at a time, all of them in flight: as many warps as that needs
    const int at_once = ahead(p.M <= 8 ? 8 : p.M <= 16 ? 16 : 32);
    p.warps = std::min(kMaxWarps, (blocks + at_once - 1) / at_once);
    p.per_warp = (blocks + p.warps - 1) / p.warps;
    const int rows = GATED ? 8 : skinny_rows(p.N, sms);
    const dim3 grid((unsigned)((p.N + rows - 1) / rows)), block((unsigned)p.warps * 32);
    auto go = [&](auto kernel) { launch_overlapped(kernel, grid, block, 0, s, 0, p); };
    if (GATED || rows == 16) {
        if (p.M <= 8) go(skinny_kernel<KIND, F16, 16, 8, Args>);
        else if (p.M <= 16) go(skinny_kernel<KIND, F16, 16, 16, Args>);
        else go(skinny_kernel<KIND, F16, 16, 32, Args>);
    } else if constexpr (!GATED) {
        if (p.M <= 8) go(skinny_kernel<KIND, F16, 8, 8, Args>);
        else if (p.M <= 16) go(skinny_kernel<KIND, F16, 8, 16, Args>);
        else go(skinny_kernel<KIND, F16, 8, 32, Args>);
    }
}

// The rows of an operand along K in 16-byte pieces.
bool rows_in_pieces(const lb_tensor& t) { return (uintptr_t)t.ptr % 16 == 0 && t.stride[1] == 1 && (t.shape[0] <= 1 || t.stride[0] % 8 == 0); }

SkinnyArgs skinny_args(const lb_tensor& x, const lb_tensor& w, const lb_tensor& out) {
    SkinnyArgs p{};
    p.x = x.ptr, p.ld_x = x.stride[0], p.w = w.ptr, p.ld_w = w.stride[0], p.out = out.ptr, p.ld_out = out.stride[0];
    p.M = (int)x.shape[0], p.K = (int)x.shape[1], p.N = (int)out.shape[1];
    return p;
}

}  // namespace

// Every block reads all tokens, from the L2: with more than eight of them that is what grows, and beyond 64 MB of it 128-row tiles are the better choice.
// us of a gated block in a graph, bfloat16, width x hidden, tiles -> these: 4 tokens 1024 x 4096 22.4 -> 5.7, 16 (17 MB) 22.2 -> 9.1, 32 (34 MB) 22.1 -> 12.9,
// 32 of 512 x 2048 12.8 -> 6.4, 4 of 2048 x 8192 33.5 -> 20.5; 9 of it (38 MB) 32 -> 29.8, 16 (67 MB) 31.9 -> 32.6, 32 (134 MB) 28.8 -> 47.0.
bool skinny_takes(const lb_tensor& x, const lb_tensor& w) {
    const long long M = x.shape[0], K = x.shape[1], N = w.shape[0];
    return M <= kMaxTokens && K % 8 == 0 && (x.dtype == LB_BF16 || x.dtype == LB_F16) && rows_in_pieces(x) && rows_in_pieces(w) &&
           (M <= 8 || M * K * 2 * (N / 16) < 64LL << 20);
}
void skinny_gated(const lb_tensor& x, const lb_tensor& w, const lb_tensor& h, const lb_tensor* kept, int act, void* stream) {
    driver();
    SkinnyArgs p = skinny_args(x, w, h);
    p.act = act;
    if (kept) p.kept = kept->ptr, p.ld_kept = kept->stride[0];
    if (x.dtype == LB_F16) launch_skinny<SKINNY_GATED, true>(p, device_info().sms, (cudaStream_t)stream);
    else launch_skinny<SKINNY_GATED, false>(p, device_info().sms, (cudaStream_t)stream);
}
void skinny_product(const lb_tensor& x, const lb_tensor& w, const lb_tensor& out, const lb_tensor* add, void* stream) {
    driver();
    SkinnyArgs p = skinny_args(x, w, out);
    if (add) p.add = add->ptr, p.ld_add = add->stride[0];
    if (x.dtype == LB_F16) launch_skinny<SKINNY_PLAIN, true>(p, device_info().sms, (cudaStream_t)stream);
    else launch_skinny<SKINNY_PLAIN, false>(p, device_info().sms, (cudaStream_t)stream);
}

int skinny_spans(long long N) {
    const int rows = skinny_rows(N, sm_count_hint());
    return (int)((N + rows - 1) / rows);
}
void skinny_loss(const lb_tensor& x, const lb_tensor& w, const Targets& targets, SpanSum* spans, float* hit, void* stream) {
    driver();
    SkinnyLossArgs p{};
    (SkinnyArgs&)p = skinny_args(x, w, w);
    p.N = (int)w.shape[0], p.out = nullptr, p.targets = targets, p.spans = spans, p.hit = hit;
    if (x.dtype == LB_F16) launch_skinny<SKINNY_LOSS, true>(p, sm_count_hint(), (cudaStream_t)stream);
    else launch_skinny<SKINNY_LOSS, false>(p, sm_count_hint(), (cudaStream_t)stream);
}

}  // namespace lb
