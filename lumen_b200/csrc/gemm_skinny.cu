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
#include "parts.cuh"

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

// The span sum of WIDTH lanes' logits.
template <int WIDTH>
__device__ __forceinline__ SpanSum span_of(float z, bool in) {
    float most = in ? z : -INFINITY;
#pragma unroll
    for (int d = WIDTH / 2; d; d >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, d));
    const float base = base_of(most);
    float sum = in ? exp2_approx((z - base) * kLog2e) : 0.0f;
#pragma unroll
    for (int d = WIDTH / 2; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    return {most, sum};
}

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
            const SpanSum sum = span_of<COLS>(z, in);
            if (m < p.M) {
                if (c == 0) p.spans[(long long)blockIdx.x * p.M + m] = sum;
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

struct FloatLossArgs : SkinnyLossArgs {
    float* logits;  // [M][ld_out], instead of the span sums; null: those
};

// The linear cross entropy's products of up to 32 float32 tokens, on the tensor cores: both operands go into registers as they are and become three parts of bfloat16 there, six of whose
// products are added up; those of the first parts by themselves, and both sums to what was before after every two blocks of K, rounded, since the tensor cores drop what lies below a sum's last
// place. A block's ROWS classes are a span.
//
// Bound by the time that loads take and, with more tokens, by parting x, which every block does anew, and the products. us in a graph for 8, 16 and 32 tokens; the weights' bytes alone; what the
// CUDA cores and, from 17 on, the parts in memory took:
//   1024 x 32768    32, 43, 68     20.5   46, 71, 127
//   344 x 116036    53, 65, 110    24.4   64, 95, 207
//   3576 x 12593    40, 54, 91     27.5   87, 157, 342
// Two blocks of K on their way: with three 10 - 15 % more, with four and six as much, since fewer warps find a place.
constexpr int kFloatWarps = 8, kFloatAhead = 2;
template <int ROWS, int TOKENS>
__global__ void __launch_bounds__(kFloatWarps * 32, 2) skinny_float_kernel(const FloatLossArgs p) {
    __shared__ float sums[kFloatWarps][ROWS][TOKENS + 1];
    grid_wait();
    constexpr int TILES = TOKENS / 8, EIGHTS = ROWS / 8, AHEAD = kFloatAhead, PAIR = TILES < 2 ? 1 : 2;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, row0 = blockIdx.x * ROWS;
    const float *w[EIGHTS], *token[TILES];
    bool row_in[EIGHTS], token_in[TILES];
#pragma unroll
    for (int h = 0; h < EIGHTS; h++) row_in[h] = row0 + 8 * h + g < p.N, w[h] = (const float*)p.w + (long long)(row_in[h] ? row0 + 8 * h + g : 0) * p.ld_w + 4 * t;
#pragma unroll
    for (int n = 0; n < TILES; n++) token_in[n] = 8 * n + g < p.M, token[n] = (const float*)p.x + (long long)(token_in[n] ? 8 * n + g : 0) * p.ld_x + 4 * t;
    float all[ROWS / 16][TILES][4];
    const int blocks = (p.K + 15) / 16, first = warp * p.per_warp, last = min(blocks, first + p.per_warp);
    // The warp's sums; whether the lane's are finite. ANY: see parts_of.
    auto pass = [&](auto any) {
        constexpr bool ANY = decltype(any)::value;
#pragma unroll
        for (int m = 0; m < ROWS / 16; m++)
#pragma unroll
            for (int n = 0; n < TILES; n++)
#pragma unroll
                for (int j = 0; j < 4; j++) all[m][n][j] = 0.0f;
        constexpr int PLACES = ANY ? 1 : AHEAD;
        uint4 a[PLACES][EIGHTS], x[PLACES][TILES];  // in turn: a place is loaded anew as soon as it has been used
        auto load = [&](int i, int block) {
            const int k = block * 16;
            const bool in = block < last && k + 4 * t < p.K;
#pragma unroll
            for (int h = 0; h < EIGHTS; h++) a[i][h] = load_if<true>(w[h] + k, in && row_in[h]);
#pragma unroll
            for (int n = 0; n < TILES; n++) x[i][n] = load_if<false>(token[n] + k, in && token_in[n]);
        };
#pragma unroll
        for (int i = 0; i < PLACES && !ANY; i++) load(i, first + i);
        for (int k0 = first; k0 < last; k0 += AHEAD) {
            float most[ROWS / 16][TILES][4] = {}, rest[ROWS / 16][TILES][4] = {};
#pragma unroll(ANY ? 1 : AHEAD)
            for (int step = 0; step < AHEAD; step++) {
                const int i = ANY ? 0 : step;
                if (ANY) load(i, k0 + step);
                uint32_t ap[EIGHTS][3][2];
#pragma unroll
                for (int h = 0; h < EIGHTS; h++) parts_of<ANY>((const float*)&a[i][h], ap[h]);
#pragma unroll
                for (int n0 = 0; n0 < TILES; n0 += PAIR) {  // tiles and products in an order that has none wait for the one before
                    uint32_t b[PAIR][3][2];
#pragma unroll
                    for (int n = 0; n < PAIR; n++) parts_of<ANY>((const float*)&x[i][n0 + n], b[n]);
                    auto add = [&](float (*d)[TILES][4], int u, int v) {
#pragma unroll
                        for (int n = 0; n < PAIR; n++)
#pragma unroll
                            for (int m = 0; m < ROWS / 16; m++)
                                mma_16x8<false>(d[m][n0 + n], ap[2 * m][u][0], ap[2 * m + 1][u][0], ap[2 * m][u][1], ap[2 * m + 1][u][1], b[n][v][0], b[n][v][1]);
                    };
                    add(rest, 0, 2), add(most, 0, 0), add(rest, 2, 0), add(rest, 1, 1), add(rest, 0, 1), add(rest, 1, 0);
                }
                if (!ANY) load(i, k0 + AHEAD + i);
            }
#pragma unroll
            for (int m = 0; m < ROWS / 16; m++)
#pragma unroll
                for (int n = 0; n < TILES; n++)
#pragma unroll
                    for (int j = 0; j < 4; j++) all[m][n][j] += most[m][n][j] + rest[m][n][j];
        }
        bool finite = true;
#pragma unroll
        for (int m = 0; m < ROWS / 16; m++)
#pragma unroll
            for (int n = 0; n < TILES; n++)
#pragma unroll
                for (int j = 0; j < 4; j++) finite = finite && fabsf(all[m][n][j]) < INFINITY;
        return finite;
    };
    // A value that is infinite, or is rounded to it, leaves NaN in its whole row of sums. That is rare enough to be met by going over all of it again (looked for in the loop, 16
    // tokens of 1024 x 32768 took 61 us where they take 51, the L2 empty).
    if (!__all_sync(0xffffffffu, pass(std::false_type{}))) pass(std::true_type{});
#pragma unroll
    for (int m = 0; m < ROWS / 16; m++)
#pragma unroll
        for (int n = 0; n < TILES; n++)
#pragma unroll
            for (int j = 0; j < 4; j++) sums[warp][16 * m + 8 * (j / 2) + g][8 * n + 2 * t + j % 2] = all[m][n][j];
    __syncthreads();
    for (int i = threadIdx.x; i < ROWS * TOKENS; i += blockDim.x) {
        const int c = i % ROWS, m = i / ROWS;
        float z = 0.0f;
        for (int k = 0; k < p.warps; k++) z += sums[k][c][m];
        const bool in = row0 + c < p.N;
        if (p.logits) {
            if (in && m < p.M) p.logits[m * p.ld_out + row0 + c] = z;
            continue;
        }
        const SpanSum sum = span_of<ROWS>(z, in);
        if (m < p.M) {
            if (c == 0) p.spans[(long long)blockIdx.x * p.M + m] = sum;
            if (in && p.targets.of(m) == row0 + c) p.hit[m] = z;
        }
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

// One token, and up to four with short rows, are faster on the CUDA cores, whose loads are a warp's whole row: 1 token 31 us there and 33 here with 1024 x 32768, 22.5 and 29 with 200 x 93558,
// 36 and 46 with 3576 x 12593; 4 tokens 40 and 33, 24 and 29.6, 58 and 46.
bool skinny_float_takes(const lb_tensor& x, const lb_tensor& w) {
    if (x.shape[0] == 1 || (x.shape[0] <= 4 && x.shape[1] < 512)) return false;
    auto in_pieces = [](const lb_tensor& t) { return (uintptr_t)t.ptr % 16 == 0 && t.stride[1] == 1 && (t.shape[0] <= 1 || t.stride[0] % 4 == 0); };
    return x.dtype == LB_F32 && x.shape[0] <= kMaxTokens && x.shape[1] % 4 == 0 && in_pieces(x) && in_pieces(w);
}
// Classes of a block: 32 where that leaves every SM one and the tokens' sums leave the registers for it (32 tokens of 1024 x 32768 75 us with 16, 94 with 32; 8 of them 38 and 33).
static int float_rows(long long M, long long N) { return M <= 16 && N >= 32LL * sm_count_hint() ? 32 : 16; }
int skinny_float_spans(long long M, long long N) { return (int)((N + float_rows(M, N) - 1) / float_rows(M, N)); }
void skinny_float_loss(const lb_tensor& x, const lb_tensor& w, const Targets& targets, SpanSum* spans, float* hit, float* logits, long long ld, void* stream) {
    driver();
    FloatLossArgs p{};
    (SkinnyArgs&)p = skinny_args(x, w, w);
    p.N = (int)w.shape[0], p.out = nullptr, p.targets = targets, p.spans = spans, p.hit = hit, p.logits = logits, p.ld_out = ld;
    const int rows = float_rows(p.M, p.N), tiles = (p.N + rows - 1) / rows, blocks = (p.K + 15) / 16;
    // four warps, so that blocks start and end at different times; eight where there are too few blocks for that (8 tokens of 4096 x 2000 14.4 us with four, 12.5 with eight; 344 x 116036 51 and 68)
    const int warps = tiles <= 2 * sm_count_hint() ? kFloatWarps : kFloatWarps / 2;
    p.warps = std::min(warps, blocks);  // (those of K; the others share what is behind)
    p.per_warp = (blocks + p.warps - 1) / p.warps;
    auto go = [&](auto kernel) { launch_overlapped(kernel, dim3((unsigned)tiles), dim3((unsigned)warps * 32), 0, (cudaStream_t)stream, 0, p); };
    if (rows == 32) p.M <= 8 ? go(skinny_float_kernel<32, 8>) : go(skinny_float_kernel<32, 16>);
    else p.M <= 8 ? go(skinny_float_kernel<16, 8>) : p.M <= 16 ? go(skinny_float_kernel<16, 16>) : go(skinny_float_kernel<16, 32>);
}

}  // namespace lb
