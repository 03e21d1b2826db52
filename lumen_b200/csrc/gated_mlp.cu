// The gated feed-forward block of M tokens: a = x Wg^T, b = x Wu^T, h = f(a) b, y = h Wd^T (+ residual), and its backward pass
// dh = dy Wd, da = dh b f'(a), db = dh f(a), dx = [da db] [Wg; Wu], d[Wg; Wu] = [da db]^T x, dWd = dy^T h.
//
// Wg and Wu are one matrix of 2 F rows, so that the last three are single products with float32 sums over all they add up. [a b] is kept for the
// backward pass in the operands' dtype; h is computed from the float32 sums, not from what was kept. [da db] is rounded to the operands'
// dtype, as an operand of the tensor cores has to be.
#include <algorithm>
#include <initializer_list>

#include "convert.cuh"
#include "gate.cuh"
#include "gemm.h"
#include "launch.cuh"
#include "overlap.h"

namespace lb {
bool gemm(const lb_tensor& a, const lb_tensor& b, const lb_tensor& d, int epilogue, int kernel_choice, void* stream, void* scratch, size_t scratch_bytes,
          const lb_tensor* aux, const GemmTuning* tuning, SimtProblem* held = nullptr);

namespace {

[[noreturn]] void refuse(const std::string& why) { fail(LB_ERR_INVALID, "gated_mlp: " + why); }

template <class T, int V>
struct alignas(sizeof(T) * V) Pack {
    T v[V];
};

struct GateArgs {
    const void* in;        // forward: [a b], backward: dh; float32
    const void* gate_up;   // backward: [a b]
    void* gate_up_out;     // forward: [a b] rounded (null: not kept), backward: [da db]
    void* h;               // forward
    long long ld_in, ld_gate_up, ld_out, ld_h;
    int M, F;
};

// What lies between the products where they do not do it themselves: V columns of a row a thread, rows in turn over the grid. Bound by memory.
template <class T, int V, int ACT, bool BWD>
__global__ void __launch_bounds__(256) gate_kernel(const GateArgs p) {
    grid_wait();
    const int col = ((int)blockIdx.x * blockDim.x + threadIdx.x) * V;
    if (col >= p.F) return;
    constexpr bool FAST = sizeof(T) == 2;
    for (long long row = (long long)blockIdx.y * blockDim.y + threadIdx.y; row < p.M; row += (long long)gridDim.y * blockDim.y) {
        const float* in = (const float*)p.in + row * p.ld_in + col;
        if (!BWD) {
            const Pack<float, V> a = *(const Pack<float, V>*)in, b = *(const Pack<float, V>*)(in + p.F);
            Pack<T, V> h, a16, b16;
#pragma unroll
            for (int j = 0; j < V; j++) h.v[j] = from_float<T>(activation<ACT, FAST>(a.v[j]) * b.v[j]), a16.v[j] = from_float<T>(a.v[j]), b16.v[j] = from_float<T>(b.v[j]);
            *(Pack<T, V>*)((T*)p.h + row * p.ld_h + col) = h;
            if (p.gate_up_out) {
                T* out = (T*)p.gate_up_out + row * p.ld_out + col;
                *(Pack<T, V>*)out = a16, *(Pack<T, V>*)(out + p.F) = b16;
            }
        } else {
            const T* kept = (const T*)p.gate_up + row * p.ld_gate_up + col;
            const Pack<float, V> dh = *(const Pack<float, V>*)in;
            const Pack<T, V> a = *(const Pack<T, V>*)kept, b = *(const Pack<T, V>*)(kept + p.F);
            Pack<T, V> da, db;
#pragma unroll
            for (int j = 0; j < V; j++) {
                float slope;
                const float value = activation_slope<ACT, FAST>(to_float(a.v[j]), slope);
                da.v[j] = from_float<T>(dh.v[j] * to_float(b.v[j]) * slope), db.v[j] = from_float<T>(dh.v[j] * value);
            }
            T* out = (T*)p.gate_up_out + row * p.ld_out + col;
            *(Pack<T, V>*)out = da, *(Pack<T, V>*)(out + p.F) = db;
        }
    }
}

template <class T, bool BWD>
void run_gate(const GateArgs& p, int act, cudaStream_t s) {
    auto vec = [&](const void* ptr, long long ld, int item) { return !ptr || ((uintptr_t)ptr % (4 * item) == 0 && ld % 4 == 0); };
    const int item = (int)sizeof(T);
    const bool whole = p.F % 4 == 0 && vec(p.in, p.ld_in, 4) && vec(p.gate_up, p.ld_gate_up, item) && vec(p.gate_up_out, p.ld_out, item) && vec(p.h, p.ld_h, item);
    const int cols = whole ? (p.F + 3) / 4 : p.F;
    int tx = 32;
    while (tx < 256 && tx < cols) tx *= 2;
    const dim3 block((unsigned)tx, (unsigned)(256 / tx));
    const unsigned gx = (unsigned)((cols + tx - 1) / tx);
    const long long rows = (p.M + block.y - 1) / block.y;
    const dim3 grid(gx, (unsigned)std::min<long long>(rows, std::max(1u, (unsigned)device_info().sms * 16 / gx)));
    auto go = [&](auto kernel4, auto kernel1) {
        auto kernel = whole ? kernel4 : kernel1;
        launch_overlapped(kernel, grid, block, 0, s, 0, p);
    };
    if (act == ACT_SILU) go(gate_kernel<T, 4, ACT_SILU, BWD>, gate_kernel<T, 1, ACT_SILU, BWD>);
    else if (act == ACT_GELU) go(gate_kernel<T, 4, ACT_GELU, BWD>, gate_kernel<T, 1, ACT_GELU, BWD>);
    else go(gate_kernel<T, 4, ACT_RELU, BWD>, gate_kernel<T, 1, ACT_RELU, BWD>);
}
template <bool BWD>
void run_gate(int dtype, const GateArgs& p, int act, cudaStream_t s) {
    if (p.M == 0 || p.F == 0) return;
    if (dtype == LB_F32) run_gate<float, BWD>(p, act, s);
    else if (dtype == LB_BF16) run_gate<__nv_bfloat16, BWD>(p, act, s);
    else run_gate<__half, BWD>(p, act, s);
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
// A tensor of rank 2 and more as the matrix of its rows, which have to be evenly spaced.
lb_tensor as_rows(const lb_tensor* t, const char* what) {
    if (!t) refuse(format("%s is missing", what));
    if (t->rank < 2 || t->rank > LB_MAX_RANK) refuse(format("%s must have rank 2 or more", what));
    const int last = t->rank - 1;
    long long rows = 1, step = 0;
    for (int d = 0; d < t->rank; d++)
        if (t->shape[d] < 0) refuse(format("%s has a negative size", what));
    for (int d = 0; d < last; d++)
        if (t->shape[d] == 0) rows = 0;  // no rows: nothing about their spacing
    for (int d = last - 1; d >= 0 && rows; d--) {
        if (t->shape[d] == 1) continue;
        if (rows != 1 && t->stride[d] != step * rows) fail(LB_ERR_UNSUPPORTED, format("gated_mlp: the rows of %s are not evenly spaced", what));
        if (rows == 1) step = t->stride[d];
        rows *= t->shape[d];
    }
    lb_tensor m = matrix(t->ptr, t->dtype, rows, t->shape[last], step);
    m.stride[1] = t->stride[last];
    if (rows <= 1) m.stride[0] = m.stride[1] == 1 ? m.shape[1] : 1;
    return m;
}
void written(const lb_tensor& t, const char* what) {
    if (t.shape[1] > 1 && t.stride[1] != 1) fail(LB_ERR_UNSUPPORTED, format("gated_mlp: %s must be row-major", what));
    if (t.shape[0] > 1 && t.stride[0] < t.shape[1]) refuse(format("the rows of %s overlap", what));
}
void sized(const lb_tensor& t, long long rows, long long cols, int dtype, const char* what) {
    if (t.shape[0] != rows || t.shape[1] != cols || t.dtype != dtype)
        refuse(format("%s must be [%lld, %lld] of the operands' dtype, got %s[%lld, %lld]", what, rows, cols, dtype_name(t.dtype), (long long)t.shape[0], (long long)t.shape[1]));
    if (rows && cols && (!t.ptr || (uintptr_t)t.ptr % dtype_size(dtype))) refuse(format("%s has no memory or is not aligned to its elements", what));
}
// What is written shares no memory with what is read, or written.
void keep_apart(std::initializer_list<const lb_tensor*> results, std::initializer_list<const lb_tensor*> operands) {
    Extent read[8], written[4];
    int k = 0, r = 0;
    for (const lb_tensor* o : operands) read[k++] = extent(*o);
    for (auto out = results.begin(); out != results.end(); ++out, r++) {
        written[r] = extent(**out);
        k = 0;
        for (const lb_tensor* o : operands)
            if (written[r].meets(read[k++]) && share_memory(**out, *o)) refuse("a result shares memory with an operand");
        k = 0;
        for (auto other = results.begin(); other != out; ++other)
            if (written[r].meets(written[k++]) && share_memory(**out, **other)) refuse("two results share memory");
    }
}

// Whether the pairs' products with the gate in their epilogue are taken, where the layouts are theirs and (forward) narrow tiles are too many: where enough SMs
// get a tile (of 128 rows by 128 columns of h, backward by 256), since lb_gemm's own choices cut K and take narrower tiles. us of a pass in a graph, products apart -> these, bfloat16, width x hidden:
// forward 200 tokens 512 x 2048 (32 tiles) 17.6 -> 20.3, 128 of 1024 x 4096 (32) 20.6 -> 24.4, 384 of 512 x 2048 (48) 17.4 -> 16.0, 200 of 1024 x 4096 (64)
// 21.4 -> 20.1, 128 of 2048 x 8192 (64) 36.1 -> 31.5, 1024 of 1024 x 4096 41.7 -> 34.4; backward 200 of 1024 x 4096 (32) 35.1 -> 39.3, 384 (48) 46.5 -> 47.1,
// 512 (64) 51.5 -> 50.8, 1024 of 512 x 2048 (64) 39.4 -> 38.9, 200 of 2048 x 8192 (64) 77.9 -> 79.6, 1024 of it 177 -> 174, 16384 of 1024 x 4096 837 -> 761.
bool gated_tiles(long long M, long long F) { return (M + 127) / 128 * ((F + 127) / 128) >= 48; }
bool sloped_tiles(long long M, long long F) { return (M + 127) / 128 * ((F + 255) / 256) >= 64; }

size_t up(size_t bytes) { return (bytes + 255) / 256 * 256; }
size_t product_scratch(const lb_tensor& a, const lb_tensor& b) { return lb_gemm_operands_scratch_bytes(&a, &b); }

// The operands of a call, checked, and where what lies between its kernels goes.
struct Block {
    int act, dtype;
    long long M, D, F;
    lb_tensor x, wgu, wd;
    void* scratch = nullptr;
    size_t products = 0;  // scratch of the products, behind the rest

    Block(int activation, const lb_tensor* x_t, const lb_tensor* wgu_t, const lb_tensor* wd_t) : act(activation) {
        if (act < ACT_SILU || act > ACT_RELU) refuse("unknown activation");
        x = as_rows(x_t, "x"), wgu = as_rows(wgu_t, "w_gate_up"), wd = as_rows(wd_t, "w_down");
        dtype = x.dtype;
        if (dtype != LB_F32 && dtype != LB_BF16 && dtype != LB_F16) refuse("float16, bfloat16 or float32 operands");
        if (wgu_t->rank != 2 || wd_t->rank != 2) refuse("the weights must have rank 2");
        wgu = *wgu_t, wd = *wd_t;
        M = x.shape[0], D = x.shape[1], F = wgu.shape[0] / 2;
        if (wgu.shape[0] % 2) refuse("w_gate_up must have an even number of rows: the gate's, then the other projection's");
        if (D < 1 || F < 1) refuse("a width or hidden size of zero");
        sized(x, M, D, dtype, "x"), sized(wgu, 2 * F, D, dtype, "w_gate_up"), sized(wd, D, F, dtype, "w_down");
        if (M > INT32_MAX || D > INT32_MAX || F > INT32_MAX / 2) fail(LB_ERR_UNSUPPORTED, "gated_mlp: sizes of at most 2^31 - 1");
    }
};

struct Forward : Block {
    lb_tensor y, gate_up{}, h;
    bool keeps, few = false, fused = false;
    size_t sums = 0;  // bytes of [a b] in float32

    Forward(int act, const lb_tensor* x_t, const lb_tensor* wgu_t, const lb_tensor* wd_t, const lb_tensor* y_t, const lb_tensor* gate_up_t, const lb_tensor* h_t)
        : Block(act, x_t, wgu_t, wd_t), y(as_rows(y_t, "y")), h(as_rows(h_t, "h")), keeps(gate_up_t) {
        sized(y, M, D, dtype, "y"), written(y, "y"), sized(h, M, F, dtype, "h"), written(h, "h");
        if (keeps) gate_up = as_rows(gate_up_t, "gate_up"), sized(gate_up, M, 2 * F, dtype, "gate_up"), written(gate_up, "gate_up");
        if (M == 0) return;
        few = skinny_takes(x, wgu) && skinny_takes(h, wd);
        if (few) return;
        fused = gemm_gated_takes(x, wgu, h, keeps ? &gate_up : nullptr) && (gemm_gated_ranges(x, wgu) || gated_tiles(M, F));
        if (!fused && (dtype != LB_F32 || !keeps)) sums = up((size_t)M * 2 * F * 4);
        products = std::max(fused ? 0 : product_scratch(x, transposed(wgu)), product_scratch(h, transposed(wd)));
    }
    size_t bytes() const { return sums + products; }
    void run(const lb_tensor* residual, void* stream) {
        char* more = (char*)scratch + sums;
        if (few) {
            skinny_gated(x, wgu, h, keeps ? &gate_up : nullptr, act, stream);
            skinny_product(h, wd, y, residual, stream);
            return;
        }
        if (fused) {
            gemm_gated(x, wgu, h, keeps ? &gate_up : nullptr, act, stream);
            gemm(h, transposed(wd), y, residual ? EPI_ADD : EPI_NONE, 0, stream, more, products, residual, nullptr);
            return;
        }
        const lb_tensor pre = sums ? matrix(scratch, LB_F32, M, 2 * F, 2 * F) : gate_up;
        gemm(x, transposed(wgu), pre, EPI_NONE, 0, stream, more, products, nullptr, nullptr);
        GateArgs g{};
        g.in = pre.ptr, g.ld_in = pre.stride[0], g.h = h.ptr, g.ld_h = h.stride[0], g.M = (int)M, g.F = (int)F;
        if (keeps && sums) g.gate_up_out = gate_up.ptr, g.ld_out = gate_up.stride[0];
        run_gate<false>(dtype, g, act, (cudaStream_t)stream);
        gemm(h, transposed(wd), y, residual ? EPI_ADD : EPI_NONE, 0, stream, more, products, residual, nullptr);
    }
};

struct Backward : Block {
    lb_tensor dy, gate_up, h, dx, dwgu, dwd;
    bool fused = false, grouped = false;
    size_t sums = 0, slopes = 0;  // bytes of dh in float32 and of [da db]

    Backward(int act, const lb_tensor* dy_t, const lb_tensor* x_t, const lb_tensor* wgu_t, const lb_tensor* wd_t, const lb_tensor* gate_up_t, const lb_tensor* h_t,
             const lb_tensor* dx_t, const lb_tensor* dwgu_t, const lb_tensor* dwd_t)
        : Block(act, x_t, wgu_t, wd_t), dy(as_rows(dy_t, "d_y")), gate_up(as_rows(gate_up_t, "gate_up")), h(as_rows(h_t, "h")), dx(as_rows(dx_t, "d_x")),
          dwgu(as_rows(dwgu_t, "d_w_gate_up")), dwd(as_rows(dwd_t, "d_w_down")) {
        sized(dy, M, D, dtype, "d_y"), sized(gate_up, M, 2 * F, dtype, "gate_up"), sized(h, M, F, dtype, "h");
        if (gate_up.stride[1] != 1) fail(LB_ERR_UNSUPPORTED, "gated_mlp: gate_up must be row-major");
        sized(dx, M, D, dtype, "d_x"), written(dx, "d_x");
        sized(dwgu, 2 * F, D, dtype, "d_w_gate_up"), written(dwgu, "d_w_gate_up"), sized(dwd, D, F, dtype, "d_w_down"), written(dwd, "d_w_down");
        fused = M && gemm_sloped_takes(dy, wd, gate_up, matrix(nullptr, dtype, M, 2 * F, 2 * F)) && (gemm_sloped_ranges(dy, wd) || sloped_tiles(M, F));
        sums = fused ? 0 : up((size_t)M * F * 4), slopes = up((size_t)M * 2 * F * dtype_size(dtype));
        const lb_tensor d = slope(), a[] = {d, transposed(d), transposed(dy)}, b[] = {wgu, x, h};
        grouped = M && gemm_group_pays(a, b, 3);
        products = fused ? 0 : product_scratch(dy, wd);
        for (int k = 0; k < 3 && !grouped; k++) products = std::max(products, product_scratch(a[k], b[k]));
    }
    lb_tensor slope() const { return matrix((char*)scratch + sums, dtype, M, 2 * F, 2 * F); }
    size_t bytes() const { return sums + slopes + products; }
    void run(void* stream) {
        char* more = (char*)scratch + sums + slopes;
        const lb_tensor d = slope();
        if (fused) {
            gemm_sloped(dy, wd, gate_up, d, act, stream);
        } else {
            const lb_tensor dh = matrix(scratch, LB_F32, M, F, F);
            gemm(dy, wd, dh, EPI_NONE, 0, stream, more, products, nullptr, nullptr);
            GateArgs g{};
            g.in = scratch, g.ld_in = F, g.gate_up = gate_up.ptr, g.ld_gate_up = gate_up.stride[0], g.gate_up_out = d.ptr, g.ld_out = 2 * F, g.M = (int)M, g.F = (int)F;
            run_gate<true>(dtype, g, act, (cudaStream_t)stream);
        }
        const lb_tensor a[] = {d, transposed(d), transposed(dy)}, b[] = {wgu, x, h}, out[] = {dx, dwgu, dwd};
        if (grouped) return gemm_group(a, b, out, 3, stream);
        for (int k = 0; k < 3; k++) gemm(a[k], b[k], out[k], EPI_NONE, 0, stream, more, products, nullptr, nullptr);
    }
};

void give_scratch(Block& b, size_t need, void* scratch, size_t bytes) {
    if (need && (!scratch || bytes < need || (uintptr_t)scratch % 16)) refuse(format("%zu bytes of scratch are needed, 16-byte aligned", need));
    b.scratch = scratch;
}

}  // namespace
}  // namespace lb

extern "C" {

int lb_gated_mlp_fwd_scratch_bytes(int activation, const lb_tensor* x, const lb_tensor* w_gate_up, const lb_tensor* w_down, const lb_tensor* y,
                                   const lb_tensor* gate_up, const lb_tensor* h, size_t* bytes) {
    return lb::guarded([&] {
        if (!bytes) lb::refuse("null argument");
        *bytes = lb::Forward(activation, x, w_gate_up, w_down, y, gate_up, h).bytes();
    });
}

int lb_gated_mlp_fwd(int activation, const lb_tensor* x, const lb_tensor* w_gate_up, const lb_tensor* w_down, const lb_tensor* residual, const lb_tensor* y,
                     const lb_tensor* gate_up, const lb_tensor* h, void* scratch, size_t scratch_bytes, void* stream) {
    return lb::guarded([&] {
        lb::Forward f(activation, x, w_gate_up, w_down, y, gate_up, h);
        lb_tensor r{};
        if (residual) {
            r = lb::as_rows(residual, "residual");
            lb::sized(r, f.M, f.D, f.dtype, "residual");
            if (f.dtype == LB_F32) lb::fail(LB_ERR_UNSUPPORTED, "gated_mlp: a residual is added to 16-bit results");
            if (r.stride[1] != 1 && f.D > 1) lb::fail(LB_ERR_UNSUPPORTED, "gated_mlp: residual must be row-major");
        }
        const lb_tensor& add = residual ? r : f.x;
        if (f.keeps) lb::keep_apart({&f.y, &f.h, &f.gate_up}, {&f.x, &f.wgu, &f.wd, &add});
        else lb::keep_apart({&f.y, &f.h}, {&f.x, &f.wgu, &f.wd, &add});
        lb::give_scratch(f, f.bytes(), scratch, scratch_bytes);
        if (f.M) f.run(residual ? &r : nullptr, stream);
    });
}

int lb_gated_mlp_bwd_scratch_bytes(int activation, const lb_tensor* d_y, const lb_tensor* x, const lb_tensor* w_gate_up, const lb_tensor* w_down,
                                   const lb_tensor* gate_up, const lb_tensor* h, const lb_tensor* d_x, const lb_tensor* d_w_gate_up, const lb_tensor* d_w_down,
                                   size_t* bytes) {
    return lb::guarded([&] {
        if (!bytes) lb::refuse("null argument");
        *bytes = lb::Backward(activation, d_y, x, w_gate_up, w_down, gate_up, h, d_x, d_w_gate_up, d_w_down).bytes();
    });
}

int lb_gated_mlp_bwd(int activation, const lb_tensor* d_y, const lb_tensor* x, const lb_tensor* w_gate_up, const lb_tensor* w_down, const lb_tensor* gate_up,
                     const lb_tensor* h, const lb_tensor* d_x, const lb_tensor* d_w_gate_up, const lb_tensor* d_w_down, void* scratch, size_t scratch_bytes,
                     void* stream) {
    return lb::guarded([&] {
        lb::Backward b(activation, d_y, x, w_gate_up, w_down, gate_up, h, d_x, d_w_gate_up, d_w_down);
        lb::keep_apart({&b.dx, &b.dwgu, &b.dwd}, {&b.dy, &b.x, &b.wgu, &b.wd, &b.gate_up, &b.h});
        lb::give_scratch(b, b.bytes(), scratch, scratch_bytes);
        b.run(stream);
    });
}
}
