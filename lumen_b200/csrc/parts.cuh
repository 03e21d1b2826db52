// float32 values as operands of the tensor cores.
#pragma once
#include <cuda_bf16.h>
#include <stdint.h>

namespace lb {

// Four values in three parts of bfloat16 each, two of them a word: the value rounded, what that leaves rounded, and the rest, 24 bits in all. A product is the sum of those of parts (first, third),
// (third, first), (second, second), (first, second), (second, first) and (first, first). NaN is NaN in every part. ANY: an infinity's parts are one, zero and the infinity, with its sign: with the
// third only first parts are multiplied, which are zero only where the value is, so that a product with it is what it should be, infinite, and NaN with zero; and what would be rounded
// to infinity has the largest finite value as its first part. Without ANY both have parts that are NaN.
template <bool ANY>
__device__ __forceinline__ void parts_of(const float* x, uint32_t (*part)[2]) {
    float v[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
    for (int k = 0; k < 3; k++)
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
            const uint32_t w = *(const uint32_t*)&h;
            part[k][j] = w;
            if (k < 2) v[2 * j] -= __uint_as_float(w << 16), v[2 * j + 1] -= __uint_as_float(w & 0xffff0000u);
        }
    constexpr float most = 3.3895313892515355e38f;  // bfloat16's
    if (ANY && __builtin_expect(fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3]))) > most, 0)) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if (!(fabsf(x[j]) > most)) continue;
            const bool infinite = fabsf(x[j]) == INFINITY;
            const float first = copysignf(infinite ? 1.0f : most, x[j]), second = infinite ? 0.0f : x[j] - first;
            const __nv_bfloat16 rounded = __float2bfloat16_rn(second);
            const uint32_t of[3] = {__float_as_uint(first) >> 16, __bfloat16_as_ushort(rounded), __bfloat16_as_ushort(__float2bfloat16_rn(infinite ? x[j] : second - __bfloat162float(rounded)))};
#pragma unroll
            for (int k = 0; k < 3; k++) part[k][j / 2] = j % 2 ? (part[k][j / 2] & 0xffffu) | of[k] << 16 : (part[k][j / 2] & 0xffff0000u) | of[k];
        }
    }
}

}  // namespace lb
