// Division by a number that is the same for a whole launch.
#pragma once
#include <stdint.h>

namespace lb {

// n / d for 0 <= n < 2^31 as a multiply and a shift (Granlund and Montgomery's round-up method): where a tile lies is worked out by
// every warp between two tiles, and six integer divisions took 1200 cycles there.
struct Divisor {
    uint32_t d = 1, mul = 1, shift = 0;
    void set(uint32_t by) {
        d = by, shift = 0;
        while ((1ull << shift) < d) shift++;
        mul = (uint32_t)(((1ull << 32) * ((1ull << shift) - d)) / d + 1);
    }
    __device__ __forceinline__ uint32_t div(uint32_t n) const { return (__umulhi(n, mul) + n) >> shift; }
};

}  // namespace lb
