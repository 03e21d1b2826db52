// How the tiles of two products of one launch are shared out to the CTA pairs that work on them.
#pragma once
#include <algorithm>
#include <cstdint>

namespace lb {

constexpr int kListed = 8192, kNone = 0xffff;  // entries of the table; a unit that there is not

// The units of two products in the order of the longer K, each to the pair that has least to do so far: us as in pairs_us, `slots` units a pair at most. False where the table
// does not hold them. Pairs are of two kinds, those that the first product's last round reaches and the others, and within a kind all alike: what has least is a kind. Taken in turn
// instead, a pair would have up to 1024 blocks of K of a piece of 16384 x 8192 x 1024 where the mean is 886. us of both products of 2600 x 840 x 10007, two launches -> one: 128 -> 74; of that
// piece 188 and 193 -> 381.
inline bool share_units(const long long* tiles, const long long* blocks, int pairs, uint16_t* table, int& slots, double& us) {
    if (tiles[0] + tiles[1] >= std::min(kListed, kNone)) return false;
    const double cost[2] = {0.3 * (double)blocks[0] + 2.0, 0.3 * (double)blocks[1] + 2.0};
    const int whole = (int)(tiles[0] / pairs), reached = (int)(tiles[0] % pairs);
    struct Kind {
        int first, size, units;
        double load;
    } kinds[2] = {{0, reached, whole + 1, (whole + 1) * cost[0]}, {reached, pairs - reached, whole, whole * cost[0]}};
    us = reached ? kinds[0].load : kinds[1].load;
    slots = reached ? whole + 1 : whole;
    int unit = 0;
    auto put = [&](int slot, int pair) {
        if (table && (slot + 1) * pairs <= kListed) table[slot * pairs + pair] = (uint16_t)unit;
        unit++;
    };
    for (int k = 0; k < tiles[0] && table; k++) put(k / pairs, k % pairs);
    for (long long left = tiles[1]; left > 0;) {
        Kind& kind = kinds[reached && kinds[0].load <= kinds[1].load ? 0 : 1];
        const int n = (int)std::min<long long>(left, kind.size);
        for (int k = 0; k < n && table; k++) put(kind.units, kind.first + k);
        left -= n, kind.units++, kind.load += cost[1];
        us = std::max(us, kind.load), slots = std::max(slots, kind.units);
    }
    us += 3.0 + 0.1 * (double)(tiles[0] * blocks[0] + tiles[1] * blocks[1]) / pairs;
    return (long long)slots * pairs <= kListed;
}

}  // namespace lb
