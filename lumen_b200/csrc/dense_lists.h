// Lists of dense tensors: what a call on all of a model's tensors looks at.
#pragma once
#include <algorithm>
#include <vector>

#include "common.h"

namespace lb {

// The number of elements of a tensor that fills its memory without gaps, in any order of its dimensions, -1 for others and for one with a negative size.
inline long long dense_elements(const lb_tensor& t) {
    long long n = 1;
    for (int d = 0; d < t.rank; d++) {
        if (t.shape[d] < 0) return -1;
        n *= t.shape[d];
    }
    if (n <= 1) return n;
    long long step = 1;
    bool used[LB_MAX_RANK] = {};
    for (int found = 0; step < n;) {  // the dimension that strides by what is filled so far
        int next = -1;
        for (int d = 0; d < t.rank && next < 0; d++)
            if (!used[d] && t.shape[d] > 1 && t.stride[d] == step) next = d;
        if (next < 0 || found++ > LB_MAX_RANK) return -1;
        used[next] = true, step *= t.shape[next];
    }
    return n;
}

// Whether two dense tensors' elements lie in the same order.
inline bool same_order(const lb_tensor& a, const lb_tensor& b) {
    bool same = a.rank == b.rank;
    for (int d = 0; same && d < a.rank; d++) same = a.shape[d] == b.shape[d] && (a.stride[d] == b.stride[d] || a.shape[d] == 1);
    return same;
}

// The tensor that chunk `c` of a table lies in: the last whose first chunk is not behind it (an empty tensor has none).
#ifdef __CUDACC__
template <class Table>
__device__ __forceinline__ int tensor_of(const Table& t, int c) {
    int lo = 0, hi = t.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (t.first[mid] <= c) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}
#endif

// The memory of the tensors of a call, to find two places that share some of it: `index` and `what` are the caller's.
struct Place {
    uintptr_t from, to;
    uint32_t index : 24, what : 7, written : 1;
};
// Two places of which one is written and that share memory; false where there are none. Sorts the places.
inline bool meeting(std::vector<Place>& places, const Place*& a, const Place*& b) {
    std::sort(places.begin(), places.end(), [](const Place& x, const Place& y) { return x.from < y.from; });
    const Place *read = nullptr, *written = nullptr;  // the ones so far that reach furthest
    for (const Place& p : places) {
        if (p.from == p.to) continue;
        b = &p;
        if (written && p.from < written->to) return a = written, true;
        if (p.written && read && p.from < read->to) return a = read, true;
        const Place*& last = p.written ? written : read;
        if (!last || p.to > last->to) last = &p;
    }
    return false;
}

}  // namespace lb
