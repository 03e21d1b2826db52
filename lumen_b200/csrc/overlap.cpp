// An element's bytes are base + sum of i_d s_d + p, 0 <= i_d < n_d, 0 <= p < the element's size. Two tensors share a byte where the difference of
// their bases is a sum of one's strides, each as often as its indices say, less a sum of the other's: a linear equation in bounded integers. It is solved from the
// largest stride down; what the smaller ones can still reach leaves one to three values for each in layouts that nest.
#include "overlap.h"

#include <algorithm>

namespace lb {
namespace {

typedef __int128 Wide;

struct Term {
    Wide step, lo, hi;  // step > 0, taken lo .. hi times
};
struct Sum {
    Term term[2 * LB_MAX_RANK + 1];
    int terms = 0;
    Wide least[2 * LB_MAX_RANK + 2], most[2 * LB_MAX_RANK + 2];  // of the terms from one on
    int steps = 4096;

    void add(Wide step, Wide lo, Wide hi) {
        for (int k = 0; k < terms; k++)
            if (term[k].step == step) {
                term[k].lo += lo, term[k].hi += hi;
                return;
            }
        term[terms++] = {step, lo, hi};
    }
    void order() {
        std::sort(term, term + terms, [](const Term& a, const Term& b) { return a.step > b.step; });
        least[terms] = most[terms] = 0;
        for (int k = terms; k-- > 0;) least[k] = least[k + 1] + term[k].step * term[k].lo, most[k] = most[k + 1] + term[k].step * term[k].hi;
    }
    // Whether terms `from` and on can add up to `value`; the last term is the bytes of an element, with a step of one.
    bool reaches(int from, Wide value) {
        if (value < least[from] || value > most[from]) return false;
        if (from >= terms - 1 || --steps < 0) return true;
        const Term& t = term[from];
        auto down = [](Wide n, Wide d) { return n >= 0 ? n / d : -((-n + d - 1) / d); };
        const Wide first = std::max(t.lo, -down(-(value - most[from + 1]), t.step)), last = std::min(t.hi, down(value - least[from + 1], t.step));
        for (Wide v = first; v <= last; v++)
            if (reaches(from + 1, value - v * t.step)) return true;
        return false;
    }
};

// The lowest address and, by `add(step, n)`, every dimension with more than one place; false for an empty tensor.
template <class Add>
bool places(const lb_tensor& t, Wide& base, Add add) {
    base = (Wide)(uintptr_t)t.ptr;
    const int item = dtype_size(t.dtype);
    for (int d = 0; d < t.rank; d++)
        if (t.shape[d] <= 0) return false;
    for (int d = 0; d < t.rank; d++) {
        const Wide step = (Wide)t.stride[d] * item, n = t.shape[d];
        if (n == 1 || step == 0) continue;
        if (step < 0) base += step * (n - 1);
        add(step < 0 ? -step : step, n);
    }
    return true;
}

}  // namespace

Extent extent(const lb_tensor& t) {
    Wide from, bytes = dtype_size(t.dtype);
    if (!places(t, from, [&](Wide step, Wide n) { bytes += step * (n - 1); })) return {0, 0};
    return {from, from + bytes};
}

bool share_memory(const lb_tensor& a, const lb_tensor& b) {
    if (!extent(a).meets(extent(b))) return false;
    Wide from_a, from_b;
    Sum sum;
    places(a, from_a, [&](Wide step, Wide n) { sum.add(step, 0, n - 1); });
    places(b, from_b, [&](Wide step, Wide n) { sum.add(step, 1 - n, 0); });
    sum.add(1, 1 - dtype_size(b.dtype), dtype_size(a.dtype) - 1);
    sum.order();
    return sum.reaches(0, from_b - from_a);
}

bool overlaps_itself(const lb_tensor& t) {
    Wide base, step[LB_MAX_RANK], n[LB_MAX_RANK];
    int dims = 0;
    if (!places(t, base, [&](Wide s, Wide count) { step[dims] = s, n[dims++] = count; })) return false;
    for (int d = 0; d < t.rank; d++)
        if (t.shape[d] > 1 && t.stride[d] == 0) return true;
    // where each dimension's step is beyond all that the smaller ones reach, as in any slice of a dense tensor, there is nothing to solve
    for (int d = 1; d < dims; d++)
        for (int k = d; k > 0 && step[k] < step[k - 1]; k--) std::swap(step[k], step[k - 1]), std::swap(n[k], n[k - 1]);
    Wide reach = dtype_size(t.dtype);
    bool nested = true;
    for (int d = 0; d < dims && nested; d++) nested = step[d] >= reach, reach += step[d] * (n[d] - 1);
    if (nested) return false;
    // two elements differ first in one dimension, the later of them by one or more there, and by anything in those behind it
    for (int first = 0; first < dims; first++) {
        Sum sum;
        sum.add(step[first], 0, n[first] - 2);
        for (int d = first + 1; d < dims; d++) sum.add(step[d], 1 - n[d], n[d] - 1);
        sum.add(1, 1 - dtype_size(t.dtype), dtype_size(t.dtype) - 1);
        sum.order();
        if (sum.reaches(0, -step[first])) return true;
    }
    return false;
}

bool same_places(const lb_tensor& a, const lb_tensor& b) {
    bool same = a.ptr == b.ptr && a.dtype == b.dtype && a.rank == b.rank;
    for (int d = 0; same && d < a.rank; d++) same = a.shape[d] == b.shape[d] && (a.stride[d] == b.stride[d] || a.shape[d] <= 1);
    return same;
}

}  // namespace lb
