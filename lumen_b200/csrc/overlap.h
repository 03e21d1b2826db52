// Whether strided tensors share memory: what is written by some threads while others read it has to lie apart.
#pragma once
#include "common.h"

namespace lb {

// The bytes from a tensor's first element to its last one's end; `to` is not behind `from` where there is none.
struct Extent {
    __int128 from, to;  // wide enough for whatever a caller says
    bool meets(const Extent& other) const { return from < to && other.from < other.to && from < other.to && other.from < to; }
};
Extent extent(const lb_tensor& t);
// Whether a byte belongs to an element of both. Exact for the layouts that views of one buffer have (columns, heads, rows, batches of it, in any order);
// where that would take more than a few thousand steps the answer is yes. Shapes and strides of any sign; an empty tensor shares nothing.
bool share_memory(const lb_tensor& a, const lb_tensor& b);
// Whether two elements of `t` share a byte; the same bound.
bool overlaps_itself(const lb_tensor& t);
// Whether both are the same elements in the same places, index for index.
bool same_places(const lb_tensor& a, const lb_tensor& b);

}  // namespace lb
