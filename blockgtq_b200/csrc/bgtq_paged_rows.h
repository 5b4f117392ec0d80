// Whether rows of 128 elements of 16 bits, (n, h) of them at strides in elements, lie apart.
#pragma once
#include <stdint.h>

namespace bgtq {

struct PagedRows {
    uintptr_t at;
    int64_t n, h, st, sh;
    int64_t along(int dim) const { return dim ? h : n; }
    int64_t bytes(int dim) const { return 2 * (dim ? sh : st); }
    int64_t span(int dim) const { return along(dim) > 1 ? (along(dim) - 1) * bytes(dim) + 256 : 256; }      // of the rows along one dimension
};

// from one another: the rows of the dimension with the smaller stride fit between two steps of the other
inline bool paged_rows_apart(const PagedRows& x) {
    const int near = x.n > 1 && (x.h <= 1 || x.st < x.sh) ? 0 : 1;
    return (x.along(near) <= 1 || x.bytes(near) >= 256) && (x.along(1 - near) <= 1 || x.bytes(1 - near) >= x.span(near));
}
// from those of another tensor of this shape: elsewhere, or between its rows, both with the same stride along one dimension
inline bool paged_rows_apart(const PagedRows& x, const PagedRows& y) {
    auto end = [](const PagedRows& r) { return r.at + (uintptr_t)(r.span(0) + r.span(1) - 256); };
    if (end(x) <= y.at || end(y) <= x.at) return true;
    for (int dim = 0; dim < 2; ++dim) {
        const int64_t step = x.bytes(dim);
        if (x.along(dim) <= 1 || step <= 0 || step != y.bytes(dim)) continue;
        const int64_t ahead = (int64_t)(x.at > y.at ? x.at - y.at : y.at - x.at) % step;
        const int64_t behind = x.at > y.at && ahead ? step - ahead : ahead;             // y's first row behind one of x's, within a step
        if (behind >= x.span(1 - dim) && behind + y.span(1 - dim) <= step) return true;
    }
    return false;
}

}  // namespace bgtq
