// Whether what a call writes lies apart from itself and from what the call reads.
#pragma once
#include <stdint.h>

namespace bgtq {

// Rows of 128 elements of 16 bits, (n, h) of them at strides in elements.
struct PagedRows {
    uintptr_t at;
    int64_t n, h, st, sh;
    int64_t along(int dim) const { return dim ? h : n; }
    int64_t bytes(int dim) const { return 2 * (dim ? sh : st); }
    int64_t span(int dim) const { return along(dim) > 1 ? (along(dim) - 1) * bytes(dim) + 256 : 256; }      // of the rows along one dimension
};

// Places of `row` bytes, (n, h) of them at strides st and sh in bytes, do not overlap one another: those along the smaller stride fit into a step of
// the larger.
inline bool paged_apart(int64_t n, int64_t h, int64_t st, int64_t sh, int64_t row) {
    const bool rows_near = n > 1 && (h <= 1 || st < sh);
    const int64_t near_n = rows_near ? n : h, near_st = rows_near ? st : sh, far_n = rows_near ? h : n, far_st = rows_near ? sh : st;
    return (near_n <= 1 || near_st >= row) && (far_n <= 1 || far_st >= (near_n > 1 ? (near_n - 1) * near_st : 0) + row);
}
inline bool paged_rows_apart(const PagedRows& x) { return paged_apart(x.n, x.h, x.bytes(0), x.bytes(1), 256); }
// The rows of two tensors of one shape lie apart: elsewhere, or between its rows, both with the same stride along one dimension
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
