// Sets of rows at two strides, and whether two of them share memory: what a call writes may lie between what it reads (parts of one
// fused projection) but not over it. Arithmetic only, for the host.
#pragma once

#include <cstdint>

namespace qs3 {

// Rows i * s0 + j * s1 .. + width of i < n0, j < n1, in bytes; n0, n1, width positive, strides not negative.
struct RowSet {
    const void* data;
    int64_t n0, n1, s0, s1, width;

    int64_t span() const { return (n0 - 1) * s0 + (n1 - 1) * s1 + width; }
    int64_t begin() const { return static_cast<int64_t>(reinterpret_cast<intptr_t>(data)); }
};

// No two rows of the set share memory.
inline bool rows_apart(const RowSet& a)
{
    if ((a.n1 > 1 && a.s1 < a.width) || (a.n0 > 1 && a.s0 < a.width))
        return false;
    return a.n0 == 1 || a.n1 == 1 || a.s0 >= (a.n1 - 1) * a.s1 + a.width || a.s1 >= (a.n0 - 1) * a.s0 + a.width;
}

// The same rows in the same order.
inline bool same_rows(const RowSet& a, const RowSet& b)
{
    return a.data == b.data && a.n0 == b.n0 && a.n1 == b.n1 && a.width == b.width && (a.n0 == 1 || a.s0 == b.s0) && (a.n1 == 1 || a.s1 == b.s1);
}

// Some row of a shares memory with some row of b. Exact where both have the same strides, else true where their spans meet and
// their rows do not fall into different parts of a common first stride.
inline bool rows_meet(const RowSet& a, const RowSet& b)
{
    const int64_t shift = b.begin() - a.begin();
    if (shift >= a.span() || -shift >= b.span())
        return false;
    // a stride that leads nowhere is the other set's
    const int64_t s0 = a.n0 > 1 ? a.s0 : b.n0 > 1 ? b.s0 : 0, s1 = a.n1 > 1 ? a.s1 : b.n1 > 1 ? b.s1 : 0;
    if (b.n0 > 1 && b.s0 != s0)
        return true;
    if (s0 > 0) {
        const int64_t at = (shift % s0 + s0) % s0;
        if (at >= (a.n1 - 1) * a.s1 + a.width && at + (b.n1 - 1) * b.s1 + b.width <= s0)
            return false;
    }
    if (b.n1 > 1 && b.s1 != s1)
        return true;
    for (int64_t j = 1 - a.n1; j < b.n1; ++j) { // steps of the second stride from a row of a to one of b
        const int64_t base = shift + j * s1;
        int64_t i = 1 - a.n0; // and of the first: the least one that brings the row's end behind a's beginning
        if (s0 > 0 && base + i * s0 <= -b.width)
            i += (-b.width - (base + i * s0)) / s0 + 1;
        if (i < b.n0 && base + i * s0 > -b.width && base + i * s0 < a.width)
            return true;
    }
    return false;
}

} // namespace qs3
