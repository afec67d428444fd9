// overlap.hpp -- whether two buffers, each rows at a pitch, have a byte in common.
#pragma once

#include <algorithm>
#include <cstdint>

namespace sili {

// n rows of `width` bytes each, `pitch` bytes apart (of either sign), from p on.
struct Rows {
    const void *p;
    int64_t n;
    __int128 width, pitch;
};

// Exact for rows of one pitch, and for one row: x and y may be columns of one matrix.
// Rows of two pitches meet where the ranges that they span do.
inline bool meet(Rows x, Rows y) {
    if (!x.p || !y.p || x.n <= 0 || y.n <= 0 || x.width <= 0 || y.width <= 0) return false;
    if (x.n == 1) x.pitch = y.pitch;
    if (y.n == 1) y.pitch = x.pitch;
    auto lowest = [](const Rows &r) {
        return (__int128) reinterpret_cast<uintptr_t>(r.p) + std::min<__int128>(0, (r.n - 1) * r.pitch);
    };
    auto size = [](__int128 v) { return v < 0 ? -v : v; };
    const __int128 a = lowest(x), b = lowest(y), p = size(x.pitch), q = size(y.pitch);
    if (a + (x.n - 1) * p + x.width <= b || b + (y.n - 1) * q + y.width <= a) return false;
    if (p != q || p == 0) return true;
    // row i of x and row j of y, k = j - i: -y.width < b - a + k p < x.width
    const __int128 gap = -y.width - (b - a);
    const __int128 k = std::max<__int128>(gap / p - (gap % p < 0 ? 1 : 0) + 1, 1 - x.n);
    return k <= y.n - 1 && b - a + k * p < x.width;
}

}  // namespace sili
