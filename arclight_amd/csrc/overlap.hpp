// Whether two strided operands share a byte (host code only, without HIP, so
// that it is tested without a GPU).
#pragma once

#include <algorithm>

#include "../../include/arclight_fattn.h"

// The bytes of an operand: blocks of `bytes`, repeated over dimensions whose
// strides are no less than what lies within them, the innermost first. Operands
// whose dimensions run into one another with gaps between are taken as the
// whole range.
struct ByteSet {
    typedef __int128 wide;                      // (strides may be anything)
    wide base = 0, bytes = 0;                   // 0 bytes: empty
    int dims = 0;
    wide n[3], step[3];

    ByteSet() = default;
    // t's first dimension is dense, of elements of `size` bytes.
    ByteSet(const al_tensor & t, const int size) : base((wide) (uintptr_t) t.data), bytes((wide) t.ne[0] * size) {
        if (!t.data || t.ne[0] < 1 || t.ne[1] < 1 || t.ne[2] < 1 || t.ne[3] < 1) {
            bytes = 0;
            return;
        }
        int order[3] = {1, 2, 3};
        std::sort(order, order + 3, [&](int a, int b) { return t.nb[a] < t.nb[b]; });
        for (const int i : order) {
            if (t.ne[i] == 1) continue;
            const wide s = (wide) t.nb[i], inner = extent(dims);
            if (s > inner || (s == inner && dims)) {
                n[dims] = t.ne[i];
                step[dims++] = s;
            } else {                            // no gap but those within
                bytes = inner + (t.ne[i] - 1) * s;
                dims = 0;
            }
        }
    }
    wide extent(const int d) const {            // of the blocks over the first d dimensions
        wide x = bytes;
        for (int i = 0; i < d; ++i) x += (n[i] - 1) * step[i];
        return x;
    }
    wide blocks() const {
        wide x = 1;
        for (int i = 0; i < dims; ++i) x *= n[i];
        return x;
    }
    // Whether a byte of [from, to) is one of those over the first d dimensions from `at` on.
    bool has(const wide from, const wide to, const wide at, const int d) const {
        const wide e = extent(d);
        if (to <= at || from >= at + e) return false;
        if (d == 0) return true;
        const wide s = step[d - 1], inner = extent(d - 1);
        // the copies of what is within that reach into it
        const wide lo = std::max<wide>(0, from - at - inner < 0 ? 0 : (from - at - inner) / s + 1);
        const wide hi = std::min<wide>(n[d - 1] - 1, (to - 1 - at) / s);
        if (lo > hi) return false;
        if (hi - lo > 1) return true;           // one lies within it as a whole
        return has(from, to, at + lo * s, d - 1) || (hi > lo && has(from, to, at + hi * s, d - 1));
    }
};

inline bool overlap(const ByteSet & x, const ByteSet & y) {
    if (!x.bytes || !y.bytes || x.base >= y.base + y.extent(y.dims) || y.base >= x.base + x.extent(x.dims)) return false;
    const ByteSet &a = x.blocks() <= y.blocks() ? x : y, &b = x.blocks() <= y.blocks() ? y : x;
    ByteSet::wide i[3] = {0, 0, 0};
    for (;;) {
        ByteSet::wide at = a.base;
        for (int d = 0; d < a.dims; ++d) at += i[d] * a.step[d];
        if (b.has(at, at + a.bytes, b.base, b.dims)) return true;
        int d = 0;
        while (d < a.dims && ++i[d] == a.n[d]) i[d++] = 0;
        if (d == a.dims) return false;
    }
}

// Whether one of the first `outs` operands, all of 4-byte elements, shares memory
// with another one. (One may lie in another's gaps.)
template <int N>
bool outputs_overlap(const al_tensor * const (&operands)[N], const int outs) {
    ByteSet x[N];
    for (int i = 0; i < N; ++i) x[i] = ByteSet(*operands[i], 4);
    for (int i = 0; i < outs; ++i)
        for (int j = i + 1; j < N; ++j)
            if (overlap(x[i], x[j])) return true;
    return false;
}
