// g4b_overlap.h -- do the buffers of a call overlap?  Plain C++, for the checks of arguments.
#pragma once
#include <stddef.h>
#include <stdint.h>

namespace g4b {

// Rows of `width` bytes, `stride` bytes from one to the next.
struct Rows {
    const void* p;
    long long rows, stride, width;
};
inline Rows flat(const void* p, size_t bytes) { return {p, 1, (long long)bytes, (long long)bytes}; }

// A byte in both?  Two views of columns of one wider buffer have none, though their ranges cross.  Buffers whose ranges
// cross and whose strides differ are taken to overlap.
inline bool rows_overlap(const Rows& a, const Rows& b) {
    const long long pa = (long long)(uintptr_t)a.p, pb = (long long)(uintptr_t)b.p;
    if (!pa || !pb || pa + (a.rows - 1) * a.stride + a.width <= pb || pb + (b.rows - 1) * b.stride + b.width <= pa)
        return false;
    if (a.stride != b.stride) return true;
    const long long d = ((pb - pa) % a.stride + a.stride) % a.stride;      // b's first column, seen from a's
    return d < a.width || d + b.width > a.stride;
}

}  // namespace g4b
