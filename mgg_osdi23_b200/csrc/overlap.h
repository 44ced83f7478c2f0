// Which outputs share memory with which inputs.  The kernels read and write rows in no order that a caller could rely on, so
// that a call whose output lies partly over an input has no defined result; it is refused.
#pragma once
#include <cstdint>

namespace mggb {

inline bool runs_meet(const void* p, uint64_t p_bytes, const void* q, uint64_t q_bytes) {
    const uint64_t a = (uint64_t)p, b = (uint64_t)q;
    return a < b + q_bytes && b < a + p_bytes;
}

// Two matrices of n rows of `row` bytes, ld_p and ld_q bytes apart.  Exact where the strides are equal (columns of one matrix
// side by side do not meet) or one of the matrices has no gaps; two with gaps and strides of their own are taken as apart.
inline bool rows_meet(const void* p, uint64_t ld_p, const void* q, uint64_t ld_q, uint64_t n, uint64_t row) {
    if (n == 0 || !runs_meet(p, (n - 1) * ld_p + row, q, (n - 1) * ld_q + row)) return false;
    if (n == 1) return true;
    const uint64_t a = (uint64_t)p, b = (uint64_t)q;
    if (ld_p == ld_q) {
        const uint64_t off = (a > b ? a - b : b - a) % ld_p;
        return off < row || ld_p - off < row;
    }
    // rows of the matrix with gaps that reach into the other's run
    auto reach = [&](uint64_t first, uint64_t ld, uint64_t lo) {
        const uint64_t i = first + row > lo ? 0 : (lo - first - row) / ld + 1;       // the first row that ends behind lo
        return i < n && first + i * ld < lo + n * row;
    };
    if (ld_p == row) return reach(b, ld_q, a);
    if (ld_q == row) return reach(a, ld_p, b);
    return false;
}

}  // namespace mggb
