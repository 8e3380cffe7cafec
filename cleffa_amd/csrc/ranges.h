// Whether what a call writes shares bytes with what it reads: host checks over strided rows. Exact for rows; for heads of rows
// exact where both have rows equally far apart, else by whole rows.
#pragma once
#include <limits.h>
#include <stdint.h>

namespace clef_hip {

// n runs of `bytes` bytes, the first at `at`, `stride` bytes apart (one run: no matter). Callers keep spans below kMaxSpan.
constexpr long kMaxSpan = 1L << 44;
struct Rows {
    uintptr_t at;
    long n, stride, bytes;
    uintptr_t end() const { return at + (uintptr_t)((n - 1) * stride + bytes); }
};
inline bool span_ok(long n, long stride, long size) { return n <= 1 || (stride >= 0 && stride <= kMaxSpan / size / (n - 1)); }

// whether a run has bytes in [lo, hi)
inline bool meets(const Rows &r, uintptr_t lo, uintptr_t hi) {
    if (r.n <= 0 || r.bytes <= 0 || lo >= hi || hi <= r.at || lo >= r.end()) return false;
    if (lo < r.at + (uintptr_t)r.bytes) return true;      // the first run does: it begins before hi
    if (r.stride == 0) return false;
    const long first = (long)((lo - r.at - (uintptr_t)r.bytes) / (uintptr_t)r.stride) + 1;    // the first that ends behind lo
    return first < r.n && r.at + (uintptr_t)(first * r.stride) < hi;
}
inline bool meet(const Rows &a, const Rows &b) {
    if (a.n <= 0 || b.n <= 0 || a.bytes <= 0 || b.bytes <= 0 || a.end() <= b.at || b.end() <= a.at) return false;
    if (a.n > 1 && b.n > 1 && a.stride == b.stride && a.bytes <= a.stride && b.bytes <= a.stride) {
        // the later one's first run lies before the other's end, so it meets a run there or none does
        const Rows &lo = a.at <= b.at ? a : b, &hi = a.at <= b.at ? b : a;
        const long d = (long)((hi.at - lo.at) % (uintptr_t)a.stride);
        return d < lo.bytes || (d > a.stride - hi.bytes && (uintptr_t)((lo.n - 1) * lo.stride) > hi.at - lo.at);
    }
    const Rows &few = a.n <= b.n ? a : b, &many = a.n <= b.n ? b : a;
    for (long i = 0; i < few.n; i++) {
        const uintptr_t at = few.at + (uintptr_t)(i * few.stride);
        if (meets(many, at, at + (uintptr_t)few.bytes)) return true;
    }
    return false;
}

// `rows` times `heads` runs of `bytes` bytes
struct Heads {
    uintptr_t at;
    long rows, row, heads, head, bytes;
    // as runs over the outer of both, each from the first to the last byte of the inner one's
    bool by_row() const { return rows <= 1 || heads <= 1 ? rows > 1 : row >= head; }
    Rows hull() const { return by_row() ? Rows{at, rows, row, (heads - 1) * head + bytes} : Rows{at, heads, head, (rows - 1) * row + bytes}; }
};
inline bool meet(const Heads &a, const Heads &b) {
    if (a.rows <= 0 || b.rows <= 0 || a.heads <= 0 || b.heads <= 0) return false;
    const Rows x = a.hull(), y = b.hull();
    if (!meet(x, y)) return false;
    const bool lone = a.rows <= 1 && b.rows <= 1;         // one row each: heads against heads
    if (lone) return meet(Rows{a.at, a.heads, a.head, a.bytes}, Rows{b.at, b.heads, b.head, b.bytes});
    if (a.rows > 1 && b.rows > 1 && a.row != b.row) return true;
    for (long i = 0; i < a.heads; i++)
        for (long j = 0; j < b.heads; j++)
            if (meet(Rows{a.at + (uintptr_t)(i * a.head), a.rows, a.row, a.bytes}, Rows{b.at + (uintptr_t)(j * b.head), b.rows, b.row, b.bytes})) return true;
    return false;
}

}  // namespace clef_hip
