// overlap.h -- whether a call's buffers share memory (host).
#pragma once
#include <algorithm>
#include <cstdint>

namespace nllb {

// `n` rows of `len` bytes, `ld` >= len apart, from address `at` on.  (Two rows 2^38 bytes apart are in no GPU's memory: of
// 2^24 rows the addresses stay in 64 bits.)
struct MemRows {
    long long at, n, ld, len;
    MemRows(const void* p, long long rows, long long stride, long long bytes)
        : at((long long)reinterpret_cast<uintptr_t>(p)), n(rows), ld(rows > 1 ? std::min(stride, 1LL << 38) : bytes), len(bytes) {}
    long long end() const { return at + (n - 1) * ld + len; }
};

// Whether one of the bytes [from, to) is a row's.
inline bool in_rows(long long from, long long to, const MemRows& r) {
    if (to <= r.at || from >= r.end()) return false;
    const long long j = std::min(r.n - 1, (to - 1 - r.at) / r.ld);  // the last row that starts before `to`
    return r.at + j * r.ld + r.len > from;
}

// Whether two sets of rows share a byte.  Rows at the same distance, as the columns of one matrix have them, are told apart by
// how many rows lie between; others one by one, where what they span overlaps at all.
inline bool meet(const MemRows& a, const MemRows& b) {
    if (a.n <= 0 || b.n <= 0 || a.len <= 0 || b.len <= 0 || a.end() <= b.at || b.end() <= a.at) return false;
    if (a.n > b.n) return meet(b, a);
    if (a.n > 1 && a.ld == b.ld) {
        // row i of a and row i + t of b: they meet where -b.len < d + t ld < a.len, d being b's distance from a
        const long long d = b.at - a.at;
        auto floor_of = [&](long long x) { return x / a.ld - (x % a.ld < 0); };
        const long long first = std::max(-(a.n - 1), floor_of(-b.len - d) + 1), last = std::min(b.n - 1, floor_of(a.len - 1 - d));
        return first <= last;
    }
    for (long long i = 0; i < a.n; ++i)
        if (in_rows(a.at + i * a.ld, a.at + i * a.ld + a.len, b)) return true;
    return false;
}

}  // namespace nllb
