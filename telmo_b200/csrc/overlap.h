// overlap.h -- whether matrices that a call is given share memory in a way that its kernels cannot bear (host code
// alone).
#pragma once

#include <cstddef>
#include <cstdint>

namespace telmo {

// Rows of `row` bytes, `pitch` bytes apart, from `p` on.
struct Span {
    const void* p;
    size_t pitch, row, rows;
    uintptr_t begin() const { return reinterpret_cast<uintptr_t>(p); }
    uintptr_t end() const { return begin() + (rows - 1) * pitch + row; }
    bool empty() const { return !p || row == 0 || rows == 0; }
};

inline bool apart(const Span& a, const Span& b) {
    return a.empty() || b.empty() || a.end() <= b.begin() || b.end() <= a.begin();
}

// Whether they share a byte. Matrices of one pitch may lie side by side; of two pitches, their ranges must be apart.
inline bool overlap(const Span& a, const Span& b) {
    if (apart(a, b)) return false;
    if (a.pitch != b.pitch || (a.rows == 1 && b.rows == 1)) return true;
    const uintptr_t a0 = a.begin(), b0 = b.begin();
    const uintptr_t behind = b0 >= a0 ? (b0 - a0) % a.pitch : (a.pitch - (a0 - b0) % a.pitch) % a.pitch;
    return behind < a.row || a.pitch - behind < b.row;
}

// Whether a row of `out` shares a byte with another row of `in` (as many rows each): an output that is written once
// its own row has been read may lie there, but not where other rows' inputs do.
inline bool overlaps_other_rows(const Span& in, const Span& out) {
    if (apart(in, out) || out.rows == 1) return false;
    if (in.pitch != out.pitch) return true;
    const int64_t pitch = static_cast<int64_t>(in.pitch);
    const int64_t d = static_cast<int64_t>(out.begin()) - static_cast<int64_t>(in.begin());
    // out's row r begins `rest` bytes behind the begin of in's row r + rows_on.
    const int64_t rows_on = d >= 0 ? d / pitch : -((-d + pitch - 1) / pitch), rest = d - rows_on * pitch;
    return (rest < static_cast<int64_t>(in.row) && rows_on != 0) ||
           (pitch - rest < static_cast<int64_t>(out.row) && rows_on != -1);
}

}  // namespace telmo
