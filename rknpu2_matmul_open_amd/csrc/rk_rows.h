// Memory that strided rows lie in, and whether two of them share a byte.  Arithmetic on addresses alone.
#ifndef RK_ROWS_H
#define RK_ROWS_H

#include <cstdint>

namespace rkhost {

// `rows` rows of `width` bytes, `pitch` >= width apart; nothing at all without an address, rows or bytes.
struct Span {
    uintptr_t from = 0, to = 0; // [from, to): the first row's first byte to the last row's last
    uintptr_t pitch = 0, width = 0;
    Span() = default;
    Span(const void* p, int64_t rows, int64_t row_pitch, int64_t row_width) {
        if (!p || rows <= 0 || row_width <= 0) return;
        from = reinterpret_cast<uintptr_t>(p);
        to = from + (uintptr_t)((rows - 1) * row_pitch + row_width);
        pitch = rows > 1 ? (uintptr_t)row_pitch : 0;
        width = (uintptr_t)row_width;
    }
    // Rows of one pitch (a single row takes the other's) may lie between each other's, as column slices of one buffer do: with o's
    // first row d bytes behind the start of one of these rows, they meet if it begins inside that row or reaches the next one.  (Where the ranges
    // meet, such rows do exist on both sides.)  Rows of two pitches are told apart by their ranges alone.
    bool meets(const Span& o) const {
        if (from == to || o.from == o.to || from >= o.to || o.from >= to) return false;
        if (pitch && o.pitch && pitch != o.pitch) return true;
        const uintptr_t p = pitch ? pitch : o.pitch;
        if (!p) return true;
        if (width > p || o.width > p) return true; // (a single row across several of the other's)
        const uintptr_t d = o.from >= from ? (o.from - from) % p : (p - (from - o.from) % p) % p;
        return d < width || d + o.width > p;
    }
};

} // namespace rkhost

#endif // RK_ROWS_H
