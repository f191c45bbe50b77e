"""Whether two sets of strided rows share a byte: what the host layer decides from addresses, against the bytes one by one."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r"""
#include <cstdio>
#include <vector>
#include "rk_rows.h"
using rkhost::Span;

static const int64_t BASE = 1000;

static Span span(int64_t at, int64_t rows, int64_t pitch, int64_t width) { return Span(reinterpret_cast<const void*>(at), rows, pitch, width); }
static bool share_a_byte(int64_t at, int64_t rows, int64_t pitch, int64_t width, int64_t at2, int64_t rows2, int64_t pitch2, int64_t width2) {
    std::vector<char> taken(400);
    for (int64_t r = 0; r < rows; ++r)
        for (int64_t i = 0; i < width; ++i) taken[at + r * pitch + i - BASE + 100] = 1;
    for (int64_t r = 0; r < rows2; ++r)
        for (int64_t i = 0; i < width2; ++i)
            if (taken[at2 + r * pitch2 + i - BASE + 100]) return true;
    return false;
}

int main() {
    long cases = 0, apart_inside = 0;
    // equal pitches, and single rows against any: exact
    for (int64_t pitch = 1; pitch <= 7; ++pitch)
        for (int64_t width = 1; width <= pitch; ++width)
            for (int64_t width2 = 1; width2 <= pitch; ++width2)
                for (int64_t rows = 0; rows <= 4; ++rows)
                    for (int64_t rows2 = 0; rows2 <= 4; ++rows2)
                        for (int64_t at = BASE - 40; at <= BASE + 40; ++at) {
                            const Span a = span(BASE, rows, pitch, width), b = span(at, rows2, pitch, width2);
                            const bool want = share_a_byte(BASE, rows, pitch, width, at, rows2, pitch, width2);
                            if (a.meets(b) != want || b.meets(a) != want) {
                                std::printf("pitch %ld: %ld x %ld at 0, %ld x %ld at %ld: %d\n", (long)pitch, (long)rows, (long)width, (long)rows2, (long)width2, (long)(at - BASE), want);
                                return 1;
                            }
                            ++cases;
                            apart_inside += !want && rows > 1 && rows2 > 1 && a.from < b.to && b.from < a.to;
                        }
    for (int64_t pitch = 2; pitch <= 6; ++pitch) // a single row that is wider than the other's pitch, whatever its own is said to be
        for (int64_t width = 1; width <= pitch; ++width)
            for (int64_t width2 = 1; width2 <= 15; ++width2)
                for (int64_t at = BASE - 20; at <= BASE + 40; ++at) {
                    const Span a = span(BASE, 4, pitch, width), b = span(at, 1, 99, width2);
                    const bool want = share_a_byte(BASE, 4, pitch, width, at, 1, 99, width2);
                    if (a.meets(b) != want || b.meets(a) != want) return 2;
                }
    for (int64_t pitch2 = 3; pitch2 <= 9; ++pitch2) // two pitches: never told apart where a byte is shared
        for (int64_t at = BASE - 30; at <= BASE + 30; ++at)
            if (share_a_byte(BASE, 3, 5, 2, at, 4, pitch2, 3) && !span(BASE, 3, 5, 2).meets(span(at, 4, pitch2, 3))) return 3;
    if (span(0, 3, 4, 4).meets(span(BASE, 1, 4, 4)) || Span().meets(span(BASE, 1, 4, 4))) return 4;
    // far apart in a large buffer, beyond 32 bits
    const int64_t far = INT64_C(1) << 33;
    if (span(BASE, 5, far, far / 2).meets(span(BASE + far / 2, 5, far, far / 2))) return 5;
    if (!span(BASE, 5, far, far / 2 + 1).meets(span(BASE + far / 2, 5, far, far / 2))) return 6;
    std::printf("%ld %ld\n", cases, apart_inside);
    return 0;
}
"""


def test_rows_meet_where_they_share_a_byte(tmp_path):
    src = tmp_path / "spans.cpp"
    src.write_text(PROGRAM)
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-I", os.path.join(ROOT, "rknpu2_matmul_open_amd", "csrc"), str(src), "-o", str(tmp_path / "spans")])
    cases, apart_inside = map(int, subprocess.check_output([str(tmp_path / "spans")]).split())
    assert cases > 100000 and apart_inside > 1000
