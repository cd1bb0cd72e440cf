"""Rows at any address are read as aligned granules of 16 bytes: no byte outside the buffer is read, and none of it is missed.
The arithmetic (csrc/granule.h) is run on the host for every buffer that matters; that the loads go through it is read off the
sources."""
import os
import re
import subprocess

import llm720_b200

CSRC = os.path.join(os.path.dirname(llm720_b200.__file__), "csrc")

PROGRAM = r"""
#include <cstdio>
#include <initializer_list>
#include "granule.h"
using namespace peer;
long wrong = 0, tried = 0;
void check(bool good) { ++tried; wrong += !good; }
int main() {
    // the bytes of a granule that belong to a buffer
    for (int size : {1, 2, 4})
        for (uintptr_t begin = 4096; begin < 4112; begin += size)
            for (int values = 1; values <= 40; ++values) {
                const uintptr_t end = begin + values * size;
                for (uintptr_t g = 4080; g < end + 32; g += 16) {
                    const GranulePart p = granule_part(g, begin, end);
                    check(granule_inside(g, begin, end) == (p.first == 0 && p.last == 16));
                    for (int b = 0; b < 16; ++b) check((g + b >= begin && g + b < end) == (b >= p.first && b < p.last));
                    check(p.first % size == 0 && p.last % size == 0);
                }
            }
    // rows of a table (rows of D values behind one another), copied to rows at any address
    for (int size : {2, 4})
        for (uintptr_t buf = 4096; buf < 4112; buf += size)
            for (int D = 1; D <= 40; ++D)
                for (int V : {1, 2, 5}) {
                    const int N = 16 / size;
                    const uintptr_t buf_end = buf + V * D * size;
                    for (int r = 0; r < V; ++r)
                        for (uintptr_t dst = 0; dst < 16; dst += size) {
                            const uintptr_t row = buf + r * D * size;
                            const PieceRange p = piece_range(row, dst, D, size, buf, buf_end);
                            check(0 <= p.begin && p.begin <= p.end && p.end <= D && (p.end - p.begin) % N == 0);
                            check(p.begin < 16 && D - p.end < 16);      // what sixteen threads take at either end
                            for (int64_t c = p.begin; c < p.end; c += N) {
                                const uintptr_t at = row + c * size - p.shift;
                                check((dst + c * size) % 16 == 0 && at % 16 == 0 && granule_inside(at, buf, buf_end));
                                check(p.shift == 0 || granule_inside(at + 16, buf, buf_end));
                            }
                        }
                    // and read by threads whose pieces begin anywhere
                    for (int r = 0; r < V; ++r)
                        for (int at = -N; at < D + N; ++at) {
                            const uintptr_t row = buf + r * D * size;
                            const GranuleWants w = granule_wants(row, at, D, size);
                            check(w.first % 16 == 0 && w.first + w.shift == row + at * size);
                            for (int q = 0; q < N; ++q)                 // every value of the row is in a granule that is wanted
                                if (at + q >= 0 && at + q < D) check(w.shift + q * size < 16 ? w.lo : w.hi);
                            // and a wanted one holds some of the buffer: the rest of it is left out by granule_part
                            for (int k = 0; k < 2; ++k)
                                if (k ? w.hi : w.lo) {
                                    const GranulePart part = granule_part(w.first + 16 * k, buf, buf_end);
                                    check(part.first < part.last);
                                }
                        }
                }
    std::printf("%ld %ld\n", tried, wrong);
}
"""


def _source(name):
    return re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, name)).read())


def _function(text, name):
    at = text.index(name + "(")
    at = text.index("{", text.index(")", at))
    depth = 0
    for i in range(at, len(text)):
        depth += {"{": 1, "}": -1}.get(text[i], 0)
        if depth == 0:
            return text[at:i + 1]
    raise AssertionError(name)


def test_the_parts_of_granules_that_belong_to_a_buffer(tmp_path):
    source, program = tmp_path / "granules.cpp", tmp_path / "granules"
    source.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", f"-I{CSRC}", str(source), "-o", str(program)], check=True)
    tried, wrong = map(int, subprocess.run([str(program)], check=True, capture_output=True, text=True).stdout.split())
    assert tried > 1000 and wrong == 0


def test_granules_are_loaded_through_it():
    shift = _source("row_shift.cuh")
    partial = _function(shift, "partial_granule")
    assert "granule_part" in partial and partial.count("__ldg(") == 1
    edge = _function(shift, "load_edge_granules")
    assert edge.count("granule_inside") == edge.count("__ldg(") == edge.count("partial_granule<T>(") == 2
    plain = _function(shift, "load_granules")                   # for rows away from the ends
    assert plain.count("__ldg(") == 2
    assert shift.count("__ldg(") == 5                           # those alone
    fetch = _function(shift, "fetch_row")
    assert re.search(r"if \(HEAD && gt == 0 && first < static_cast<const char\*>\(begin\)\) \{[^}]*partial_granule<", fetch)
    for name, rings in (("layer_norm.cu", 2), ("row_pack.cu", 2)):
        text = _source(name)
        assert text.count("fetch(std::true_type());") == rings and text.count("first_row_alone(") >= 2
        for at in re.finditer(r"fetch\(std::true_type\(\)\);", text):     # the first fetch of each
            assert "fetch(std::" not in text[text.rindex("auto fetch", 0, at.start()):at.start()]
    sums = _source("row_sum.cu")
    assert sums.count("load_granules(") == sums.count("load_edge_granules(") == 1
    assert re.search(r"edge \|= j < p\.n && at - p\.edge >= p\.inner", sums)
    assert re.search(r"else if \(!edges\) \{[^}]*load_granules\([^}]*\} else \{[^}]*load_edge_granules\(", sums)
    lookup = _function(_source("embedding.cu"), "embed_kernel")
    assert lookup.index("piece_range(") < lookup.index("__ldg(at)")
