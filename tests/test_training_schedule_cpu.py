"""Which cluster takes which tile of the training products: every tile once.

The header that the kernel includes is compiled for the host and its numbering
followed cluster by cluster."""
import ctypes
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SOURCE = r"""
#include "hb_schedule.hpp"
#include <vector>
using namespace hb::train;

// 0: each of the items once, and every cluster's numbering ends; the rounds and places taken in *branches:
// 1 a whole round of the first job, 2 a part round beside which the second's go, 4 the second's go on after it,
// 8 the first's rounds are whole
extern "C" int two(unsigned clusters, unsigned items0, unsigned length0, unsigned items1, unsigned length1, int *branches) {
    std::vector<unsigned char> seen(items0 + items1, 0);
    for (unsigned c = 0; c < clusters; c++) {
        unsigned k = 0;
        for (;; k++) {
            if (k > items0 + items1) return 1;
            const unsigned i = nth_of_two(k, c, clusters, items0, length0, items1, length1);
            if (i == kNoItem) break;
            if (i >= items0 + items1 || seen[i]++) return 2;
        }
        for (unsigned j = 1; j < 4; j++)  // nothing comes after the end
            if (nth_of_two(k + j, c, clusters, items0, length0, items1, length1) != kNoItem) return 3;
    }
    for (unsigned char s : seen)
        if (!s) return 4;
    const unsigned rest = items0 % clusters, beside = (length0 + length1 - 1) / length1 * (clusters - rest);
    *branches = (items0 >= clusters) | (rest ? 2 : 8) | (rest && items1 > beside ? 4 : 0);
    return 0;
}
extern "C" int one(unsigned clusters, unsigned items) {
    std::vector<unsigned char> seen(items, 0);
    for (unsigned c = 0; c < clusters; c++)
        for (unsigned k = 0, i; (i = nth_of_one(k, c, clusters, items)) != kNoItem; k++)
            if (i >= items || seen[i]++) return 1;
    for (unsigned char s : seen)
        if (!s) return 2;
    return 0;
}
extern "C" int tiles(unsigned m, unsigned n) {
    std::vector<unsigned char> seen(m * n, 0);
    for (unsigned i = 0; i < m * n; i++) {
        int mt = -1, nt = -1;
        tile_at(i, m, n, mt, nt);
        if (mt < 0 || nt < 0 || mt >= (int)m || nt >= (int)n || seen[mt * n + nt]++) return 1;
    }
    return 0;
}
extern "C" int parts(int depth, int splits) {
    int at = 0;
    for (int s = 0; s < splits; s++) {
        int k0 = -1, k1 = -1;
        part_of(depth, s, splits, k0, k1);
        if (k0 != at || k1 < k0 || k1 - k0 > depth / splits + 1) return 1;
        at = k1;
    }
    return at != depth;
}
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("schedule")
    (d / "s.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-I", os.path.join(ROOT, "helrm_b200", "csrc"),
                    str(d / "s.cpp"), "-o", str(d / "s.so")], check=True)
    return ctypes.CDLL(str(d / "s.so"))


def test_two_products_in_one_launch(lib):
    got = set()
    b = ctypes.c_int(0)
    for clusters in (1, 2, 3, 74):
        sizes = sorted({1, 2, clusters - 1, clusters, clusters + 1, 2 * clusters, 2 * clusters + 1, 3 * clusters - 1, 5 * clusters + 7}
                       - {0})
        for items0 in sizes:
            for items1 in sizes + [11 * clusters + 3]:
                for length0, length1 in ((2, 2), (3, 2), (34, 6), (66, 66), (7, 1), (5, 4)):
                    assert lib.two(clusters, items0, length0, items1, length1, ctypes.byref(b)) == 0, \
                        (clusters, items0, length0, items1, length1)
                    if clusters == 74:
                        got.add(b.value)
    # with and without a whole round; beside a part round with and without room for all; whole rounds alone
    assert got == {2, 2 | 4, 1 | 2, 1 | 2 | 4, 1 | 8}


def test_one_product(lib):
    for clusters in (1, 3, 74):
        for items in (1, 2, 73, 74, 75, 148, 1000):
            assert lib.one(clusters, items) == 0


def test_tiles(lib):
    for m in list(range(1, 26)) + [40, 64, 67]:
        for n in (1, 2, 3, 7, 8, 9, 48):
            assert lib.tiles(m, n) == 0, (m, n)


def test_parts_of_a_depth(lib):
    for depth in (0, 1, 3, 15, 16, 17, 64, 1000):
        for splits in (1, 2, 3, 7, 18, 74):
            assert lib.parts(depth, splits) == 0, (depth, splits)
