"""The host's look at whether the row lists of a call share memory (csrc/row_lists.h), against sets of bytes."""
import ctypes as C
import os
import shutil
import subprocess

import numpy as np
import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "voxcpm.cpp_b200", "csrc")
SOURCE = """
#include "row_lists.h"
using namespace vox;
static RowLists lists(const long * x) { return RowLists((void *) x[0], x[1], {{x[2], (size_t) x[3]}, {x[4], (size_t) x[5]}, {x[6], (size_t) x[7]}}); }
extern "C" int overlap(const long * x) { return lists(x).overlap(); }
extern "C" int shifted(const long * x, long other) { return lists(x).overlap_shifted((void *) other); }
extern "C" int meets(const long * x, long at, long size) { return lists(x).meets((void *) at, size); }
extern "C" int ranges(long a, long n, long b, long m) { return ranges_meet((void *) a, n, (void *) b, m); }
"""


@pytest.fixture(scope="module")
def fn(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("no g++")
    at = tmp_path_factory.mktemp("row_lists")
    (at / "t.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover", "-shared", "-fPIC", "-I", CSRC,
                    str(at / "t.cpp"), "-o", str(at / "t.so")], check=True)
    lib = C.CDLL(str(at / "t.so"))

    class Calls:
        @staticmethod
        def x(base, size, dims):
            flat = [base, size] + [int(v) for d in dims for v in d]
            return (C.c_long * 8)(*flat)

        def overlap(self, *a):
            return bool(lib.overlap(self.x(*a)))

        def shifted(self, other, *a):
            return bool(lib.shifted(self.x(*a), C.c_long(other)))

        def meets(self, at, size, *a):
            return bool(lib.meets(self.x(*a), C.c_long(at), C.c_long(size)))

        def ranges(self, *a):
            return bool(lib.ranges(*[C.c_long(v) for v in a]))

    return Calls()


def starts(base, dims):
    at = np.array([base])
    for n, s in dims:
        at = (at[:, None] + s * np.arange(n)).ravel()
    return at


def draws(seed, n=400):
    """Layouts with extents of one to five: packed and padded ones in any order, ones that interleave, and random strides."""
    rng = np.random.default_rng(seed)
    for _ in range(n):
        size, dims = int(rng.integers(1, 9)), [(int(rng.integers(1, 6)), int(rng.integers(0, 60))) for _ in range(3)]
        if rng.random() < 0.6:
            span, strides = size + int(rng.integers(0, 3) * rng.integers(0, 12)), [0, 0, 0]
            for d in rng.permutation(3):
                strides[d] = span
                span = span * dims[d][0] + int(rng.integers(0, 2) * rng.integers(0, 9))
            if rng.random() < 0.3:
                strides[int(rng.integers(3))] += int(rng.integers(-3, 4))
            dims = [(n_, max(0, s)) for (n_, _), s in zip(dims, strides)]
        yield rng, 1 << 20, size, dims


@pytest.mark.parametrize("seed", range(8))
def test_lists_over_one_another_are_seen(seed, fn):
    seen = set()
    for rng, base, size, dims in draws(seed):
        at = np.sort(starts(base, dims))
        want = bool((np.diff(at) < size).any())
        assert fn.overlap(base, size, dims) == want, (size, dims)
        seen.add(want)
    assert seen == {True, False}


@pytest.mark.parametrize("seed", range(8))
def test_lists_over_those_of_another_base_are_seen(seed, fn):
    seen = set()
    for rng, base, size, dims in draws(seed):
        a = starts(base, dims)
        span = int(a.max() - a.min()) + size
        for other in (base + int(rng.integers(-span - 9, span + 10)), base + size, base - size, base + span, base - span, base, base + size - 1):
            want = bool((np.abs(a[:, None] - starts(other, dims)[None]) < size).any())
            assert fn.shifted(other, base, size, dims) == want, (size, dims, other - base)
            seen.add(want)
    assert seen == {True, False}


@pytest.mark.parametrize("seed", range(8))
def test_a_buffer_in_a_list_is_seen(seed, fn):
    seen = set()
    for rng, base, size, dims in draws(seed):
        a = starts(base, dims)
        for _ in range(6):
            at, n = int(rng.integers(base - 20, a.max() + size + 20)), int(rng.integers(1, 12))
            want = bool(((a < at + n) & (a + size > at)).any())
            assert fn.meets(at, n, base, size, dims) == want, (size, dims, at - base, n)
            seen.add(want)
    assert seen == {True, False}


def test_layouts_of_a_user(fn):
    f, rows, HK, S, L = 4, 1000, 2, 64, 30
    packed = [(HK, rows * f), (S, HK * rows * f), (L, S * HK * rows * f)]
    assert not fn.overlap(1 << 40, rows * f, packed)
    assert fn.overlap(1 << 40, rows * f, [(HK, rows * f), (S, rows * f), (L, S * HK * rows * f)])  # equal strides of heads and streams
    assert fn.overlap(1 << 40, rows * f, [(HK, rows * f), (S, HK * rows * f), (L, rows * f)])
    assert fn.overlap(1 << 40, (rows + 1) * f, packed)
    side_by_side = [(n, 2 * s) for n, s in packed]  # a list of positions behind each list of scores
    assert not fn.overlap(1 << 40, rows * f, side_by_side)
    assert not fn.shifted((1 << 40) + rows * f, 1 << 40, rows * f, side_by_side)
    assert fn.shifted((1 << 40) + rows * f - 4, 1 << 40, rows * f, side_by_side)
    assert fn.shifted(1 << 40, 1 << 40, rows * f, packed)
    assert not fn.overlap(0, 0, [(HK, 0), (S, 0), (L, 0)])  # no rows at all
    assert not fn.meets(0, 400, 1 << 40, rows * f, packed)  # a buffer that is not given
    assert fn.ranges(100, 8, 107, 1) and not fn.ranges(100, 8, 108, 1) and not fn.ranges(100, 8, 92, 8) and not fn.ranges(0, 200, 100, 8)
