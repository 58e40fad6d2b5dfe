"""The selection's search over order keys, compiled for the host: exact and at most three steps for any keys."""
import ctypes
import math
import shutil
import subprocess
from pathlib import Path

import numpy as np
import pytest

CSRC = Path(__file__).resolve().parent.parent / "fier-2bits_b200" / "csrc"

# The kernel's loop for one row: a histogram a step, then the bin that holds the wanted rank.
HARNESS = r"""
#include "key_range.h"
using popkv::KeyRange;
extern "C" int search(const uint32_t* keys, int n, uint32_t want, uint32_t* thr, uint32_t* taken) {
    KeyRange r{0xffffffffu, 0u};
    for (int i = 0; i < n; ++i) {
        r.lo = keys[i] < r.lo ? keys[i] : r.lo;
        r.hi = keys[i] > r.hi ? keys[i] : r.hi;
    }
    uint32_t left = want;
    for (int step = 1; step <= 20; ++step) {
        static uint32_t hist[1 << KeyRange::kBits];
        for (uint32_t& h : hist) h = 0;
        const int shift = r.shift();
        for (int i = 0; i < n; ++i)
            if (r.holds(keys[i])) {
                if (r.bin(keys[i], shift) >> KeyRange::kBits) return -1;  // past the histogram
                ++hist[r.bin(keys[i], shift)];
            }
        uint32_t above = 0, pick = 0, in = 0, before = 0;
        bool found = false;
        for (int i = (1 << KeyRange::kBits) - 1; i >= 0; --i) {
            if (above < left && above + hist[i] >= left) {
                pick = i; before = above; in = hist[i]; found = true;
            }
            above += hist[i];
        }
        if (!found) return -2;  // no bin holds the rank: the kernel would go on with a stale one
        r.keep(pick, shift);
        left -= before;
        if (left == in || shift == 0) {
            *thr = r.lo;
            *taken = left == in ? 0xffffffffu : left;
            return step;
        }
    }
    return -3;  // never ends
}
"""


@pytest.fixture(scope="module")
def search(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("no host compiler")
    d = tmp_path_factory.mktemp("key_range")
    (d / "search.cpp").write_text(HARNESS)
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", f"-I{CSRC}", str(d / "search.cpp"), "-o", str(d / "s.so")],
                   check=True)
    lib = ctypes.CDLL(str(d / "s.so"))

    def run(keys, want):
        keys = np.ascontiguousarray(keys, dtype=np.uint32)
        thr, taken = ctypes.c_uint32(), ctypes.c_uint32()
        steps = lib.search(keys.ctypes.data_as(ctypes.c_void_p), len(keys), ctypes.c_uint32(want), ctypes.byref(thr),
                           ctypes.byref(taken))
        return steps, thr.value, taken.value
    return run


def order_keys(x):
    """Larger number, larger key; NaN above everything (the kernel's select_key)."""
    x = np.asarray(x, dtype=np.float32) + np.float32(0)  # -0 as +0
    u = x.view(np.uint32)
    key = np.where(u >> 31, ~u, u | np.uint32(0x80000000)).astype(np.uint32)
    return np.where(np.isnan(x), np.uint32(0xffffffff), key).astype(np.uint32)


def check(search, keys, want):
    steps, thr, taken = search(keys, want)
    assert 1 <= steps <= 3, (steps, want)
    above, equal = int((keys > thr).sum()), int((keys == thr).sum())
    if taken == 0xffffffff:
        assert int((keys >= thr).sum()) == want
    else:
        assert taken <= equal and above + taken == want


def test_a_row_of_two_numbers_and_two_nan(search):
    check(search, order_keys([-0.4257649, -0.3772625, math.nan, math.nan]), 1)


@pytest.mark.parametrize("nans", [0, 1, 2, 5, 17, 60, 199])
def test_rows_with_nan(search, nans):
    rng = np.random.default_rng(nans)
    for _ in range(60):
        n = int(rng.integers(1, 250))
        x = rng.standard_normal(n + nans).astype(np.float32) * np.float32(10.0 ** rng.uniform(-30, 30))
        x[rng.permutation(n + nans)[:nans]] = np.nan
        if rng.random() < 0.3:
            x[rng.integers(n + nans)] = np.inf
        keys = order_keys(x)
        for want in {1, max(1, nans - 1), max(1, nans), nans + 1, int(rng.integers(1, n + nans))}:
            if want < len(keys):
                check(search, keys, want)


@pytest.mark.parametrize("lo,hi", [(1, 0xffffffff), (1, 2), (0xfffffff0, 0xffffffff), (0x7fffffff, 0x80000001),
                                   (0xffdfffff, 0xffffffff), (0x40000001, 0xffffffff)])
def test_keys_at_the_ends_of_the_range(search, lo, hi):
    rng = np.random.default_rng(lo & 0xffff)
    for _ in range(60):
        keys = rng.integers(lo, hi, size=int(rng.integers(2, 300)), dtype=np.uint32, endpoint=True)
        keys[:2] = lo, hi
        keys[2:2 + int(rng.integers(0, 6))] = hi
        for want in {1, 2, len(keys) - 1, int(rng.integers(1, len(keys)))}:
            check(search, keys, want)
