"""The whole-number sums of the sampling kernel at its largest sizes, without a GPU: the constants of
``csrc/sample.cu`` and the arithmetic that its words of 32 and 64 bits do with them."""
import os
import re

import numpy as np
import pytest

SRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "dsalt_b200", "csrc", "sample.cu")


@pytest.fixture(scope="module")
def const():
    found = {}
    for line in re.findall(r"constexpr int ([^;]*);", open(SRC, encoding="utf-8").read()):
        for name, value in re.findall(r"(\w+) = (\d+)(?=,|$)", line):
            found[name] = int(value)
    return found


def shares(vocab, step=256):
    """Elements of one block's share, as the host cuts a row of this vocabulary into 1, 2, 4 or 8."""
    return {c: (vocab + 7 + c * step - 1) // (c * step) * step for c in (1, 2, 4, 8) if c == 8 or vocab / c <= 80000}


@pytest.mark.parametrize("vocab", [5, 50257, 151936, 640000, 2**20 - 7, 2**20 - 6, 2**20])
def test_a_histogram_of_one_bin_holds_a_whole_share(const, vocab):
    """Every element of a share in one bin, each with the same mass: the limbs' sums in 32-bit words give the
    sum of the masses. The masses have limbs of ones, or are the largest."""
    bits, limbs, one = const["LIMB_BITS"], const["LIMBS"], 1 << const["MASS_BITS"]
    masses = [one, one - 1, one // 2 + 1] + [(1 << n) - 1 for n in range(1, const["MASS_BITS"] + 1)]
    masses += [one // 4096 - d for d in (1, 100, 32767)]  # weights just below 2^-12
    for n in shares(vocab).values():
        assert n <= const["MAX_SHARE"]
        for m in masses:
            words = [np.uint32(n * (m >> x * bits & (1 << bits) - 1) & 0xffffffff) for x in range(limbs)]
            assert sum(int(w) << x * bits for x, w in enumerate(words)) == n * m, (n, m)


def test_a_threads_bins_hold_its_elements(const):
    # count in the upper 12 bits, mass in the lower 52; a thread has 8 elements of each of its warp's steps
    steps = -(-const["MAX_SHARE"] // 256)
    per_thread = -(-steps // (const["SAMPLE_THREADS"] // 32)) * 8
    assert per_thread < 1 << 12 and per_thread << const["MASS_BITS"] < 1 << 52
