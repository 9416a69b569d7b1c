"""CPU-only: what the plans of the real-valued products ask of an SM, over their whole range of sizes."""
import ctypes as C
import random

import pytest

from tcbnn_b200 import lib

SMS = 148
SIZES = [1, 5, 8, 16, 17, 31, 48, 64, 100, 200, 224, 256, 333, 512, 1000, 1024, 2049, 4096, 8192, 16384, 32768, 50000, 131072]


def plan(M, N, K, packed, cols=0, splits=0, out=lib.BF16):
    """(few rows' kernel taken, form, cols, splits, sets of sums, columns of tensor memory, stages, bytes of shared memory, chained sums)"""
    of = (C.c_int * 9)()
    lib.call("tcbnn_set_linear_plan", cols, splits)
    try:
        lib.call("tcbnn_linear_plan", M, N, K, int(packed), out, SMS, of)
    finally:
        lib.call("tcbnn_set_linear_plan", 0, 0)
    return tuple(of)


def sizes():
    rng = random.Random(5)
    some = [(M, N, K) for M in SIZES[:20] for N in SIZES for K in (64, 512, 4096, 16384)]
    return some + [tuple(int(2 ** rng.uniform(0, top)) for top in (13, 17, 14)) for _ in range(2000)]


def columns_read(cols, sets):
    """The epilogue reads 32 columns at a time of each set, which start `cols` apart."""
    return (sets - 1) * cols + (cols + 31) // 32 * 32


@pytest.mark.parametrize("packed", [False, True])
def test_all_columns_that_are_read_are_allocated(packed):
    for M, N, K in sizes():
        _, _, cols, _, sets, columns, _, smem, _ = plan(M, N, K, packed)
        assert columns_read(cols, sets) <= columns <= 512 and columns & (columns - 1) == 0, (M, N, K, cols, sets, columns)
        assert smem <= 227 * 1024


@pytest.mark.parametrize("packed,cols,splits", [(b, c, s) for b in (False, True) for s in (1, 2, 4, 8, -2) for c in range(16, 257, 16)
                                                if not (s == -2 and (b or c % 32)) and not (b and s > 1 and c > 128)])
def test_all_columns_of_forced_plans_are_allocated(packed, cols, splits):
    for M, N, K in [(1, 128, 64), (8, 50000, 512), (5000, 1500, 640), (4096, 16384, 4096)]:
        if splits > 1 and -(-M // cols) * -(-N // 128) * splits > 1 << 20:
            continue
        _, _, c, _, sets, columns, _, smem, _ = plan(M, N, K, packed, cols, splits)
        assert c == cols and columns_read(c, sets) <= columns <= 512
        assert smem <= 227 * 1024


def test_long_sums_of_fp32_results_are_chained():
    """Dense weights: no set of sums takes more than 768 of K.  Two sets take turns, for 64 tokens at most in a cluster's CTA, or a cluster's CTA has
    a set for each chain."""
    for M, N, K in sizes():
        _, form, cols, splits, sets, columns, _, smem, chained = plan(M, N, K, False, out=lib.FP32)
        blocks = -(-(-(-K // 64)) // splits)
        if chained:
            assert blocks > 12 and sets == 2 and (form != 1 or cols <= 64), (M, N, K, form, cols, splits)
        else:
            assert blocks <= 12 * (sets if form == 1 else 1), (M, N, K, form, cols, splits)
        assert columns_read(cols, sets) <= columns <= (256 if form == 1 else 512) and smem <= 227 * 1024
        assert not plan(M, N, K, False)[8] and not plan(M, N, K, True, out=lib.FP32)[8]


@pytest.mark.parametrize("out", [lib.BF16, lib.FP32])
@pytest.mark.parametrize("packed", [False, True])
def test_shared_sums_leave_half_an_sm_and_three_stages(packed, out):
    """A CTA of a cluster keeps to 113 KB, two to an SM, with three stages at least."""
    for M, N, K in sizes() + [(224, 4096, 4096), (1024, 1024, 4096), (566, 1504, 3560)]:
        few, form, cols, _, _, _, stages, smem, _ = plan(M, N, K, packed, out=out)
        if form == 1 and not few:
            assert stages >= 3 and smem <= 113 * 1024, (M, N, K, cols, stages, smem)
