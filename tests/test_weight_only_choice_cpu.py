"""Which kernel a product with a packed weight takes: `fos_weight_only_kernel`, the function that the entries decide with, needs no GPU. The shapes
here are those on which tests/test_weight_only_kernels_gpu.py compares every kernel with 64 bits: should the choice move, they move with it."""

from __future__ import annotations

import ctypes

import pytest

from fouroversix_b200 import _native

FEW_ROWS, PAIRS, EVEN = 1, 2, 3

# (kernel, CTAs that share K, rows, n, k): tiles of 32 to 256 rows with one tile per CTA, with more of them (a CTA's second tile) and with K
# shared; pairs with one and with two tiles each; stages dealt out evenly
FORWARD = [
    (32, 1, 17, 139, 300), (32, 2, 19, 4311, 1097), (32, 4, 19, 132, 1072), (32, 8, 18, 137, 2197),
    (64, 1, 33, 10057, 332), (64, 2, 36, 4784, 1193), (64, 4, 565, 138, 1047), (64, 8, 34, 1038, 2232),
    (128, 1, 72, 10182, 308), (128, 1, 261, 9697, 324), (128, 2, 69, 4773, 1036), (128, 4, 68, 2202, 996), (128, 8, 67, 1041, 2197),
    (256, 1, 129, 10414, 318), (256, 1, 445, 15111, 314), (256, 4, 130, 2111, 1156), (256, 8, 134, 1057, 2347),
    (PAIRS, 1, 131, 10243, 1682), (PAIRS, 1, 553, 11275, 663), (PAIRS, 1, 2049, 8001, 1100), (PAIRS, 1, 1281, 9000, 2048),
    (EVEN, 1, 17, 9573, 2779),
]
# the gradient of the input: the sum runs over n
GRADIENT = [
    (32, 1, 3, 303, 135), (32, 2, 1, 915, 4173), (32, 4, 20, 898, 128), (32, 8, 30, 2033, 132),
    (64, 1, 2524, 326, 129), (64, 2, 33, 933, 4778), (64, 4, 560, 915, 132), (64, 8, 33, 2021, 1037),
    (128, 1, 66, 327, 10676), (128, 1, 301, 304, 9690), (128, 2, 66, 905, 5499), (128, 4, 1079, 976, 130), (128, 8, 541, 2089, 142),
    (256, 1, 134, 313, 11152), (256, 1, 408, 322, 15251), (256, 4, 162, 928, 2142), (256, 8, 1121, 1940, 154),
    (PAIRS, 1, 132, 1317, 11068), (PAIRS, 1, 1706, 643, 4036), (PAIRS, 1, 2049, 1100, 8001), (PAIRS, 1, 1281, 2048, 9000),
]
# (kernel, rows, n, k, groups)
GROUPED = [(FEW_ROWS, 33, 129, 257, 9), (32, 25, 137, 311, 3), (64, 342, 782, 303, 21), (128, 917, 664, 312, 21), (256, 1835, 694, 317, 21),
           (PAIRS, 2488, 517, 1321, 21), (PAIRS, 3000, 1000, 1500, 5), (EVEN, 78, 132, 4051, 9)]


def choice(rows, n, k, groups=0, transposed=0, block=64):
    split = ctypes.c_int(0)
    kernel = _native.lib().fos_weight_only_kernel(rows, -(-n // 128) * 128, -(-k // block) * block, groups, transposed, ctypes.byref(split))
    return kernel, split.value


@pytest.mark.parametrize("block", [64, 128])                 # NVFP4 and IF4 pad K to 64, MXFP4 to 128
@pytest.mark.parametrize("case", FORWARD)
def test_forward(case, block):
    kernel, split, rows, n, k = case
    assert choice(rows, n, k, block=block) == (kernel, split)


@pytest.mark.parametrize("block", [64, 128])
@pytest.mark.parametrize("case", GRADIENT)
def test_gradient(case, block):
    kernel, split, rows, n, k = case
    assert choice(rows, n, k, transposed=1, block=block) == (kernel, split)


@pytest.mark.parametrize("block", [64, 128])
@pytest.mark.parametrize("case", GROUPED)
def test_grouped(case, block):
    kernel, rows, n, k, groups = case
    assert choice(rows, n, k, groups, block=block)[0] == kernel


def test_some_ctas_have_a_second_tile():
    """148 SMs: tiles of 128 features by the kernel's rows, or of 256 by 256 for 74 pairs."""
    for cases, columns in ((FORWARD, 3), (GRADIENT, 4)):
        for kernel in (128, 256, PAIRS):
            wide = 256 if kernel == PAIRS else kernel
            tiles = [-(-c[columns] // (256 if kernel == PAIRS else 128)) * -(-c[2] // wide) for c in cases if c[:2] == (kernel, 1)]
            assert max(tiles) > (74 if kernel == PAIRS else 148), (kernel, tiles)


def test_few_rows():
    """Up to eight rows whatever the weight, with K shared by up to eight CTAs of four steps each."""
    for rows in (1, 8):
        for n, k in ((1, 1), (4096, 4096), (28672, 8192)):
            assert choice(rows, n, k)[0] == FEW_ROWS
    assert [choice(1, n, 8192)[1] for n in (128, 128 * 112, 128 * 120, 128 * 224, 128 * 240, 128 * 480)] == [8, 8, 4, 4, 2, 1]
    assert [choice(1, 128, k)[1] for k in (512, 1024, 2048, 4096)] == [1, 2, 4, 8]


def test_refusals():
    for bad in ((0, 128, 64, 0, 0), (1, 0, 64, 0, 0), (1, 100, 64, 0, 0), (1, 128, 0, 0, 0), (1, 128, 32, 0, 0), (1, 128, 64, -1, 0), (1, 128, 64, 257, 0),
                (1, 128, 64, 4, 1)):
        assert _native.lib().fos_weight_only_kernel(*bad, None) == -1
