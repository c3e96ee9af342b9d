"""Which kernels the 8-bit operators take, on the CPU: every size that the entry points accept has a launch that the card takes."""
import pytest

from krea2_svdquant_amd.kernels.hip import lib

TILE, STRIP, ROWS = 1, 2, 3


def threads(kind, rows, cols):
    return 512 if kind == ROWS or rows * cols >= 256 * 128 or (kind == STRIP and rows == 32) else 256


@pytest.mark.parametrize("m", [1, 2, 4, 8, 15, 16, 17, 20, 32, 33, 64])
def test_product_launches_hold_fewer_than_2_32_threads(m):
    for n in (1, 16, 2 ** 20, 2 ** 26, 2 ** 27 - 16, 2 ** 27 - 15, 2 ** 27, 2 ** 28 + 1, 2 ** 29, (2 ** 24 - 1) * 64):
        for k in (1, 128, 1024):
            kind, rows, cols, head = lib.fp8_kernel(m, n, k)
            assert kind in (TILE, STRIP, ROWS) and head == 0
            assert -(-m // rows) * -(-n // cols) * threads(kind, rows, cols) < 2 ** 32, (n, k)


def test_product_kernel_is_told_of_sizes_that_are_taken_alone():
    assert lib.fp8_kernel(5, 300, 640) == (ROWS, 16, 16, 0)
    assert lib.fp8_kernel(0, 300, 640)[0] == lib.fp8_kernel(5, 0, 640)[0] == lib.fp8_kernel(5, 300, 0)[0] == 0
    assert lib.fp8_kernel(5, 300, 2 ** 22 + 1)[0] == 0 and lib.fp8_kernel(2 ** 30, 2 ** 14, 128)[0] == 0
