"""Which kernels the 8-bit operators take, on the CPU: every size that the entry points accept has a launch that the card takes."""
import pytest
import torch

from krea2_svdquant_amd.kernels.hip import lib
from krea2_svdquant_amd.quant.fp8 import quantize_fp8
from krea2_svdquant_amd.quant.pow2 import pow2
from tests import fp8_util as u

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


# ---- the converter ---------------------------------------------------------------------------------------
def test_powers_of_two():
    e = torch.arange(-149, 128)
    assert torch.equal(pow2(e).double(), torch.tensor([2.0 ** i for i in range(-149, 128)], dtype=torch.float64))


def every_exponent(g):
    """A weight of one column of blocks, a magnitude each: [257 blocks, 128, 40]."""
    amp = torch.exp2(torch.arange(-140, 117).double())[:, None, None]
    return (torch.randn(257, 128, 40, generator=g).double().clamp(-3.9, 3.9) * amp).float().flatten(0, 1)


def test_converter_at_every_exponent():
    w = every_exponent(torch.Generator().manual_seed(0))
    codes, scales = quantize_fp8(w)
    s = u.scale_of(w.double().view(257, 128, 40).abs().amax((1, 2)))
    assert torch.equal(scales[:, 0].double(), s)
    assert torch.equal(codes[:, :40].double(), u.e4m3(w.double() / s.repeat_interleave(128)[:, None]))


def test_every_product_kernel_is_tested_where_it_is_chosen():
    from tests.test_gpu_fp8_edges import DEEP, KERNELS
    every = ({(STRIP, *t) for t in ((32, 16), (32, 32), (64, 32), (48, 64), (64, 64))} |
             {(TILE, *t) for t in ((64, 64), (64, 128), (128, 128), (256, 128), (256, 256))} | {(ROWS, 16, 16)})
    for sizes in ([(m, n, 640, kernel) for m, n, kernel in KERNELS.values()], list(DEEP.values())):
        assert all(lib.fp8_kernel(m, n, k) == kernel for m, n, k, kernel in sizes)
        assert {kernel[:3] for *_, kernel in sizes} == every and any(kernel[3] for *_, kernel in sizes)


# ---- attention over the cache ----------------------------------------------------------------------------
def test_attention_plans():
    """An image over itself splits its last tiles alone; a long sequence's token is split, two thousand short ones' are not."""
    kind, splits, whole, tiles = lib.kv8_kernel(4352, 1, 73, 48, 12, 128, False)
    assert kind == 2 and splits > 1 and 0 < whole < tiles
    assert lib.kv8_kernel(4352, 1, 73, 48, 12, 128, True)[:2] == (2, 1)
    assert lib.kv8_kernel(1, 1, 2049, 48, 12, 128, True)[0] == 1 and lib.kv8_kernel(1, 1, 2049, 48, 12, 128, True)[1] > 8
    assert lib.kv8_kernel(2000, 2000, 64, 48, 12, 128, True)[:2] == (1, 1)
    assert lib.kv8_kernel(900, 5, 80, 64, 8, 64, True)[0] == 3
    for bad in ((0, 1, 1, 4, 2, 64), (1, 0, 1, 4, 2, 64), (1, 1, 0, 4, 2, 64), (1, 1, 1, 3, 2, 64), (1, 1, 1, 4, 2, 96), (2 ** 30, 1, 1, 64, 2, 64)):
        assert lib.kv8_kernel(*bad, True)[0] == 0


@pytest.mark.parametrize("causal", [False, True])
def test_attention_workspace_is_that_of_the_plan(causal):
    load = lib.load()
    for n, b, w, heads, kv, d in ((4352, 1, 73, 48, 12, 128), (1, 1, 2049, 48, 12, 128), (32, 32, 129, 48, 12, 128), (900, 5, 80, 64, 8, 64),
                                  (2140, 3, 14, 32, 2, 64), (300, 2, 3, 8, 1, 64)):
        kind, splits, whole, tiles = lib.kv8_kernel(n, b, w, heads, kv, d, causal)
        rows, pieces = (16, tiles * kv * splits if splits > 1 else 0) if kind == 1 else (128, 8 * (tiles - whole) * splits)
        assert load.svdq_kv8_attention_workspace(n, b, w, heads, kv, d, int(causal)) == pieces * rows * (d + 2) * 4
