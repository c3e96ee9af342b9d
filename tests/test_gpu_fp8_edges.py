"""The 8-bit operators at the ends of their sizes, values and launches, against their definitions in 64 bits."""
from __future__ import annotations

import pytest
import torch

from krea2_svdquant_amd.kernels.hip import ops
from tests import fp8_util as u

pytestmark = pytest.mark.gpu


def gen(seed):
    return torch.Generator().manual_seed(seed)


def normal(shape, g, amp=1.0):
    return (amp * torch.randn(shape, generator=g)).to(torch.bfloat16)


# ---- the product ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("m", [3, 12])
def test_product_of_more_columns_than_a_launch_of_few_rows_holds(dev, m):
    """16 columns a workgroup of 512 threads would be 2^32 threads and more.  One block of K: a value is one product."""
    n, g = 2 ** 27 + 5, torch.Generator(device=dev).manual_seed(m)
    w = torch.zeros((n, 128), dtype=torch.float8_e4m3fn, device=dev)
    ws = torch.ones((-(-n // 128), 1), device=dev)
    x = torch.randint(-3, 4, (m, 128), device=dev, generator=g).to(torch.bfloat16)
    parts = [slice(s, s + 200) for s in (0, 2 ** 26 - 100, 2 ** 27 - 195)]
    for p in parts:
        w[p] = torch.randint(-3, 4, (200, 128), device=dev, generator=g).float().to(torch.float8_e4m3fn)
        ws[p.start // 128:p.start // 128 + 2] = 2.0
    a, sa = ops.fp8_quantize(x)
    for y in (ops.fp8_gemm(a, sa, w, ws), ops.fp8_linear(x, w, ws)):
        for p in parts:
            s = ws[torch.arange(p.start, p.stop, device=dev) // 128].double()
            assert torch.equal(y[:, p], (x.double() @ (w[p].double() * s).T).to(torch.bfloat16))
        assert not y[:, 300:400].any() and not y[:, 2 ** 26 + 200:2 ** 26 + 300].any()


# ---- the converter -------------------------------------------------------------------------------------------
def test_converter_on_the_gpu_is_the_one_on_the_cpu(dev):
    from krea2_svdquant_amd.quant.fp8 import quantize_fp8
    from tests.test_fp8_edges_cpu import every_exponent
    w = every_exponent(gen(0))
    (codes, scales), (c, s) = quantize_fp8(w), quantize_fp8(w.to(dev))
    assert torch.equal(s.cpu(), scales) and torch.equal(c.cpu().view(torch.uint8), codes.view(torch.uint8))


@pytest.mark.parametrize("fmt", ["e2m1", "e4m3"])
def test_mx_converter_on_the_gpu_is_the_one_on_the_cpu(dev, fmt):
    """Every exponent of a block's scale, and values between two codes."""
    from krea2_svdquant_amd.quant.mx import dequantize_mx, quantize_mx
    amp = torch.exp2(torch.arange(-140, 116).float())[:, None]
    for x in (torch.randn(256, 32, generator=gen(1)), torch.randint(-24, 25, (256, 32), generator=gen(2)) / 4):
        codes, scales = quantize_mx(x * amp, fmt)
        c, s = quantize_mx((x * amp).to(dev), fmt)
        assert torch.equal(c.cpu().view(torch.uint8), codes.view(torch.uint8))
        assert torch.equal(s.cpu().view(torch.uint8), scales.view(torch.uint8))
        assert torch.equal(dequantize_mx(c, s, 32).cpu(), dequantize_mx(codes, scales, 32))
