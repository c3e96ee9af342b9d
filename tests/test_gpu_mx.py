"""The microscaled operators on the GPU against 64-bit numpy.  Quantising is exact; products are held to float32's
rounding of their sums; the norm's and the SwiGLU product's codes to those of values within float32's rounding."""
import numpy as np
import pytest
import torch

from krea2_svdquant_amd.kernels.hip import lib, ops
from krea2_svdquant_amd.quant.mx import quantize_mx
from oracle import mx
from tests.mx_util import (check_blocks, check_product, dropped, f64, random_mx, to_device, to_oracle, values)

pytestmark = pytest.mark.gpu
FMTS = list(mx.FORMATS)
EPS = 1e-6


def _act(dev, *shape, seed=0, dtype=torch.bfloat16):
    gen = torch.Generator(device=dev).manual_seed(seed)
    x = torch.randn(shape, device=dev, generator=gen)
    return (x * torch.where(torch.rand(shape[-1], device=dev, generator=gen) < 0.02, 16.0, 1.0)).to(dtype)


def _check_quantized(x, fmt):
    codes, scales = ops.mx_quantize(x, fmt)
    assert codes.shape[:-1] == x.shape[:-1] and (codes.shape[-1], scales.shape[-1]) == ops.mx_shapes(x.shape[-1], fmt)
    want_c, want_s = mx.quantize(f64(x).reshape(-1, x.shape[-1]), fmt)
    got_c, got_s, _ = to_oracle(codes, scales)
    assert np.array_equal(got_s, want_s)
    assert np.array_equal(got_c, want_c)
    back = ops.mx_dequantize(codes, scales, x.shape[-1])
    want = torch.from_numpy(mx.dequantize(want_c, want_s, fmt)[:, :x.shape[-1]]).to(torch.bfloat16)
    assert back.shape == x.shape and torch.equal(back.cpu().view(torch.int16).reshape(want.shape).masked_fill(want.isnan(), 0),
                                                 want.view(torch.int16).masked_fill(want.isnan(), 0))
    assert torch.equal(back.cpu().reshape(want.shape).isnan(), want.isnan())


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("m,k", [(1, 1), (1, 8), (3, 31), (2, 32), (5, 33), (7, 127), (4, 128), (3, 136), (2, 511),
                                 (2, 512), (3, 520), (33, 1000), (1, 6144), (65, 1187), (3, 16384), (17000, 40), (16999, 41)])
def test_quantize(dev, fmt, m, k):
    _check_quantized(_act(dev, m, k, seed=k), fmt)


@pytest.mark.parametrize("fmt", FMTS)
def test_quantize_every_bf16_value(dev, fmt):
    # every bit pattern as a block's largest magnitude, with smaller companions that reach ties and zeros
    bits = torch.arange(65536, device=dev, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    f = torch.tensor([1, -1, 0.5, 0.25, -0.125, 0.0625, 0.75, -0.6, 0.4, 0.3, 0.2, 0.15, 0.1, 1 / 24, 3 / 16, 5 / 6,
                      7 / 12, 5 / 12, 7 / 24, 1 / 48, 1 / 100, 1 / 300, 1 / 900, 1e-4, 0, -0.0, 0.9, -0.8, 0.7, 0.55,
                      0.45, 0.35], device=dev)
    x = (bits.float()[:, None] * f).to(torch.bfloat16)
    x[:, 0] = bits
    _check_quantized(x.reshape(2048, 1024), fmt)


@pytest.mark.parametrize("fmt", FMTS)
def test_quantize_layouts(dev, fmt):
    base = _act(dev, 40, 1100, seed=3)
    for x in (base[:, 3:1003], base[:, 8:1032], base[::2, :1024], base.t()[:512], base[5, :768].expand(6, 768),
              base[:30].reshape(2, 3, 5, 1100)[:, 1:, ::2, :96], base.flatten()[1:1 + 64 * 65].view(65, 64), base[7, :100]):
        codes, scales = ops.mx_quantize(x, fmt)
        want = ops.mx_quantize(x.contiguous().clone(), fmt)
        assert codes.shape == want[0].shape
        assert torch.equal(codes.view(torch.uint8), want[0].view(torch.uint8))
        assert torch.equal(scales.view(torch.uint8), want[1].view(torch.uint8))
        _check_quantized(x, fmt)


@pytest.mark.parametrize("fmt", FMTS)
def test_dequantize_every_code_and_scale(dev, fmt):
    n = 16 if fmt == "e2m1" else 256
    codes = np.tile(np.arange(n, dtype=np.uint8), (256, 512 // n))
    scales = np.repeat(np.arange(256, dtype=np.uint8)[:, None], 16, 1)
    c, s = to_device(codes, scales, fmt, dev)
    want = torch.from_numpy(mx.dequantize(codes, scales, fmt)).to(torch.bfloat16)
    got = ops.mx_dequantize(c, s, 512).cpu()
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got.nan_to_num(0), want.nan_to_num(0))


@pytest.mark.parametrize("fmt", FMTS)
def test_no_rows(dev, fmt):
    x = torch.empty(0, 200, device=dev, dtype=torch.bfloat16)
    codes, scales = ops.mx_quantize(x, fmt)
    assert codes.shape == (0, ops.mx_shapes(200, fmt)[0]) and scales.shape == (0, 16)
    assert ops.mx_dequantize(codes, scales, 200).shape == (0, 200)
    w, ws = ops.mx_quantize(_act(dev, 24, 200))
    assert ops.mx_gemm(codes, scales, w, ws).shape == (0, 24)
    assert ops.mx_linear(x, w, ws, fmt=fmt).shape == (0, 24)
    assert ops.silu_mul_mx(x, x, fmt)[0].shape == codes.shape
    v = torch.ones(200, device=dev, dtype=torch.bfloat16)
    assert ops.rms_norm_modulate_mx(x, v, v, EPS, fmt)[1].shape == scales.shape
    assert ops.residual_rms_norm_modulate_mx(x, x, v, v, v, EPS, fmt)[0].shape == (0, 200)


# ---- product ----
SIZES = [(1, 1, 1), (1, 17, 128), (3, 64, 129), (16, 128, 640), (17, 33, 1000), (31, 1001, 512), (32, 256, 2176),
         (33, 96, 384), (64, 64, 6144), (65, 130, 768), (77, 1536, 1187), (100, 40, 16384), (128, 256, 896),
         (129, 257, 1152), (255, 384, 1024), (300, 520, 640), (513, 1030, 256), (700, 2049, 384)]


def _product_case(dev, m, n, k, fmt, seed=0, narrow=False):
    a, sa = random_mx(m, k, fmt, seed + 1, narrow)
    w, sw = random_mx(n, k, "e2m1", seed + 2)
    return (*to_device(a, sa, fmt, dev), *to_device(w, sw, "e2m1", dev)), mx.dequantize(a, sa, fmt), mx.dequantize(
        w, sw, "e2m1")


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("m,n,k", SIZES)
def test_product(dev, fmt, m, n, k):
    t, a, w = _product_case(dev, m, n, k, fmt, seed=m)
    bias = _act(dev, n, seed=9)
    check_product(ops.mx_gemm(*t, None, True), a, w)
    check_product(ops.mx_gemm(*t, bias, True), a, w, f64(bias))
    y = ops.mx_gemm(*t, bias)
    check_product(y, a, w, f64(bias), dropped(a, w) if fmt == "e4m3" else 0)
    assert torch.equal(y, ops.mx_gemm(*t, bias))   # the same bits every time
    if fmt == "e4m3":   # codes between which nothing is dropped: the plain bound
        t, a, w = _product_case(dev, m, n, k, fmt, seed=m, narrow=True)
        check_product(ops.mx_gemm(*t, bias), a, w, f64(bias))


# sizes that each kernel is chosen for, with ragged edges on both sides: (kind, rows, columns) as lib.mx_tile gives them
TILES = {"e2m1": {(2, 8, 16): (7, 1000), (2, 16, 16): (13, 1000), (1, 64, 64): (70, 3000), (1, 128, 64): (250, 6100),
                  (1, 128, 128): (500, 8100), (1, 256, 256): (1990, 8100)},
         "e4m3": {(2, 8, 16): (7, 1000), (1, 64, 64): (70, 3000), (1, 64, 128): (250, 6100), (1, 128, 128): (500, 8100),
                  (1, 256, 256): (1990, 8100)}}


@pytest.mark.parametrize("k", [128, 384, 640, 1000, 2304, 2432])   # one stage, halves of one, ends within a chunk of scales
@pytest.mark.parametrize("fmt,tile", [(f, t) for f in FMTS for t in TILES[f]])
def test_every_tile(dev, fmt, tile, k):
    _check_tile(dev, fmt, tile, *TILES[fmt][tile], k)


@pytest.mark.parametrize("fmt", FMTS)
def test_last_rows_on_smaller_tiles(dev, fmt):
    _check_tile(dev, fmt, (3, 256, 256), 2200, 8100, 3000)


def _check_tile(dev, fmt, tile, m, n, k):
    assert lib.mx_tile(m, n, k, ops.MX_FORMATS[fmt]) == tile
    x, w = _act(dev, m, k, seed=1), _act(dev, n, k, seed=2)
    a, b = ops.mx_quantize(x, fmt), ops.mx_quantize(w)
    bias = _act(dev, n, seed=3)
    av, bv = (torch.from_numpy(values(*t)).to(dev) for t in (a, b))   # float64 on the card: torch's product there
    y, mag = av @ bv.T + bias.double(), av.abs() @ bv.abs().T + bias.double().abs()
    bound = 1.01 * (av.shape[1] + 1) * 2.0 ** -24 * mag   # as mx_util.product_bound
    got = ops.mx_gemm(*a, *b, bias, True).double()
    assert ((got - y).abs() <= bound).all()
    if fmt == "e4m3":
        ma, mb = (t.abs().reshape(len(t), -1, mx.BLOCK).amax(-1) for t in (av, bv))
        bound = bound + 4 * 7 * 2.0 ** -13 * 2 * (ma @ mb.T)   # as mx_util.dropped
    bound = bound + 2.0 ** -8 * (y.abs() + bound)
    got = ops.mx_gemm(*a, *b, bias).double()
    assert ((got - y).abs() <= bound).all()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("m,n", [(5, 40), (40, 72), (300, 300)])
def test_product_is_blockwise(dev, fmt, m, n):
    # blocks with scales of their own over 40 powers of two, exactly representable sums: any mistake in which scale
    # goes with which block, or which code with which, moves the result
    k = 1024
    rng = np.random.default_rng(m)
    a = rng.integers(0, 8, (m, k)).astype(np.uint8) if fmt == "e2m1" else rng.integers(0x30, 0x48, (m, k)).astype(np.uint8)
    a |= (rng.integers(0, 2, (m, k)) * (8 if fmt == "e2m1" else 128)).astype(np.uint8)
    w = rng.integers(0, 16, (n, k)).astype(np.uint8)
    sa = np.zeros((m, 32), np.uint8)
    sw = np.zeros((n, 32), np.uint8)
    one = rng.integers(0, 32)   # a single block counts: its scales are 2^0 to 2^3, all others 2^-40
    sa[:], sw[:] = 107, 107
    sa[:, one] = rng.integers(127, 131, m)
    sw[:, one] = rng.integers(127, 131, n)
    t = (*to_device(a, sa, fmt, dev), *to_device(w, sw, "e2m1", dev))
    av, wv = mx.dequantize(a, sa, fmt), mx.dequantize(w, sw, "e2m1")
    check_product(ops.mx_gemm(*t, None, True), av, wv)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("m", [2, 40, 200])
def test_product_of_blocks_that_are_not_numbers(dev, fmt, m):
    t, a, w = _product_case(dev, m, 70, 384, fmt)
    scales_a, scales_w = t[1].view(torch.uint8), t[3].view(torch.uint8)
    scales_a[1, 3] = 255
    scales_w[69, 11] = 255
    scales_a[0, 12:] = 255   # the padding of a row's scales is not read
    scales_w[0, 12:] = 255
    a[1] = np.nan
    w[69] = np.nan
    y = f64(ops.mx_gemm(*t, None, True))
    bad = np.zeros((m, 70), bool)
    bad[1], bad[:, 69] = True, True
    assert np.array_equal(np.isnan(y), bad)
    assert np.array_equal(y[0, :69], f64(ops.mx_gemm(*_product_case(dev, m, 70, 384, fmt)[0], None, True))[0, :69])


@pytest.mark.parametrize("fmt", FMTS)
def test_product_of_zeros_and_of_extreme_scales(dev, fmt):
    for m in (3, 90):
        t, a, w = _product_case(dev, m, 50, 256, fmt)
        z, sz = ops.mx_quantize(torch.zeros(m, 256, device=dev, dtype=torch.bfloat16), fmt)
        assert (sz.view(torch.uint8) == 0).all()
        assert torch.equal(ops.mx_gemm(z, sz, t[2], t[3], None, True), torch.zeros(m, 50, device=dev))
        t[1].view(torch.uint8)[:, :8] = 0        # 2^-127 against 2^120: an ordinary result
        t[3].view(torch.uint8)[:, :8] = 247
        av, wv = values(t[0], t[1]), values(t[2], t[3])
        check_product(ops.mx_gemm(*t, None, True), av, wv)


def test_product_shapes_and_rows_behind(dev):
    (a, sa, w, sw), av, wv = _product_case(dev, 24, 96, 256, "e4m3", narrow=True)
    y = ops.mx_gemm(a.view(2, 3, 4, 256), sa.view(2, 3, 4, 16), w, sw)
    assert y.shape == (2, 3, 4, 96)
    check_product(y.view(24, 96), av, wv)
    y1 = ops.mx_gemm(a[5], sa[5], w, sw, None, True)
    assert y1.shape == (96,)
    check_product(y1.view(1, 96), av[5:6], wv)
    # a wider destination through the C entry: columns and rows behind the product stay as they were
    for m, n in ((24, 96), (3, 90), (23, 95)):
        out = torch.full((m + 2, n + 5), 7.0, device=dev, dtype=torch.bfloat16)
        st = torch.cuda.current_stream().cuda_stream
        lib.call("svdq_mx_gemm", a.data_ptr(), sa.data_ptr(), lib.SVDQ_MX_E4M3, w.data_ptr(), sw.data_ptr(), None, m, n,
                 256, out.data_ptr(), n + 5, 0, st)
        assert torch.equal(out[:m, :n], ops.mx_gemm(a[:m].contiguous(), sa[:m].contiguous(), w[:n].contiguous(),
                                                    sw[:n].contiguous()))
        assert (out[m:] == 7).all() and (out[:, n:] == 7).all()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("m,n,k", [(1, 64, 256), (20, 100, 1000), (77, 512, 640), (200, 96, 129)])
def test_linear(dev, fmt, m, n, k):
    x = _act(dev, m, k, seed=4)
    w, sw = quantize_mx(_act(dev, n, k, seed=5, dtype=torch.float32) * 0.02)
    bias = _act(dev, n, seed=6)
    y = ops.mx_linear(x, w, sw, bias, fmt)
    assert torch.equal(y, ops.mx_gemm(*ops.mx_quantize(x, fmt), w, sw, bias))
    a = mx.dequantize(*mx.quantize(f64(x), fmt), fmt)
    check_product(y, a, values(w, sw), f64(bias), dropped(a, values(w, sw)) if fmt == "e4m3" else 0)
    check_product(ops.mx_linear(x, w, sw, bias, fmt, True), a, values(w, sw), f64(bias))
    wide = torch.zeros(m, k + 9, device=dev, dtype=torch.bfloat16)
    wide[:, 5:5 + k] = x
    assert torch.equal(y, ops.mx_linear(wide[:, 5:5 + k], w, sw, bias, fmt))
    assert ops.mx_linear(x.view(m, 1, k), w, sw, None, fmt, True).shape == (m, 1, n)


# ---- norm ----
def _norm64(x, w, shift, eps):
    """y, and how far float32's evaluation may be from it.  The mean of squares adds positive terms, at most
    K / 256 + 16 of them one after another, rsqrt, the product with x and the fma round once each: under
    K / 512 + 16 roundings of 2^-24 of the two terms' magnitudes."""
    t = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w
    return t + shift, (x.shape[1] / 512 + 16) * 2.0 ** -24 * (np.abs(t) + np.abs(shift))


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("m,h", [(1, 8), (2, 104), (5, 128), (3, 1000), (4, 2048), (2, 2056), (3, 6144), (9, 8192),
                                 (2, 8200), (2, 16384)])
def test_norm(dev, fmt, m, h):
    x, v = _act(dev, m, h, seed=1), _act(dev, m, h, seed=2)
    if m > 2:
        x[1], v[1] = 0, 0
    gate, w, shift = (_act(dev, h, seed=s) for s in (3, 4, 5))
    codes, scales = ops.rms_norm_modulate_mx(x, w, shift, EPS, fmt)
    check_blocks(codes, scales, *_norm64(f64(x), f64(w), f64(shift), EPS))
    xo, codes, scales = ops.residual_rms_norm_modulate_mx(x, v, gate, w, shift, EPS, fmt)
    want, _ = ops.residual_rms_norm_modulate(x, v, gate, w, shift, EPS)
    assert torch.equal(xo, want)   # the residual stream's bits do not depend on the output's form
    check_blocks(codes, scales, *_norm64(f64(xo), f64(w), f64(shift), EPS))


@pytest.mark.parametrize("fmt", FMTS)
def test_norm_layouts_and_rows_that_are_not_finite(dev, fmt):
    base = _act(dev, 12, 1200, seed=8)
    w, shift, gate = (_act(dev, 1032, seed=s)[1:1025] for s in (3, 4, 5))   # vectors of any alignment
    for x in (base[:, 8:1032], base[:, 3:1027], base[::3, :1024], base[2, :1024].expand(4, 1024),
              base[:, :1024].reshape(2, 6, 1024)):
        got = ops.residual_rms_norm_modulate_mx(x, x, gate, w, shift, EPS, fmt)
        c = x.contiguous().clone()
        want = ops.residual_rms_norm_modulate_mx(c, c, gate.clone(), w.clone(), shift.clone(), EPS, fmt)
        for g, t in zip(got, want):
            assert g.shape == t.shape and torch.equal(g.view(torch.uint8), t.view(torch.uint8))
    x = base[:3, :1024].clone()
    x[1, 700] = float("nan")
    x[2, 5] = float("inf")
    codes, scales = ops.rms_norm_modulate_mx(x, w, shift, EPS, fmt)
    y = ops.mx_dequantize(codes, scales, 1024).float()
    assert y[0].isfinite().all() and y[1].isnan().all()
    assert y[2, :32].isnan().all()   # inf * 0; the rest of the row is the shift
    t = ops.rms_norm_modulate_mx(torch.zeros_like(x), w, shift, EPS, fmt)
    assert torch.equal(y[2, 32:], ops.mx_dequantize(*t, 1024).float()[2, 32:])


@pytest.mark.parametrize("fmt", FMTS)
def test_norm_of_rows_of_any_size(dev, fmt):
    # magnitudes whose squares, sums and products with the weight leave float32's range
    scale = torch.tensor([1e-38, 1e-30, 1e-20, 1.0, 1e15, 1e25, 1e37], device=dev)
    x = (_act(dev, 7, 640, seed=1, dtype=torch.float32).clamp(-20, 20) * scale[:, None]).to(torch.bfloat16)
    w, shift = _act(dev, 640, seed=4), _act(dev, 640, seed=5)
    for eps in (0.0, 1e-6):
        check_blocks(*ops.rms_norm_modulate_mx(x, w, shift, eps, fmt), *_norm64(f64(x), f64(w), f64(shift), eps))


# ---- SwiGLU product ----
def _silu64(g, u):
    """y, and how far float32's evaluation may be from it: exp to 2 units of 2^-23, the sum, the quotient and the
    product to 2^-24 each (under 8 x 2^-24 together, exp's share of the denominator being at most 1); where exp
    overflows the result is 0 for a magnitude under 2^-118 |u|."""
    with np.errstate(over="ignore"):
        y = g / (1 + np.exp(-g)) * u
    return y, 8 * 2.0 ** -24 * np.abs(y) + 2.0 ** -118 * np.abs(u)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("m,k", [(1, 1), (3, 31), (2, 32), (3, 130), (7, 1000), (2, 1187), (5, 6144), (2, 16384), (16999, 41)])
def test_silu(dev, fmt, m, k):
    g, u = _act(dev, m, k, seed=1) * 3, _act(dev, m, k, seed=2)
    codes, scales = ops.silu_mul_mx(g, u, fmt)
    check_blocks(codes, scales, *_silu64(f64(g), f64(u)))


@pytest.mark.parametrize("fmt", FMTS)
def test_silu_layouts_and_extremes(dev, fmt):
    both = _act(dev, 9, 2000, seed=7)
    for g, u in ((both[:, :1000], both[:, 1000:]), (both[:, 1:513], both[:, 513:1025]), (both[::2, :96], both[1::2, :96].new_ones(5, 96)),
                 (both[:, :256].reshape(3, 3, 256), both[:, 256:512].reshape(3, 3, 256))):
        got, want = ops.silu_mul_mx(g, u, fmt), ops.silu_mul_mx(g.contiguous().clone(), u.contiguous().clone(), fmt)
        for a, b in zip(got, want):
            assert a.shape == b.shape and torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    g = torch.linspace(-300, 300, 4096, device=dev).to(torch.bfloat16).view(4, 1024)
    u = _act(dev, 4, 1024, seed=3)
    check_blocks(*ops.silu_mul_mx(g, u, fmt), *_silu64(f64(g), f64(u)))
    g[1, 40], u[2, 100] = float("nan"), float("inf")
    y = ops.mx_dequantize(*ops.silu_mul_mx(g, u, fmt), 1024)
    bad = torch.zeros(4, 1024, dtype=torch.bool, device=dev)
    bad[1, 32:64], bad[2, 96:128] = True, True
    assert torch.equal(y.isnan(), bad)


@pytest.mark.parametrize("fmt", FMTS)
def test_silu_whole_range(dev, fmt):
    # Gates from -700 to 80 with up of 2^-120 .. 2^127: gate * up passes float32's range where the product does not, and a
    # far negative gate leaves an ordinary product of a large up.  Relative as in _silu64 (under 8 x 2^-24), and below
    # float32's normal range half its smallest step, 2^-150, twice (the product's rounding and the last scaling's).
    g = torch.cat([torch.linspace(-700, -60, 1600), torch.linspace(-100, 80, 1600), torch.linspace(-4, 4, 800)])
    g = g.to(torch.bfloat16).repeat(8, 1)
    e = torch.tensor([127, 126, 124, 120, 100, 60, -60, -120], dtype=torch.float64)[:, None]
    u = (2.0 ** e * (1 + torch.arange(4000, dtype=torch.float64) % 128 / 128)).to(torch.bfloat16)
    u[:, 1::2] *= -1
    with np.errstate(over="ignore"):
        y = f64(g) / (1 + np.exp(-f64(g))) * f64(u)
    inside = np.abs(y) < 2.0 ** 128 * (1 - 2.0 ** -20)   # what float32 holds; elsewhere a gate of zero stands instead
    g, y = g.masked_fill(~torch.from_numpy(inside), 0.0), np.where(inside, y, 0.0)
    codes, scales = ops.silu_mul_mx(g.to(dev), u.to(dev), fmt)
    check_blocks(codes, scales, y, 8 * 2.0 ** -24 * np.abs(y) + 2.0 ** -149)
    # an infinite gate gives no number, like the formula
    x = torch.ones(1, 64, device=dev, dtype=torch.bfloat16)
    for at in (-float("inf"), float("inf")):
        bad = x.clone()
        bad[0, 3] = at
        out = ops.mx_dequantize(*ops.silu_mul_mx(bad, x, fmt), 64)
        assert out[:, :32].isnan().all() and out[:, 32:].isfinite().all()


# ---- together ----
def _ff_weights(dev, h, f):
    return {name: quantize_mx(_act(dev, n, k, seed=i, dtype=torch.float32) * 0.05)
            for i, (name, n, k) in enumerate((("gate", f, h), ("up", f, h), ("down", h, f)))}


def _ff(x, v, vecs, w):
    xo, a, s = ops.residual_rms_norm_modulate_mx(x, v, *vecs, EPS, "e4m3")
    g, u = ops.mx_gemm(a, s, *w["gate"]), ops.mx_gemm(a, s, *w["up"])
    f, fs = ops.silu_mul_mx(g, u, "e2m1")
    return xo, a, s, g, u, f, fs, ops.mx_gemm(f, fs, *w["down"])


@pytest.mark.parametrize("m", [1, 45, 300])
def test_feed_forward(dev, m):
    h, f = 520, 1160
    x, v = _act(dev, m, h, seed=1), _act(dev, m, h, seed=2)
    vecs = [_act(dev, h, seed=s) for s in (3, 4, 5)]
    w = _ff_weights(dev, h, f)
    xo, a, s, g, u, fc, fs, y2 = _ff(x, v, vecs, w)
    check_blocks(a, s, *_norm64(f64(xo), f64(vecs[1]), f64(vecs[2]), EPS))
    for y, name in ((g, "gate"), (u, "up")):
        wv = values(*w[name])
        check_product(y, values(a, s), wv, None, dropped(values(a, s), wv))
    check_blocks(fc, fs, *_silu64(f64(g), f64(u)))
    check_product(y2, values(fc, fs), values(*w["down"]))


def test_streams_and_graphs(dev):
    h, f = 512, 1024
    vecs = [_act(dev, h, seed=s) for s in (3, 4, 5)]
    w = _ff_weights(dev, h, f)
    xs = [(_act(dev, m, h, seed=m), _act(dev, m, h, seed=m + 1)) for m in (4, 70)]
    want = [_ff(x, v, vecs, w)[-1] for x, v in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]   # two calls at once
    got = []
    for st, (x, v) in zip(streams, xs):
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            got.append(_ff(x, v, vecs, w)[-1])
    for st in streams:
        torch.cuda.current_stream().wait_stream(st)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs = []
    for x, v in xs:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = _ff(x, v, vecs, w)[-1]
        graphs.append((gr, out))
    for r in range(4):   # replays with new inputs, eager work between them
        for i, ((gr, out), (x, v)) in enumerate(zip(graphs, xs)):
            x.copy_(_act(dev, *x.shape, seed=50 + 2 * r + i))
            eager = _ff(x, v, vecs, w)[-1].clone()
            gr.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, eager)


@pytest.mark.parametrize("activation", FMTS)
def test_module(dev, activation):
    from krea2_svdquant_amd import MXLinear
    dense = _act(dev, 200, 300, seed=1, dtype=torch.float32) * 0.05
    bias = _act(dev, 200, seed=2)
    layer = MXLinear.from_dense(dense, bias, activation=activation)
    x = _act(dev, 5, 7, 300, seed=3)
    y = layer(x)
    assert torch.equal(y, ops.mx_linear(x, *quantize_mx(dense), bias, activation))
    assert torch.equal(y, layer.forward_mx(*layer.quantize(x)))
    assert torch.equal(layer.dense_weight(), torch.from_numpy(values(*quantize_mx(dense))[:, :300]).float().to(dev))
    moved = MXLinear.from_dense(torch.zeros_like(dense), torch.zeros_like(bias), activation=activation)
    moved.load_state_dict(layer.cpu().state_dict())
    assert torch.equal(moved.to(dev, torch.bfloat16)(x), y)   # byte buffers do not change type
    with pytest.raises(ValueError, match="300"):
        moved(x[..., :299])


def test_block_on_mx_layers(dev):
    from krea2_svdquant_amd.runtime import krea2_standin as ks
    dims = ks.Krea2Dims(layers=2, hidden=256, heads=2, kv_heads=1, head_dim=128, mlp=520)
    model = ks.Krea2StandInTransformer.random(dims, linears="mx", device=dev, seed=5)
    x = _act(dev, 70, 256, seed=1)
    cos, sin = ks.rope_tables(70, 128, dev, torch.bfloat16)
    t, pending = x, None
    for blk in model.transformer_blocks:   # the block's operators one by one
        shift_a, scale_a, gate_a, shift_f, scale_f, gate_f = blk.modulation
        lin = blk.linears()
        if pending is None:
            a = ops.rms_norm_modulate_mx(t, 1 + scale_a, shift_a, EPS, "e4m3")
        else:
            t, *a = ops.residual_rms_norm_modulate_mx(t, pending[1], pending[0], 1 + scale_a, shift_a, EPS, "e4m3")
        q, k, v, g = (lin[f"attn.to_{n}"].forward_mx(*a) for n in ("q", "k", "v", "gate"))
        q, k, v = (z.view(70, -1, 128) for z in (q, k, v))
        o = ks.attention(ks.head_norm_rope(q, cos, sin), ks.head_norm_rope(k, cos, sin), v)
        o = lin["attn.to_out.0"](ks.gate_mul_sigmoid(o, g))
        t, *a = ops.residual_rms_norm_modulate_mx(t, o, gate_a, 1 + scale_f, shift_f, EPS, "e4m3")
        f = ops.silu_mul_mx(lin["ff.gate"].forward_mx(*a), lin["ff.up"].forward_mx(*a), "e4m3")
        pending = gate_f, lin["ff.down"].forward_mx(*f)
    want = torch.addcmul(t, *pending)
    assert want.isfinite().all()
    assert torch.equal(model(x), want)
    # the linears alone replaced: the norms and products are rounded to bf16 ahead of their quantising
    calls = []
    model(x, linear=lambda name, mod, z: calls.append(name) or mod(z))
    assert len(calls) == 16
    with pytest.raises(NotImplementedError):
        model(x, fused=True)


@pytest.mark.parametrize("kinds", [("e2m1", "e2m1"), ("e2m1", "e4m3")])
def test_block_keeps_its_layers_formats(dev, kinds):
    # Zero modulation shifts and scales of one: norms and products of the block in the formats that its layers name, whole
    # blocks of one format on the operators with MX outputs, siblings of two formats each on its own quantised input.
    from krea2_svdquant_amd.runtime import krea2_standin as ks
    dims = ks.Krea2Dims(layers=1, hidden=256, heads=2, kv_heads=1, head_dim=128, mlp=520)
    model = ks.Krea2StandInTransformer.random(dims, linears="mx", device=dev, seed=5)
    blk = model.transformer_blocks[0]
    lin = blk.linears()
    for i, m in enumerate(lin.values()):
        m.activation = kinds[i % 2]
    seen = []
    hooks = {n: getattr(ops, n) for n in ("mx_linear", "rms_norm_modulate_mx", "residual_rms_norm_modulate_mx", "silu_mul_mx")}
    try:
        for n, f in hooks.items():
            setattr(ops, n, lambda *args, n=n, f=f: seen.append((n, args[-1])) or f(*args))
        y = model(_act(dev, 70, 256, seed=1))
    finally:
        for n, f in hooks.items():
            setattr(ops, n, f)
    assert y.isfinite().all()
    if kinds[0] == kinds[1]:
        assert {n for n, _ in seen} == set(hooks) and {fmt for _, fmt in seen} == {"e2m1"}
    else:
        assert sorted(fmt for n, fmt in seen if n == "mx_linear") == ["e2m1"] * 4 + ["e4m3"] * 4 and len(seen) == 8
    blk.ff.down = torch.nn.Linear(520, 256, device=dev, dtype=torch.bfloat16)   # some MX layers
    with pytest.raises(NotImplementedError):
        model(_act(dev, 70, 256, seed=1), fused=True)


def test_refusals(dev):
    x = _act(dev, 4, 256)
    codes, scales = ops.mx_quantize(x)
    vec = torch.ones(256, device=dev, dtype=torch.bfloat16)
    with pytest.raises(TypeError):
        ops.mx_quantize(x.float())
    with pytest.raises(ValueError):
        ops.mx_quantize(x[:, :0])
    with pytest.raises(ValueError, match="fmt"):
        ops.mx_quantize(x, "e5m2")
    with pytest.raises(ValueError):
        ops.mx_dequantize(codes, scales, 257)
    with pytest.raises(ValueError):
        ops.mx_dequantize(codes, scales[:, :8].contiguous(), 256)
    with pytest.raises(TypeError):
        ops.mx_dequantize(codes.int(), scales, 256)
    with pytest.raises(TypeError):
        ops.mx_dequantize(codes, scales.float(), 256)
    with pytest.raises(ValueError, match="contiguous"):
        ops.mx_dequantize(codes[:, ::2], scales, 128)
    with pytest.raises(TypeError):   # an 8-bit weight
        ops.mx_gemm(codes, scales, *ops.mx_quantize(x, "e4m3"))
    with pytest.raises(ValueError):   # another K
        ops.mx_gemm(codes, scales, *ops.mx_quantize(x[:, :100]))
    with pytest.raises(ValueError):
        ops.mx_gemm(codes, scales, codes, scales, vec)
    with pytest.raises(TypeError):
        ops.mx_gemm(codes, scales, codes, scales, torch.ones(4, device=dev))
    with pytest.raises(ValueError):
        ops.mx_gemm(codes, scales, codes[0], scales[0])
    with pytest.raises(ValueError):
        ops.mx_gemm(codes.cpu().to(dev), scales.cpu(), codes, scales)
    with pytest.raises(ValueError):
        ops.mx_linear(x[:, :100], codes, scales)
    with pytest.raises(ValueError):
        ops.silu_mul_mx(x, x[:2])
    with pytest.raises(TypeError):
        ops.silu_mul_mx(x, x.half())
    with pytest.raises(ValueError):   # rows of 252
        ops.rms_norm_modulate_mx(x[:, :252], vec[:252], vec[:252], EPS)
    with pytest.raises(ValueError):
        ops.rms_norm_modulate_mx(x, vec[:8], vec, EPS)
    with pytest.raises(lib.SVDQError):
        ops.rms_norm_modulate_mx(x, vec, vec, -1.0)
    with pytest.raises(ValueError):
        ops.residual_rms_norm_modulate_mx(x, x[:2], vec, vec, vec, EPS)
    misaligned = torch.empty(codes.numel() + 1, device=dev, dtype=torch.uint8)[1:].view(codes.shape)
    with pytest.raises(lib.SVDQError, match="16-byte"):
        ops.mx_dequantize(misaligned, scales, 256)
    with pytest.raises(RuntimeError):   # no gradient is defined
        ops.mx_linear(x.clone().requires_grad_(), codes, scales).float().sum().backward()
