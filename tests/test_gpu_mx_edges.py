"""Microscaled operators at the ends of their ranges: rows of the smallest values, rows longer than a workgroup keeps,
calls in place, products that drop nothing on every tile, equal bits from every tile, layers that were moved to another
type, blocks whose layers carry hooks."""
import numpy as np
import pytest
import torch

from krea2_svdquant_amd.kernels.hip import lib, ops
from oracle import mx
from tests.mx_util import check_blocks, f64, to_oracle, values

pytestmark = pytest.mark.gpu
FMTS = list(mx.FORMATS)


def _randn(dev, *shape, seed, dtype=torch.bfloat16):
    return torch.randn(shape, device=dev, generator=torch.Generator(device=dev).manual_seed(seed)).to(dtype)


def _norm64(x, w, shift, eps):
    """y = t + shift, t = x w / root, and how far the kernel may be from it: t is (x w 2^k) (r0 + r1), x w 2^k exact
    (16 bits) and r0 + r1 the root's reciprocal to 2^-47; two fused products round to float32, 2^-24 of their result
    each (of y up to 2^-24 of t), or half of 2^-149 below its normal range.  The reference here is off by a few 2^-53
    of t and shift: taken with the 2^-46 of t."""
    t = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w
    y = t + shift
    return y, 2.1 * 2.0 ** -24 * np.abs(y) + 2.0 ** -46 * (np.abs(t) + np.abs(shift)) + 2.0 ** -149


@pytest.mark.parametrize("fmt", FMTS)
def test_norm_of_the_smallest_rows(dev, fmt):
    # without eps the reciprocal root of a row of bf16 subnormals passes float32's range; the normed row does not
    scale = torch.tensor([2.0 ** -133, 3e-40, 1e-39, 3e-39, 1e-38], device=dev)
    x = (_randn(dev, 5, 640, seed=1, dtype=torch.float32).clamp(-20, 20) * scale[:, None]).to(torch.bfloat16)
    x[0] = 0
    x[0, 77] = 2.0 ** -133   # the smallest bf16 alone
    assert (x != 0).any(1).all()
    w, shift = _randn(dev, 640, seed=2), _randn(dev, 640, seed=3)
    for eps in (0.0, 1e-6):
        check_blocks(*ops.rms_norm_modulate_mx(x, w, shift, eps, fmt), *_norm64(f64(x), f64(w), f64(shift), eps))
    # a row of zeros without eps has no direction: NaN, as the formula's 0 / 0
    codes, scales = ops.rms_norm_modulate_mx(torch.zeros_like(x), w, shift, 0.0, fmt)
    assert ops.mx_dequantize(codes, scales, 640).isnan().all()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("m,h", [(3, 6144), (2, 16384), (3, 16392), (2, 20000), (5, 33000)])
def test_norm_of_long_rows(dev, fmt, m, h):
    # beyond 16384 values a row's chunks are read again after the mean
    x, v = _randn(dev, m, h, seed=1), _randn(dev, m, h, seed=2)
    gate, w, shift = (_randn(dev, h, seed=s) for s in (3, 4, 5))
    check_blocks(*ops.rms_norm_modulate_mx(x, w, shift, 1e-6, fmt), *_norm64(f64(x), f64(w), f64(shift), 1e-6))
    xo, codes, scales = ops.residual_rms_norm_modulate_mx(x, v, gate, w, shift, 1e-6, fmt)
    assert torch.equal(xo, torch.addcmul(x, gate, v))
    check_blocks(codes, scales, *_norm64(f64(xo), f64(w), f64(shift), 1e-6))


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("m,h,ld", [(1, 8, 8), (70, 512, 520), (300, 6144, 6144), (9, 20000, 20008)])
def test_norm_in_place(dev, fmt, m, h, ld):
    buf, v = _randn(dev, m, ld, seed=1), _randn(dev, m, h, seed=2)
    gate, w, shift = (_randn(dev, h, seed=s) for s in (3, 4, 5))
    want = ops.residual_rms_norm_modulate_mx(buf[:, :h], v, gate, w, shift, 1e-6, fmt)
    behind = buf[:, h:].clone()
    codes, scales = torch.empty_like(want[1]), torch.empty_like(want[2])
    lib.call("svdq_residual_rms_norm_modulate_mx", buf.data_ptr(), ld, v.data_ptr(), h, gate.data_ptr(), w.data_ptr(),
             shift.data_ptr(), m, h, 1e-6, ops.MX_FORMATS[fmt], buf.data_ptr(), ld, codes.data_ptr(), scales.data_ptr(),
             torch.cuda.current_stream().cuda_stream)
    assert torch.equal(buf[:, :h], want[0]) and torch.equal(buf[:, h:], behind)
    assert torch.equal(codes.view(torch.uint8), want[1].view(torch.uint8))
    assert torch.equal(scales.view(torch.uint8), want[2].view(torch.uint8))


# ---- layers ----
@pytest.mark.parametrize("move", ["float", "half", "double", "bfloat16"])
def test_layer_after_a_move_to_another_type(dev, move):
    from krea2_svdquant_amd import MXLinear
    bias = _randn(dev, 200, seed=2)
    bias[:3] = torch.tensor([1e6, 1e-9, -3e38], device=dev)   # bf16 values that float16 does not hold
    layer = MXLinear.from_dense(_randn(dev, 200, 300, seed=1, dtype=torch.float32) * 0.05, bias)
    x = _randn(dev, 5, 300, seed=3)
    want = layer(x)
    getattr(layer, move)()
    assert torch.equal(layer(x), want)
    assert torch.equal(layer.forward_mx(*layer.quantize(x)), want)


def test_inputs_that_ask_for_gradients(dev):
    # forward works and gives the same bits; no gradient is defined
    x, v, w = (_randn(dev, *s, seed=i) for i, s in enumerate(((4, 256), (4, 256), (256,))))
    codes, scales = ops.mx_quantize(_randn(dev, 40, 256, seed=9))
    calls = (lambda x: ops.mx_quantize(x), lambda x: ops.mx_quantize(x, "e4m3"), lambda x: (ops.mx_linear(x, codes, scales),),
             lambda x: ops.silu_mul_mx(x, v), lambda x: ops.rms_norm_modulate_mx(x, w, w, 1e-6),
             lambda x: ops.residual_rms_norm_modulate_mx(x, v, w, w, w, 1e-6))
    for call in calls:
        for got, want in zip(call(x.clone().requires_grad_()), call(x)):
            assert torch.equal(got.detach().view(torch.uint8), want.view(torch.uint8))


# ---- blocks ----
def _block_model(dev):
    from krea2_svdquant_amd.runtime import krea2_standin as ks
    dims = ks.Krea2Dims(layers=1, hidden=256, heads=2, kv_heads=1, head_dim=128, mlp=520)
    return ks, ks.Krea2StandInTransformer.random(dims, linears="mx", device=dev, seed=5), _randn(dev, 70, 256, seed=1)


def test_block_runs_the_hooks_of_its_layers(dev):
    ks, model, x = _block_model(dev)
    lin = model.transformer_blocks[0].linears()
    want = model(x)
    one_by_one = model(x, linear=lambda name, mod, z: mod(z))   # bf16 activations between the layers
    seen = []
    handles = [m.register_forward_hook(lambda mod, args, out, n=n: seen.append((n, args[0].dtype, out.shape[-1])))
               for n, m in lin.items()]
    assert torch.equal(model(x), one_by_one)
    assert sorted(seen) == sorted(((n, torch.bfloat16, m.out_features) for n, m in lin.items()), key=lambda t: t[0])
    for h in handles:
        h.remove()
    assert torch.equal(model(x), want)
    for siblings in ("grouped", "concurrent", True, False):
        assert torch.equal(model(x, siblings=siblings), want)


def test_block_calls_the_forward_of_a_subclass(dev):
    ks, model, x = _block_model(dev)
    blk = model.transformer_blocks[0]

    class Doubled(ks.MXLinear):
        def forward(self, z):
            return 2 * super().forward(z)
    up = blk.ff.up
    blk.ff.up = Doubled(up.weight_codes, up.weight_scales, None, in_features=256, activation=up.activation)
    want = model(x, linear=lambda name, mod, z: mod(z))
    assert torch.equal(model(x), want)


@pytest.mark.parametrize("switch", ["NORMS", "GATES"])
def test_block_follows_the_switches(dev, switch, monkeypatch):
    ks, model, x = _block_model(dev)
    monkeypatch.setattr(ks, switch, "torch")
    assert torch.equal(model(x), model(x, linear=lambda name, mod, z: mod(z)))


# ---- products ----
def _narrow(dev, m, k, seed):
    """bf16 values with magnitudes of 0.026 to 0.99: E4M3 codes of 8 and more under a scale of 2^-9, whose products with
    E2M1 codes are multiples of 1/2 of at most 2688, so the matrix instruction drops nothing."""
    gen = torch.Generator(device=dev).manual_seed(seed)
    x = torch.rand(m, k, device=dev, generator=gen) * 0.964 + 0.026
    return (x * torch.where(torch.rand(m, k, device=dev, generator=gen) < 0.5, -1.0, 1.0)).to(torch.bfloat16)


# rows and columns that each kernel is chosen for, as lib.mx_tile names it
E4M3_TILES = {(2, 8, 16): (7, 1000), (1, 64, 64): (70, 3000), (1, 64, 128): (250, 6100), (1, 128, 128): (500, 8100),
              (1, 256, 256): (1990, 8100)}


def _check_narrow(dev, tile, m, n, k):
    assert lib.mx_tile(m, n, k, lib.SVDQ_MX_E4M3) == tile
    a, b = ops.mx_quantize(_narrow(dev, m, k, 1), "e4m3"), ops.mx_quantize(_randn(dev, n, k, seed=2))
    assert (a[1].view(torch.uint8)[:, :k // 32] == 127 - 9).all()
    bias = _randn(dev, n, seed=3)
    av, bv = (torch.from_numpy(values(*t)).to(dev) for t in (a, b))
    y, mag = av @ bv.T + bias.double(), av.abs() @ bv.abs().T + bias.double().abs()
    bound = 1.01 * (av.shape[1] + 1) * 2.0 ** -24 * mag   # as mx_util.product_bound; then one rounding to bf16
    assert ((ops.mx_gemm(*a, *b, bias).double() - y).abs() <= bound + 2.0 ** -8 * (y.abs() + bound)).all()


@pytest.mark.parametrize("k", [128, 384, 1000, 2432])
@pytest.mark.parametrize("tile", E4M3_TILES)
def test_every_e4m3_tile_where_nothing_is_dropped(dev, tile, k):
    _check_narrow(dev, tile, *E4M3_TILES[tile], k)


def test_last_rows_on_smaller_e4m3_tiles_where_nothing_is_dropped(dev):
    _check_narrow(dev, (3, 256, 256), 2200, 8100, 3000)


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("k", [384, 1000, 2432])
def test_bits_do_not_depend_on_the_tile(dev, fmt, f32, k):
    # every output sums K in one order, whichever block tile holds it
    sizes = [(70, 3000), (250, 6100), (500, 8100), (1990, 8100), (2200, 8100)]
    a, b = ops.mx_quantize(_randn(dev, 2200, k, seed=1), fmt), ops.mx_quantize(_randn(dev, 8100, k, seed=2))
    bias = _randn(dev, 8100, seed=3)
    kinds = {lib.mx_tile(m, n, k, ops.MX_FORMATS[fmt]) for m, n in sizes}
    assert len(kinds) >= 4 and all(kind != 2 for kind, _, _ in kinds)
    whole = ops.mx_gemm(*a, *b, bias, f32)
    for m, n in sizes[:-1]:
        part = ops.mx_gemm(a[0][:m], a[1][:m], b[0][:n], b[1][:n], bias[:n].clone(), f32)
        assert torch.equal(part, whole[:m, :n])


@pytest.mark.parametrize("fmt", FMTS)
def test_norm_next_to_the_borders_of_codes(dev, fmt):
    # shifts in the middle of two codes, at a code and at a power of two (a block's scale), and normed values of 2^-25 to
    # 2^-38 of them on either side, which float32's sum does not hold: every code and scale is that of the sum itself
    h = 640
    x = torch.zeros(8, h, dtype=torch.float64)
    sign = torch.where(torch.arange(h) % 3 == 0, -1.0, 1.0)
    for r in range(8):
        x[r] = sign * (1 if r % 2 else -1) * 2.0 ** (-25 - 2 * (r // 2)) * (1 + torch.arange(h) % 5 / 8)
        x[r, 32 * r] = 25.0   # the root mean square is about 1
    shift = torch.tensor([1.25, 1.75, 1.0625, 1.1875, 2.0, 1.0, 0.875, 0.15625, 1.9375, 0.4375, 0.3125, 2.0 ** -9 * 1.5, 1.5,
                          0.625, -1.25, -2.0, -0.6875], dtype=torch.float64)[torch.arange(h) % 17]
    shift[::64] *= 4   # blocks with a largest value of other scales
    x, shift = x.to(torch.bfloat16), shift.to(torch.bfloat16)
    w = torch.ones(h, dtype=torch.bfloat16)
    w[::7] = 0.5
    codes, scales = ops.rms_norm_modulate_mx(x.to(dev), w.to(dev), shift.to(dev), 1e-6, fmt)
    y, _ = _norm64(f64(x), f64(w), f64(shift), float(np.float32(1e-6)))
    want_c, want_s = mx.quantize(y, fmt)
    as_f32 = mx.quantize(y.astype(np.float32).astype(np.float64), fmt)
    assert (as_f32[0] != want_c).sum() > 100 and (as_f32[1] != want_s).any()   # what float32 alone would give
    got_c, got_s, _ = to_oracle(codes, scales)
    assert np.array_equal(got_s, want_s) and np.array_equal(got_c, want_c)
