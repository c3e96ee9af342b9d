"""Microscaled blocks on the CPU: the oracle against the element types' published values and torch's float8, the
converter against the oracle, shape functions, and the refusals of the C entry points (no GPU call is made)."""
import ctypes

import numpy as np
import pytest
import torch

from krea2_svdquant_amd.kernels.hip import lib, ops
from krea2_svdquant_amd.quant.mx import dequantize_mx, quantize_mx
from oracle import mx
from tests import mx_util


def test_element_values():
    assert mx.MAGNITUDES["e2m1"].tolist() == [0, 0.5, 1, 1.5, 2, 3, 4, 6]
    codes = torch.arange(256, dtype=torch.uint8)
    want = codes.view(torch.float8_e4m3fn).double().numpy()
    got = mx.decode(codes.numpy(), "e4m3")
    assert np.array_equal(got, want, equal_nan=True)


def test_oracle_encoding_is_the_nearest_value():
    # every midpoint, its neighbours, every value, by brute force over all values
    for fmt in mx.FORMATS:
        mags = mx.MAGNITUDES[fmt]
        mids = (mags[1:] + mags[:-1]) / 2
        v = np.concatenate([mags, mids, np.nextafter(mids, 0), np.nextafter(mids, 1e9), [mags[-1] * 1.5]])
        c = mx.encode(v, fmt)
        dist = np.abs(v[:, None] - mags[None, :])
        assert np.array_equal(np.abs(v - mags[c]), dist.min(1))
        ties = (dist == dist.min(1, keepdims=True)).sum(1) == 2
        assert (c[ties] % 2 == 0).all() and ties.sum() == len(mids)
        assert np.array_equal(mx.encode(-v, fmt), c | (8 if fmt == "e2m1" else 128))
    # torch's own rounding to float8
    v = np.random.default_rng(0).standard_normal(10000) * 50
    t = torch.from_numpy(v.astype(np.float32)).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(mx.encode(v.astype(np.float32).astype(np.float64), "e4m3"), t)


@pytest.mark.parametrize("fmt", mx.FORMATS)
@pytest.mark.parametrize("k", [1, 31, 32, 128, 129, 700])
def test_converter_matches_the_oracle(fmt, k):
    rng = np.random.default_rng(k)
    x = (rng.standard_normal((5, k)) * 10.0 ** rng.integers(-3, 4, (5, k))).astype(np.float32)
    x[1] = 0
    x[2, k // 2] = np.inf
    x[3, k - 1] = np.nan
    codes, scales = quantize_mx(torch.from_numpy(x), fmt)
    want_c, want_s = mx.quantize(x.astype(np.float64), fmt)
    got_c, got_s, got_fmt = mx_util.to_oracle(codes, scales)
    assert got_fmt == fmt and np.array_equal(got_s, want_s)
    assert np.array_equal(got_c, want_c)
    back = dequantize_mx(codes, scales, k).numpy()
    assert np.array_equal(back, mx.dequantize(want_c, want_s, fmt)[:, :k].astype(np.float32), equal_nan=True)
    assert tuple(c.shape[-1] for c in (codes, scales)) == ops.mx_shapes(k, fmt)


def test_converter_refusals():
    with pytest.raises(ValueError, match="fmt"):
        quantize_mx(torch.zeros(1, 32), "e5m2")
    with pytest.raises(TypeError):
        quantize_mx(torch.zeros(1, 32, dtype=torch.int32))
    with pytest.raises(ValueError):
        quantize_mx(torch.zeros(4, 0))
    codes, scales = quantize_mx(torch.zeros(1, 32))
    with pytest.raises(ValueError):
        dequantize_mx(codes, scales, 129)
    with pytest.raises(TypeError):
        dequantize_mx(codes.int(), scales, 32)


def test_operators_refuse_the_cpu_and_unknown_formats():
    x = torch.zeros(2, 64, dtype=torch.bfloat16)
    codes, scales = quantize_mx(x)
    for call in (lambda: ops.mx_quantize(x), lambda: ops.mx_dequantize(codes, scales, 64),
                 lambda: ops.mx_gemm(codes, scales, codes, scales), lambda: ops.mx_linear(x, codes, scales),
                 lambda: ops.silu_mul_mx(x, x), lambda: ops.rms_norm_modulate_mx(x, x, x, 1e-6),
                 lambda: ops.residual_rms_norm_modulate_mx(x, x, x, x, x, 1e-6)):
        with pytest.raises(RuntimeError, match="GPU"):
            call()
    with pytest.raises(ValueError, match="fmt"):
        ops.mx_shapes(64, "int4")


@pytest.mark.skipif(not lib.TORCH_LIB_PATH.exists(), reason="library not built")
def test_shape_functions():
    from torch._subclasses.fake_tensor import FakeTensorMode
    native = ops.load_native()
    e2m1, e4m3 = lib.SVDQ_MX_E2M1, lib.SVDQ_MX_E4M3
    with FakeTensorMode():
        x = torch.empty(2, 3, 520, dtype=torch.bfloat16)
        c, s = native["mx_quantize"](x, e2m1)
        assert c.shape == (2, 3, 320) and c.dtype == torch.uint8
        assert s.shape == (2, 3, 32) and s.dtype == torch.float8_e8m0fnu
        c8, _ = native["silu_mul_mx"](x, x, e4m3)
        assert c8.shape == (2, 3, 640) and c8.dtype == torch.float8_e4m3fn
        y = native["mx_dequantize"](c, s, 520)
        assert y.shape == (2, 3, 520) and y.dtype == torch.bfloat16
        w = torch.empty(40, 320, dtype=torch.uint8)
        ws = torch.empty(40, 32, dtype=torch.float8_e8m0fnu)
        y = native["mx_gemm"](c, s, w, ws, None, True)
        assert y.shape == (2, 3, 40) and y.dtype == torch.float32
        assert native["mx_linear"](x, w, ws, None, e2m1, False).dtype == torch.bfloat16
        xo, c, s = native["residual_rms_norm_modulate_mx"](x, x, x, x, x, 1e-6, e4m3)
        assert xo.shape == x.shape and c.shape == (2, 3, 640) and s.shape == (2, 3, 32)
        c, _ = native["rms_norm_modulate_mx"](x, x, x, 1e-6, e2m1)
        assert c.shape == (2, 3, 320)


P = ctypes.c_void_p(0x1000)    # never read: the calls below fail on the host
ODD = ctypes.c_void_p(0x1001)
EIGHT = ctypes.c_void_p(0x1008)


@pytest.mark.parametrize("fn,args,status,needle", [
    ("svdq_mx_quantize", (P, 64, 2, 64, 7, P, P), -1, "format 7"),
    ("svdq_mx_quantize", (P, 64, -1, 64, 0, P, P), -2, "M=-1"),
    ("svdq_mx_quantize", (P, 64, 2, 0, 0, P, P), -2, "K=0"),
    ("svdq_mx_quantize", (P, 63, 2, 64, 0, P, P), -2, "ldx=63"),
    ("svdq_mx_quantize", (None, 64, 2, 64, 0, P, P), -1, "null"),
    ("svdq_mx_quantize", (P, 64, 2, 64, 0, None, P), -1, "null"),
    ("svdq_mx_quantize", (P, 64, 2, 64, 0, P, EIGHT), -3, "16-byte"),
    ("svdq_mx_quantize", (ODD, 64, 2, 64, 0, P, P), -3, "2-byte"),
    ("svdq_mx_dequantize", (P, P, 2, 64, 0, None), -1, "null"),
    ("svdq_mx_dequantize", (EIGHT, P, 2, 64, 0, P), -3, "16-byte"),
    ("svdq_mx_gemm", (P, P, 2, P, P, None, 2, 8, 64, P, 8, 0), -1, "format 2"),
    ("svdq_mx_gemm", (P, P, 0, P, P, None, 2, 0, 64, P, 8, 0), -2, "N=0"),
    ("svdq_mx_gemm", (P, P, 0, P, P, None, 2, 8, 64, P, 7, 0), -2, "ldy=7"),
    ("svdq_mx_gemm", (P, P, 0, P, P, None, 2, 8, 64, P, 8, 2), -1, "out_f32"),
    ("svdq_mx_gemm", (P, P, 0, None, P, None, 2, 8, 64, P, 8, 0), -1, "null"),
    ("svdq_mx_gemm", (P, P, 0, P, EIGHT, None, 2, 8, 64, P, 8, 0), -3, "16-byte"),
    ("svdq_mx_gemm", (P, P, 0, P, P, ODD, 2, 8, 64, P, 8, 0), -3, "elements"),
    ("svdq_silu_mul_mx", (P, 64, P, 32, 2, 64, 0, P, P), -2, "ldu=32"),
    ("svdq_silu_mul_mx", (P, 64, None, 64, 2, 64, 0, P, P), -1, "null"),
    ("svdq_rms_norm_modulate_mx", (P, 64, P, P, 2, 60, ctypes.c_float(0), 0, P, P), -2, "H=60"),
    ("svdq_rms_norm_modulate_mx", (P, 64, P, P, 2, 64, ctypes.c_float(-1), 0, P, P), -1, "eps"),
    ("svdq_rms_norm_modulate_mx", (P, 68, P, P, 2, 64, ctypes.c_float(0), 0, P, P), -3, "multiples of 8"),
    ("svdq_residual_rms_norm_modulate_mx", (P, 64, None, 64, P, P, P, 2, 64, ctypes.c_float(0), 0, P, 64, P, P), -1,
     "null"),
    ("svdq_residual_rms_norm_modulate_mx", (P, 64, P, 56, P, P, P, 2, 64, ctypes.c_float(0), 0, P, 64, P, P), -3,
     "multiples of 8"),
])
def test_c_entries_refuse_before_any_launch(fn, args, status, needle):
    with pytest.raises(lib.SVDQError, match=needle) as e:
        lib.call(fn, *args, None)
    assert e.value.status == status


MANY = 2 ** 24    # a workgroup of 256 threads per row: 2^32 threads


@pytest.mark.parametrize("fn,args", [
    ("svdq_mx_quantize", (P, 8, 2 ** 26, 8, 0, P, P)),                     # a wave of 64 threads per row
    ("svdq_mx_quantize", (P, 1024, 2 ** 25, 1024, 1, P, P)),
    ("svdq_mx_dequantize", (P, P, 2 ** 26, 8, 0, P)),
    ("svdq_silu_mul_mx", (P, 8, P, 8, 2 ** 26, 8, 0, P, P)),
    ("svdq_rms_norm_modulate_mx", (P, 8, P, P, MANY, 8, ctypes.c_float(0), 0, P, P)),
    ("svdq_residual_rms_norm_modulate_mx", (P, 8, P, 8, P, P, P, MANY, 8, ctypes.c_float(0), 0, P, 8, P, P)),
    ("svdq_mx_gemm", (P, P, 0, P, P, None, 2 ** 30, 2 ** 14, 64, P, 2 ** 14, 0)),
])
def test_c_entries_refuse_launches_of_too_many_threads(fn, args):
    with pytest.raises(lib.SVDQError, match="too many") as e:
        lib.call(fn, *args, None)
    assert e.value.status == -2


def test_c_entries_take_no_rows():
    zero = ctypes.c_float(0)
    lib.call("svdq_mx_quantize", None, 64, 0, 64, 0, None, None, None)
    lib.call("svdq_mx_dequantize", None, None, 0, 64, 1, None, None)
    lib.call("svdq_mx_gemm", None, None, 0, P, P, None, 0, 8, 64, None, 8, 0, None)
    lib.call("svdq_silu_mul_mx", None, 64, None, 64, 0, 64, 1, None, None, None)
    lib.call("svdq_rms_norm_modulate_mx", None, 64, None, None, 0, 64, zero, 0, None, None, None)
    lib.call("svdq_residual_rms_norm_modulate_mx", None, 64, None, 64, None, None, None, 0, 64, zero, 0, None, 64, None,
             None, None)


def test_module_on_the_cpu():
    from krea2_svdquant_amd import MXLinear
    w = torch.randn(6, 40)
    layer = MXLinear.from_dense(w, torch.zeros(6))
    assert layer.weight_codes.shape == (6, 64) and layer.weight_scales.dtype == torch.uint8 and layer.bias.dtype == torch.bfloat16
    assert torch.equal(layer.dense_weight(), dequantize_mx(*quantize_mx(w), 40))
    assert set(layer.state_dict()) == {"weight_codes", "weight_scales", "bias"}
    with pytest.raises(RuntimeError, match="GPU"):
        layer(torch.zeros(2, 40, dtype=torch.bfloat16))
    with pytest.raises(ValueError):
        layer(torch.zeros(2, 41, dtype=torch.bfloat16))
    with pytest.raises(ValueError):
        MXLinear.from_dense(w, activation="int8")
    with pytest.raises(ValueError):
        MXLinear(layer.weight_codes, layer.weight_scales, in_features=200)
    with pytest.raises(ValueError):
        MXLinear(layer.weight_codes, layer.weight_scales[:, :8], in_features=40)
    with pytest.raises(ValueError):
        MXLinear(layer.weight_codes, layer.weight_scales, torch.zeros(5), in_features=40)
    with pytest.raises(ValueError):
        MXLinear.from_dense(w[0])


@pytest.mark.skipif(not lib.LIB_PATH.exists(), reason="library not built")
def test_kernels_stay_in_registers():
    from tests.test_kernel_resources import _kernel_metadata
    meta = {k: v["private_segment_fixed_size"] for k, v in _kernel_metadata().items() if "mx_" in k or "_mx_" in k}
    names = ("mx_quantize_kernel", "mx_dequantize_kernel", "rms_norm_mx_kernel", "mx_gemm_rows_kernel")
    for name in names:
        assert any(name in k for k in meta), name
        assert all(v == 0 for k, v in meta.items() if name in k), name
    # the largest block tiles use all 512 registers and keep a few addresses of their epilogue in scratch
    tiles = [v for k, v in meta.items() if "mx_gemm_tile_kernel" in k]
    assert len(tiles) >= 16 and max(tiles) <= 32
