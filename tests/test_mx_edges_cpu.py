"""Microscaled operators on the CPU: launches at the end of what a grid holds, calls in place, the layer's bias under
moves to another type, and when a block takes its operators with microscaled outputs."""
import ctypes

import pytest
import torch

from krea2_svdquant_amd import MXLinear
from krea2_svdquant_amd.kernels.hip import lib

P = ctypes.c_void_p(0x1000)    # never read: the calls below fail on the host
Q = ctypes.c_void_p(0x2000)
ZERO = ctypes.c_float(0)


@pytest.mark.skipif(not lib.LIB_PATH.exists(), reason="library not built")
@pytest.mark.parametrize("m,k", [(2 ** 26 - 1, 8), (2 ** 26 - 3, 512), (2 ** 25 - 1, 1024)])
def test_swiglu_refuses_the_last_partial_workgroup_beyond_a_launch(m, k):
    # workgroups of 256 threads take four units of 512 columns: 2^24 of them hold 2^32 threads
    with pytest.raises(lib.SVDQError, match="too many") as e:
        lib.call("svdq_silu_mul_mx", P, k, P, k, m, k, 0, P, P, None)
    assert e.value.status == -2


@pytest.mark.skipif(not lib.LIB_PATH.exists(), reason="library not built")
def test_norm_refuses_rows_of_another_stride_in_place():
    # a row would be written over another workgroup's
    args = lambda xo, ldxo: (P, 64, Q, 64, Q, Q, Q, 2, 64, ZERO, 0, xo, ldxo, Q, Q, None)
    with pytest.raises(lib.SVDQError, match="ldxo") as e:
        lib.call("svdq_residual_rms_norm_modulate_mx", *args(P, 72))
    assert e.value.status == -2


@pytest.mark.parametrize("move", [lambda m: m.half(), lambda m: m.float(), lambda m: m.to(torch.float64),
                                  lambda m: m.half().float().bfloat16(), lambda m: torch.nn.Sequential(m).half()[0]])
def test_bias_stays_bf16(move):
    bias = torch.tensor([1e6, 1e-9, -3e38, 0.1, 0, 7]).bfloat16()   # values that float16 does not hold among them
    layer = MXLinear.from_dense(torch.randn(6, 40), bias)
    moved = move(layer)
    assert moved.bias.dtype == torch.bfloat16 and torch.equal(moved.bias, bias)
    assert moved.weight_codes.dtype == torch.uint8
    assert moved.to("meta").bias.device.type == "meta" and moved.bias.dtype == torch.bfloat16


def test_bias_of_another_type_is_taken_as_bf16():
    layer = MXLinear.from_dense(torch.randn(6, 40), torch.zeros(6))
    state = {**layer.state_dict(), "bias": torch.full((6,), 0.3)}
    layer.load_state_dict(state, assign=True)
    assert layer.bias.dtype == torch.bfloat16 and torch.equal(layer.bias, torch.full((6,), 0.3).bfloat16())


def test_block_takes_microscaled_outputs_only_where_nothing_is_passed_by():
    from krea2_svdquant_amd.runtime import krea2_standin as ks
    dims = ks.Krea2Dims(layers=1, hidden=64, heads=2, kv_heads=1, head_dim=32, mlp=96)
    blk = ks.Krea2StandInTransformer.random(dims, linears="mx", device="cpu", seed=5).transformer_blocks[0]
    assert blk._on_mx()
    for register in ("register_forward_hook", "register_forward_pre_hook"):
        for m in blk.linears().values():
            handle = getattr(m, register)(lambda *args: None)
            assert not blk._on_mx()
            handle.remove()
        handle = getattr(torch.nn.modules.module, register.replace("register_", "register_module_"))(lambda *args: None)
        assert not blk._on_mx()
        handle.remove()
    up = blk.ff.up
    up.forward = lambda x: x   # replaced on the instance
    assert not blk._on_mx()
    del up.forward
    assert blk._on_mx()

    class Other(MXLinear):
        pass
    blk.ff.up = Other(up.weight_codes, up.weight_scales, in_features=64, activation=up.activation)
    assert not blk._on_mx()
    blk.ff.up = up
    for switch in ("NORMS", "GATES"):
        before = getattr(ks, switch)
        setattr(ks, switch, "torch")
        try:
            assert not blk._on_mx()
        finally:
            setattr(ks, switch, before)
    assert blk._on_mx()


@pytest.mark.skipif(not lib.LIB_PATH.exists(), reason="library not built")
def test_no_tile_is_named_for_a_product_that_is_refused():
    assert lib.mx_tile(2 ** 30, 2 ** 14, 64, 0)[0] == 0
    with pytest.raises(lib.SVDQError, match="too many"):
        lib.call("svdq_mx_gemm", P, P, 0, P, P, None, 2 ** 30, 2 ** 14, 64, P, 2 ** 14, 0, None)
    assert lib.mx_tile(2 ** 16, 2 ** 14, 64, 0)[0] != 0


def test_converter_refuses_scales_that_are_not_the_codes():
    from krea2_svdquant_amd.quant.mx import dequantize_mx, quantize_mx
    codes, scales = quantize_mx(torch.randn(3, 512))
    with pytest.raises(TypeError, match="scales"):   # four bytes each: their bytes are no scales
        dequantize_mx(codes, torch.ones(3, 4), 512)
    for wrong in (scales[:, :1], scales[:1], scales[:2], torch.cat([scales, scales], 1)):   # the first two broadcast
        with pytest.raises(ValueError, match="scales"):
            dequantize_mx(codes, wrong, 512)
    assert torch.equal(dequantize_mx(codes, scales, 512), dequantize_mx(codes, scales.view(torch.uint8), 512))
