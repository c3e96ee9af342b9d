"""The 8-bit operators on the CPU: the definitions against brute force and torch's float8, the converter and the module, shape
functions, and the refusals of the C entry points (no GPU call is made)."""
import ctypes
import math

import pytest
import torch

from krea2_svdquant_amd import FP8Linear
from krea2_svdquant_amd.kernels.hip import lib, ops
from krea2_svdquant_amd.quant.fp8 import dequantize_fp8, quantize_fp8
from tests import fp8_util as u


# ---- the definitions ---------------------------------------------------------------------------------
def test_definition_of_an_element():
    values = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    values = values[~torch.isnan(values)].unique()
    mids = (values[1:] + values[:-1]) / 2
    x = torch.cat([values, mids, torch.nextafter(mids, mids + 1), torch.nextafter(mids, mids - 1)])
    q = u.e4m3(x)
    dist = (x[:, None] - values).abs()
    assert torch.equal((x - q).abs(), dist.amin(1))
    assert torch.equal(q[len(values):len(values) + len(mids)].float().to(torch.float8_e4m3fn).view(torch.uint8) & 1,
                       torch.zeros(len(mids), dtype=torch.uint8))   # ties go to the even code
    x = torch.randn(10000, generator=torch.Generator().manual_seed(0)) * 60
    assert torch.equal(u.e4m3(x.clamp(-448, 448).double()), x.clamp(-448, 448).to(torch.float8_e4m3fn).double())


def test_definition_of_a_scale():
    for top in (448.0, 449.0, 1.0, 1.75, 1.7501, 1e-30, 3e38, 2.0 ** -130):
        s = u.scale_of(torch.tensor(top, dtype=torch.float64)).item()
        assert math.frexp(s)[0] == 0.5 and top <= 448 * s and (s == 2.0 ** -126 or top > 224 * s)
    assert u.scale_of(torch.zeros(1, dtype=torch.float64)).item() == 2.0 ** -126


def test_attention_definition_against_a_softmax():
    g = torch.Generator().manual_seed(1)
    kc, vc, s = u.pages(3, 2, 64, g)
    q = torch.randn(4, 4, 64, generator=g).to(torch.bfloat16)
    o, bound = u.attention(q, [0, 4], [100], [[2, 0]], kc.float().double(), vc.float().double(), s.double(), 0.125, True)
    pages = torch.tensor([2, 0])
    k = (kc.float().double() * s[..., 0, None, None])[pages].transpose(0, 1).reshape(2, 128, 64)[:, :100].repeat_interleave(2, 0)
    v = (vc.float().double() * s[..., 1, None, None])[pages].permute(1, 0, 3, 2).reshape(2, 128, 64)[:, :100].repeat_interleave(2, 0)
    mask = torch.arange(100) <= torch.arange(4)[:, None] + 96
    want = torch.nn.functional.scaled_dot_product_attention(q.double().transpose(0, 1), k, v, attn_mask=mask, scale=0.125)
    assert (o - want.transpose(0, 1)).abs().max() < 1e-12 and (bound > 0).all() and bound.max() < 0.05 * o.abs().max()


def test_the_bounds_find_a_wrong_value():
    """A page of another sequence, a missing token and a scale of the wrong head are further off than the bounds."""
    g = torch.Generator().manual_seed(2)
    kc, vc, s = u.pages(4, 2, 64, g)
    kc, vc, s = kc.float().double(), vc.float().double(), s.double()
    q = torch.randn(3, 4, 64, generator=g).to(torch.bfloat16)
    args = (kc, vc, s, 0.125, True)
    want, bound = u.attention(q, [0, 3], [150], [[0, 1, 2]], *args)
    for offsets, lengths, table, cache in (([0, 3], [150], [[0, 3, 2]], args), ([0, 3], [149], [[0, 1, 2]], args),
                                           ([0, 3], [150], [[0, 1, 2]], (kc, vc, s.flip(1), 0.125, True))):
        got, _ = u.attention(q, offsets, lengths, table, *cache)
        with pytest.raises(AssertionError):
            u.check(got, want, bound)
    a, sa = u.quantize(torch.randn(5, 256, generator=g))
    w = torch.randint(-100, 100, (130, 256), generator=g).float().to(torch.float8_e4m3fn).float()
    ws = torch.rand(2, 2, generator=g)
    want, bound = u.product(a, sa, w, ws)
    got, _ = u.product(a, sa.flip(0), w, ws)
    with pytest.raises(AssertionError):
        u.check(got, want, bound)


# ---- the converter and the module ------------------------------------------------------------------------
@pytest.mark.parametrize("n,k", [(1, 1), (128, 128), (129, 127), (300, 260)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float64])
def test_converter(n, k, dtype):
    g = torch.Generator().manual_seed(n + k)
    w = (torch.randn(n, k, generator=g) * torch.exp2(torch.randint(-20, 20, (n, 1), generator=g).float())).to(dtype)
    w[n // 2, k - 1], w[0, 0] = math.inf, 0.0
    codes, scales = quantize_fp8(w)
    kp = -(-k // 128) * 128
    assert codes.shape == (n, kp) and codes.dtype == torch.float8_e4m3fn and scales.dtype == torch.float32
    assert scales.shape == (-(-n // 128), kp // 128) and not codes[:, k:].float().any()
    for i in range(scales.shape[0]):
        for j in range(scales.shape[1]):
            b = w[128 * i:128 * i + 128, 128 * j:128 * j + 128].float().double()
            s = u.scale_of(u.finite_top(b, (0, 1)))
            assert scales[i, j].item() == s.item()
            got = codes[128 * i:128 * i + 128, 128 * j:128 * j + 128].float().double()[:, :b.shape[1]]
            want = u.e4m3(b / s)
            assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got.nan_to_num(), want.nan_to_num())
    back = dequantize_fp8(codes, scales, k)
    ok = torch.isfinite(w)
    step = scales.repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
    # half a step: 2^-4 of the value, 2^-10 of the scale below the smallest normal value
    assert ((back - w.float()).abs() <= torch.maximum(w.float().abs() * 2.0 ** -4, step * 2.0 ** -10))[ok].all()


def test_converter_refusals():
    with pytest.raises(TypeError):
        quantize_fp8(torch.zeros(4, 4, dtype=torch.int32))
    for shape in ((4,), (0, 4), (4, 0), (2, 3, 4)):
        with pytest.raises(ValueError):
            quantize_fp8(torch.zeros(shape))
    codes, scales = quantize_fp8(torch.zeros(130, 64))
    with pytest.raises(TypeError):
        dequantize_fp8(codes.float(), scales, 64)
    with pytest.raises(ValueError):
        dequantize_fp8(codes, scales, 129)
    with pytest.raises(ValueError):
        dequantize_fp8(codes, scales[:1], 64)


def test_module_on_the_cpu():
    w = torch.randn(130, 40)
    layer = FP8Linear.from_dense(w, torch.zeros(130))
    assert layer.weight_codes.shape == (130, 128) and layer.weight_codes.dtype == torch.uint8
    assert layer.weight_scales.shape == (2, 1) and layer.bias.dtype == torch.bfloat16
    assert torch.equal(layer.dense_weight(), dequantize_fp8(*quantize_fp8(w), 40))
    assert set(layer.state_dict()) == {"weight_codes", "weight_scales", "bias"}
    before = {k: v.clone() for k, v in layer.state_dict().items()}
    layer.weight_scales.mul_(1.2345678)   # not a power of two, so that half precision would show
    before["weight_scales"] = layer.weight_scales.clone()
    for kept in (layer.half(), layer.to(torch.bfloat16), layer.float(), layer.double()):
        for name, t in kept.state_dict().items():
            assert t.dtype == before[name].dtype and torch.equal(t, before[name])
    other = FP8Linear.from_dense(torch.zeros(130, 40), torch.ones(130))
    state = dict(layer.state_dict(), weight_codes=layer.weight_codes.view(torch.float8_e4m3fn))
    for assign in (False, True):   # codes as float8 or as bytes
        other.load_state_dict(state, assign=assign)
        assert other.weight_codes.dtype == torch.uint8 and torch.equal(other.weight_codes, layer.weight_codes)
        assert torch.equal(other.weight_scales, layer.weight_scales)
    with pytest.raises(RuntimeError, match="GPU"):
        layer(torch.zeros(2, 40, dtype=torch.bfloat16))
    with pytest.raises(ValueError):
        layer(torch.zeros(2, 41, dtype=torch.bfloat16))
    with pytest.raises(ValueError):
        FP8Linear.from_dense(w[0])
    codes, scales = layer.weight_codes, layer.weight_scales
    for bad in (dict(in_features=200), dict(in_features=0), dict(in_features=40, bias=torch.zeros(5)),
                dict(in_features=40, weight_scales=scales[:1]), dict(in_features=40, weight_scales=scales.half()),
                dict(in_features=40, weight_codes=codes.int())):
        with pytest.raises(ValueError):
            FP8Linear(**{"weight_codes": codes, "weight_scales": scales, **bad})


def test_stand_in_takes_them():
    from krea2_svdquant_amd.runtime import krea2_standin as ks
    dims = ks.Krea2Dims(layers=1, hidden=128, heads=1, kv_heads=1, head_dim=128, mlp=200)
    model = ks.Krea2StandInTransformer.random(dims, linears="fp8", device="cpu")
    assert all(type(m) is FP8Linear for m in model.transformer_blocks[0].linears().values())
    with pytest.raises(ValueError, match="fp8"):
        ks.Krea2StandInTransformer.random(dims, linears="fp6", device="cpu")


# ---- operators ------------------------------------------------------------------------------------------------
def test_operators_refuse_the_cpu():
    x = torch.zeros(2, 128, dtype=torch.bfloat16)
    w, ws = quantize_fp8(torch.zeros(8, 128))
    h = torch.zeros(2, 1, 64, dtype=torch.bfloat16)
    tab = torch.zeros(2, 32)
    i = torch.zeros(2, dtype=torch.int32)
    kc, vc, s = u.pages(1, 1, 64, torch.Generator().manual_seed(0))
    cache = (i, i[:1], i[:1, None], kc, vc, s)
    for call in (lambda: ops.fp8_quantize(x), lambda: ops.fp8_gemm(w, ws, w, ws), lambda: ops.fp8_linear(x, w, ws),
                 lambda: ops.qk_norm_rope(h, h, None, None, tab, tab, 1e-6), lambda: ops.kv8_append(h, h, *cache),
                 lambda: ops.kv8_attention(h, *cache, 0.125)):
        with pytest.raises(RuntimeError, match="GPU"):
            call()


@pytest.mark.skipif(not lib.TORCH_LIB_PATH.exists(), reason="library not built")
def test_shape_functions():
    from torch._subclasses.fake_tensor import FakeTensorMode
    native = ops.load_native()
    with FakeTensorMode():
        x = torch.empty(2, 3, 520, dtype=torch.bfloat16)
        c, s = native["fp8_quantize"](x)
        assert c.shape == (2, 3, 640) and c.dtype == torch.float8_e4m3fn and s.shape == (5, 6) and s.dtype == torch.float32
        w, ws = torch.empty(40, 640, dtype=torch.float8_e4m3fn), torch.empty(1, 5)
        for y in (native["fp8_gemm"](c, s, w, ws, None), native["fp8_linear"](x, w, ws, None)):
            assert y.shape == (2, 3, 40) and y.dtype == torch.bfloat16
        q, k = torch.empty(7, 8, 64, dtype=torch.bfloat16), torch.empty(7, 2, 64, dtype=torch.bfloat16)
        tab = torch.empty(10, 32)
        assert [t.shape for t in native["qk_norm_rope"](q, k, None, None, tab, tab, 1e-6, None, False)] == [q.shape, k.shape]
        i = torch.empty(2, dtype=torch.int32)
        kc, vc = (torch.empty(s, dtype=torch.float8_e4m3fn) for s in ((4, 2, 64, 64), (4, 2, 64, 64)))
        cache = (i, i[:1], i[:1, None], kc, vc, torch.empty(4, 2, 2))
        assert native["kv8_append"](k, k, *cache) is None
        assert native["kv8_attention"](q, *cache, 0.125, True).shape == q.shape


P = ctypes.c_void_p(0x1000)    # never read: the calls below fail on the host
ODD = ctypes.c_void_p(0x1001)
EIGHT = ctypes.c_void_p(0x1008)
ZERO, EPS = ctypes.c_float(0), ctypes.c_float(1e-6)


def qk(**change):
    a = dict(q=P, ldq=512, hsq=64, k=P, ldk=512, hsk=64, qw=None, kw=None, cos=P, sin=P, ldcs=32, P=9, wide=1, at=None, T=4,
             H=4, Hkv=2, D=64, eps=EPS, pairs=0, qo=P, ko=P)
    return "svdq_qk_norm_rope", tuple({**a, **change}.values())


def append(**change):
    a = dict(k=P, ldk=128, v=P, ldv=128, N=4, offsets=P, lengths=P, table=P, B=2, W=3, kc=P, vc=P, scales=P, P=5, Hkv=2, D=64)
    return "svdq_kv8_append", tuple({**a, **change}.values())


def attend(**change):
    a = dict(q=P, ldq=256, N=4, offsets=P, lengths=P, table=P, B=2, W=3, kc=P, vc=P, scales=P, P=5, H=4, Hkv=2, D=64,
             scale=ZERO, causal=1, o=P, work=P)
    return "svdq_kv8_attention", tuple({**a, **change}.values())


def gemm(**change):
    a = dict(a=P, sa=P, w=P, ws=P, bias=None, M=2, N=8, K=128, y=P, ldy=8)
    return "svdq_fp8_gemm", tuple({**a, **change}.values())


def linear(**change):
    a = dict(x=P, ldx=128, w=P, ws=P, bias=None, M=2, N=8, K=128, y=P, ldy=8, work=P)
    return "svdq_fp8_linear", tuple({**a, **change}.values())


@pytest.mark.parametrize("call,status,needle", [
    (("svdq_fp8_quantize", (P, 64, -1, 64, P, P)), -2, "M=-1"),
    (("svdq_fp8_quantize", (P, 64, 2, 0, P, P)), -2, "K=0"),
    (("svdq_fp8_quantize", (P, 63, 2, 64, P, P)), -2, "ldx=63"),
    (("svdq_fp8_quantize", (None, 64, 2, 64, P, P)), -1, "null"),
    (("svdq_fp8_quantize", (P, 64, 2, 64, P, None)), -1, "null"),
    (("svdq_fp8_quantize", (P, 64, 2, 64, EIGHT, P)), -3, "16-byte"),
    (("svdq_fp8_quantize", (ODD, 64, 2, 64, P, P)), -3, "elements"),
    (("svdq_fp8_quantize", (P, 64, 2 ** 31 - 1, 2 ** 20, P, P)), -2, "ldx=64"),
    (("svdq_fp8_quantize", (P, 2 ** 20, 2 ** 31 - 1, 2 ** 20, P, P)), -2, "too many"),
    (gemm(N=0), -2, "N=0"), (gemm(ldy=7), -2, "ldy=7"), (gemm(K=2 ** 22 + 1), -2, "2.22"), (gemm(a=None), -1, "null"),
    (gemm(w=None), -1, "null"), (gemm(y=None), -1, "null"), (gemm(a=EIGHT), -3, "16-byte"), (gemm(w=EIGHT), -3, "16-byte"),
    (gemm(ws=ODD), -3, "elements"), (gemm(sa=ODD), -3, "elements"),
    (gemm(bias=ODD), -3, "elements"),
    (gemm(M=2 ** 30, N=2 ** 14, ldy=2 ** 14), -2, "too many"),
    (linear(N=0), -2, "N=0"), (linear(ldx=127), -2, "ldx=127"), (linear(x=None), -1, "null"), (linear(ws=None), -1, "null"),
    (linear(x=ODD), -3, "elements"), (linear(work=None), -1, "workspace"), (linear(work=EIGHT), -3, "16-byte"),
    (linear(K=2 ** 23), -2, "2.22"), (linear(M=2 ** 30, N=2 ** 14, ldy=2 ** 14), -2, "too many"),
    (qk(D=60), -2, "D=60"), (qk(D=272), -2, "D=272"), (qk(H=0), -2, "H=0"), (qk(P=3), -2, "3 table rows"),
    (qk(ldcs=28), -2, "ldcs=28"), (qk(wide=2), -1, "wide=2"), (qk(pairs=3), -1, "pairs=3"),
    (qk(eps=ctypes.c_float(math.nan)), -1, "eps"), (qk(q=None), -1, "null"), (qk(ko=None), -1, "null"), (qk(q=EIGHT), -3, "16-byte"),
    (qk(hsq=60), -3, "16-byte"), (qk(ldcs=34), -3, "16-byte"), (qk(at=ODD), -3, "16-byte"),
    (qk(T=2 ** 27, P=2 ** 27), -2, "too many"),
    (append(D=96), -4, "D=96"), (append(B=0), -2, "B=0"), (append(W=0), -2, "W=0"), (append(W=2 ** 24 + 1), -2, "W="),
    (append(P=0), -2, "P=0"), (append(N=-1), -2, "N=-1"), (append(offsets=None), -1, "null"), (append(k=None), -1, "null"),
    (append(kc=EIGHT), -3, "16-byte"), (append(table=ODD), -3, "elements"), (append(ldk=100), -3, "multiples of 8"),
    (append(N=2 ** 30), -2, "too many"),
    (attend(D=32), -4, "D=32"), (attend(H=3), -2, "H=3"), (attend(causal=2), -1, "causal=2"), (attend(q=None), -1, "null"),
    (attend(scales=None), -1, "null"), (attend(q=EIGHT), -3, "16-byte"), (attend(ldq=100), -3, "multiple of 8"),
    (attend(work=None, W=1000), -1, "workspace"), (attend(work=EIGHT), -3, "16-byte"), (attend(lengths=ODD), -3, "elements"),
    (attend(N=2 ** 30, H=64), -2, "too many"),
])
def test_c_entries_refuse_before_any_launch(call, status, needle):
    fn, args = call
    with pytest.raises(lib.SVDQError, match=needle) as e:
        lib.call(fn, *args, None)
    assert e.value.status == status


def test_c_entries_take_no_rows():
    lib.call("svdq_fp8_quantize", None, 64, 0, 64, None, None, None)
    for fn, args in (gemm(M=0, a=None, y=None), linear(M=0, x=None, y=None, work=None), qk(T=0, q=None, qo=None),
                     append(N=0, k=None, v=None), attend(N=0, q=None, o=None, work=None)):
        lib.call(fn, *args, None)


def test_workspaces():
    load = lib.load()
    assert load.svdq_fp8_linear_workspace(77, 6100) == 77 * 6144 + 77 * 48 * 4
    assert load.svdq_fp8_linear_workspace(-1, 8) == 0 and load.svdq_fp8_linear_workspace(2, 2 ** 23) == 0
    assert load.svdq_kv8_attention_workspace(1, 1, 2048, 48, 12, 128, 1) > 0
    assert load.svdq_kv8_attention_workspace(1, 1, 2048, 48, 7, 128, 1) == 0


@pytest.mark.skipif(not lib.LIB_PATH.exists(), reason="library not built")
def test_kernels_stay_in_registers():
    from tests.test_kernel_resources import _kernel_metadata
    meta = {k: v["private_segment_fixed_size"] for k, v in _kernel_metadata().items()}
    for name, count in (("fp8_quantize_kernel", 2), ("fp8_gemm_rows_kernel", 2), ("fp8_linear_rows_kernel", 1),
                        ("fp8_gemm_tile_kernel", 5), ("fp8_gemm_strip_kernel", 5), ("qk_norm_rope_kernel", 1),
                        ("kv8_append_kernel", 2), ("kv8_rows_kernel", 2), ("kv8_many_kernel", 2), ("kv8_join_kernel", 4)):
        found = [v for k, v in meta.items() if name in k]
        assert len(found) >= count and not any(found), name
