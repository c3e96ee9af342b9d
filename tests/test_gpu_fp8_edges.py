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


# ---- the cache and its attention -----------------------------------------------------------------------------
def i32(dev, x):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def mean_of(v, seen):
    """(o, bound) of equal probabilities of the keys `seen` [keys]: rounded to bf16 times their page's scale, which the sum
    shares (fp8_util.attention), and the result's rounding."""
    x = v[..., seen].double()
    o, size = x.mean(-1), x.abs().mean(-1)
    near = u.HALF / (1 - u.HALF) * (size + o.abs()) + size * 2.0 ** -17
    return o, near + u.HALF * (o.abs() + near)


@pytest.mark.parametrize("n", [3, 130])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("level", [2.0 ** 12, 2.0 ** 24, 2.0 ** 40, 2.0 ** 100])
def test_attention_of_scores_of_any_size(dev, n, d, level):
    """Scores of whole multiples of a level, far apart: the largest share the result evenly, whatever their page's scale; with
    pages in every order of their largest scores."""
    g = gen(d)
    k = torch.randint(-6, 4, (4, 1, 64, d), generator=g).float()
    for page, top in enumerate((2, 5, 5, 4)):
        k[page, 0, :, 0] = torch.randint(-6, top, (64,), generator=g).float()
        k[page, 0, 7:60:10 + page, 0] = top
    v = torch.randint(-100, 100, (4, 1, d, 64), generator=g).float().to(torch.float8_e4m3fn)
    s = torch.ones(4, 1, 2)
    s[:, 0, 1] = torch.tensor([0.7, 0.013, 3.0, 1.0])
    q = torch.zeros(n, 4, d)
    q[..., 0] = level
    for order in ([0, 1, 2, 3], [2, 3, 0, 1], [3, 0, 1, 2]):
        for sign in (1.0, -1.0):
            o = ops.kv8_attention((sign * q).to(torch.bfloat16).to(dev), i32(dev, [0, n]), i32(dev, [256]), i32(dev, [order]),
                                  k.to(torch.float8_e4m3fn).to(dev), v.to(dev), s.to(dev), 0.3, False)
            kv = sign * k[order, 0, :, 0].flatten()
            vv = (v.float() * s[..., 1:, None])[order, 0].permute(1, 0, 2).flatten(1)
            want, bound = mean_of(vv, kv == kv.max())
            u.check(o, want.expand(n, 4, d), bound.expand(n, 4, d))


@pytest.mark.parametrize("n", [3, 130])
@pytest.mark.parametrize("order", [[0, 1, 2], [1, 0, 2]])
def test_attention_of_a_page_whose_scores_pass_float32(dev, n, order):
    """-infinity for every key of a page (the first one, too) leaves the others their part."""
    k = torch.full((3, 1, 64, 64), -2.0 ** -9)
    k[0] = -448.0
    v = torch.randint(-100, 100, (3, 1, 64, 64), generator=gen(n)).float().to(torch.float8_e4m3fn)
    q = torch.full((n, 4, 64), 3e37).to(torch.bfloat16)
    o = ops.kv8_attention(q.to(dev), i32(dev, [0, n]), i32(dev, [192]), i32(dev, [order]), k.to(torch.float8_e4m3fn).to(dev),
                          v.to(dev), torch.ones(3, 1, 2, device=dev), 0.125, False)
    vv = v.float()[order, 0].permute(1, 0, 2).flatten(1)
    want, bound = mean_of(vv, torch.tensor(order).repeat_interleave(64) != 0)
    u.check(o, want.expand(n, 4, 64), bound.expand(n, 4, 64))


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("had", [-0.3, -2.0 ** -6, -3.7e-5, -1e30, 0.3, 2.5e-9])
def test_append_behind_a_page_scale_of_any_sign(dev, d, had):
    """The scale that is larger in magnitude holds the older tokens and the new ones."""
    g = gen(d)
    kc, vc, s = u.pages(1, 2, d, g)
    s[:] = had
    s[0, 1] *= 0.5
    k, v = normal((9, 2, d), g), normal((9, 2, d), g, 0.01)
    K, V, S = kc.to(dev), vc.to(dev), s.to(dev)
    ops.kv8_append(k.to(dev), v.to(dev), i32(dev, [0, 9]), i32(dev, [21]), i32(dev, [[0]]), K, V, S)
    for w, (x, codes, got) in enumerate(((k, kc, K.cpu()), (v, vc.transpose(2, 3), V.cpu().transpose(2, 3)))):
        x, old, got = x.double().transpose(0, 1), codes.double()[0], got.double()[0]
        need, before = u.scale_of(x.abs().amax((1, 2))), s[0, :, w].double()
        after = torch.where(before.abs() >= need, before, need)
        assert torch.equal(S.cpu().double()[0, :, w], after)
        factor = (before / after).float().double()[:, None, None]   # rounded to float32
        assert torch.equal(got[:, :21], u.e4m3(old[:, :21] * factor))
        assert torch.equal(got[:, 21:30], u.e4m3(x / after[:, None, None]))
        assert torch.equal(got[:, 30:], old[:, 30:])


# ---- the product's kernels, each at a size that it is taken for (K = 640): (M, N) and lib.fp8_kernel's answer ----
KERNELS = {
    "8 rows": (5, 130, (3, 16, 16, 0)), "16 rows": (12, 131, (3, 16, 16, 0)),
    "strip 32 x 16": (17, 50, (2, 32, 16, 0)), "strip 32 x 32": (33, 2081, (2, 32, 32, 0)),
    "strip 64 x 32": (34, 4127, (2, 64, 32, 0)), "strip 48 x 64": (18, 8249, (2, 48, 64, 0)),
    "strip 64 x 64": (50, 8321, (2, 64, 64, 0)), "tile 64 x 64": (5501, 262, (1, 64, 64, 0)),
    "tile 64 x 128": (17, 16424, (1, 64, 128, 0)), "tile 128 x 128": (259, 16918, (1, 128, 128, 0)),
    "tile 256 x 128": (133, 22092, (1, 256, 128, 0)), "tile 256 x 256": (337, 21920, (1, 256, 256, 0)),
    "two launches": (1802, 17685, (1, 64, 128, 1792))}


def product_on(a, sa, w, sw, bias=None):
    """fp8_util.product on the operands' device, block by block."""
    n, kb = w.shape[0], sa.shape[0]
    y = mag = lost = 0.0
    for b in range(kb):
        p = a[:, 128 * b:128 * b + 128].double() * sa[b].double()[:, None]
        q = w[:, 128 * b:128 * b + 128].double() * sw[:, b].double().repeat_interleave(128)[:n, None]
        y, mag = y + p @ q.T, mag + p.abs() @ q.abs().T
        lost = lost + 16 * 7 * 2.0 ** -13 * p.abs().amax(-1)[:, None] * q.abs().amax(-1)
    if bias is not None:
        y, mag = y + bias.double(), mag + bias.double().abs()
    near = (131 + kb) * 2.0 ** -24 * mag + lost
    return y, near + u.HALF * (y.abs() + near) + 2.0 ** -133


def check_on(got, want, bound):
    assert torch.isfinite(got).all() and torch.isfinite(want).all()
    worst = ((got.double() - want).abs() / bound.clamp_min(1e-300)).max().item()   # 0: rows that see nothing
    assert worst <= 1.0, f"off by {worst:.3g} of the bound"


# codes' magnitude, the scales' exponents, and what a block may be off where the scales' product is subnormal: half of its last bit,
# 2^-150, times a sum of 128 products of 448 x 448
FAR_SCALES = {"product up to 2^127": (2.0 ** -8, 110, 15, 0.0), "product from 2^-126": (448.0, -126, 0, 0.0),
              "subnormal activations": (448.0, -135, 20, 0.0), "subnormal weights": (8.0, 124, -138, 0.0),
              "product of 2^-138": (448.0, -126, -12, 128 * 448.0 ** 2 * 2.0 ** -150)}


@pytest.mark.parametrize("size", KERNELS)
@pytest.mark.parametrize("far", FAR_SCALES)
def test_product_of_scales_at_the_ends_of_float32(dev, size, far):
    """Results are ordinary; rows, columns and blocks of zeros, of codes and of scales, among them."""
    from krea2_svdquant_amd.kernels.hip import lib
    m, n, kernel = KERNELS[size]
    assert lib.fp8_kernel(m, n, 640) == kernel
    amp, ea, ew, off = FAR_SCALES[far]
    g = torch.Generator(device=dev).manual_seed(m)
    a, w = ((torch.randn((r, 640), device=dev, generator=g) * amp / 3).clamp(-amp, amp).to(torch.float8_e4m3fn) for r in (m, n))
    sa = ((1 + torch.rand((5, m), device=dev, generator=g).double()) * 2.0 ** ea).float()
    sw = ((1 + torch.rand((-(-n // 128), 5), device=dev, generator=g).double()) * 2.0 ** ew).float()
    for t in (a.view(torch.uint8)[0], a.view(torch.uint8)[1, 128:256], w.view(torch.uint8)[n - 1]):
        t.zero_()
    sa[3, 2], sw[0, 4] = 0.0, -sw[0, 4]
    want, bound = product_on(a, sa, w, sw)
    check_on(ops.fp8_gemm(a, sa, w, sw), want, bound + 5 * off)


# Each kernel at 66 blocks of K (the weights' scales are looked up 64 at a time), and layer sizes of the denoiser's.
DEEP = {
    "8 rows": (5, 130, 8448, (3, 16, 16, 0)), "16 rows": (12, 131, 8448, (3, 16, 16, 0)),
    "strip 32 x 16": (17, 50, 8448, (2, 32, 16, 0)), "strip 32 x 32": (33, 2065, 8448, (2, 32, 32, 0)),
    "strip 64 x 32": (33, 4107, 8448, (2, 64, 32, 0)), "strip 48 x 64": (18, 8198, 8448, (2, 48, 64, 0)),
    "strip 64 x 64": (49, 8418, 8448, (2, 64, 64, 0)), "tile 64 x 64": (5634, 263, 8448, (1, 64, 64, 0)),
    "tile 64 x 128": (65, 8207, 8448, (1, 64, 128, 0)), "tile 128 x 128": (260, 19949, 8448, (1, 128, 128, 0)),
    "tile 256 x 128": (145, 23076, 8448, (1, 256, 128, 0)), "tile 256 x 256": (520, 18194, 8448, (1, 256, 256, 0)),
    "two launches": (1285, 18151, 8448, (1, 64, 128, 768)),
    "prompt": (77, 6144, 6144, (2, 48, 64, 0)), "128 tokens": (128, 6144, 6144, (2, 64, 64, 0)),
    "320 tokens": (320, 6144, 6144, (1, 64, 128, 0)), "image, up": (4352, 16384, 6144, (1, 64, 128, 4096)),
    "image, down": (4352, 6144, 16384, (1, 256, 256, 0))}


@pytest.mark.parametrize("size", DEEP)
@pytest.mark.parametrize("bias", [False, True])
def test_product_of_small_whole_numbers_on_every_kernel(dev, size, bias):
    """Codes and scales of which every sum is a whole number below 2^24, so only the store rounds; scales differ from block to
    block."""
    from krea2_svdquant_amd.kernels.hip import lib
    m, n, k, kernel = DEEP[size]
    assert lib.fp8_kernel(m, n, k) == kernel
    kb, g = k // 128, torch.Generator(device=dev).manual_seed(m + bias)
    a, w = (torch.randint(-3, 4, (r, k), device=dev, generator=g).float() for r in (m, n))
    sa = torch.randint(1, 4, (kb, m), device=dev, generator=g).float()
    sw = torch.randint(1, 4, (-(-n // 128), kb), device=dev, generator=g).float()
    b = torch.randint(-100, 101, (n,), device=dev, generator=g).to(torch.bfloat16) if bias else None
    y = ops.fp8_gemm(a.to(torch.float8_e4m3fn), sa, w.to(torch.float8_e4m3fn), sw, b)
    ab = (a.view(m, kb, 128) * sa.T[..., None]).view(m, k).double()
    wb = (w.view(n, kb, 128) * sw.repeat_interleave(128, 0)[:n, :, None]).view(n, k).double()
    want = ab @ wb.T
    if bias:
        want += b.double()
    assert torch.equal(y, want.to(torch.bfloat16))


# ---- attention of which a card's last tiles alone are split ------------------------------------------------------
def attention_on(q, offsets, lengths, table, kc, vc, scales, scale, causal):
    """fp8_util.attention of pages that are all there and hold numbers, on the operands' device."""
    heads, d, group = q.shape[1], q.shape[2], q.shape[1] // kc.shape[1]
    out, bound = (torch.zeros(q.shape, dtype=torch.float64, device=q.device) for _ in range(2))
    for b, length in enumerate(lengths):
        row, n = offsets[b], offsets[b + 1] - offsets[b]
        if not n or not length:
            continue
        pages = torch.tensor(table[b][:-(-length // u.PAGE)], device=q.device)
        last = torch.arange(n, device=q.device)[:, None] + length - n if causal else torch.full((n, 1), length, device=q.device)
        hidden = torch.arange(length, device=q.device) > last
        for h in range(heads):
            kv = h // group
            k = (kc[pages, kv].double() * scales[pages, kv, 0].double()[:, None, None]).reshape(-1, d)[:length]
            v = (vc[pages, kv].double() * scales[pages, kv, 1].double()[:, None, None]).transpose(1, 2).reshape(-1, d)[:length]
            x = q[row:row + n, h].double()
            s = (x @ k.T * scale).masked_fill_(hidden, -float("inf"))
            mag = (x.abs() @ k.abs().T * abs(scale)).masked_fill_(hidden, 0).amax(-1, keepdim=True)
            p = torch.exp(s - s.amax(-1, keepdim=True).clamp_min(-1e300))
            total = p.sum(-1, keepdim=True)
            p = p / torch.where(total == 0, 1.0, total)
            o, size = p @ v, p @ v.abs()
            off = 2 * ((d + 8) * 2.0 ** -24 * 1.4427 * mag + 2.0 ** -20)
            near = u.HALF / (1 - u.HALF) * (size + o.abs()) + size * (2 * off + 2.0 ** -18)
            out[row:row + n, h] = o
            bound[row:row + n, h] = near + u.HALF * (o.abs() + near) + 2.0 ** -133
    return out, bound


# key heads, query heads of each, sequences (new tokens, tokens held): more than the 64 tiles that an XCD runs at a time, and a few
ROUNDS = {
    "8 heads": (8, 4, [(700, 500), (0, 300), (900, 640), (560, 64)]), "12 heads": (12, 4, [(500, 700), (300, 1), (0, 0), (900, 333)]),
    "2 heads": (2, 16, [(2140, 700)]), "3 heads": (3, 8, [(1500, 64), (1350, 700)]), "1 head": (1, 64, [(50, 700), (1000, 129)])}


@pytest.mark.parametrize("name", ROUNDS)
@pytest.mark.parametrize("d", [64, 128])
def test_attention_of_which_the_last_tiles_are_split(dev, name, d):
    from krea2_svdquant_amd.kernels.hip import lib
    from tests.test_gpu_fp8 import Cache
    kv, group, seqs = ROUNDS[name]
    c = Cache(dev, seqs, kv, d, len(name), width=3)
    rows, heads = c.offsets[-1], kv * group
    kind, splits, whole, tiles = lib.kv8_kernel(rows, len(seqs), len(c.table[0]), heads, kv, d, False)
    assert kind == 2 and splits > 1 and 0 < whole < tiles
    q = normal((rows + 70, heads, d), c.g).to(dev)[:rows + 5]   # the last rows are no sequence's
    args = c.device()
    o = ops.kv8_attention(q, *args, d ** -0.5, False)
    check_on(o, *attention_on(q, c.offsets, c.lengths(), c.table, *args[3:], d ** -0.5, False))
    assert not o[rows:].any()


@pytest.mark.parametrize("prompt,singles,kernel", [(1500, 40, 1), (3000, 63, 1), (2100, 7, 3), (2100, 31, 3), (3000, 64, 2)])
@pytest.mark.parametrize("d", [64, 128])
def test_attention_of_a_prompt_among_single_tokens(dev, prompt, singles, kernel, d):
    """A batch takes one kernel, by its rows in the mean: the prompt on that for few rows (1), single tokens on that for many
    (2, 3: in pieces of about one length)."""
    from krea2_svdquant_amd.kernels.hip import lib
    from tests.test_gpu_fp8 import Cache
    seqs = [(1, 1 + 97 * b % 2000) for b in range(singles)]
    seqs.insert(singles // 3, (prompt, prompt + 500))
    c = Cache(dev, seqs, 2, d, singles, width=1)
    rows = c.offsets[-1]
    group = 4 if kernel == 1 else 8
    assert lib.kv8_kernel(rows, len(seqs), len(c.table[0]), 2 * group, 2, d, True)[0] == kernel
    q = normal((rows, 2 * group, d), c.g).to(dev)
    args = c.device()
    for causal in (True, False):
        o = ops.kv8_attention(q, *args, d ** -0.5, causal)
        check_on(o, *attention_on(q, c.offsets, c.lengths(), c.table, *args[3:], d ** -0.5, causal))


# ---- layers that read the same input -----------------------------------------------------------------------------
def test_grouped_layers_are_not_asked_for_a_shared_8_bit_activation(dev, monkeypatch):
    """SVDQuant layers take their one launch without looking for 8-bit ones first; those share their activation as before."""
    from krea2_svdquant_amd import FP8Linear, SVDQuantLinear
    from krea2_svdquant_amd.runtime import krea2_standin as ks, siblings
    asked = []
    share = siblings._share_fp8
    monkeypatch.setattr(siblings, "_share_fp8", lambda x, layers: asked.append(1) or share(x, layers))
    g = torch.Generator(device=dev).manual_seed(0)
    x = torch.randn((40, 256), device=dev, generator=g).to(torch.bfloat16)
    layers = [SVDQuantLinear(ks.random_quantized_state(n, 256, rank=32, group_size=64, device=dev, generator=g), backend="hip_gfx950")
              for n in (256, 128)]
    assert [y.shape for y in siblings.run_grouped(x, layers)] == [(40, 256), (40, 128)] and not asked
    layers = [FP8Linear.from_dense(torch.randn((n, 256), device=dev, generator=g)) for n in (256, 130)]
    quantized = []
    monkeypatch.setattr(FP8Linear, "quantize", lambda self, z: quantized.append(1) or ops.fp8_quantize(z))
    for y, layer in zip(siblings.run_grouped(x, layers), layers):
        assert torch.equal(y, ops.fp8_linear(x, layer._codes(), layer.weight_scales))
    assert len(quantized) == 1 and asked


def test_linear_of_rows_in_any_layout(dev):
    """Repeated, transposed, unaligned, single and no rows: as their contiguous copy."""
    g = gen(80)
    w, ws = torch.randint(-100, 100, (130, 256), generator=g).float().to(torch.float8_e4m3fn).to(dev), torch.rand((2, 2), generator=g).to(dev)
    base = normal((300, 40), g).to(dev)
    for x in (normal((1, 256), g).to(dev).expand(5, 256), base[:256].T, base.view(-1)[3:3 + 256], base[:256, 5:6].T, base[:256].T[:0],
              base.view(-1)[1:1 + 6 * 256].view(2, 3, 256)):
        y = ops.fp8_linear(x, w, ws)
        assert y.shape == (*x.shape[:-1], 130) and torch.equal(y, ops.fp8_linear(x.contiguous().clone(), w, ws))
        codes, scales = ops.fp8_quantize(x)
        assert torch.equal(y, ops.fp8_gemm(codes, scales, w, ws))


# ---- the largest sizes ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("m,n", [(3, 50), (12, 50), (20, 50), (1100, 130)])
def test_product_of_the_longest_rows(dev, m, n):
    """K = 2^22: codes of 1 and -1 and scales of 1, so that sums are whole numbers below 2^24."""
    k, g = 2 ** 22, torch.Generator(device=dev).manual_seed(m)
    a, w = (torch.randint(0, 2, (r, k), device=dev, generator=g, dtype=torch.uint8) * 128 + 0x38 for r in (m, n))
    sa, sw = torch.ones((k // 128, m), device=dev), torch.ones((-(-n // 128), k // 128), device=dev)
    y = ops.fp8_gemm(a.view(torch.float8_e4m3fn), sa, w.view(torch.float8_e4m3fn), sw)
    want = torch.zeros((m, n), device=dev, dtype=torch.float64)
    for c in range(0, k, 2 ** 17):
        want += (1 - (a[:, c:c + 2 ** 17] >> 7).double() * 2) @ (1 - (w[:, c:c + 2 ** 17] >> 7).double() * 2).T
    assert torch.equal(y, want.to(torch.bfloat16))


def test_quantize_a_row_of_2_30_columns(dev):
    g = torch.Generator(device=dev).manual_seed(0)
    x = torch.zeros((1, 2 ** 30), dtype=torch.bfloat16, device=dev)
    parts = (0, 2 ** 29 - 4096, 2 ** 30 - 8192)
    for p in parts:
        x[0, p:p + 8192] = torch.randn(8192, device=dev, generator=g).to(torch.bfloat16)
    codes, scales = ops.fp8_quantize(x)
    for p in parts:
        c, s = ops.fp8_quantize(x[:, p:p + 8192].contiguous())
        assert torch.equal(codes[:, p:p + 8192].view(torch.uint8), c.view(torch.uint8))
        assert torch.equal(scales[p // 128:p // 128 + 64], s)
    assert not codes[:, 10000:20000].view(torch.uint8).any()


def test_head_norms_whose_output_passes_32_bits(dev):
    t, h, kv, d = 600000, 48, 12, 64
    g = torch.Generator(device=dev).manual_seed(1)
    x = torch.empty((t, h + kv, d), dtype=torch.bfloat16, device=dev)
    x[:] = torch.randn((1000, h + kv, d), device=dev, generator=g).to(torch.bfloat16).repeat(600, 1, 1)
    tab = torch.randn((700, d // 2), device=dev, generator=g)
    at = torch.randint(0, 700, (t,), device=dev, generator=g)
    qo, ko = ops.qk_norm_rope(x[:, :h], x[:, h:], None, None, tab, tab, 1e-6, at)
    for p in (0, t // 2, t - 100):
        q, k = ops.qk_norm_rope(x[p:p + 100, :h], x[p:p + 100, h:], None, None, tab, tab, 1e-6, at[p:p + 100])
        assert torch.equal(qo[p:p + 100], q) and torch.equal(ko[p:p + 100], k)


def test_attention_whose_output_passes_32_bits(dev):
    """1000 sequences of 300 tokens of 64 heads, which share their pages; the last ones against the definition."""
    from tests.test_gpu_fp8 import Cache
    n, heads, d, count = 300, 64, 128, 1000
    c = Cache(dev, [(n, 310)], 8, d, 90)
    _, _, _, k, v, s = c.device()
    q = normal((n, heads, d), c.g).to(dev).repeat(count, 1, 1)
    o = ops.kv8_attention(q, i32(dev, [n * b for b in range(count + 1)]), i32(dev, [310] * count), i32(dev, c.table * count), k, v, s,
                          d ** -0.5)
    want, bound = attention_on(q[:n], [0, n], [310], c.table, k, v, s, d ** -0.5, True)
    for b in (0, count // 2, count - 1):
        check_on(o[n * b:n * b + n], want, bound)
