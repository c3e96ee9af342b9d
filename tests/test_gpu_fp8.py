"""The 8-bit linear, the head norms with rotation and the 8-bit cache against their definitions in 64 bits."""
from __future__ import annotations

import math

import pytest
import torch

from krea2_svdquant_amd.kernels.hip import ops
from tests import fp8_util as u

pytestmark = pytest.mark.gpu


def gen(seed):
    return torch.Generator().manual_seed(seed)


def normal(shape, g, amp=1.0):
    return (amp * torch.randn(shape, generator=g)).to(torch.bfloat16)


# ---- quantising ------------------------------------------------------------------------------------
def same_codes(got, want):
    got = got.cpu().float().double()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got.nan_to_num(), want.nan_to_num())


def test_quantize_every_bf16_value(dev):
    """All bit patterns, one exponent a row of blocks, so that every magnitude meets its neighbours' scale, and mixed."""
    bits = torch.arange(65536, dtype=torch.int32).to(torch.uint16).view(torch.bfloat16)
    for x in (bits.view(512, 128), bits.view(128, 512), bits[torch.randperm(65536, generator=gen(0))].view(64, 1024)):
        codes, scales = ops.fp8_quantize(x.to(dev))
        want, s = u.quantize(x)
        assert torch.equal(scales.cpu().double(), s)
        same_codes(codes, want)


@pytest.mark.parametrize("m,k", [(1, 1), (1, 127), (3, 128), (5, 129), (2, 513), (77, 1000), (33, 1187), (4, 6144)])
def test_quantize_sizes(dev, m, k):
    x = normal((m, k), gen(m + k))
    x[:, ::7] *= 40
    codes, scales = ops.fp8_quantize(x.to(dev))
    want, s = u.quantize(x)
    assert torch.equal(scales.cpu().double(), s)
    same_codes(codes, want)


def test_quantize_strided_and_leading(dev):
    wide = normal((4, 6, 300), gen(1)).to(dev)
    for x in (wide[..., 5:290], wide[:, ::2, :256], wide.transpose(0, 1)):
        codes, scales = ops.fp8_quantize(x)
        want, s = u.quantize(x.cpu().reshape(-1, x.shape[-1]))
        assert codes.shape[:-1] == x.shape[:-1] and torch.equal(scales.cpu().double(), s)
        same_codes(codes.reshape(want.shape), want)


# ---- the product ---------------------------------------------------------------------------------------
def weight(n, k, g):
    """E4M3 codes [n, kp], zero beyond k, and any float32 scales."""
    w = torch.zeros((n, (k + 127) // 128 * 128))
    w[:, :k] = torch.randn((n, k), generator=g) * 60
    s = torch.rand(((n + 127) // 128, w.shape[1] // 128), generator=g) * 1e-3 + 1e-4
    return w.clamp(-448, 448).to(torch.float8_e4m3fn), s


@pytest.mark.parametrize("m,n,k,bias", [
    (1, 1, 1, False), (1, 64, 128, True), (1, 1000, 2048, True), (3, 130, 257, False), (8, 256, 1024, True),
    (9, 300, 640, True), (16, 128, 8448, False), (17, 129, 384, True), (64, 64, 128, False), (65, 200, 1187, True),
    (128, 384, 512, False), (200, 1001, 640, True), (333, 257, 1187, True), (700, 520, 256, False)])
def test_product(dev, m, n, k, bias):
    g = gen(m * 7 + n * 3 + k)
    x = normal((m, k), g)
    x[:, ::13] *= 20
    w, ws = weight(n, k, g)
    b = normal((n,), g) if bias else None
    a, sa = ops.fp8_quantize(x.to(dev))
    y = ops.fp8_gemm(a, sa, w.to(dev), ws.to(dev), None if b is None else b.to(dev))
    want, bound = u.product(a.cpu().float(), sa.cpu(), w.float(), ws, b)
    u.check(y, want, bound)
    assert torch.equal(ops.fp8_linear(x.to(dev), w.to(dev), ws.to(dev), None if b is None else b.to(dev)), y)


@pytest.mark.parametrize("m,n", [(2, 200), (16, 96), (40, 130), (130, 260), (1100, 4100), (4352, 4096)])
def test_product_of_small_whole_numbers_is_exact(dev, m, n):
    """Codes 0, 1, 2 and 3 and scales of 1 and 2: sums are whole numbers below 2^24, so only the store rounds.  The last sizes
    fill the card with the largest tiles, to the edges and past them."""
    k, g = 640, torch.Generator(device=dev).manual_seed(m)
    a, w = (torch.randint(-3, 4, (r, k), device=dev, generator=g).float() for r in (m, n))
    sa = torch.randint(1, 3, (k // 128, m), device=dev, generator=g).float()
    sw = torch.randint(1, 3, ((n + 127) // 128, k // 128), device=dev, generator=g).float()
    y = ops.fp8_gemm(a.to(torch.float8_e4m3fn), sa, w.to(torch.float8_e4m3fn), sw)
    ab = (a.view(m, -1, 128) * sa.T[..., None]).view(m, k).double()
    wb = (w.view(n, -1, 128) * sw.repeat_interleave(128, 0)[:n, :, None]).view(n, k).double()
    assert torch.equal(y, (ab @ wb.T).to(torch.bfloat16))


@pytest.mark.parametrize("m,n,k,bias", [(20, 130, 4096, True), (33, 1001, 2048, True), (77, 256, 6144, False), (17, 3, 16384, False)])
def test_product_in_pieces_of_k(dev, m, n, k, bias):
    """Few tiles: K is cut into pieces, whose sums are joined."""
    test_product(dev, m, n, k, bias)


@pytest.mark.parametrize("m", [1, 2, 3, 4, 5, 8, 9])
@pytest.mark.parametrize("n,k", [(1, 128), (100, 640), (1000, 6144)])
def test_linear_of_few_rows_is_the_product_of_the_quantized_ones(dev, m, n, k):
    """Bit for bit, whichever kernel encodes: rows on 16 bytes and off them, of all magnitudes, zeros, infinities and NaN."""
    g = gen(m + n)
    x = normal((m, k + 8), g) * torch.exp2(torch.randint(-130, 100, (m, k + 8), generator=g).float()).to(torch.bfloat16)
    x[m - 1, :130] = 0
    x[m // 2, 64] = math.inf
    x[0, k - 1] = math.nan
    w, ws = (t.to(dev) for t in weight(n, k, g))
    b = normal((n,), g).to(dev)
    for z in (x.to(dev)[:, :k], x.to(dev)[:, 3:3 + k], x.to(dev)[:, 8:].contiguous()):
        y = ops.fp8_linear(z, w, ws, b)
        want = ops.fp8_gemm(*ops.fp8_quantize(z), w, ws, b)
        assert torch.equal(torch.isnan(y), torch.isnan(want))
        assert torch.equal(y.nan_to_num(), want.nan_to_num())


def test_product_whose_output_passes_32_bits(dev):
    m, n = 140000, 16384   # one block of K: a value is one product, whatever the tile
    g = torch.Generator(device=dev).manual_seed(0)
    a, w = (torch.randint(-3, 4, (r, 128), device=dev, generator=g).float().to(torch.float8_e4m3fn) for r in (m, n))
    sa, sw = torch.rand(1, m, device=dev, generator=g), torch.rand(n // 128, 1, device=dev, generator=g)
    y = ops.fp8_gemm(a, sa, w, sw)
    for at in (0, 131071, m - 300):
        assert torch.equal(y[at:at + 300], ops.fp8_gemm(a[at:at + 300], sa[:, at:at + 300].contiguous(), w, sw))


def test_product_of_more_rows_than_a_grid_has_in_y(dev):
    m, n = 2200000, 20   # one block of K, as above
    g = torch.Generator(device=dev).manual_seed(1)
    a, w = (torch.randint(-3, 4, (r, 128), device=dev, generator=g).float().to(torch.float8_e4m3fn) for r in (m, n))
    sa, sw = torch.rand(1, m, device=dev, generator=g), torch.rand(1, 1, device=dev, generator=g)
    y = ops.fp8_gemm(a, sa, w, sw)
    for at in (0, 2097100, m - 300):
        assert torch.equal(y[at:at + 300], ops.fp8_gemm(a[at:at + 300], sa[:, at:at + 300].contiguous(), w, sw))


def test_product_passes_nan_and_zero_scales(dev):
    x = normal((5, 256), gen(3))
    x[1, 40], x[2, 200] = math.nan, math.inf
    w, ws = weight(130, 256, gen(4))
    ws[1, 1] = 0.0
    y = ops.fp8_linear(x.to(dev), w.to(dev), ws.to(dev)).cpu()
    assert torch.isnan(y[1:3]).all() and torch.isfinite(y[[0, 3, 4]]).all()


def test_product_of_no_rows(dev):
    w, ws = weight(130, 256, gen(4))
    assert ops.fp8_linear(torch.zeros((0, 256), dtype=torch.bfloat16, device=dev), w.to(dev), ws.to(dev)).shape == (0, 130)


# ---- norms of heads, and rotation ---------------------------------------------------------------------------
@pytest.mark.parametrize("d", [16, 32, 48, 64, 96, 128, 192, 256])
@pytest.mark.parametrize("pairs", [False, True])
@pytest.mark.parametrize("wide", [False, True])
def test_qk_norm_rope(dev, d, pairs, wide):
    g = gen(d + pairs)
    t, h, kv = 37, 6, 2
    x = normal((t, h + 2 * kv, d), g, 3.0)
    x[:, 0] *= 1e-4
    x[5, 1] = 0
    q, k = x.to(dev)[:, :h], x.to(dev)[:, h:h + kv]
    qw, kw = normal((d,), g) + 1, normal((d,), g)
    ang = torch.rand((50, d // 2 + 3), generator=g) * 6.3
    cos, sin = (f(ang).to(torch.float32 if wide else torch.bfloat16) for f in (torch.cos, torch.sin))
    at = torch.randint(0, 50, (t,), generator=g)
    for weights, pos in (((qw, kw), at), ((qw, None), at.int()), ((None, None), None)):
        got = ops.qk_norm_rope(q, k, *(None if w is None else w.to(dev) for w in weights), cos.to(dev), sin.to(dev), 1e-6,
                               None if pos is None else pos.to(dev), pairs)
        for y, z, w in zip(got, (q, k), weights):
            u.check(y, *u.qk(z.cpu(), w, cos, sin, 1e-6, pos, pairs))


@pytest.mark.parametrize("d", [16, 64, 256])
@pytest.mark.parametrize("eps", [0.0, 1e-6, 0.5])
def test_qk_norm_rope_of_any_magnitude(dev, d, eps):
    """Heads whose squares pass the ends of float32 beside ordinary ones."""
    g = gen(d)
    q, k = normal((12, 5, d), g), normal((12, 1, d), g)
    for i, amp in enumerate((1e38, 1e25, 1e19, 1e-15, 1e-25, 1e-36)):
        q[2 * i + 1, :3] = (torch.rand((3, d), generator=g) * 2 - 1).mul(amp).to(torch.bfloat16)
    tab = torch.randn((12, d // 2), generator=g)
    for y, z in zip(ops.qk_norm_rope(q.to(dev), k.to(dev), None, None, tab.to(dev), tab.to(dev), eps), (q, k)):
        u.check(y, *u.qk(z, None, tab, tab, eps, None, False))


def test_qk_norm_rope_positions_that_are_not_there(dev):
    q, k = normal((4, 2, 64), gen(0)).to(dev), normal((4, 1, 64), gen(1)).to(dev)
    tab = torch.rand(10, 32, device=dev)
    qo, ko = ops.qk_norm_rope(q, k, None, None, tab, tab, 1e-6, torch.tensor([0, 10, -1, 9], device=dev))
    for y in (qo, ko):
        assert torch.isnan(y[1:3]).all() and torch.isfinite(y[[0, 3]]).all()


# ---- the cache -------------------------------------------------------------------------------------------------
class Cache:
    """A cache on both sides: device tensors and the oracle's float64 copy."""

    def __init__(self, dev, seqs, kv, d, seed, *, stale=False, width=0):
        """seqs: (new tokens, tokens held) of each sequence; pages in any order, -1 behind the last."""
        g = gen(seed)
        need = [-(-held // u.PAGE) for _, held in seqs]
        order = torch.randperm(sum(need) + 3, generator=g).tolist()
        w = max(max(need), 1) + width
        self.table, at = [], 0
        for n in need:
            self.table.append(order[at:at + n] + [-1] * (w - n))
            at += n
        self.k, self.v, self.s = u.pages(len(order), kv, d, g, stale=stale)
        self.seqs, self.kv, self.d, self.g = seqs, kv, d, g
        self.offsets = [0]
        for n, _ in seqs:
            self.offsets.append(self.offsets[-1] + n)
        self.dev = dev

    def lengths(self, before=False):
        return [held - (n if before else 0) for n, held in self.seqs]

    def device(self, before=False):
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=self.dev)   # noqa: E731
        return (i32(self.offsets), i32(self.lengths(before)), i32(self.table), self.k.to(self.dev), self.v.to(self.dev),
                self.s.to(self.dev))

    def oracle(self):
        return self.k.float().double(), self.v.float().double(), self.s.double()


SEQS = {
    "one": [(1, 1)],
    "page": [(64, 64)],
    "edges": [(1, 64), (1, 65), (63, 63), (64, 100), (65, 129), (2, 66)],
    "empty": [(0, 0), (0, 70), (5, 5), (0, 0), (3, 200), (0, 1)],
    "prompts": [(150, 150), (7, 300), (129, 333)],
}


@pytest.mark.parametrize("name", SEQS)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("kv", [1, 3])
def test_append(dev, name, d, kv):
    c = Cache(dev, SEQS[name], kv, d, len(name) + d, width=1)
    c.s = torch.exp2(torch.randint(-9, 3, c.s.shape, generator=c.g).float())
    rows = c.offsets[-1]
    k, v = normal((rows, kv, d), c.g), normal((rows, 2 * kv, d), c.g, 300.0)[:, ::2][:, :kv]
    k[:, :, 5] *= 1000
    if rows > 2:
        k[1, 0, 3], v[2, 0, 1], v[0, 0, 2] = math.nan, math.inf, -math.inf
    want = c.oracle()
    u.append(k, v, c.offsets, c.lengths(True), c.table, *want)
    args = c.device(before=True)
    for _ in range(2):   # the second call finds the scales that the first one left, and changes nothing
        ops.kv8_append(k.to(dev), v.to(dev), *args)
        same_codes(args[3], want[0])
        same_codes(args[4], want[1])
        assert torch.equal(args[5].cpu().double(), want[2])


def test_append_drops_what_has_no_page(dev):
    c = Cache(dev, [(10, 64), (70, 100)], 2, 64, 0)
    c.table = [[-1, 0], [c.table[1][0], 9999]]
    rows = c.offsets[-1]
    k = normal((rows, 2, 64), c.g)
    args = c.device(before=True)
    lengths = torch.tensor([54, 60], dtype=torch.int32, device=dev)   # the second one runs past its table
    want = c.oracle()
    u.append(k, k, c.offsets, [54, 60], c.table, *want)
    ops.kv8_append(k.to(dev), k.to(dev), args[0], lengths, *args[2:])
    same_codes(args[3], want[0])
    same_codes(args[4], want[1])
    assert torch.equal(args[5].cpu(), want[2].float())


def attend(c, heads, causal, scale=None, q=None):
    q = normal((c.offsets[-1], heads, c.d), c.g) if q is None else q
    scale = c.d ** -0.5 if scale is None else scale
    got = ops.kv8_attention(q.to(c.dev), *c.device(), scale, causal)
    want, bound = u.attention(q, c.offsets, c.lengths(), c.table, *c.oracle(), scale, causal)
    u.check(got, want, bound)
    return got


@pytest.mark.parametrize("n", [3, 130])
def test_offsets_that_do_not_ascend_stay_in_range(dev, n):
    """What such a batch means is not defined; nothing is read or written out of range, and other sequences' pages stay."""
    c = Cache(dev, [(n, 200), (n, 200), (n, 200)], 2, 64, 70)
    args = c.device(before=True)
    q, x = normal((3 * n, 8, 64), c.g).to(dev), normal((3 * n, 2, 64), c.g).to(dev)
    before = args[3].view(torch.uint8).clone()
    free = [p for p in range(len(before)) if not any(p in row for row in c.table)]
    for offsets in ([0, 2 * n, n, 3 * n], [3 * n, 2 * n, n, 0], [-5, 10 ** 9, -7, 2 ** 31 - 1], [n, n, n, n]):
        args = (torch.tensor(offsets, dtype=torch.int32, device=dev), *args[1:])
        ops.kv8_append(x, x, *args)
        ops.kv8_attention(q, *args, 0.125)
        torch.cuda.synchronize()
    assert torch.equal(args[3].view(torch.uint8)[free], before[free])


def attend_gpu(c, heads, causal):
    q = normal((c.offsets[-1], heads, c.d), c.g)
    return ops.kv8_attention(q.to(c.dev), *c.device(), c.d ** -0.5, causal)


@pytest.mark.parametrize("name", SEQS)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("heads,kv", [(1, 1), (6, 2), (12, 3), (40, 2)])
@pytest.mark.parametrize("causal", [True, False])
def test_attention(dev, name, d, heads, kv, causal):
    """Slots behind a sequence's tokens, and pages of nobody, hold codes that are not numbers."""
    c = Cache(dev, SEQS[name], kv, d, len(name) + heads, stale=True, width=2)
    own = torch.zeros(c.k.shape[0], u.PAGE, dtype=torch.bool)
    for row, (_, held) in zip(c.table, c.seqs):
        for i in range(held):
            own[row[i // u.PAGE], i % u.PAGE] = True
    for t, m in ((c.k, own[:, None, :, None]), (c.v, own[:, None, None, :])):
        b = t.view(torch.uint8)
        b[m.expand(b.shape) & ((b & 127) == 127)] = 17
    attend(c, heads, causal)


@pytest.mark.parametrize("n", [1, 3, 40, 200])
@pytest.mark.parametrize("d", [64, 128])
def test_attention_long(dev, n, d):
    """Long sequences, which are cut along the keys and joined."""
    attend(Cache(dev, [(n, 9000 + n)], 1, d, n), 4, True)
    attend(Cache(dev, [(n, 5000), (n, 9001), (n, n)], 2, d, n), 4, n != 3)


@pytest.mark.parametrize("n", [2, 70])
def test_attention_nan_reaches_only_rows_that_see_it(dev, n):
    c = Cache(dev, [(n, 150)], 1, 64, 5)
    k, v = c.k.view(torch.uint8), c.v.view(torch.uint8)
    k[c.table[0][2], 0, 20, 7] = 255      # token 148
    v[c.table[0][2], 0, 9, 21] = 127      # token 149, one channel
    if n > 2:
        v[c.table[0][1], 0, 40, 30] = 127     # token 94
    attend(c, 4, True)


def test_attention_nothing_visible(dev):
    """More new tokens than the sequence holds: the first ones see nothing; rows behind the last sequence neither."""
    c = Cache(dev, [(10, 4), (3, 0), (90, 20)], 2, 64, 6, width=1)
    got = attend(c, 4, True)
    assert not got[:6].any() and not got[10:13].any()
    args = c.device()
    got = ops.kv8_attention(normal((200, 4, 64), c.g).to(dev), *args, 0.125, False)
    assert not got[103:].any() and got[:10].any()


@pytest.mark.parametrize("seqs", [[(300, 0), (200, 4)], [(500, 0)], [(0, 70), (300, 0), (100, 64), (60, 70)]])
@pytest.mark.parametrize("causal", [True, False])
def test_attention_nothing_visible_in_pieces(dev, seqs, causal):
    """Many rows over a wide table of which little or nothing is held."""
    c = Cache(dev, seqs, 1, 64, 71, width=60)
    got = attend(c, 8, causal)
    if all(held == 0 for _, held in seqs):
        assert not got.any()


def test_attention_pages_and_lengths_out_of_range(dev):
    c = Cache(dev, [(5, 200), (1, 130)], 2, 64, 7)
    c.table[0][1], c.table[1][2] = 10 ** 6, -7
    attend(c, 4, True)
    c.seqs = [(5, 10 ** 6), (1, 130)]     # beyond the table: as much as it names
    q = normal((6, 4, 64), c.g)
    got = ops.kv8_attention(q.to(dev), *c.device(), 0.125, False)
    c.seqs = [(5, len(c.table[0]) * u.PAGE), (1, 130)]
    assert torch.equal(got, ops.kv8_attention(q.to(dev), *c.device(), 0.125, False))


@pytest.mark.parametrize("amp", [0.0, 30.0, -3.0])
def test_attention_scales(dev, amp):
    """A scale of 0 (the mean), a sharp one and a negative one."""
    attend(Cache(dev, [(3, 200), (80, 90)], 1, 128, 8), 4, True, scale=amp / 128)


def test_attention_queries_sliced_from_a_projection(dev):
    c = Cache(dev, [(30, 100)], 2, 64, 9)
    wide = normal((30, 12, 64), c.g)
    assert torch.equal(attend(c, 8, True, q=wide[:, 2:10]), attend(c, 8, True, q=wide[:, 2:10].contiguous()))


def shared(dev, n, held, heads, kv, d, count, seed):
    """`count` sequences of the same tokens that read the same pages: one of them against the definition, all alike."""
    c = Cache(dev, [(n, held)], kv, d, seed)
    q = normal((n, heads, d), c.g)
    want, bound = u.attention(q, c.offsets, c.lengths(), c.table, *c.oracle(), d ** -0.5, True)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)   # noqa: E731
    _, _, _, k, v, s = c.device()
    got = ops.kv8_attention(q.to(dev).repeat(count, 1, 1), i32([n * b for b in range(count + 1)]), i32([held] * count),
                            i32(c.table * count), k, v, s, d ** -0.5)
    u.check(got, want.repeat(count, 1, 1), bound.repeat(count, 1, 1))


@pytest.mark.parametrize("n,heads,count", [(1, 1, 129), (9, 32, 100)])
def test_attention_of_many_sequences_over_more_pages_than_a_look_up(dev, n, heads, count):
    """More sequences than lanes, and each piece longer than the 64 pages that are looked up at a time."""
    shared(dev, n, 17000, heads, 1, 64, count, 20)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("seqs", [[(300, 5000), (100, 640), (0, 300), (129, 2100), (200, 900)], [(400, 400), (330, 4700)]])
def test_attention_of_a_ragged_batch(dev, seqs, d, causal):
    """Long sequences in pieces about as long as the short ones; the last rows of each against the definition."""
    c = Cache(dev, seqs, 8, d, 23)
    q = normal((c.offsets[-1], 64, d), c.g)
    got = ops.kv8_attention(q.to(dev), *c.device(), d ** -0.5, causal).cpu()
    assert torch.isfinite(got).all()
    last = [min(n, 5) for n, _ in seqs]
    rows = torch.cat([torch.arange(end - n, end) for n, end in zip(last, c.offsets[1:])])
    offsets = [0, *torch.tensor(last).cumsum(0).tolist()]
    u.check(got[rows], *u.attention(q[rows], offsets, c.lengths(), c.table, *c.oracle(), d ** -0.5, causal))


@pytest.mark.parametrize("n", [1, 100])
def test_many_sequences(dev, n):
    """64 and more sequences, some empty; few rows and many."""
    seqs = [(0, 3) if b % 7 == 3 else (n + b % 3, n + 3 * b) for b in range(75)]
    attend(Cache(dev, seqs, 2, 64, 21, stale=False), 8, True)
    c = Cache(dev, seqs, 2, 64, 22)
    k, v = normal((c.offsets[-1], 2, 64), c.g), normal((c.offsets[-1], 2, 64), c.g)
    c.s = torch.exp2(torch.randint(-9, 3, c.s.shape, generator=c.g).float())
    want = c.oracle()
    u.append(k, v, c.offsets, c.lengths(True), c.table, *want)
    args = c.device(before=True)
    ops.kv8_append(k.to(dev), v.to(dev), *args)
    same_codes(args[3], want[0])
    same_codes(args[4], want[1])
    assert torch.equal(args[5].cpu().double(), want[2])


@pytest.mark.parametrize("n", [3, 130])
@pytest.mark.parametrize("d", [64, 128])
def test_attention_page_scales_of_any_kind(dev, n, d):
    """Negative, zero, far from 1, and not a number in a page that only the last tokens see."""
    c = Cache(dev, [(n, 700)], 2, d, 30)
    t = c.table[0]
    c.s[t[0], 0, 0], c.s[t[1], 1, 0] = 0.0, -0.003
    c.s[t[2], 0, 1], c.s[t[3], 1, 1], c.s[t[4], 0, 1], c.s[t[5], 1, 1] = 0.0, -0.01, 2.0 ** -100, 2.0 ** 100
    attend(c, 8, True)
    c.s[t[10], 0, 0], c.s[t[10], 1, 1] = math.nan, math.nan   # tokens 640 ..
    attend(c, 8, True)
    c.s[t[10]] = 0.01
    c.s[t[3], 1, 1], c.s[t[10], 1, 0] = math.inf, -math.inf   # head 1: NaN throughout
    c.s[t[10], 0, 1] = math.nan
    got = attend_gpu(c, 8, True)
    assert torch.isnan(got[:, 4:]).all()
    seen = max(0, n - 60)   # rows that see token 640
    assert torch.isnan(got[n - min(n, 60):, :4]).all() and torch.isfinite(got[:seen, :4]).all()


@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("n", [12, 130])
def test_attention_scale_that_is_no_number_reaches_only_rows_that_see_it(dev, n, bad, which):
    c = Cache(dev, [(n, 136)], 1, 64, 33)   # the last page: tokens 128 to 135, seen by the last 8 rows
    c.s[c.table[0][2], 0, which] = bad
    got = attend_gpu(c, 4, True).cpu()
    assert torch.isnan(got[n - 8:]).all() and torch.isfinite(got[:n - 8]).all()
    c.s[c.table[0][2], 0, which] = math.nan   # as the definition has it
    attend(c, 4, True)


@pytest.mark.parametrize("n", [3, 130])
@pytest.mark.parametrize("d", [64, 128])
def test_attention_scores_far_apart_and_a_missing_first_page(dev, n, d):
    """Scores whose exponents are hundreds apart, in any order; then without the first page, or the first four."""
    c = Cache(dev, [(n, 700)], 2, d, 31)
    attend(c, 8, True, scale=4.0)
    c.table[0][0] = -1
    attend(c, 8, True, scale=4.0)
    attend(c, 8, False)
    c.table[0][:4] = [-1, 10 ** 6, -5, -1]
    attend(c, 8, True)
    c.table[0][:] = [-1] * len(c.table[0])
    assert not attend(c, 8, True).any()


@pytest.mark.parametrize("n", [1, 130])
def test_attention_of_infinite_queries_stays_in_its_rows(dev, n):
    c = Cache(dev, [(n, 300)], 1, 64, 32)
    q = normal((n, 4, 64), c.g)
    want = ops.kv8_attention(q.to(dev), *c.device(), 0.125)
    q[0, 1, 5], q[n - 1, 2, 0] = math.inf, math.nan
    got = ops.kv8_attention(q.to(dev), *c.device(), 0.125)
    hit = torch.zeros(n, 4, dtype=torch.bool)
    hit[0, 1] = hit[n - 1, 2] = True
    # a matrix tile of which some row is not finite may be summed in another order
    assert torch.isnan(got.cpu()[hit]).all() and torch.isfinite(got.cpu()[~hit]).all()
    wanted, bound = u.attention(q[:, [0, 3]], c.offsets, c.lengths(), c.table, *c.oracle(), 0.125, True)
    u.check(got[:, [0, 3]], wanted, bound)
    assert torch.isfinite(want).all()


@pytest.mark.parametrize("n", [1, 80])
def test_cache_that_passes_32_bits(dev, n):
    """Pages at the end of a cache of more than 2^32 codes: as those of a small one."""
    c = Cache(dev, [(n, 400)], 4, 128, 40)
    count, kv, d = 140000, 4, 128
    used = torch.tensor(c.table[0], device=dev)
    cu, before, table, k, v, s = c.device(before=True)
    big_k = torch.empty((count, kv, u.PAGE, d), dtype=torch.float8_e4m3fn, device=dev)
    big_v = torch.empty((count, kv, d, u.PAGE), dtype=torch.float8_e4m3fn, device=dev)
    big_s = torch.zeros((count, kv, 2), device=dev)
    far = count - 1 - 2 * torch.arange(len(used), device=dev)
    for big, small in ((big_k.view(torch.uint8), k.view(torch.uint8)), (big_v.view(torch.uint8), v.view(torch.uint8)), (big_s, s)):
        for i, j in zip(far.tolist(), used.tolist()):
            big[i] = small[j]
    x = normal((n, 2 * kv, d), c.g).to(dev)
    q = normal((n, 8, d), c.g).to(dev)
    outs = []
    for tab, cache in ((table, (k, v, s)), (far.int()[None], (big_k, big_v, big_s))):
        ops.kv8_append(x[:, :kv], x[:, kv:], cu, before, tab, *cache)
        outs.append(ops.kv8_attention(q, cu, before + n, tab, *cache, d ** -0.5))
    assert torch.equal(*outs) and outs[0].any()
    for i, j in zip(far.tolist(), used.tolist()):
        assert torch.equal(big_k[i].view(torch.uint8), k[j].view(torch.uint8)) and torch.equal(big_s[i], s[j])
        assert torch.equal(big_v[i].view(torch.uint8), v[j].view(torch.uint8))


def test_strides_that_pass_32_bits(dev):
    """Two tokens 2^31 + 64 values apart."""
    far = torch.zeros(2 ** 31 + 4096, dtype=torch.bfloat16, device=dev)
    x = far.as_strided((2, 4, 64), (2 ** 31 + 64, 64, 1))
    dense = normal((2, 4, 64), gen(41)).to(dev)
    x.copy_(dense)
    rows, drows = x.as_strided((2, 256), (2 ** 31 + 64, 1)), dense.view(2, 256)
    for a, b in zip(ops.fp8_quantize(rows), ops.fp8_quantize(drows)):
        assert torch.equal(a.float(), b.float())
    w, ws = (t.to(dev) for t in weight(130, 256, gen(42)))
    assert torch.equal(ops.fp8_linear(rows, w, ws), ops.fp8_linear(drows, w, ws))
    tab = torch.rand(2, 32, device=dev)
    for a, b in zip(ops.qk_norm_rope(x[:, :2], x[:, 2:], None, None, tab, tab, 1e-6),
                    ops.qk_norm_rope(dense[:, :2], dense[:, 2:], None, None, tab, tab, 1e-6)):
        assert torch.equal(a, b)
    c = Cache(dev, [(2, 30)], 2, 64, 43)
    outs = []
    for t in (x, dense):
        args = c.device(before=True)
        ops.kv8_append(t[:, :2], t[:, 2:], *args)
        outs.append((args[3].float(), args[4].float(), args[5], ops.kv8_attention(t, args[0], args[1] + 2, *args[2:], 0.125)))
    for a, b in zip(*outs):
        assert torch.equal(a, b)


def test_calls_on_two_streams_at_once(dev):
    """Split along the keys and along K, so that each call has partial results of its own."""
    c = Cache(dev, [(1, 9000)], 2, 64, 44)
    args = c.device()
    q = [normal((1, 8, 64), c.g).to(dev) for _ in range(2)]
    w, ws = (t.to(dev) for t in weight(256, 6144, gen(45)))
    x = [normal((40, 6144), c.g).to(dev) for _ in range(2)]
    want = [(ops.kv8_attention(a, *args, 0.125), ops.fp8_linear(b, w, ws)) for a, b in zip(q, x)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append((ops.kv8_attention(q[i], *args, 0.125), ops.fp8_linear(x[i], w, ws)))
    torch.cuda.synchronize()
    for i in range(2):
        for o, y in got[i]:
            assert torch.equal(o, want[i][0]) and torch.equal(y, want[i][1])


def test_graph_of_split_calls_replayed(dev):
    c = Cache(dev, [(1, 9000), (1, 400)], 2, 64, 46)
    args = c.device()
    q = normal((2, 8, 64), c.g).to(dev)
    w, ws = (t.to(dev) for t in weight(256, 6144, gen(47)))
    x = normal((40, 6144), c.g).to(dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.kv8_attention(q, *args, 0.125), ops.fp8_linear(x, w, ws)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, y = ops.kv8_attention(q, *args, 0.125), ops.fp8_linear(x, w, ws)
    for i in range(5):
        q.copy_(normal(q.shape, c.g))
        x.copy_(normal(x.shape, c.g))
        args[1].copy_(torch.tensor([9000 - 700 * i, 1 + 90 * i]))
        want = ops.kv8_attention(q, *args, 0.125), ops.fp8_linear(x, w, ws)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, want[0]) and torch.equal(y, want[1])


def test_nothing_to_do(dev):
    c = Cache(dev, [(0, 5), (0, 0)], 2, 64, 48)
    args = c.device()
    none = torch.zeros((0, 2, 64), dtype=torch.bfloat16, device=dev)
    assert ops.kv8_attention(none, *args, 0.125).shape == (0, 2, 64)
    before = [t.float().clone() for t in args[3:]]
    ops.kv8_append(none, none, *args)
    assert all(torch.equal(a.float().nan_to_num(), b.nan_to_num()) for a, b in zip(args[3:], before))
    tab = torch.zeros(1, 32, device=dev)
    assert [t.shape for t in ops.qk_norm_rope(none, none, None, None, tab, tab, 1e-6)] == [(0, 2, 64)] * 2


# ---- together ------------------------------------------------------------------------------------------------------
def test_a_layer_step_by_step(dev):
    """Projection, norms and rotation, cache and attention over a prompt and five single tokens, eager and as one captured
    graph that is replayed with new inputs: the graph's results are the eager ones."""
    g = gen(11)
    hidden, h, kv, d = 512, 8, 2, 64
    w, ws = weight((h + 2 * kv) * d, hidden, g)
    wo, wos = weight(hidden, h * d, g)
    w, ws, wo, wos = (t.to(dev) for t in (w, ws, wo, wos))
    qw, kw = (normal((d,), g, 0.1) + 1).to(dev), (normal((d,), g, 0.1) + 1).to(dev)
    ang = torch.arange(400)[:, None] * 10000.0 ** (-torch.arange(0, d, 2) / d)
    cos, sin = torch.cos(ang).to(dev), torch.sin(ang).to(dev)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)   # noqa: E731

    def layer(x, cu, before, table, pages, at):
        y = ops.fp8_linear(x, w, ws).view(len(x), -1, d)
        q, k = ops.qk_norm_rope(y[:, :h], y[:, h:h + kv], qw, kw, cos, sin, 1e-6, at)
        ops.kv8_append(k, y[:, h + kv:], cu, before, table, *pages)
        new = (cu[1:] - cu[:-1]).int()
        o = ops.kv8_attention(q, cu, before + new, table, *pages, d ** -0.5)
        return ops.fp8_linear(o.view(len(x), -1), wo, wos)

    def pages():
        return [t.to(dev) for t in u.pages(8, kv, d, gen(12))]

    table = i32([[3, 0, 5, -1], [7, 1, 2, 4]])
    prompt, tokens = normal((170, hidden), g).to(dev), normal((5, 2, hidden), g).to(dev)
    lens = [70, 100]

    def run(step):
        held, cache = list(lens), pages()
        out = [layer(prompt, i32([0, 70, 170]), i32([0, 0]), table, cache, torch.cat([torch.arange(n) for n in lens]).to(dev))]
        for x in tokens:
            out.append(step(x, held, cache).clone())
            held = [n + 1 for n in held]
        return out, cache

    eager, cache_a = run(lambda x, held, cache: layer(x, i32([0, 1, 2]), i32(held), table, cache, torch.tensor(held, device=dev)))
    assert all(torch.isfinite(t).all() for t in eager)

    buf, before, at, graph = tokens[0].clone(), i32(lens), torch.tensor(lens, device=dev), None
    cu, static = i32([0, 1, 2]), {}

    def replayed(x, held, cache):
        if "graph" not in static:
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                layer(buf, cu, before, table, pages(), at)
            torch.cuda.current_stream().wait_stream(side)
            static["graph"] = torch.cuda.CUDAGraph()
            with torch.cuda.graph(static["graph"]):
                static["y"] = layer(buf, cu, before, table, cache, at)
        buf.copy_(x)
        before.copy_(i32(held))
        at.copy_(torch.tensor(held))
        torch.cuda.synchronize()
        static["graph"].replay()
        return static["y"]

    again, cache_b = run(replayed)
    for a, b in zip(eager, again):
        assert torch.equal(a, b)
    for a, b in zip(cache_a, cache_b):
        assert torch.equal(a.view(torch.uint8) if a.element_size() == 1 else a, b.view(torch.uint8) if b.element_size() == 1 else b)


# ---- modules -----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("m", [1, 5, 40])
def test_module(dev, m):
    from krea2_svdquant_amd import FP8Linear
    from krea2_svdquant_amd.quant.fp8 import quantize_fp8
    g = gen(50 + m)
    dense, bias = normal((200, 300), g, 0.05), normal((200,), g)
    layer = FP8Linear.from_dense(dense.to(dev), bias.to(dev))
    x = normal((2, m, 300), g).to(dev)
    y = layer(x)
    codes, scales = quantize_fp8(dense)
    assert torch.equal(layer.weight_codes.cpu(), codes.view(torch.uint8)) and torch.equal(layer.weight_scales.cpu(), scales)
    assert y.shape == (2, m, 200) and torch.equal(y, ops.fp8_linear(x, codes.to(dev), scales.to(dev), bias.to(dev)))
    assert torch.equal(y, layer.forward_fp8(*layer.quantize(x)))
    a, sa = ops.fp8_quantize(x)
    want, bound = u.product(a.cpu().float().view(2 * m, -1), sa.cpu(), codes.float(), scales, bias)
    u.check(y.view(2 * m, -1), want, bound)
    moved = FP8Linear.from_dense(torch.zeros(200, 300), torch.zeros(200))
    moved.load_state_dict(layer.cpu().state_dict())
    assert torch.equal(moved.to(dev, torch.bfloat16)(x), y)


def test_block_on_fp8_layers(dev):
    from krea2_svdquant_amd.runtime import krea2_standin as ks
    dims = ks.Krea2Dims(layers=2, hidden=256, heads=2, kv_heads=1, head_dim=128, mlp=520)
    model = ks.Krea2StandInTransformer.random(dims, linears="fp8", device=dev, seed=5)
    x = normal((70, 256), gen(60)).to(dev)
    y = model(x)
    assert torch.isfinite(y).all() and y.shape == x.shape
    # each layer called by itself: the quantised activation that they share changes nothing
    calls = []
    assert torch.equal(model(x, linear=lambda name, mod, z: calls.append(name) or mod(z)), y) and len(calls) == 16
    assert torch.equal(model(x, siblings=True), y)
    layer = model.transformer_blocks[0].attn.to_k
    seen = []
    hook = layer.register_forward_hook(lambda mod, args, out: seen.append(out))
    assert torch.equal(model(x), y) and len(seen) == 1
    hook.remove()
    with pytest.raises(NotImplementedError, match="FP8Linear"):
        model(x, fused=True)


def test_block_on_fp8_layers_captured(dev):
    from krea2_svdquant_amd.runtime import krea2_standin as ks
    dims = ks.Krea2Dims(layers=1, hidden=256, heads=2, kv_heads=1, head_dim=128, mlp=520)
    model = ks.Krea2StandInTransformer.random(dims, linears="fp8", device=dev, seed=6)
    x = normal((33, 256), gen(61)).to(dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        model(x)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = model(x)
    for i in range(3):
        x.copy_(normal(x.shape, gen(62 + i)))
        want = model(x)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)


# ---- refusals -----------------------------------------------------------------------------------------------------------
def test_refusals_of_the_linear(dev):
    x = normal((4, 256), gen(0)).to(dev)
    w, ws = (t.to(dev) for t in weight(130, 256, gen(1)))
    a, sa = ops.fp8_quantize(x)
    with pytest.raises(TypeError):
        ops.fp8_quantize(x.float())
    for kind, call in ((TypeError, lambda: ops.fp8_linear(x.half(), w, ws)), (TypeError, lambda: ops.fp8_linear(x, w.view(torch.uint8), ws)),
                       (TypeError, lambda: ops.fp8_linear(x, w, ws.half())), (ValueError, lambda: ops.fp8_linear(x[:, :100], w, ws)),
                       (ValueError, lambda: ops.fp8_linear(x, w, ws[:1])), (ValueError, lambda: ops.fp8_linear(x, w, ws, x[0, :129])),
                       (TypeError, lambda: ops.fp8_linear(x, w, ws, torch.zeros(130, device=dev))),
                       (ValueError, lambda: ops.fp8_linear(x, w, ws.cpu())), (ValueError, lambda: ops.fp8_linear(x, w[:, :128], ws)),
                       (ValueError, lambda: ops.fp8_gemm(a, sa[:1], w, ws)), (TypeError, lambda: ops.fp8_gemm(a, sa.half(), w, ws)),
                       (ValueError, lambda: ops.fp8_gemm(a[:, :100].contiguous(), sa, w, ws)),
                       (TypeError, lambda: ops.fp8_gemm(x, sa, w, ws))):
        with pytest.raises(kind):
            call()


def test_refusals_of_the_norms(dev):
    q, k = normal((4, 2, 64), gen(0)).to(dev), normal((4, 1, 64), gen(1)).to(dev)
    tab = torch.rand(4, 32, device=dev)
    i = torch.arange(4, device=dev)
    for kind, args in ((TypeError, (q.half(), k, None, None, tab, tab, 1e-6)), (ValueError, (q, k[:3], None, None, tab, tab, 1e-6)),
                       (ValueError, (q[0], k, None, None, tab, tab, 1e-6)), (ValueError, (q, k, q[0, 0, :60], None, tab, tab, 1e-6)),
                       (TypeError, (q, k, None, None, tab, tab.bfloat16(), 1e-6)), (ValueError, (q, k, None, None, tab[:3], tab[:3], 1e-6)),
                       (ValueError, (q, k, None, None, tab[:, :31], tab[:, :31], 1e-6)), (ValueError, (q, k, None, None, tab, tab[:3], 1e-6)),
                       (ValueError, (q, k, None, None, tab, tab, 1e-6, i[:3])), (TypeError, (q, k, None, None, tab, tab, 1e-6, i.float())),
                       (ValueError, (q, k, None, None, tab, tab, 1e-6, i.cpu())), (ValueError, (q[..., :60], k[..., :60], None, None, tab, tab, 1e-6))):
        with pytest.raises(kind):
            ops.qk_norm_rope(*args)
    with pytest.raises(Exception, match="eps"):
        ops.qk_norm_rope(q, k, None, None, tab, tab, -1.0)


def test_refusals_of_the_cache(dev):
    c = Cache(dev, [(3, 100)], 2, 64, 0)
    good = c.device()
    x, q = normal((3, 2, 64), c.g).to(dev), normal((3, 4, 64), c.g).to(dev)
    before = good[3].float().clone()
    names = ("cu_seqlens", "lengths", "block_table", "k_codes", "v_codes", "scales")
    bad = [(TypeError, 0, good[0].long()), (ValueError, 0, good[0][:1]), (TypeError, 1, good[1].float()), (ValueError, 1, good[1].cpu()),
           (ValueError, 2, good[2][0]), (ValueError, 2, good[2][:0]), (TypeError, 3, good[3].view(torch.uint8)),
           (ValueError, 3, good[3][..., :32].contiguous()), (ValueError, 3, good[3].transpose(0, 1)), (ValueError, 4, good[4][:1]),
           (TypeError, 5, good[5].half()), (ValueError, 5, good[5][..., 0])]
    for kind, at, t in bad:
        args = [*good[:at], t, *good[at + 1:]]
        for call in (lambda: ops.kv8_append(x, x, *args), lambda: ops.kv8_attention(q, *args, 0.125)):
            with pytest.raises(kind):
                call()
                raise AssertionError(names[at])
    for kind, k, v in ((ValueError, x, x[:2]), (ValueError, x[:, :1], x[:, :1]), (TypeError, x.float(), x.float()),
                       (ValueError, x.cpu(), x), (ValueError, x[..., :32], x[..., :32])):
        with pytest.raises(kind):
            ops.kv8_append(k, v, *good)
    with pytest.raises(RuntimeError, match="gradient"):
        ops.kv8_append(x.clone().requires_grad_(), x, *good)
    for kind, z in ((ValueError, q[:, :3]), (TypeError, q.float()), (ValueError, q[0])):
        with pytest.raises(kind):
            ops.kv8_attention(z, *good, 0.125)
    assert torch.equal(good[3].float().nan_to_num(), before.nan_to_num())


def test_append_marks_the_cache_as_changed(dev):
    c = Cache(dev, [(3, 100)], 2, 64, 0)
    args = c.device(before=True)
    versions = [t._version for t in args[3:]]
    ops.kv8_append(*(normal((3, 2, 64), c.g).to(dev) for _ in range(2)), *args)
    assert all(t._version > v for t, v in zip(args[3:], versions))
    x = normal((3, 2, 64), c.g).to(dev).requires_grad_()
    y = ops.kv8_attention(x, *args, 0.125)
    with pytest.raises(RuntimeError):
        y.sum().backward()
