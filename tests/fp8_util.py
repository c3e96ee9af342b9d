"""The 8-bit operators in 64 bits, on the CPU, and the bounds that their kernels are held to."""
from __future__ import annotations

import math

import torch

PAGE = 64
HALF = 2.0 ** -8   # half a bf16 step, relative


def scale_of(top: torch.Tensor) -> torch.Tensor:
    """The smallest power of two >= 2^-126 with top <= 448 of it (float64)."""
    m, e = torch.frexp(top)
    e = torch.where(m <= 0.875, e - 9, e - 8)
    return torch.ldexp(torch.ones_like(top), torch.where(top > 0, e, -126).clamp_min(-126))


def e4m3(x: torch.Tensor) -> torch.Tensor:
    """float64 at the nearest E4M3 value, ties to even; what is not finite is NaN."""
    mag = torch.where(torch.isfinite(x), x.abs(), 0.0)
    step = torch.exp2(torch.floor(torch.log2(mag.clamp_min(2.0 ** -6))) - 3)
    q = torch.copysign((torch.round(mag / step) * step).clamp_max(448.0), x)
    return torch.where(torch.isfinite(x), q, math.nan)


def finite_top(x: torch.Tensor, dims) -> torch.Tensor:
    return torch.where(torch.isfinite(x), x.abs(), 0.0).amax(dims)


def quantize(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows [M, K] -> the codes' values [M, kp] and scales [kp / 128, M], float64."""
    x = torch.nn.functional.pad(x.double(), (0, -x.shape[1] % 128))
    b = x.view(x.shape[0], -1, 128)
    s = scale_of(finite_top(b, -1))
    return e4m3(b / s[..., None]).view(x.shape), s.T.contiguous()


def product(a, a_scales, w, w_scales, bias=None):
    """(y, bound) in float64 from codes' values: 128 + blocks + 3 float32 roundings of sums no larger than the sum of
    magnitudes; what the matrix instruction drops, in each of a block's 16 groups of 8 up to 7 products' share below 2^-13 of
    a power of two that is at most the largest product; and the result's rounding."""
    kb, n = a.shape[1] // 128, w.shape[0]
    ab = a.double().view(-1, kb, 128) * a_scales.double().T[..., None]
    wb = w.double().view(n, kb, 128) * w_scales.double().repeat_interleave(128, 0)[:n, :, None]
    y, mag = (torch.einsum("mbk,nbk->mn", p, q) for p, q in ((ab, wb), (ab.abs(), wb.abs())))
    lost = 16 * 7 * 2.0 ** -13 * ab.abs().amax(-1) @ wb.abs().amax(-1).T
    if bias is not None:
        y, mag = y + bias.double(), mag + bias.double().abs()
    near = (131 + kb) * 2.0 ** -24 * mag + lost
    return y, near + HALF * (y.abs() + near) + 2.0 ** -133


def qk(x, weight, cos, sin, eps, positions, pairs):
    """(y, bound): a sum of D squares, the root, three products and the rotation's two, each a few float32 roundings of 2^-24."""
    x = x.double()
    d = x.shape[-1]
    n = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps)
    if weight is not None:
        n = n * weight.double()
    at = torch.arange(x.shape[0]) if positions is None else positions.long()
    c, s = cos.double()[at, None, :d // 2], sin.double()[at, None, :d // 2]
    a, b = (n[..., 0::2], n[..., 1::2]) if pairs else (n[..., :d // 2], n[..., d // 2:])
    parts = (a * c - b * s, b * c + a * s, (a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs())
    y, mag = (torch.stack(p, -1).flatten(-2) if pairs else torch.cat(p, -1) for p in (parts[:2], parts[2:]))
    near = (d / 2 + 16) * 2.0 ** -24 * mag
    return y, near + HALF * (y.abs() + near) + 2.0 ** -133


def append(k, v, offsets, lengths, table, kc, vc, scales):
    """In place on float64 codes' values [P, Hkv, 64, D], [P, Hkv, D, 64] and scales [P, Hkv, 2]."""
    for b in range(len(lengths)):
        row, end, place = offsets[b], offsets[b + 1], lengths[b]
        while row < end and place < len(table[b]) * PAGE:
            page, slot = table[b][place // PAGE], place % PAGE
            count = min(PAGE - slot, end - row)
            if 0 <= page < len(kc):
                for i, (codes, x) in enumerate(((kc[page], k), (vc[page].transpose(1, 2), v))):
                    x = x[row:row + count].double().transpose(0, 1)
                    s = scale_of(finite_top(x, (1, 2)))
                    if slot:
                        before = scales[page, :, i].clone()
                        s = torch.maximum(s, before)
                        codes[:, :slot] = e4m3(codes[:, :slot] * (before / s)[:, None, None])
                    codes[:, slot:slot + count] = e4m3(x / s[:, None, None])
                    scales[page, :, i] = s
            row, place = row + count, place + count


def attention(q, offsets, lengths, table, kc, vc, scales, scale, causal):
    """(o, bound): a probability is off by its score's error (D + 4 roundings of the sum of magnitudes; exp2's argument and value)
    and a bf16 rounding e <= 2^-8, which the numerator and the sum share:
        (sum p (1 + e) v) / (sum p (1 + e)) - o = (sum p e (v - o)) / (sum p (1 + e)),
    at most 2^-8 / (1 - 2^-8) (sum p |v| + |o|), and less where the sum takes p itself; then the result's rounding."""
    q = q.double()
    heads, d, kv = q.shape[1], q.shape[2], kc.shape[1]
    out, bound = torch.zeros_like(q), torch.zeros_like(q)
    for b in range(len(lengths)):
        row, n = offsets[b], offsets[b + 1] - offsets[b]
        length = min(lengths[b], len(table[b]) * PAGE)
        pages = table[b][:-(-length // PAGE)]
        there = torch.tensor([0 <= p < len(kc) for p in pages], dtype=torch.bool).repeat_interleave(PAGE)[:length]
        pages = torch.tensor([p if 0 <= p < len(kc) else 0 for p in pages], dtype=torch.long)
        if not n or not length:
            continue
        k = (kc[pages] * scales[pages, :, 0, None, None]).transpose(0, 1).reshape(kv, -1, d)[:, :length]
        v = (vc[pages] * scales[pages, :, 1, None, None]).permute(1, 0, 3, 2).reshape(kv, -1, d)[:, :length]
        k, v = (t.repeat_interleave(heads // kv, 0) for t in (k, v))
        qb = q[row:row + n].transpose(0, 1)
        seen = there.expand(n, -1)
        if causal:
            seen = seen & (torch.arange(length) <= torch.arange(n)[:, None] + length - n)
        s = (qb @ k.transpose(1, 2) * scale).masked_fill(~seen, -math.inf)
        mag = (qb.abs() @ k.nan_to_num().abs().transpose(1, 2) * abs(scale)).masked_fill(~seen, 0).amax(-1, keepdim=True)
        top = s.amax(-1, keepdim=True)
        p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
        total = p.sum(-1, keepdim=True)
        p = p / torch.where(total == 0, 1.0, total)
        # what no row sees counts for nothing, whatever it holds
        o = torch.stack([p[:, i, seen[i]].unsqueeze(1) @ v[:, seen[i]] for i in range(n)], 1).squeeze(2)
        size = p.nan_to_num() @ v.nan_to_num().abs()
        off = 2 * ((d + 8) * 2.0 ** -24 * 1.4427 * mag + 2.0 ** -20)
        near = HALF / (1 - HALF) * (size + o.nan_to_num().abs()) + size * (2 * off + 2.0 ** -18)
        out[row:row + n] = o.transpose(0, 1)
        bound[row:row + n] = (near + HALF * (o.nan_to_num().abs() + near) + 2.0 ** -133).transpose(0, 1)
    return out, bound


def check(got: torch.Tensor, want: torch.Tensor, bound: torch.Tensor) -> None:
    got = got.double().cpu()
    assert got.shape == want.shape
    assert torch.equal(torch.isnan(got), torch.isnan(want)), "NaN at other places"
    off = torch.where(torch.isnan(want), 0.0, (got - want).abs())
    worst = (off / bound.clamp_min(1e-300)).max().item() if off.numel() else 0.0
    assert worst <= 1.0, f"off by {worst:.3g} of the bound"


def pages(p, kv, d, gen, *, stale=False):
    """Random codes (every byte a value, some NaN where ``stale``) and scales of either kind."""
    k, v = (torch.randint(0, 256, s, generator=gen, dtype=torch.uint8) for s in ((p, kv, PAGE, d), (p, kv, d, PAGE)))
    for t in (k, v):
        t[(t & 127) > 118] -= 16           # up to 240, none NaN
        if stale:
            t[torch.rand(t.shape, generator=gen) < 0.02] = 127
    s = torch.rand((p, kv, 2), generator=gen) * 0.01 + 0.002
    return k.view(torch.float8_e4m3fn), v.view(torch.float8_e4m3fn), s
