"""Dense weights into microscaled (MX) blocks (torch, any device): the converter's side of the format, not the
forward path.

Blocks of 32 consecutive values of a row share an E8M0 scale 2^(s - 127); elements are E2M1 (``"e2m1"``, two per
byte, the even column in the low half) or E4M3 (``"e4m3"``).  The storage is that of ``kernels.hip.ops.mx_quantize``,
bit for bit on bf16 inputs; float32 weights are quantised as they are, float64
ones from their float32 values.  The reference has no such format.
"""
from __future__ import annotations

import torch
import torch.nn.functional as F

BLOCK = 32
EMAX = {"e2m1": 2, "e4m3": 8}


def quantize_mx(x: torch.Tensor, fmt: str = "e2m1") -> tuple[torch.Tensor, torch.Tensor]:
    """Rows of ``x`` [..., K] (floating point) into MX blocks: ``(codes, scales)``.  A block with an infinity or a
    NaN gets the scale that is not a number and zero codes."""
    if fmt not in EMAX:
        raise ValueError(f"fmt must be one of {sorted(EMAX)}, got {fmt!r}")
    if not x.is_floating_point():
        raise TypeError(f"expected a floating-point tensor, got {x.dtype}")
    if x.ndim < 1 or x.shape[-1] == 0:
        raise ValueError(f"expected [..., K] with K > 0, got {tuple(x.shape)}")
    k = x.shape[-1]
    b = F.pad(x.float(), (0, -k % 128)).unflatten(-1, (-1, BLOCK))
    amax = b.abs().amax(-1)
    finite = torch.isfinite(amax)
    b = torch.where(finite[..., None], b, 0.0)
    e = torch.frexp(torch.where(finite, amax, 1.0)).exponent - 1 - EMAX[fmt]
    e = torch.where(amax > 0, e, -127).clamp(-127, 127)
    v = torch.ldexp(b, -e[..., None]).flatten(-2)
    s = F.pad(torch.where(finite, e + 127, 255).to(torch.uint8), (0, -e.shape[-1] % 16))
    scales = s.contiguous().view(torch.float8_e8m0fnu)
    if fmt == "e4m3":
        return v.clamp(-448, 448).to(torch.float8_e4m3fn), scales
    a = v.abs()
    # midpoints of 0, 0.5, 1, 1.5, 2, 3, 4, 6; a tie goes to the even code
    code = torch.signbit(v).byte() * 8
    for i, mid in enumerate((0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)):
        code += (a >= mid if i % 2 else a > mid).byte()
    return code[..., 0::2] | (code[..., 1::2] << 4), scales


def dequantize_mx(codes: torch.Tensor, scales: torch.Tensor, k: int, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values [..., k] that MX blocks hold."""
    if codes.dtype == torch.uint8:
        c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
        table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], device=codes.device)
        v = table[c.int()]
    elif codes.dtype == torch.float8_e4m3fn:
        v = codes.float()
    else:
        raise TypeError(f"codes must be uint8 (E2M1) or float8_e4m3fn, got {codes.dtype}")
    kp = v.shape[-1]
    if not 0 < k <= kp or -(-k // 128) * 128 != kp:
        raise ValueError(f"k={k} does not pad to the codes' {kp} columns")
    if scales.element_size() != 1:
        raise TypeError(f"scales must be float8_e8m0fnu or their bytes, got {scales.dtype}")
    want = (*codes.shape[:-1], -(-kp // 512) * 16)
    if tuple(scales.shape) != want:
        raise ValueError(f"scales must be {want}, got {tuple(scales.shape)}")
    s = scales.view(torch.uint8)[..., :kp // BLOCK].int()
    f = torch.where(s == 255, float("nan"), torch.ldexp(torch.ones((), device=codes.device), s - 127))
    return (v.unflatten(-1, (-1, BLOCK)) * f[..., None]).flatten(-2)[..., :k].to(dtype)
