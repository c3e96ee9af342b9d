"""Dense weights into E4M3 blocks of 128 x 128 (torch, any device): the converter's side of the format, not the forward
path.

Each block of a weight [out, in] has a float32 scale, the smallest power of two (2^-126 at least) under which its largest
finite magnitude is at most 448; its codes are the nearest E4M3 values, ties to even, and values that are not finite become NaN.
Rows are padded to a multiple of 128 columns with zeros.  Float32 weights are quantised as they are, float64 ones from their
float32 values.  The product takes any float32 scales, so checkpoints with others need no conversion.  The reference has
no such format.
"""
from __future__ import annotations

import torch
import torch.nn.functional as F

from .pow2 import pow2

BLOCK = 128


def quantize_fp8(w: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``w`` [N, K] (floating point) as ``(codes [N, kp], scales [ceil(N / 128), kp / 128])``."""
    if not w.is_floating_point():
        raise TypeError(f"expected a floating-point tensor, got {w.dtype}")
    if w.ndim != 2 or 0 in w.shape:
        raise ValueError(f"expected [N, K] with N, K > 0, got {tuple(w.shape)}")
    n, k = w.shape
    b = F.pad(w.float(), (0, -k % BLOCK, 0, -n % BLOCK)).unflatten(1, (-1, BLOCK)).unflatten(0, (-1, BLOCK))   # [nb, 128, kb, 128]
    finite = torch.isfinite(b)
    amax = torch.where(finite, b.abs(), 0.0).amax((1, 3))
    m, e = torch.frexp(amax)
    e = torch.where(amax > 0, torch.where(m <= 0.875, e - 9, e - 8), -126).clamp_min(-126)
    v = torch.where(finite, b, float("nan")) * pow2(-e)[:, None, :, None]
    codes = v.flatten(2).flatten(0, 1)[:n].to(torch.float8_e4m3fn)
    return codes.contiguous(), pow2(e)


def dequantize_fp8(codes: torch.Tensor, scales: torch.Tensor, k: int, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values [N, k] that E4M3 blocks hold."""
    if codes.dtype != torch.float8_e4m3fn or codes.ndim != 2:
        raise TypeError(f"codes must be float8_e4m3fn [N, kp], got {codes.dtype} {tuple(codes.shape)}")
    n, kp = codes.shape
    if not 0 < k <= kp or -(-k // BLOCK) * BLOCK != kp:
        raise ValueError(f"k={k} does not pad to the codes' {kp} columns")
    if tuple(scales.shape) != (-(-n // BLOCK), kp // BLOCK):
        raise ValueError(f"scales must be {(-(-n // BLOCK), kp // BLOCK)}, got {tuple(scales.shape)}")
    s = scales.float().repeat_interleave(BLOCK, 0)[:n, :, None]
    return (codes.float().unflatten(1, (-1, BLOCK)) * s).flatten(1)[:, :k].to(dtype)
