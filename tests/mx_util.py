"""Device MX tensors <-> the oracle's element codes and scale bytes."""
from __future__ import annotations

import numpy as np
import torch

from oracle import mx


def to_oracle(codes: torch.Tensor, scales: torch.Tensor) -> tuple[np.ndarray, np.ndarray, str]:
    c = codes.view(torch.uint8).reshape(-1, codes.shape[-1]).cpu().numpy()
    s = scales.view(torch.uint8).reshape(-1, scales.shape[-1]).cpu().numpy()
    return (mx.unpack(c), s, "e2m1") if codes.dtype == torch.uint8 else (c, s, "e4m3")


def to_device(codes: np.ndarray, scales: np.ndarray, fmt: str, dev) -> tuple[torch.Tensor, torch.Tensor]:
    c = torch.from_numpy(mx.pack(codes) if fmt == "e2m1" else codes).to(dev)
    s = torch.from_numpy(scales).to(dev).view(torch.float8_e8m0fnu)
    return (c if fmt == "e2m1" else c.view(torch.float8_e4m3fn)), s


def values(codes: torch.Tensor, scales: torch.Tensor) -> np.ndarray:
    return mx.dequantize(*to_oracle(codes, scales))


def random_mx(m: int, k: int, fmt: str, seed: int, narrow: bool = False) -> tuple[np.ndarray, np.ndarray]:
    """Quantised normal values with a few large columns, as the oracle's codes and scales.  ``narrow``: magnitudes
    of a block within a factor of 40, so that E4M3 codes are 8 and more, and their products with E2M1 codes
    multiples of 1/2 of at most 2^12: nothing lies below 2^-13 of the largest power of two among them."""
    rng = np.random.default_rng(seed)
    if narrow:
        return mx.quantize(rng.choice([-1.0, 1.0], (m, k)) * rng.uniform(0.026, 1.0, (m, k)), fmt)
    x = rng.standard_normal((m, k)) * np.where(rng.random(k) < 0.02, 16.0, 1.0)
    return mx.quantize(x, fmt)


def dropped(a: np.ndarray, w: np.ndarray) -> np.ndarray:
    """What an E4M3 x E2M1 product with bf16 output may lose: in each group of 8 of a block, up to 7 products lose
    less than 2^-13 of a power of two that is at most twice (0.5 counts as 1) the largest product."""
    ma, mw = (np.abs(t).reshape(t.shape[0], -1, mx.BLOCK).max(-1) for t in (a, w))
    return 4 * 7 * 2.0 ** -13 * 2 * (ma @ mw.T)


def f64(t: torch.Tensor) -> np.ndarray:
    return t.detach().double().cpu().numpy()


def product_bound(a: np.ndarray, w: np.ndarray, bias=None) -> tuple[np.ndarray, np.ndarray]:
    """(y, bound) of y = a w^T + bias for float32 sums in any order: every product of two codes and its scale is
    exact in float32, each of the kp + 1 additions rounds by at most 2^-24 of a partial sum's magnitude, and no
    partial sum exceeds the sum of magnitudes (with room of 1 % for the rounding of those)."""
    y, mag = a @ w.T, np.abs(a) @ np.abs(w).T
    if bias is not None:
        y, mag = y + bias, mag + np.abs(bias)
    return y, 1.01 * (a.shape[1] + 1) * 2.0 ** -24 * mag


def check_product(got: torch.Tensor, a: np.ndarray, w: np.ndarray, bias=None, lost=0.0) -> None:
    y, bound = product_bound(a, w, bias)
    bound = bound + lost
    if got.dtype == torch.bfloat16:
        bound = bound + 2.0 ** -8 * (np.abs(y) + bound)   # one rounding to bf16: half a step
    err = np.abs(f64(got).reshape(y.shape) - y)
    assert (err <= bound).all(), f"off by {np.max(err / np.maximum(bound, 1e-300)):.3g} of the bound"


def check_blocks(codes: torch.Tensor, scales: torch.Tensor, y: np.ndarray, delta: np.ndarray) -> None:
    """Codes and scales are a quantisation of values within ``delta`` of y [M, K]: a block's scale is one that its
    largest magnitude's interval gives, and each code lies between those of y - delta and y + delta under it
    (rounding is monotone).  Padding: zero codes, the smallest scale."""
    c, s, fmt = to_oracle(codes, scales)
    m, k = y.shape
    kp, sp = mx.padded(k)
    assert c.shape == (m, kp) and s.shape == (m, sp)
    yb, db = np.zeros((m, kp)), np.zeros((m, kp))
    yb[:, :k], db[:, :k] = y, delta
    yb, db = (t.reshape(m, -1, mx.BLOCK) for t in (yb, db))
    lo = mx.scale_bytes(np.maximum(np.abs(yb) - db, 0).max(-1))[fmt]
    hi = mx.scale_bytes((np.abs(yb) + db).max(-1))[fmt]
    got = s[:, :kp // mx.BLOCK]
    assert ((lo <= got) & (got <= hi)).all()
    assert (s[:, kp // mx.BLOCK:] == 0).all()
    f = (2.0 ** (got.astype(np.float64) - 127))[..., None]
    q = mx.decode(c, fmt).reshape(m, -1, mx.BLOCK)
    least, most = mx.decode(mx.encode((yb - db) / f, fmt), fmt), mx.decode(mx.encode((yb + db) / f, fmt), fmt)
    assert ((least <= q) & (q <= most)).all()
