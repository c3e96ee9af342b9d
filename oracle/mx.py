"""Microscaled (MX) blocks in 64-bit numpy, from the format definitions (OCP Microscaling specification v1.0):
blocks of 32 values share a scale 2^(s - 127) (s = 255: not a number), elements E2M1 or E4M3."""
from __future__ import annotations

import numpy as np

BLOCK = 32
FORMATS = ("e2m1", "e4m3")


def _magnitudes(exp_bits: int, man_bits: int, bias: int) -> np.ndarray:
    """Non-negative values of a sign / exponent / mantissa format by code, its special codes included as numbers."""
    c = np.arange(1 << (exp_bits + man_bits))
    e, m = c >> man_bits, (c & ((1 << man_bits) - 1)) / 2.0 ** man_bits
    return np.where(e == 0, m * 2.0 ** (1 - bias), (1 + m) * 2.0 ** (e - bias))


# E2M1: bias 1, no special values.  E4M3: bias 7, the last code is NaN.
MAGNITUDES = {"e2m1": _magnitudes(2, 1, 1), "e4m3": _magnitudes(4, 3, 7)[:-1]}
EMAX = {"e2m1": 2, "e4m3": 8}


def padded(k: int) -> tuple[int, int]:
    """(columns of codes, bytes of scales) of a row of k values."""
    return -(-k // 128) * 128, -(-k // 512) * 16


def scale_bytes(amax: np.ndarray) -> dict:
    """Scale byte of blocks by format, from their largest magnitude (255 where it is not finite)."""
    out = {}
    for fmt in FORMATS:
        finite = np.isfinite(amax)
        a = np.where(finite & (amax > 0), amax, 1.0)
        e = np.frexp(a)[1] - 1 - EMAX[fmt]
        s = np.where(amax > 0, np.clip(e, -127, 127) + 127, 0)
        out[fmt] = np.where(finite, s, 255).astype(np.uint8)
    return out


def encode(v: np.ndarray, fmt: str) -> np.ndarray:
    """Codes (sign bit above the magnitude's) of finite values already divided by their scale: nearest, ties to the
    even code, saturating."""
    mags = MAGNITUDES[fmt]
    a = np.abs(v)
    lo = np.clip(np.searchsorted(mags, a, side="right") - 1, 0, len(mags) - 1)
    hi = np.minimum(lo + 1, len(mags) - 1)
    mid = (mags[lo] + mags[hi]) / 2
    up = (a > mid) | ((a == mid) & (lo % 2 == 1))
    code = np.where(up, hi, lo)
    return (code | np.where(np.signbit(v), 8 if fmt == "e2m1" else 128, 0)).astype(np.uint8)


def decode(codes: np.ndarray, fmt: str) -> np.ndarray:
    sign = 8 if fmt == "e2m1" else 128
    mags = MAGNITUDES[fmt]
    if fmt == "e4m3":
        mags = np.append(mags, np.nan)
    return np.where(codes & sign, -1.0, 1.0) * mags[codes & (sign - 1)]


def quantize(x: np.ndarray, fmt: str) -> tuple[np.ndarray, np.ndarray]:
    """[M, K] -> element codes uint8 [M, kp] (one per byte, both formats) and scale bytes [M, sp]."""
    m, k = x.shape
    kp, sp = padded(k)
    b = np.zeros((m, kp))
    b[:, :k] = x
    b = b.reshape(m, kp // BLOCK, BLOCK)
    with np.errstate(invalid="ignore"):
        amax = np.abs(b).max(-1)
    s = scale_bytes(amax)[fmt]
    good = s != 255
    v = np.where(good[..., None], b, 0.0) / 2.0 ** (np.where(good, s, 127).astype(np.float64) - 127)[..., None]
    scales = np.zeros((m, sp), np.uint8)
    scales[:, :kp // BLOCK] = s
    return encode(v, fmt).reshape(m, kp), scales


def dequantize(codes: np.ndarray, scales: np.ndarray, fmt: str) -> np.ndarray:
    """float64 [M, kp] of element codes (one per byte) and their scale bytes."""
    m, kp = codes.shape
    s = scales[:, :kp // BLOCK].astype(np.float64)
    f = np.where(s == 255, np.nan, 2.0 ** (s - 127))
    return (decode(codes, fmt).reshape(m, -1, BLOCK) * f[..., None]).reshape(m, kp)


def pack(codes: np.ndarray) -> np.ndarray:
    """E2M1 codes, one per byte -> two per byte, the even column in the low half."""
    return codes[:, 0::2] | (codes[:, 1::2] << 4)


def unpack(packed: np.ndarray) -> np.ndarray:
    out = np.empty((packed.shape[0], packed.shape[1] * 2), np.uint8)
    out[:, 0::2], out[:, 1::2] = packed & 15, packed >> 4
    return out
