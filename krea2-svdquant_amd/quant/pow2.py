"""Powers of two for the converters, exact on every device."""
from __future__ import annotations

import torch


def pow2(e: torch.Tensor) -> torch.Tensor:
    """float32 2^e of whole numbers ``e`` from -149 to 127, by their bits: torch.ldexp takes pow(2, e), which is off by a
    rounding for some exponents on the GPU."""
    e = e.int()
    return torch.where(e >= -126, (e + 127) << 23, 1 << (e + 149).clamp(0, 22)).view(torch.float32)
