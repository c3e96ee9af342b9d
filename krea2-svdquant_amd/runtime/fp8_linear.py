"""``FP8Linear``: a linear layer with an 8-bit floating-point weight, a scale for each block of 128 x 128, and activations of
the same type with a scale for each 128 values.

Beside ``SVDQuantLinear`` and ``MXLinear`` where 4 bits of a weight are too few: half of a bf16 weight's bytes.  Layers that read
the same input share one quantised activation (``forward_fp8``).  The reference has no such layer.
"""
from __future__ import annotations

import torch
from torch import nn

from ..kernels.hip import ops
from ..quant.fp8 import BLOCK, dequantize_fp8, quantize_fp8


class FP8Linear(nn.Module):
    """``y = x w^T + bias`` with ``w`` held as E4M3 codes and ``x`` quantised by the call; bf16 in and out, sums in float32.

    Buffers: ``weight_codes`` uint8 [out, kp] (the E4M3 bytes), ``weight_scales`` float32 [ceil(out / 128), kp / 128] (any
    values), ``bias`` bf16 [out] or None.  All keep their type under ``.to(dtype)``, ``.half()`` and ``.float()``: what the layer
    computes does not follow the model's type."""

    def __init__(self, weight_codes: torch.Tensor, weight_scales: torch.Tensor, bias: torch.Tensor | None = None, *,
                 in_features: int):
        super().__init__()
        if in_features <= 0:
            raise ValueError(f"in_features={in_features}")
        n, kp = weight_codes.shape[0], -(-in_features // BLOCK) * BLOCK
        if weight_codes.element_size() != 1 or tuple(weight_codes.shape) != (n, kp) or n == 0:
            raise ValueError(f"weight_codes must be float8_e4m3fn or its bytes, [out, {kp}] for in_features={in_features}, got "
                             f"{weight_codes.dtype} {tuple(weight_codes.shape)}")
        want = (-(-n // BLOCK), kp // BLOCK)
        if weight_scales.dtype != torch.float32 or tuple(weight_scales.shape) != want:
            raise ValueError(f"weight_scales must be float32 {list(want)}, got {weight_scales.dtype} {tuple(weight_scales.shape)}")
        if bias is not None and tuple(bias.shape) != (n,):
            raise ValueError(f"bias must be [{n}], got {tuple(bias.shape)}")
        self.in_features, self.out_features = int(in_features), int(n)
        self.register_buffer("weight_codes", weight_codes.contiguous().view(torch.uint8), persistent=True)
        self.register_buffer("weight_scales", weight_scales.contiguous(), persistent=True)
        if bias is None:
            self.bias = None
        else:
            self.register_buffer("bias", bias.detach().to(torch.bfloat16).contiguous(), persistent=True)

    @classmethod
    def from_dense(cls, weight: torch.Tensor, bias: torch.Tensor | None = None) -> "FP8Linear":
        """The layer of a dense ``weight`` [out, in], quantised on its device."""
        if weight.ndim != 2:
            raise ValueError("linear weight must be [out_features, in_features]")
        codes, scales = quantize_fp8(weight.detach())
        return cls(codes, scales, bias, in_features=weight.shape[1])

    def dense_weight(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The weight [out, in] that the codes and scales stand for."""
        return dequantize_fp8(self._codes(), self.weight_scales, self.in_features, dtype)

    def quantize(self, x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        """``x`` [..., in] as codes and scales, for ``forward_fp8`` of this layer and of layers beside it."""
        self._check(x)
        return ops.fp8_quantize(x)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        self._check(x)
        return ops.fp8_linear(x, self._codes(), self.weight_scales, self.bias)

    def forward_fp8(self, codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
        """The layer on an activation that is quantised already (``quantize``); the same result as ``forward``'s."""
        return ops.fp8_gemm(codes, scales, self._codes(), self.weight_scales, self.bias)

    def _codes(self) -> torch.Tensor:
        return self.weight_codes.view(torch.float8_e4m3fn)

    def _apply(self, fn, *args, **kwargs):
        kept = {name: t for name, t in self._buffers.items() if t is not None and t.is_floating_point()}
        super()._apply(fn, *args, **kwargs)
        for name, t in kept.items():
            if self._buffers[name].dtype != t.dtype:   # moved, with the values it had
                self._buffers[name] = t.to(self._buffers[name].device)
        return self

    def _load_from_state_dict(self, state_dict, prefix, *args, **kwargs):
        codes = state_dict.get(prefix + "weight_codes")
        if codes is not None and codes.dtype == torch.float8_e4m3fn:   # by their bytes, not their values
            state_dict = {**state_dict, prefix + "weight_codes": codes.view(torch.uint8)}
        super()._load_from_state_dict(state_dict, prefix, *args, **kwargs)
        self.weight_scales = self.weight_scales.float()   # assigned from a checkpoint of another type
        if self.bias is not None:
            self.bias = self.bias.to(torch.bfloat16)

    def _check(self, x: torch.Tensor) -> None:
        if x.shape[-1] != self.in_features:
            raise ValueError(f"expected [..., {self.in_features}] activation, got shape {tuple(x.shape)}")

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}"
