"""``MXLinear``: a linear layer with a microscaled 4-bit weight and microscaled 4- or 8-bit activations.

Beside ``SVDQuantLinear`` for dense weights without calibration data: no smoothing scale and no low-rank branch, so
the scale of 32 consecutive values is all there is, and layers that read the same input share one quantised
activation (``forward_mx``).  The reference has no such layer.
"""
from __future__ import annotations

import torch
from torch import nn

from ..kernels.hip import ops
from ..quant.mx import dequantize_mx, quantize_mx


class MXLinear(nn.Module):
    """``y = x w^T + bias`` with ``w`` held as E2M1 MX blocks and ``x`` quantised to ``activation`` MX blocks
    (``"e4m3"`` or ``"e2m1"``) by the call; bf16 in and out, sums in float32.

    Buffers: ``weight_codes`` uint8 [out, kp / 2], ``weight_scales`` uint8 [out, sp] (the E8M0 bytes), ``bias`` bf16 [out]
    or None.  All keep their type under ``.to(dtype)``, ``.half()`` and ``.float()``: what the layer computes does not
    follow the model's type."""

    def __init__(self, weight_codes: torch.Tensor, weight_scales: torch.Tensor, bias: torch.Tensor | None = None, *,
                 in_features: int, activation: str = "e4m3"):
        super().__init__()
        cols, sp = ops.mx_shapes(in_features, "e2m1")
        ops.mx_shapes(in_features, activation)   # a known format
        n = weight_codes.shape[0]
        if weight_codes.dtype != torch.uint8 or tuple(weight_codes.shape) != (n, cols):
            raise ValueError(f"weight_codes must be uint8 [out, {cols}] for in_features={in_features}, got "
                             f"{weight_codes.dtype} {tuple(weight_codes.shape)}")
        if weight_scales.element_size() != 1 or tuple(weight_scales.shape) != (n, sp):
            raise ValueError(f"weight_scales must be bytes [{n}, {sp}], got {weight_scales.dtype} "
                             f"{tuple(weight_scales.shape)}")
        if bias is not None and tuple(bias.shape) != (n,):
            raise ValueError(f"bias must be [{n}], got {tuple(bias.shape)}")
        self.in_features, self.out_features = int(in_features), int(n)
        self.activation = activation
        self.register_buffer("weight_codes", weight_codes.contiguous(), persistent=True)
        self.register_buffer("weight_scales", weight_scales.contiguous().view(torch.uint8), persistent=True)
        if bias is None:
            self.bias = None
        else:
            self.register_buffer("bias", bias.detach().to(torch.bfloat16).contiguous(), persistent=True)

    @classmethod
    def from_dense(cls, weight: torch.Tensor, bias: torch.Tensor | None = None, *,
                   activation: str = "e4m3") -> "MXLinear":
        """The layer of a dense ``weight`` [out, in], quantised on its device."""
        if weight.ndim != 2:
            raise ValueError("linear weight must be [out_features, in_features]")
        codes, scales = quantize_mx(weight.detach(), "e2m1")
        return cls(codes, scales, bias, in_features=weight.shape[1], activation=activation)

    def dense_weight(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The weight [out, in] that the codes and scales stand for."""
        return dequantize_mx(self.weight_codes, self.weight_scales, self.in_features, dtype)

    def quantize(self, x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        """``x`` [..., in] as this layer's activation blocks, for ``forward_mx`` of it and of layers beside it."""
        self._check(x)
        return ops.mx_quantize(x, self.activation)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        self._check(x)
        return ops.mx_linear(x, self.weight_codes, self.weight_scales, self.bias, self.activation)

    def forward_mx(self, codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
        """The layer on MX blocks [..., in] of either format (``quantize``, or the output of
        ``ops.rms_norm_modulate_mx``, ``ops.residual_rms_norm_modulate_mx`` or ``ops.silu_mul_mx``)."""
        return ops.mx_gemm(codes, scales, self.weight_codes, self.weight_scales, self.bias)

    def _apply(self, fn, *args, **kwargs):
        bias = self.bias
        super()._apply(fn, *args, **kwargs)
        if bias is not None and self.bias.dtype != bias.dtype:   # moved, with the values it had
            self.bias = bias.to(self.bias.device)
        return self

    def _load_from_state_dict(self, *args, **kwargs):
        super()._load_from_state_dict(*args, **kwargs)
        if self.bias is not None:   # assigned from a checkpoint of another type
            self.bias = self.bias.to(torch.bfloat16)

    def _check(self, x: torch.Tensor) -> None:
        if x.shape[-1] != self.in_features:
            raise ValueError(f"expected [..., {self.in_features}] activation, got shape {tuple(x.shape)}")

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}, activation={self.activation!r}"
