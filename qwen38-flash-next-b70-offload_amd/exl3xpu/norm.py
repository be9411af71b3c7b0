"""The root-mean-square norm before a layer's linears, with the residual's addition (torch.ops.exl3xpu_C.rms_norm).

  norm = RmsNorm(weight, eps=1e-6, unit_offset=False)
  y = norm(x)                                   x / sqrt(mean(x^2) + eps) * weight, of x's dtype
  y, h = norm(x, residual)                      h = x + residual in the residual's dtype, y the norm of h, of x's dtype
  q, s = norm.quant(x)                          the norm as e4m3 rows, as Fp8Linear.quantised takes them
  q, s, h = norm.quant(x, residual, "fp4")      as 4-bit rows, as Fp4Linear.quantised and Fp4Mlp.quantised take them
  q, s, y, h = norm.quant(x, residual, "fp8", rows=True)     y as well: the router and the EXL3 experts take it

One launch, each input read once (rows of more than 32,768 columns again for their outputs). h is added in fp32 and rounded once,
to the residual's dtype (x's or fp32), and the norm is that of the rounded h, so that it is the same as a norm of h by itself; it
is computed in 64 bits, rounded to 32, and from there to x's dtype. q, s are those of the norm before it is rounded to x's dtype,
in the forms of exl3xpu.fp8 and exl3xpu.fp4. Rows may lie inside wider ones at a uniform stride, and x [tokens, heads, k] inside
the rows of a fused projection. A row with an infinite element is NaN there and 0 elsewhere, one with a NaN element NaN. Calls run
on the device's current stream, keep no state and can be captured into a graph. They are for inference: inputs that require
gradients (while gradients are on) or carry tangents are refused, and the weight is detached when the norm is made, so that a
parameter given to it gets no gradient.
"""
from __future__ import annotations

import torch

from .linear import C as _C

__all__ = ["RmsNorm"]

_FORMS = {"fp8": 1, "fp4": 2}


class RmsNorm:
    def __init__(self, weight: torch.Tensor | None = None, eps: float = 1e-6, unit_offset: bool = False, device=None):
        """weight: [k] or None, kept as fp32 on `device` (its own by default); with unit_offset the norm is multiplied by 1 + weight,
        which is added in 64 bits. Raises ValueError on arguments that no rows could go with."""
        if weight is not None and (weight.dim() != 1 or not weight.numel()):
            raise ValueError(f"exl3xpu: weight [k], got {tuple(weight.shape)}")
        if not 2.0 ** -126 <= eps <= 3.0e38:
            raise ValueError(f"exl3xpu: eps positive and finite in fp32, got {eps}")
        if unit_offset and weight is None:
            raise ValueError("exl3xpu: unit_offset without a weight")
        if weight is not None:
            weight = weight.detach().to(weight.device if device is None else torch.device(device), torch.float32).contiguous()
        self.weight, self.eps, self.unit_offset = weight, float(eps), bool(unit_offset)
        self._op = _C().rms_norm.default

    def __call__(self, x: torch.Tensor, residual: torch.Tensor | None = None):
        """x [..., k] fp16 / bf16 / fp32 -> y, or (y, h) with a residual [..., k]."""
        out = self._op(x, residual, self.weight, self.eps, 0, True, self.unit_offset)
        return out[0] if residual is None else tuple(out)

    def quant(self, x: torch.Tensor, residual: torch.Tensor | None = None, form: str = "fp8", rows: bool = False):
        """-> (q, s) in the form "fp8" or "fp4", then y with rows=True, then h with a residual."""
        if form not in _FORMS:
            raise ValueError(f"exl3xpu: form 'fp8' or 'fp4', got {form!r}")
        return tuple(self._op(x, residual, self.weight, self.eps, _FORMS[form], rows, self.unit_offset))
