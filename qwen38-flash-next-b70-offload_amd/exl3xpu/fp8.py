"""The 8-bit float linear beside the EXL3 one: weights in e4m3 with one fp32 scale per 128 x 128 block, rows quantised to
e4m3 with one fp32 scale per 128 columns, fp32 sums (torch.ops.exl3xpu_C.fp8_*). For layers whose weights are in that form
next to EXL3 experts: projections, and the shared expert of an MoE layer. The caller's model builds and calls them; no loader
here makes them out of a checkpoint.

  y = Fp8Linear(weight, weight_scale, bias=None)(x)        x [..., k] -> [..., n] of x's dtype
  y = Fp8Mlp(gate_up, down)(x)                             down(silu(gate) * up) of two Fp8Linear
  q, s = quant(x)                                          rows as the linear quantises them
  q, s = silu_mul_quant(gate_up)                           the same of silu(gate) * up of gate|up rows

q is float8_e4m3fn [..., k rounded up to 128] (zeros behind k), s fp32 [..., ceil(k / 128)], q s the value: s = max(amax /
448, 2^-80), q = x / s rounded to the nearest, halves to even. Calls run on the device's current stream, keep no state and
can be captured into a graph. How many rows a call has picks the order of a product's sums: a row alone and the same row
in a batch may differ in the last bits.
"""
from __future__ import annotations

import functools

import torch

from .linear import C as _C

__all__ = ["BLOCK", "Fp8Linear", "Fp8Mlp", "quant", "silu_mul_quant"]

BLOCK = 128


@functools.cache
def _op(name: str):
    return getattr(_C(), name).default


def quant(x: torch.Tensor):
    """x [..., k] fp16 / bf16 / fp32 -> (q, s)."""
    return _op("fp8_quant")(x)


def silu_mul_quant(gate_up: torch.Tensor):
    """gate|up rows [..., 2 k] -> (q, s) of silu(gate) * up, computed in fp32."""
    return _op("fp8_silu_mul_quant")(gate_up)


class Fp8Linear:
    """x @ weight^T + bias for weight [n, k] in float8_e4m3fn with weight_scale fp32 [ceil(n / 128), ceil(k / 128)] (the
    value is weight * its block's scale). Weights whose k is no multiple of 128 are padded with zeros here, and those that do not
    start on 16 bytes copied, once."""

    def __init__(self, weight: torch.Tensor, weight_scale: torch.Tensor, bias: torch.Tensor | None = None, device=None):
        """Tensors move to `device` (the weight's by default). Raises ValueError on shapes or types that do not fit."""
        if weight.dim() != 2 or weight.dtype != torch.float8_e4m3fn or 0 in weight.shape:
            raise ValueError(f"exl3xpu: weight float8_e4m3fn [n, k], got {weight.dtype} {tuple(weight.shape)}")
        self.n, self.k = weight.shape
        blocks = (-(-self.n // BLOCK), -(-self.k // BLOCK))
        if tuple(weight_scale.shape) != blocks:
            raise ValueError(f"exl3xpu: weight_scale {blocks}, got {tuple(weight_scale.shape)}")
        if bias is not None and tuple(bias.shape) != (self.n,):
            raise ValueError(f"exl3xpu: bias ({self.n},), got {tuple(bias.shape)}")
        device = weight.device if device is None else torch.device(device)
        pad = blocks[1] * BLOCK - self.k
        raw = weight.detach().to(device).view(torch.uint8)
        raw = torch.nn.functional.pad(raw, (0, pad)) if pad else raw.contiguous()
        # (the op takes weights that start on 16 bytes; a view into a larger buffer may not)
        self.weight = (raw.clone() if raw.data_ptr() % 16 else raw).view(torch.float8_e4m3fn)
        self.weight_scale = weight_scale.detach().to(device, torch.float32).contiguous()
        self.bias = None if bias is None else bias.detach().to(device, torch.float32).contiguous()
        self._linear, self._matmul = _op("fp8_linear"), _op("fp8_matmul")

    def __call__(self, x: torch.Tensor) -> torch.Tensor:
        """x [..., k] fp16 / bf16 / fp32 -> [..., n] of x's dtype."""
        if x.size(-1) != self.k:                  # (the op takes any k that the padded weight has room for)
            raise ValueError(f"exl3xpu: rows of {self.k}, got {tuple(x.shape)}")
        return self._linear(x, self.weight, self.weight_scale, self.bias)

    def quantised(self, q: torch.Tensor, s: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
        """The product of rows that are quantised already (q, s of quant or silu_mul_quant) -> [..., n] of dtype. Its sums are
        held in 32 bits for torch.float32; for fp16 and bf16 the e4m3 matrix instruction drops what is 13 bits below the
        largest of 8 products, 1.5e-5 of the outputs' root mean square for normal values."""
        return self._matmul(q, s, self.weight, self.weight_scale, self.bias, dtype)


class Fp8Mlp:
    """down(silu(gate) * up) with gate|up one fused linear [2 I, k]: the shared expert of an MoE layer, whose output is
    added to the routed experts'."""

    def __init__(self, gate_up: Fp8Linear, down: Fp8Linear):
        if gate_up.n != 2 * down.k:
            raise ValueError(f"exl3xpu: gate|up of {gate_up.n} columns does not fit a down of {down.k} inputs")
        self.gate_up, self.down = gate_up, down
        self._weights = [t for lin in (gate_up, down) for t in (lin.weight, lin.weight_scale, lin.bias)]
        self._op = _op("fp8_mlp")

    def __call__(self, x: torch.Tensor) -> torch.Tensor:
        """x [..., k] -> [..., n] of x's dtype; gate|up is rounded to x's dtype between the two products."""
        if x.size(-1) != self.gate_up.k:
            raise ValueError(f"exl3xpu: rows of {self.gate_up.k}, got {tuple(x.shape)}")
        return self._op(x, *self._weights)
