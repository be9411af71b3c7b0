"""The 4-bit float linear beside the EXL3 and the 8-bit one: weights and rows in microscaled 4-bit floats (OCP MX: e2m1 with one
power of two per 32 columns), fp32 sums (torch.ops.exl3xpu_C.fp4_*). For layers whose weights are in that form next to EXL3
experts: projections, and the shared expert of an MoE layer. The caller's model builds and calls them; no loader here makes
them out of a checkpoint.

  y = Fp4Linear(weight, weight_scale, bias=None)(x)        x [..., k] -> [..., n] of x's dtype
  y = Fp4Mlp(gate_up, down)(x)                             down(silu(gate) * up) of two Fp4Linear
  q, s = quant(x)                                          rows as the linear quantises them
  q, s = silu_mul_quant(gate_up)                           the same of silu(gate) * up of gate|up rows
  x = dequant(q, s, dtype, k)                              the values that they stand for

q is uint8 [..., kp / 2] with kp = k rounded up to 128: two codes to a byte, the first in the low half, zeros behind k. A code is
0, 0.5, 1, 1.5, 2, 3, 4 or 6, with 8 added for the negative ones. s is uint8 [..., ceil(k / 256), 8], whose byte [..., b, j] is the exponent
+ 127 of the scale of columns 256 b + 32 j to 256 b + 32 j + 31 (255: NaN; 0 behind k); in memory the stages b are outermost. The
scale is 2^(floor(log2(amax)) - 2), 2^-126 at the least; x / scale is rounded to the nearest code, halves to even, 6 at the most. A
block with an infinite or NaN element is NaN. Calls run on the device's current stream, keep no state and can be captured into a
graph. They are for inference: inputs that require gradients (while gradients are on) or carry tangents are refused, and weights and
biases are detached when a linear is made, so that parameters given to it get no gradients. How many rows a call has picks the order
of a product's sums: a row alone and the same row in a batch may differ in the last bits.
"""
from __future__ import annotations

import functools

import torch

from .linear import C as _C

__all__ = ["BLOCK", "Fp4Linear", "Fp4Mlp", "dequant", "quant", "silu_mul_quant"]

BLOCK = 32
_COLS, _STAGE = 128, 256


@functools.cache
def _op(name: str):
    return getattr(_C(), name).default


def quant(x: torch.Tensor):
    """x [..., k] fp16 / bf16 / fp32 -> (q, s)."""
    return _op("fp4_quant")(x)


def silu_mul_quant(gate_up: torch.Tensor):
    """gate|up rows [..., 2 k] -> (q, s) of silu(gate) * up, computed in fp32."""
    return _op("fp4_silu_mul_quant")(gate_up)


def dequant(q: torch.Tensor, s: torch.Tensor, dtype: torch.dtype = torch.float32, k: int | None = None) -> torch.Tensor:
    """(q, s) of k columns (all that q holds by default) -> [..., k] of dtype."""
    return _op("fp4_dequant")(q, s, 2 * q.size(-1) if k is None else k, dtype)


def _bytes(t: torch.Tensor, *others: torch.dtype) -> torch.Tensor:
    return t.detach().view(torch.uint8) if t.dtype in others else t.detach()


class Fp4Linear:
    """x @ weight^T + bias for weight [n, k] in the form above: codes uint8 (or float4_e2m1fn_x2) [n, ceil(k / 2)], scales uint8 (or
    float8_e8m0fnu) [n, ceil(k / 32)], as a checkpoint has them; or (q, s) of quant(weight) with k=. Both are laid out here, once."""

    def __init__(self, weight: torch.Tensor, weight_scale: torch.Tensor, bias: torch.Tensor | None = None, k: int | None = None,
                 device=None):
        """Tensors move to `device` (the weight's by default). Raises ValueError on shapes or types that do not fit."""
        w = _bytes(weight, torch.float4_e2m1fn_x2)
        sw = _bytes(weight_scale, torch.float8_e8m0fnu)
        if w.dim() != 2 or w.dtype != torch.uint8 or 0 in w.shape:
            raise ValueError(f"exl3xpu: weight uint8 [n, k / 2], got {weight.dtype} {tuple(weight.shape)}")
        self.n, self.k = w.size(0), 2 * w.size(1) if k is None else int(k)
        blocks, stages, cols = -(-self.k // BLOCK), -(-self.k // _STAGE), -(-self.k // _COLS) * _COLS
        if self.k <= 0 or w.size(1) not in (-(-self.k // 2), cols // 2):
            raise ValueError(f"exl3xpu: weight of {w.size(1)} bytes a row does not hold k={self.k}")
        if sw.dtype != torch.uint8 or tuple(sw.shape) not in ((self.n, blocks), (self.n, stages, 8)):
            raise ValueError(f"exl3xpu: weight_scale uint8 ({self.n}, {blocks}), got {weight_scale.dtype} {tuple(sw.shape)}")
        if bias is not None and tuple(bias.shape) != (self.n,):
            raise ValueError(f"exl3xpu: bias ({self.n},), got {tuple(bias.shape)}")
        device = weight.device if device is None else torch.device(device)
        raw, used = w.to(device), -(-self.k // 2)
        if used < cols // 2 or self.k % 2:
            raw = torch.nn.functional.pad(raw[:, :used], (0, cols // 2 - used))
            raw[:, used - 1] &= 15 if self.k % 2 else 255
        # (the op takes weights that start on 16 bytes; a view into a larger buffer may not)
        raw = raw.contiguous()
        self.weight = raw.clone() if raw.data_ptr() % 16 else raw
        flat = sw.to(device).reshape(self.n, -1)[:, :blocks]
        flat = torch.nn.functional.pad(flat, (0, 8 * stages - blocks)).view(self.n, stages, 8)
        self.weight_scale = flat.movedim(1, 0).clone(memory_format=torch.contiguous_format).movedim(0, 1)   # stages outermost
        self.bias = None if bias is None else bias.detach().to(device, torch.float32).contiguous()
        self._linear, self._matmul = _op("fp4_linear"), _op("fp4_matmul")

    def __call__(self, x: torch.Tensor) -> torch.Tensor:
        """x [..., k] fp16 / bf16 / fp32 -> [..., n] of x's dtype."""
        if x.size(-1) != self.k:                  # (the op takes any k that the padded weight has room for)
            raise ValueError(f"exl3xpu: rows of {self.k}, got {tuple(x.shape)}")
        return self._linear(x, self.weight, self.weight_scale, self.bias)

    def quantised(self, q: torch.Tensor, s: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
        """The product of rows that are quantised already (q, s of quant, silu_mul_quant or RmsNorm.quant) -> [..., n] of dtype."""
        return self._matmul(q, s, self.weight, self.weight_scale, self.bias, dtype)


class Fp4Mlp:
    """down(silu(gate) * up) with gate|up one fused linear [2 I, k]: the shared expert of an MoE layer, whose output is added to the
    routed experts'. gate|up stays in fp32 until silu(gate) * up is quantised. The gate|up weights are copied, in an order in which
    every 32 gates have their ups next to them: the linear that they came from is not needed any more."""

    def __init__(self, gate_up: Fp4Linear, down: Fp4Linear):
        if gate_up.n != 2 * down.k:
            raise ValueError(f"exl3xpu: gate|up of {gate_up.n} columns does not fit a down of {down.k} inputs")
        if gate_up.weight.device != down.weight.device:
            raise ValueError(f"exl3xpu: gate|up on {gate_up.weight.device}, down on {down.weight.device}")
        self.k, self.I, self.n = gate_up.k, down.k, down.n
        # (row 2 I stands for the zeros behind the last gate and the last up)
        i = torch.arange(-(-self.I // _COLS) * _COLS, device=gate_up.weight.device).view(-1, 1, BLOCK)
        order = torch.cat([torch.where(i < self.I, i, 2 * self.I), torch.where(i < self.I, i + self.I, 2 * self.I)], 1).view(-1)

        def ordered(t):
            return torch.cat([t, t.new_zeros(1, *t.shape[1:])])[order]
        bias = None if gate_up.bias is None else ordered(gate_up.bias)
        scale = ordered(gate_up.weight_scale).movedim(1, 0).contiguous().movedim(0, 1)
        self._weights = [ordered(gate_up.weight), scale, bias, down.weight, down.weight_scale, down.bias]
        self._mlp, self._matmul = _op("fp4_mlp"), _op("fp4_mlp_matmul")

    def __call__(self, x: torch.Tensor) -> torch.Tensor:
        """x [..., k] -> [..., n] of x's dtype."""
        if x.size(-1) != self.k:
            raise ValueError(f"exl3xpu: rows of {self.k}, got {tuple(x.shape)}")
        return self._mlp(x, self.I, *self._weights)

    def quantised(self, q: torch.Tensor, s: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
        """The same of rows that are quantised already (q, s of quant or RmsNorm.quant) -> [..., n] of dtype."""
        return self._matmul(q, s, self.I, *self._weights, dtype)
