"""The router beside the routed experts: logits -> the picks of each row and their weights (torch.ops.exl3xpu_moe.moe_route).

  router = Router(topk, scoring="softmax", bias=None, n_group=1, topk_group=1, renormalize=True, scale=1.0)
  ids, w = router(logits)                  int32 / fp32 [..., topk], what ExpertStore.forward and forward_cached take
  y = store.forward_routed(key, x, logits, router)

Scores are softmax(logits) or sigmoid(logits) over the experts. The choice goes by the scores, with a bias (the load
balance's) by score + bias; with n_group > 1 only the experts of the topk_group best groups of neighbours compete, a
group's value being its largest score, or with a bias the sum of its two largest scores + bias. Picks are in descending
order, equal ones by index, and always topk different experts. The weights are the picks' scores (without the bias), with
renormalize over their sum, times scale.

An expert whose logit is -inf has score 0. Without a bias it is picked only where fewer than topk others are left; with one it
competes with its bias alone, so an expert that must not be picked needs a bias of -inf. A row of -inf gets weights of 0. (The
sigmoid of a logit below -700 counts as 0.) A NaN logit counts as the largest and gives NaN weights, but for softmax with a bias:
there a NaN or +inf logit makes every score of its row NaN, so the first topk experts of those that compete are picked, and
with renormalize the weights come from the picks' own logits.

The reference's plugin gets ids and weights from its caller's router (plugin/sglang_plugin.tier.py:531-561).
"""
from __future__ import annotations

import torch

from .moe_offload import ops as _load_ops

__all__ = ["Router"]


class Router:
    def __init__(self, topk: int, scoring: str = "softmax", bias: torch.Tensor | None = None, n_group: int = 1,
                 topk_group: int = 1, renormalize: bool = True, scale: float = 1.0):
        """bias: [E] on the device of the logits, kept as fp32. Raises ValueError on arguments that no logits could go
        with; the number of experts is checked at the call."""
        if scoring not in ("softmax", "sigmoid"):
            raise ValueError(f"exl3xpu: scoring 'softmax' or 'sigmoid', got {scoring!r}")
        if not 1 <= topk <= 64 or not 1 <= n_group <= 64 or not 1 <= topk_group <= n_group:
            raise ValueError(f"exl3xpu: topk {topk} and n_group {n_group} in 1..64, topk_group {topk_group} in 1..n_group")
        if bias is not None:
            if bias.dim() != 1 or bias.numel() % n_group:
                raise ValueError(f"exl3xpu: bias [experts], a multiple of {n_group} groups, got {tuple(bias.shape)}")
            bias = bias.detach().to(torch.float32).contiguous()
        self.topk, self.scoring, self.bias = int(topk), scoring, bias
        self.n_group, self.topk_group = int(n_group), int(topk_group)
        self.renormalize, self.scale = bool(renormalize), float(scale)
        self._op = _load_ops().moe_route.default

    def __call__(self, logits: torch.Tensor):
        """logits [..., experts] fp32 / bf16 / fp16 on the device -> (ids int32, w fp32) [..., topk]; on the device's
        current stream."""
        return self._op(logits, self.bias, self.topk, self.scoring, self.n_group, self.topk_group, self.renormalize,
                        self.scale)
