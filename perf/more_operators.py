"""Timed cases of the norm before a layer's linears and of the 4-bit float linear: what a program runs around the router,
the EXL3 experts and the 8-bit float linear.

  norm    the residual's addition and the root-mean-square norm; rows of the inputs' type, or e4m3 with one scale per 128 columns
  quant   rows -> 4-bit floats (e2m1) with one power of two per 32 columns, and the values that they stand for
  linear  x @ W^T with W in that form; x is quantised as `quant` does, or comes out of the norm in that form
  mlp     the gated MLP of a shared expert: linear (gate|up), silu(gate) * up quantised, linear (down)

Sizes are this repository's own (bench.py: hidden 2048 and 4096, intermediate 512, the dense projections of one decoder
layer, heads of 128) and ragged ones around them.
"""
from __future__ import annotations

import math
import os
import sys

import torch

own = False
DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
BLK8 = 128                    # columns of an e4m3 scale
E4M3_MAX = 448.0
TINY8 = 2.0 ** -80            # the smallest e4m3 scale: a block of zeros has it
BLK = 32                      # columns of an e2m1 scale
LEAST = -126                  # the smallest e2m1 scale's exponent: a block of zeros has it
EPS = 1e-6


def _norm(name, M, k, dtype="bf16", heads=1, residual="", out="same", offset=False):
    return {"name": name, "kind": "norm", "M": M, "k": k, "dtype": dtype, "heads": heads, "residual": residual, "out": out,
            "offset": offset}


def _quant(name, M, k, dtype="bf16"):
    return {"name": name, "kind": "quant", "M": M, "k": k, "dtype": dtype}


def _linear(name, M, k, n, bias=False, dtype="bf16", norm=False):
    return {"name": name, "kind": "linear", "M": M, "k": k, "n": n, "bias": bias, "dtype": dtype, "norm": norm}


def _mlp(name, M, k, I, dtype="bf16"):  # noqa: E741
    return {"name": name, "kind": "mlp", "M": M, "k": k, "I": I, "dtype": dtype}


def listed():
    return [
        # one user's token before an 8-bit float linear: pure latency
        _norm("norm_bs1", 1, 2048, residual="bf16", out="fp8"),
        # the queries' heads inside the rows of a fused projection, each normed by itself
        _norm("norm_heads", 1500, 128, heads=16, offset=True),
        # a ragged fp16 prompt whose residual stream is held in fp32
        _norm("norm_ragged", 333, 1000, "fp16", residual="fp32"),
        # the largest chunk of a prompt, before an 8-bit float linear
        _norm("norm_8192", 8192, 2048, residual="bf16", out="fp8"),
        # the rows of a ragged fp16 prompt, and the largest chunk
        _quant("quant_301", 301, 1000, "fp16"),
        _quant("quant_8192", 8192, 2048),
        # one user's token: the layer's norm and the widest projection group behind it
        _linear("linear_bs1", 1, 2048, 12288, norm=True),
        # a decode batch through the output projection
        _linear("linear_m40", 40, 4096, 2048),
        # a ragged chunk, sizes that end inside a block, a bias, fp32 in and out
        _linear("linear_ragged", 777, 2000, 1000, bias=True, dtype="fp32"),
        # the largest chunk through the widest projection group
        _linear("linear_8192", 8192, 2048, 12288),
        # a small decode batch through the whole shared expert, and the largest chunk
        _mlp("mlp_bs4", 4, 2048, 512),
        _mlp("mlp_8192", 8192, 2048, 512),
    ]


def draw(rng):
    def logint(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(["norm", "norm", "norm", "quant", "linear", "linear", "linear", "mlp"])
    dt = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if kind == "norm":
        if rng.random() < 0.3:
            c = _norm("", logint(1, 4096), rng.choice([64, 128, 256]), dt, rng.choice([2, 8, 16]), offset=rng.random() < 0.5)
        else:
            c = _norm("", logint(1, 8192), rng.choice([2048, 4096, logint(100, 4500)]), dt, 1,
                      rng.choice(["", dt, dt, "fp32"]), rng.choice(["same", "fp8", "fp8"]), rng.random() < 0.5)
            if c["M"] * c["k"] > 8192 * 2048:
                c["M"] //= 2
    elif kind == "quant":
        c = _quant("", logint(1, 8192), rng.choice([2048, 4096, 512, logint(100, 4500)]), dt)
    elif kind == "linear":
        k, n = rng.choice([(2048, 12288), (4096, 2048), (2048, 1024), (512, 2048), (logint(100, 4500) // 2 * 2, logint(100, 4500))])
        # (a norm's 32 bits decide which side of a border a value falls: 16-bit outputs, for which that is small)
        c = _linear("", logint(1, 8192), k, n, rng.random() < 0.3, dt, dt != "fp32" and rng.random() < 0.4)
    else:
        c = _mlp("", logint(1, 8192), rng.choice([2048, 4096]), rng.choice([512, 640, 1024]), rng.choice(["bf16", "fp16"]))
    c.pop("name", None)
    return c


# ---- inputs -----------------------------------------------------------------------------------------------------------

def _gen(seed, more):
    return torch.Generator(device=DEV).manual_seed((int(seed) % (1 << 40)) * 64 + more)


def _activations(g, M, k, dtype):
    """Normal rows with channels of unequal size, as a residual stream has them; the last of many rows is padding (0)."""
    x = torch.randn(M, k, generator=g, device=DEV) * torch.exp(0.6 * torch.randn(k, generator=g, device=DEV))
    if M > 8:
        x[-1] = 0
    return x.to(DTYPES[dtype])


def _weight(g, n, k):
    """A normal matrix as a checkpoint holds it: two codes per byte [n, k / 2], the first in the low half, and one exponent + 127
    per 32 columns [n, ceil(k / 32)]."""
    v, e = _blocks4(torch.randn(n, k, generator=g, device=DEV) / math.sqrt(k))
    a = v.abs()
    code = (torch.where(a < 2, 2 * a, torch.where(a < 4, a + 2, a / 2 + 4)) + 8 * (v < 0)).to(torch.uint8).view(n, -1)
    code = code.view(n, -1, 2)
    return (code[..., 0] | code[..., 1] << 4)[:, :k // 2].contiguous(), (e + 127).to(torch.uint8)


def prepare(case, seed):
    kind, M, k = case["kind"], case["M"], case["k"]
    g = _gen(seed, 1)
    st = {"case": case}
    if own:
        pkg = os.path.join(os.getcwd(), "qwen38-flash-next-b70-offload_amd")
        if pkg not in sys.path:
            sys.path.insert(0, pkg)
        from exl3xpu import fp4, norm
        st["fp4"] = fp4
    if kind == "norm" and case["heads"] > 1:
        # heads at the front of wider rows (keys and values behind them)
        rows = torch.randn(M, (case["heads"] + 4) * k, generator=g, device=DEV).to(DTYPES[case["dtype"]])
        st["x"] = rows[:, :case["heads"] * k].view(M, case["heads"], k)
    else:
        st["x"] = _activations(g, M, k, case["dtype"])
    if kind == "norm" or case.get("norm"):
        kept = case["residual"] if kind == "norm" else case["dtype"]
        st["residual"] = 3 * _activations(g, M, k, kept) if kept else None
        st["offset"] = bool(case.get("offset"))
        st["weight"] = 0.2 * torch.randn(k, generator=g, device=DEV) + (0.0 if st["offset"] else 1.0)
        if own:
            st["norm"] = norm.RmsNorm(st["weight"], EPS, unit_offset=st["offset"])
    if kind == "linear":
        st["w"], st["sw"] = _weight(g, case["n"], k)
        st["bias"] = 0.1 * torch.randn(case["n"], generator=g, device=DEV) if case["bias"] else None
        if own:
            st["linear"] = fp4.Fp4Linear(st["w"], st["sw"], st["bias"])
    elif kind == "mlp":
        st["wg"], st["sg"] = _weight(g, 2 * case["I"], k)
        st["wd"], st["sd"] = _weight(g, k, case["I"])
        if own:
            st["mlp"] = fp4.Fp4Mlp(fp4.Fp4Linear(st["wg"], st["sg"]), fp4.Fp4Linear(st["wd"], st["sd"]))
    return st


# ---- the plain forms ------------------------------------------------------------------------------------------------

def _plain_norm(st):
    """(y in 32 bits, the new residual or None): the sum is held in the residual's type, and the norm is that of what is held."""
    x, res = st["x"].float(), st["residual"]
    held = None
    if res is not None:
        held = (x + res.float()).to(res.dtype)
        x = held.float()
    w = st["weight"] + 1 if st["offset"] else st["weight"]
    return x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w, held


def _plain_quant8(x):
    """x fp32 [M, k] -> e4m3 [M, k up to a multiple of 128] (zeros behind k), fp32 [M, ceil(k / 128)]. Scale and quotient
    are divided in 64 bits and rounded to 32: a quotient one step off would cross the border between two e4m3 values."""
    M, k = x.shape
    kb = -(-k // BLK8)
    p = torch.zeros(M, kb * BLK8, device=x.device)
    p[:, :k] = x
    p = p.view(M, kb, BLK8)
    s = (p.abs().amax(-1).double() / E4M3_MAX).float().clamp_min(TINY8)
    return (p.double() / s[..., None].double()).float().view(M, kb * BLK8).to(torch.float8_e4m3fn), s


def _blocks4(x):
    """x fp32 [M, k] -> e2m1 values [M, blocks, 32] and the exponents of their scales [M, blocks]: 2^e is the power of two in the
    block's largest magnitude over that in 6, e2m1's largest value; values to the nearest, halves to even, above 6 to 6."""
    M, k = x.shape
    kb = -(-k // BLK)
    p = torch.zeros(M, kb * BLK, device=x.device)
    p[:, :k] = x
    p = p.view(M, kb, BLK)
    e = (torch.frexp(p.abs().amax(-1)).exponent - 3).clamp_min(LEAST)
    v = torch.ldexp(p, -e[..., None]).clamp(-6, 6)
    a = v.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    return torch.round(v / step) * step, e


def _plain_quant4(x):
    """x fp32 [M, k] -> the values that its 4-bit floats stand for."""
    v, e = _blocks4(x)
    return torch.ldexp(v, e[..., None]).view(x.size(0), -1)[:, :x.size(1)]


def _plain_weight(w, sw):
    codes = torch.stack([w & 15, w >> 4], -1).view(w.size(0), -1).long()
    values = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6], device=w.device)
    s = torch.exp2(sw.float() - 127)
    return values[codes] * s.repeat_interleave(BLK, 1)[:, :codes.size(1)]


def _plain_product(x, w, sw, bias=None):
    y = x @ _plain_weight(w, sw).t()
    return y if bias is None else y + bias


def run(st):
    c, x = st["case"], st["x"]
    kind, dt = c["kind"], x.dtype
    if own:
        if kind == "norm":
            out = st["norm"].quant(x, st["residual"]) if c["out"] == "fp8" else st["norm"](x, st["residual"])
            return out if isinstance(out, tuple) else (out,)
        if kind == "quant":
            return st["fp4"].dequant(*st["fp4"].quant(x), dt, c["k"])
        if kind == "linear" and c["norm"]:
            q, s, r = st["norm"].quant(x, st["residual"], "fp4")
            return st["linear"].quantised(q, s, dt), r
        return st[kind](x)
    if kind == "norm":
        y, held = _plain_norm(st)
        out = _plain_quant8(y) if c["out"] == "fp8" else (y.to(dt),)
        return out if held is None else (*out, held)
    if kind == "quant":
        return _plain_quant4(x.float()).to(dt)
    if kind == "linear":
        y, held = _plain_norm(st) if c["norm"] else (x.float(), None)
        y = _plain_product(_plain_quant4(y), st["w"], st["sw"], st["bias"]).to(dt)
        return y if held is None else (y, held)
    gate, up = _plain_product(_plain_quant4(x.float()), st["wg"], st["sg"]).chunk(2, dim=-1)
    return _plain_product(_plain_quant4(gate / (1 + torch.exp(-gate)) * up), st["wd"], st["sd"]).to(dt)


def work(case):
    c, kind, M, k = case, case["kind"], case["M"], case["k"]
    size = SIZE[c["dtype"]]
    if kind == "norm":
        rows = M * c["heads"]
        out = rows * -(-k // BLK8) * (BLK8 + 4) if c["out"] == "fp8" else rows * k * size
        held = 2 * rows * k * SIZE[c["residual"]] if c["residual"] else 0
        return {"bytes": rows * k * size + held + out + 4 * k, "flops": rows * k * (9 if c["out"] == "fp8" else 5)}
    if kind == "quant":
        return {"bytes": 2 * M * k * size, "flops": 3 * M * k}
    if kind == "linear":
        n = c["n"]
        return {"bytes": M * (k * (3 if c["norm"] else 1) + n) * size + n * k // 2 + n * -(-k // BLK), "flops": 2 * M * n * k}
    mats = 3 * k * c["I"]
    return {"bytes": 2 * M * k * size + mats // 2 + mats // BLK, "flops": 2 * M * mats}


# ---- 64 bits ---------------------------------------------------------------------------------------------------------

def _nearest(v, ladder):
    """v (64 bits) to the nearest of the ladder's values (ascending magnitudes), a half-way one to the entry of even place."""
    at = torch.searchsorted(ladder, v.abs().contiguous()).clamp(1, ladder.numel() - 1)
    low, high = ladder[at - 1], ladder[at]
    below, above = v.abs() - low, high - v.abs()
    take_low = (below < above) | ((below == above) & ((at - 1) % 2 == 0))
    return torch.copysign(torch.where(take_low, low, high), v)


def _exact4(x):
    """x (64 bits) -> the values of its 4-bit floats."""
    M, k = x.shape
    p = torch.nn.functional.pad(x, (0, -k % BLK)).reshape(M, -1, BLK)
    top = p.abs().amax(-1, keepdim=True)
    s = torch.exp2(torch.floor(torch.log2(torch.where(top > 0, top, 1.0)))) / 4
    # (a logarithm next to a whole number may be rounded to it)
    s = torch.where(top < 4 * s, s / 2, torch.where(top >= 8 * s, 2 * s, s))
    s = torch.where(top > 0, s, 2.0 ** LEAST).clamp_min(2.0 ** LEAST)
    ladder = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=x.device)
    return (_nearest(p / s, ladder) * s).reshape(M, -1)[:, :k]


def _exact8(x):
    """x (64 bits) -> (e4m3 values, scales): scale and quotient are held in 32 bits, so a quotient that lies between two of e4m3's
    values in 32 bits goes to the even one, as the operator says."""
    M, k = x.shape
    p = torch.nn.functional.pad(x, (0, -k % BLK8)).reshape(M, -1, BLK8)
    s = torch.maximum(p.abs().amax(-1) / E4M3_MAX, torch.full((), TINY8, dtype=torch.float64, device=x.device))
    quotient = (p / s.float().double()[..., None]).float().double()
    # steps of 2^-9 below 2^-6, of 2^(e - 3) from there
    step = torch.exp2(torch.frexp(quotient.abs().clamp_min(2.0 ** -6)).exponent.double() - 4)
    return (torch.round(quotient / step) * step).reshape(M, -1), s


def _exact_norm(st):
    h, held = st["x"].double(), None
    if st["residual"] is not None:
        held = (h + st["residual"].double()).to(st["residual"].dtype)
        h = held.double()
    gain = st["weight"].double() + (1.0 if st["offset"] else 0.0)
    return h * torch.rsqrt(h.square().sum(-1, keepdim=True) / h.size(-1) + EPS) * gain, held


def _exact_matrix(w, sw):
    n = w.size(0)
    wide = torch.empty(n, 2 * w.size(1), dtype=torch.uint8, device=w.device)
    wide[:, ::2], wide[:, 1::2] = w % 16, w // 16
    mantissa, exponent = (wide % 2).double(), (wide % 8 // 2).double()
    v = torch.where(exponent > 0, (1 + mantissa / 2) * torch.exp2(exponent - 1), mantissa / 2)
    v = torch.where(wide >= 8, -v, v)
    cols = torch.arange(v.size(1), device=w.device) // BLK
    return v * torch.exp2(sw.double() - 127)[:, cols]


def exact(case, seed):
    st = prepare(case, seed)
    c, kind = case, case["kind"]
    if kind == "norm":
        y, held = _exact_norm(st)
        out = _exact8(y) if c["out"] == "fp8" else (y,)
        return out if held is None else (*out, held)
    if kind == "quant":
        return _exact4(st["x"].double())
    if kind == "linear":
        y, held = _exact_norm(st) if c["norm"] else (st["x"].double(), None)
        y = _exact4(y) @ _exact_matrix(st["w"], st["sw"]).t()
        if st["bias"] is not None:
            y = y + st["bias"].double()
        return y if held is None else (y, held)
    gu = _exact4(st["x"].double()) @ _exact_matrix(st["wg"], st["sg"]).t()
    half = c["I"]
    h = gu[:, :half] * torch.sigmoid(gu[:, :half]) * gu[:, half:]
    return _exact4(h) @ _exact_matrix(st["wd"], st["sd"]).t()
