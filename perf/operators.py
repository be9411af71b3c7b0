"""Timed cases of the router and of the 8-bit float linear: the operators a program runs beside the EXL3 experts.

  route   logits -> the picks of each row and their weights, as the expert calls take them
  quant   rows -> e4m3 with one scale per 128 columns
  silu    silu(gate) * up of a fused gate|up row -> e4m3 with one scale per 128 columns
  linear  x @ W^T with W in e4m3 and one scale per 128 x 128 block; x is quantised as `quant` does
  mlp     the gated MLP of a shared expert: linear (gate|up), silu, linear (down)

Sizes are this repository's own (bench.py: hidden 2048 and 4096, intermediate 512, 512 experts with top-10, 128 with top-8,
the dense projections of one decoder layer) and ragged ones around them.
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
BLK = 128
E4M3_MAX = 448.0
TINY = 2.0 ** -80             # the smallest scale: a block of zeros has it


def _route(name, M, E, topk, scoring="softmax", groups=1, kept=1, bias=False, renorm=True, scale=1.0, masked=0,
           dtype="fp32"):
    return {"name": name, "kind": "route", "M": M, "E": E, "topk": topk, "scoring": scoring, "groups": groups,
            "kept": kept, "bias": bias, "renorm": renorm, "scale": scale, "masked": masked, "dtype": dtype}


def _rows(name, kind, M, k, dtype="bf16"):
    return {"name": name, "kind": kind, "M": M, "k": k, "dtype": dtype}


def _linear(name, M, k, n, bias=False, dtype="bf16"):
    return {"name": name, "kind": "linear", "M": M, "k": k, "n": n, "bias": bias, "dtype": dtype}


def listed():
    return [
        # one user's token, once per layer: pure latency
        _route("route_bs1", 1, 512, 10),
        # a decode batch's balanced router: sigmoid scores, a bias for balance, 4 of 8 groups
        _route("route_groups_200", 200, 256, 8, "sigmoid", groups=8, kept=4, bias=True, scale=2.5),
        # the largest chunk of a prompt
        _route("route_8192", 8192, 512, 10),
        # the rows of a ragged fp16 prompt, and the largest chunk
        _rows("quant_301", "quant", 301, 1000, "fp16"),
        _rows("quant_8192", "quant", 8192, 2048),
        # a decode batch's shared expert, and the largest chunk's
        _rows("silu_64", "silu", 64, 512),
        _rows("silu_8192", "silu", 8192, 512),
        # one user's token through the widest projection group
        _linear("linear_bs1", 1, 2048, 12288),
        # a decode batch through the output projection
        _linear("linear_m40", 40, 4096, 2048),
        # a ragged chunk, sizes that end inside a block, a bias, fp32 in and out
        _linear("linear_ragged", 777, 2000, 1000, bias=True, dtype="fp32"),
        # the largest chunk through the widest projection group
        _linear("linear_8192", 8192, 2048, 12288),
        # a small decode batch through the whole shared expert
        {"name": "mlp_bs4", "kind": "mlp", "M": 4, "k": 2048, "I": 512, "dtype": "bf16"},
    ]


def draw(rng):
    def logint(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(["route", "route", "quant", "silu", "linear", "linear", "linear", "mlp"])
    dt = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if kind == "route":
        E, topk, groups, kept = rng.choice([(512, 10, 1, 1), (128, 8, 1, 1), (256, 8, 8, 4), (160, 6, 8, 3), (60, 4, 1, 1)])
        c = _route("", logint(1, 8192), E, topk, rng.choice(["softmax", "sigmoid"]), groups, kept, rng.random() < 0.4,
                   rng.random() < 0.7, rng.choice([1.0, 1.0, 2.5]), rng.choice([0, 0, 0, E // 4, E - 2]), dt)
    elif kind == "quant":
        c = _rows("", kind, logint(1, 8192), rng.choice([2048, 4096, logint(100, 4500)]), dt)
    elif kind == "silu":
        c = _rows("", kind, logint(1, 8192), rng.choice([512, 640, logint(60, 2000)]), dt)
    elif kind == "linear":
        k, n = rng.choice([(2048, 12288), (4096, 2048), (2048, 1024), (512, 2048), (logint(100, 4500), logint(100, 4500))])
        c = _linear("", logint(1, 8192), k, n, rng.random() < 0.3, dt)
    else:
        c = {"kind": "mlp", "M": logint(1, 4096), "k": rng.choice([2048, 4096]), "I": rng.choice([512, 640, 1024]),
             "dtype": rng.choice(["bf16", "fp16"])}
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
    """e4m3 [n, k] and fp32 scales [ceil(n / 128), ceil(k / 128)] of a normal matrix."""
    w = torch.randn(n, k, generator=g, device=DEV) / math.sqrt(k)
    nb, kb = -(-n // BLK), -(-k // BLK)
    p = torch.zeros(nb * BLK, kb * BLK, device=DEV)
    p[:n, :k] = w
    p = p.view(nb, BLK, kb, BLK)
    s = p.abs().amax((1, 3)) / E4M3_MAX
    q = (p / s[:, None, :, None]).view(nb * BLK, kb * BLK)[:n, :k].to(torch.float8_e4m3fn).contiguous()
    return q, s


def prepare(case, seed):
    kind, M = case["kind"], case["M"]
    g = _gen(seed, 1)
    st = {"case": case}
    if own:
        pkg = os.path.join(os.getcwd(), "qwen38-flash-next-b70-offload_amd")
        if pkg not in sys.path:
            sys.path.insert(0, pkg)
        from exl3xpu import fp8, routing
        st["fp8"] = fp8
    if kind == "route":
        E = case["E"]
        # some experts are wanted more than others, in an order of their own; the last `masked` of them are not there
        rank = torch.randperm(E, generator=g, device=DEV).float()
        lg = torch.randn(M, E, generator=g, device=DEV) - 0.4 * torch.log1p(rank)
        if case["masked"]:
            lg[:, E - case["masked"]:] = -math.inf
        st["logits"] = lg.to(DTYPES[case["dtype"]])
        st["bias"] = 0.05 * torch.randn(E, generator=g, device=DEV) if case["bias"] else None
        if own:
            st["router"] = routing.Router(case["topk"], scoring=case["scoring"], bias=st["bias"], n_group=case["groups"],
                                          topk_group=case["kept"], renormalize=case["renorm"], scale=case["scale"])
    elif kind in ("quant", "silu"):
        st["x"] = _activations(g, M, case["k"] * (2 if kind == "silu" else 1), case["dtype"])
    elif kind == "linear":
        st["x"] = _activations(g, M, case["k"], case["dtype"])
        st["w"], st["sw"] = _weight(g, case["n"], case["k"])
        st["bias"] = 0.1 * torch.randn(case["n"], generator=g, device=DEV) if case["bias"] else None
        if own:
            st["linear"] = fp8.Fp8Linear(st["w"], st["sw"], st["bias"])
    else:
        k, I = case["k"], case["I"]  # noqa: E741
        st["x"] = _activations(g, M, k, case["dtype"])
        st["wg"], st["sg"] = _weight(g, 2 * I, k)
        st["wd"], st["sd"] = _weight(g, k, I)
        if own:
            st["mlp"] = fp8.Fp8Mlp(fp8.Fp8Linear(st["wg"], st["sg"]), fp8.Fp8Linear(st["wd"], st["sd"]))
    return st


# ---- the plain forms ------------------------------------------------------------------------------------------------

def _plain_route(lg, bias, c):
    M, E, topk, G = lg.size(0), lg.size(1), c["topk"], c["groups"]
    lf = lg.float()
    if c["scoring"] == "softmax":
        top = lf.amax(-1, keepdim=True)
        e = torch.exp(lf - torch.where(top == -math.inf, 0.0, top))
        total = e.sum(-1, keepdim=True)
        score = e / torch.where(total == 0, 1.0, total)
    else:
        score = 1 / (1 + torch.exp(-lf))
    if bias is None:
        key = lf + 0.0                      # both scores rise with the logit
    else:                                   # 64 bits: values next to each other decide the order
        ld = lg.double()
        if c["scoring"] == "softmax":
            top = ld.amax(-1, keepdim=True)
            e = torch.exp(ld - torch.where(top == -math.inf, 0.0, top))
            total = e.sum(-1, keepdim=True)
            key = e / torch.where(total == 0, 1.0, total) + bias.double()
        else:
            key = 1 / (1 + torch.exp(-ld)) + bias.double()
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices
    if G > 1:
        by = key.view(M, G, E // G)
        value = by.amax(-1) if bias is None else by.topk(min(2, E // G), dim=-1).values.sum(-1)
        best = torch.sort(value, dim=-1, descending=True, stable=True).indices[:, :c["kept"]]
        kept = torch.zeros(M, G, dtype=torch.int32, device=lg.device).scatter_(1, best, 1)
        there = kept.gather(1, order // (E // G))
        order = order.gather(1, torch.sort(there, dim=-1, descending=True, stable=True).indices)
    ids = order[:, :topk]
    w = score.gather(1, ids)
    if c["renorm"]:
        if c["scoring"] == "softmax":       # over the picks' own logits: nothing underflows
            p = lf.gather(1, ids)
            top = p.amax(-1, keepdim=True)
            w = torch.exp(p - torch.where(top == -math.inf, 0.0, top))
        total = w.sum(-1, keepdim=True)
        w = w / torch.where(total == 0, 1.0, total)
    return ids.to(torch.int32), w * c["scale"]


def _plain_quant(x):
    """x fp32 [M, k] -> e4m3 [M, k up to a multiple of 128] (zeros behind k), fp32 [M, ceil(k / 128)]. Scale and quotient
    are divided in 64 bits and rounded to 32: a quotient one step off would cross the border between two e4m3 values."""
    M, k = x.shape
    kb = -(-k // BLK)
    p = torch.zeros(M, kb * BLK, device=x.device)
    p[:, :k] = x
    p = p.view(M, kb, BLK)
    s = (p.abs().amax(-1).double() / E4M3_MAX).float().clamp_min(TINY)
    return (p.double() / s[..., None].double()).float().view(M, kb * BLK).to(torch.float8_e4m3fn), s


def _plain_silu(gu):
    g, u = gu.float().chunk(2, dim=-1)
    return g / (1 + torch.exp(-g)) * u


def _wide(s, n, k):
    return s.repeat_interleave(BLK, 0)[:n].repeat_interleave(BLK, 1)[:, :k]


def _plain_product(q, s, w, sw, bias, dtype):
    n, k = w.shape
    x = (q.float().view(q.size(0), -1, BLK) * s[..., None]).view(q.size(0), -1)[:, :k]
    y = x @ (w.float() * _wide(sw, n, k)).t()
    return (y if bias is None else y + bias).to(dtype)


def run(st):
    c = st["case"]
    kind = c["kind"]
    if own:
        if kind == "route":
            return st["router"](st["logits"])
        if kind == "quant":
            return st["fp8"].quant(st["x"])
        if kind == "silu":
            return st["fp8"].silu_mul_quant(st["x"])
        return st[kind](st["x"])
    if kind == "route":
        return _plain_route(st["logits"], st["bias"], c)
    if kind == "quant":
        return _plain_quant(st["x"].float())
    if kind == "silu":
        return _plain_quant(_plain_silu(st["x"]))
    x, dt = st["x"], st["x"].dtype
    if kind == "linear":
        return _plain_product(*_plain_quant(x.float()), st["w"], st["sw"], st["bias"], dt)
    gu = _plain_product(*_plain_quant(x.float()), st["wg"], st["sg"], None, dt)
    return _plain_product(*_plain_quant(_plain_silu(gu)), st["wd"], st["sd"], None, dt)


def work(case):
    c, kind, M = case, case["kind"], case["M"]
    if kind == "route":
        return {"bytes": M * c["E"] * SIZE[c["dtype"]] + 8 * M * c["topk"] + (4 * c["E"] if c["bias"] else 0),
                "flops": M * c["E"] * (6 if c["bias"] or not c["renorm"] else 1) + 8 * M * c["topk"]}
    kb = -(-c["k"] // BLK)
    if kind in ("quant", "silu"):
        read = M * c["k"] * SIZE[c["dtype"]] * (2 if kind == "silu" else 1)
        return {"bytes": read + M * kb * (BLK + 4), "flops": M * c["k"] * (8 if kind == "silu" else 3)}
    if kind == "linear":
        n = c["n"]
        return {"bytes": M * (c["k"] + n) * SIZE[c["dtype"]] + n * c["k"] + 4 * kb * -(-n // BLK), "flops": 2 * M * n * c["k"]}
    mats = 3 * c["k"] * c["I"]
    return {"bytes": 2 * M * c["k"] * SIZE[c["dtype"]] + mats + 4 * mats // BLK ** 2, "flops": 2 * M * mats}


# ---- 64 bits ---------------------------------------------------------------------------------------------------------

def _exact_e4m3(v):
    """v (64 bits) to the nearest of e4m3's values, halves to even: steps of 2^-9 below 2^-6, of 2^(e - 3) from there."""
    step = torch.exp2(torch.frexp(v.abs().clamp_min(2.0 ** -6)).exponent.double() - 4)
    return torch.round(v / step) * step


def _exact_quant(x):
    """x (64 bits) -> (q, the scale as it is held, the scale in 64 bits). The scale and the quotient x / scale are held in
    32 bits, so a quotient that lies between two of e4m3's values in 32 bits goes to the even one, as the operators say."""
    M, k = x.shape
    kb = -(-k // BLK)
    p = torch.nn.functional.pad(x, (0, kb * BLK - k)).reshape(M, kb, BLK)
    s = torch.maximum(p.abs().amax(-1) / E4M3_MAX, torch.full((), TINY, dtype=torch.float64, device=x.device))
    held = s.float().double()
    return _exact_e4m3((p / held[..., None]).float().double()), held, s


def _exact_product(x, w, sw, bias):
    n, k = w.shape
    q, held, _ = _exact_quant(x)
    a = (q * held[..., None]).reshape(x.size(0), -1)[:, :k]
    rows, cols = torch.arange(n, device=x.device) // BLK, torch.arange(k, device=x.device) // BLK
    b = w.double() * sw.double()[rows][:, cols]
    y = a @ b.t()
    return y if bias is None else y + bias.double()


def _exact_silu(gu):
    h = gu.size(1) // 2
    g, u = gu[:, :h].double(), gu[:, h:].double()
    return g * torch.sigmoid(g) * u


def exact(case, seed):
    st = prepare(case, seed)
    c, kind = case, case["kind"]
    if kind == "route":
        lg, M, E, G, topk = st["logits"].double(), c["M"], c["E"], c["groups"], c["topk"]
        gone = lg == -math.inf
        sc = torch.softmax(lg.masked_fill(gone, -1e300), -1).masked_fill(gone, 0) if c["scoring"] == "softmax" else torch.sigmoid(lg)
        key = lg if st["bias"] is None else sc + st["bias"].double()
        if G > 1:
            v = key.reshape(M, G, -1)
            v = v.max(-1).values if st["bias"] is None else v.sort(-1).values[..., -2:].sum(-1)
            # the place of each group among its row's: those above it, and its equals before it
            at = torch.arange(G, device=DEV)
            before = (v[:, None] > v[:, :, None]) | ((v[:, None] == v[:, :, None]) & (at[None, None] < at[None, :, None]))
            out = (before.sum(-1) >= c["kept"]).repeat_interleave(E // G, 1)
        else:
            out = torch.zeros_like(gone)
        # keys replaced by their place: kept groups first, then the key, then the index
        low = torch.where(out, -2e308, torch.where(key == -math.inf, -1e308, key))
        ids = torch.sort(-low, dim=-1, stable=True).indices[:, :topk]
        w = sc.gather(1, ids)
        if c["renorm"]:
            t = w.sum(-1, keepdim=True)
            w = torch.where(t > 0, w / t, torch.zeros_like(w))
        return ids.to(torch.int32), w * c["scale"]
    if kind in ("quant", "silu"):
        q, _, s = _exact_quant(st["x"].double() if kind == "quant" else _exact_silu(st["x"]))
        return q.reshape(c["M"], -1), s
    if kind == "linear":
        return _exact_product(st["x"].double(), st["w"], st["sw"], st["bias"])
    # the row between the two products is held in the activations' type
    gu = _exact_product(st["x"].double(), st["wg"], st["sg"], None).to(st["x"].dtype)
    return _exact_product(_exact_silu(gu), st["wd"], st["sd"], None)
