"""The router (torch.ops.exl3xpu_moe.moe_route, exl3xpu.routing.Router) against its definition in 64 bits, where it can go
wrong: experts around the lanes' shares, ties, masked rows, infinities and NaN, groups, biases, strides, one row and none.

ids have to be equal. A weight is a quotient of exponentials in fp32: the difference from the largest logit, its
exponential (2 units), the sum of up to 1,024 terms in ten doublings over the lanes and 16 steps in one, the quotient and
the scale, each within one rounding, with the difference d's own rounding raised by |d|: (|d| + 32) 2^-23 relative."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _router(*a, **k):
    from exl3xpu.routing import Router
    return Router(*a, **k)


def _above(a, b):
    """a before b in descending order, NaN first."""
    return (math.isnan(a) and not math.isnan(b)) or a > b


def _order(values):
    """Indices by value, descending, NaN first, equal ones by index."""
    return sorted(range(len(values)), key=lambda i: (0 if math.isnan(values[i]) else 1, 0 if math.isnan(values[i]) else -values[i], i))


def _reference(logits, topk, scoring="softmax", bias=None, n_group=1, topk_group=1, renormalize=True, scale=1.0):
    """(ids, w) in 64 bits, row by row from the definition."""
    with np.errstate(all="ignore"):
        lg = logits.double().cpu().numpy()
        M, E = lg.shape
        ids, out = np.zeros((M, topk), np.int32), np.zeros((M, topk))
        b = None if bias is None else bias.double().cpu().numpy()
        for m in range(M):
            v = lg[m]
            if scoring == "softmax":
                top = np.max(v)
                e = np.exp(v - (0 if top == -np.inf else top))
                score = e / (e.sum() if e.sum() != 0 else 1)
            else:
                score = 1 / (1 + np.exp(-v))
            key = v if b is None else score + b
            live = range(E)
            if n_group > 1:
                gs = E // n_group
                value = []
                for g in range(n_group):
                    part = [key[i] for i in (_order(key[g * gs:(g + 1) * gs]) + np.int64(g * gs))]
                    value.append(part[0] if b is None or gs == 1 else part[0] + part[1])
                kept = _order(value)[:topk_group]
                live = [i for i in range(E) if i // gs in kept]
            pick = [live[i] for i in _order([key[i] for i in live])][:topk]
            w = score[pick]
            if renormalize:
                if scoring == "softmax":
                    top = np.max(v[pick])
                    w = np.exp(v[pick] - (0 if top == -np.inf else top))
                w = w / (w.sum() if w.sum() != 0 else 1)
            ids[m], out[m] = pick, w * scale
    return ids, out


def _check(logits, topk, **k):
    ids, w = _router(topk, **k)(logits)
    torch.cuda.synchronize()
    rid, rw = _reference(logits.reshape(-1, logits.size(-1)), topk, **k)
    assert ids.dtype == torch.int32 and w.dtype == torch.float32 and ids.shape == w.shape == logits.shape[:-1] + (topk,)
    got, gw = ids.reshape(-1, topk).cpu().numpy(), w.reshape(-1, topk).double().cpu().numpy()
    np.testing.assert_array_equal(got, rid)
    lf = logits.double().reshape(-1, logits.size(-1)).cpu()
    span = torch.where(lf.isfinite() & (lf.abs() < 1e30), lf, 0.0)
    d = float(span.max() - span.min()) if lf.numel() else 0.0
    np.testing.assert_allclose(gw, rw, rtol=(min(d, 110) + 32) * 2 ** -23, atol=1e-37, equal_nan=True)
    return ids, w


@pytest.mark.parametrize("E,topk", [(1, 1), (2, 2), (7, 3), (63, 8), (64, 64), (65, 6), (128, 8), (160, 6), (257, 10),
                                    (512, 10), (513, 64), (1000, 12), (1024, 1)])
def test_route_sizes(E, topk):
    g = torch.Generator(device="cuda").manual_seed(E)
    for M in (1, 3, 4, 33):
        for dtype in DTYPES:
            lg = torch.randn(M, E, generator=g, device="cuda").mul_(2).to(dtype)
            bias = 0.1 * torch.randn(E, generator=g, device="cuda")
            for scoring in ("softmax", "sigmoid"):
                print(f"case route E={E} topk={topk} M={M} {dtype} {scoring}", flush=True)
                _check(lg, topk, scoring=scoring)
                _check(lg, topk, scoring=scoring, renormalize=False, scale=2.5)
                _check(lg, topk, scoring=scoring, bias=bias)
                _check(lg, topk, scoring=scoring, bias=bias, renormalize=False)


@pytest.mark.parametrize("E,n_group,topk_group,topk", [(256, 8, 4, 8), (160, 8, 3, 6), (96, 3, 2, 7), (64, 64, 9, 9),
                                                       (128, 32, 1, 4), (1000, 5, 2, 64), (1024, 2, 1, 3), (60, 60, 60, 60),
                                                       (6, 3, 2, 4), (512, 1, 1, 10)])
def test_route_groups(E, n_group, topk_group, topk):
    g = torch.Generator(device="cuda").manual_seed(E + n_group)
    k = dict(n_group=n_group, topk_group=topk_group)
    for dtype in DTYPES:
        lg = torch.randn(21, E, generator=g, device="cuda").to(dtype)
        lg[3] = -math.inf                                   # a row that its mask leaves empty
        lg[4, : E // 2] = -math.inf
        lg[5] = lg[5, 0]                                    # one value everywhere: the first groups, the first experts
        bias = 0.2 * torch.randn(E, generator=g, device="cuda")
        for scoring in ("softmax", "sigmoid"):
            print(f"case route groups E={E} {n_group}/{topk_group} {dtype} {scoring}", flush=True)
            _check(lg, topk, scoring=scoring, **k)
            _check(lg, topk, scoring=scoring, bias=bias, **k)


@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_route_masks_infinities_and_ties(scoring, bias):
    E, topk = 130, 9
    g = torch.Generator(device="cuda").manual_seed(5)
    lg = torch.randn(16, E, generator=g, device="cuda")
    lowest = torch.finfo(torch.float32).min
    lg[0] = -math.inf                                       # nothing left
    lg[1] = lowest                                          # the lowest finite value everywhere
    lg[2, 5:] = -math.inf                                   # fewer left than picked
    lg[3, 5:] = lowest
    lg[4, 7] = math.inf
    lg[5, [9, 120]] = math.nan
    lg[6] = math.nan
    lg[7] = 0.0
    lg[7, ::2] = -0.0                                       # the two zeros are equal
    lg[8] = lg[8].round()                                   # many ties
    lg[9, [3, 64, 65, 129]] = 50.0
    lg[10] = torch.arange(E, device="cuda").flip(0) * -1.0  # the best ones last
    lg[11, [3, 77]] = math.inf
    lg[12] *= 40
    lg[13, 1:] = -math.inf                                  # one left
    b = None
    if bias:
        b = 0.3 * torch.randn(E, generator=g, device="cuda")
        b[11] = -math.inf                                   # never wanted
        b[12] = math.inf
    for renormalize in (True, False):
        print(f"case route masks {scoring} bias={bias} renormalize={renormalize}", flush=True)
        ids, w = _check(lg, topk, scoring=scoring, bias=b, renormalize=renormalize, scale=1.5)
        assert all(len(set(r)) == topk and min(r) >= 0 and max(r) < E for r in ids.tolist())
    if not bias:
        assert ids[0].tolist() == list(range(topk)) and w[0].abs().max() == 0


@pytest.mark.parametrize("E,topk,n_group,topk_group", [(60, 60, 1, 1), (130, 9, 1, 1), (250, 12, 1, 1), (512, 10, 1, 1),
                                                       (256, 8, 8, 4), (160, 6, 8, 3)])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_route_biases_without_an_end(E, topk, n_group, topk_group, scoring):
    """Experts that the bias rules out, forces or spoils, biases that start anywhere, scores at both ends of sigmoid's range."""
    g = torch.Generator(device="cuda").manual_seed(E)
    lg = torch.randn(12, E, generator=g, device="cuda")
    lg[1] = -math.inf
    lg[2] = math.nan
    lg[3, ::3] = math.nan
    lg[4] *= 30
    lg[5, 5:] = -800.0
    lg[6, :-3] = -math.inf
    lg[7, 1::2] = 800.0
    room = torch.empty(E + 1, device="cuda")
    for at in (0, 1):
        bias = room[at:at + E]
        for kind in range(5):
            bias.copy_(0.1 * torch.randn(E, generator=g, device="cuda"))
            if kind == 1:
                bias[::4] = -math.inf
            elif kind == 2:
                bias.fill_(-math.inf)
            elif kind == 3:
                bias[[1, E - 1]] = math.inf
                bias[E // 2] = math.nan
            elif kind == 4:
                bias.zero_()
            print(f"case route bias E={E} groups={n_group} {scoring} at={at} kind={kind}", flush=True)
            _check(lg, topk, scoring=scoring, bias=bias, n_group=n_group, topk_group=topk_group)


def test_route_strides_and_shapes():
    g = torch.Generator(device="cuda").manual_seed(9)
    wide = torch.randn(12, 300, generator=g, device="cuda")
    _check(wide[:, 1:200], 8)                               # rows further apart, at an odd element
    _check(wide[:, ::3], 8)
    _check(wide.t(), 3)
    _check(wide[:1].expand(5, 300), 4)                      # one row for all
    _check(wide.view(3, 4, 300), 8)                         # leading dimensions
    _check(wide[0], 8)
    ids, w = _router(8)(wide[:0])
    assert ids.shape == w.shape == (0, 8)
    assert [t.shape for t in _router(2)(wide.view(3, 4, 300)[:, :0])] == [(3, 0, 2)] * 2


def test_route_rows_past_32_bits():
    g = torch.Generator(device="cuda").manual_seed(15)
    far = torch.zeros((1 << 31) + 600, dtype=torch.bfloat16, device="cuda")
    lg = far.as_strided((2, 512), (1 << 31, 1))
    lg.copy_(torch.randn(2, 512, generator=g, device="cuda"))
    print("case route rows 2^32 bytes apart", flush=True)
    _check(lg, 10)
    _check(lg, 10, scoring="sigmoid", bias=0.1 * torch.randn(512, generator=g, device="cuda"))


def test_route_feeds_the_experts_of_two_streams():
    """Two routers at once, each with its experts, on two streams."""
    from exl3xpu.moe_offload import ExpertStore
    from exl3xpu.synth import expert_blob
    g = torch.Generator(device="cuda").manual_seed(17)
    store = ExpertStore(256, 128, 3, 8, 8, max_layers=1)
    store.add_layer("layer0", torch.stack([expert_blob(7, e, 256, 128, 3) for e in range(8)]))
    store.make_resident("layer0", range(8))
    torch.cuda.synchronize()
    routers = [_router(2), _router(3, scoring="sigmoid", bias=0.1 * torch.randn(8, generator=g, device="cuda"))]
    lg = [torch.randn(m, 8, generator=g, device="cuda") for m in (3, 70)]
    want = [[t.clone() for t in r(x)] for r, x in zip(routers, lg)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in routers], [[], []]
    for _ in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(routers[i](lg[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for i in range(2) for pair in got[i] for a, b in zip(pair, want[i]))
    x = torch.randn(3, 256, generator=g, device="cuda").bfloat16()
    assert torch.equal(store.forward_routed("layer0", x, lg[0], routers[0], cached=False), store.forward("layer0", x, *want[0]))


def test_route_keys_closer_than_32_bits():
    """Scores + bias that differ by less than 32 bits hold: the choice is that of 64."""
    E, M = 256, 512
    g = torch.Generator(device="cuda").manual_seed(11)
    lg = torch.randn(M, E, generator=g, device="cuda")
    want = 0.5 + torch.arange(E, device="cuda").double() * 1e-9
    for m in range(4):                                      # rows whose scores + bias climb in steps of 1e-9
        lg[m] = torch.logit((want[torch.randperm(E, generator=g, device="cuda")])).float()
    _check(lg, 8, scoring="sigmoid", bias=torch.full((E,), 0.25, device="cuda"))
    _check(lg, 8, scoring="sigmoid", bias=1e-7 * torch.randn(E, generator=g, device="cuda"), n_group=8, topk_group=4)


def test_route_refusals():
    lg = torch.randn(4, 64, device="cuda")
    for k in (dict(topk=9, n_group=8, topk_group=1), dict(topk=2, n_group=7), dict(topk=65)):
        with pytest.raises((RuntimeError, ValueError)):
            _router(**k)(lg)
    with pytest.raises(RuntimeError):
        _router(2)(lg.double())
    with pytest.raises(RuntimeError):
        _router(2)(torch.randn(4, 1025, device="cuda"))
    with pytest.raises(RuntimeError):
        _router(2, bias=torch.zeros(63, device="cuda"))(lg)
    with pytest.raises(RuntimeError):
        _router(2, bias=torch.zeros(64))(lg)                # a bias in host memory
    with pytest.raises(NotImplementedError):
        _router(2)(lg.cpu())


def test_route_on_a_stream_and_in_a_graph():
    g = torch.Generator(device="cuda").manual_seed(13)
    r = _router(10, bias=0.1 * torch.randn(512, generator=g, device="cuda"), scoring="sigmoid")
    inputs = [torch.randn(5, 512, generator=g, device="cuda") for _ in range(4)]
    want = [[t.clone() for t in r(x)] for x in inputs]
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = r(inputs[1])
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want[1]))
    x = inputs[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ids, w = r(x)
    for i in (1, 2, 3, 0):
        x.copy_(inputs[i])
        graph.replay()
        r(inputs[3 - i])                                    # eager work between the replays
        torch.cuda.synchronize()
        assert torch.equal(ids, want[i][0]) and torch.equal(w, want[i][1])


@pytest.mark.parametrize("bias", [False, True])
def test_route_sigmoid_weights_far_below(bias):
    """Renormalised sigmoid weights are those of the scores also where every pick's score is far below fp32's smallest."""
    g = torch.Generator(device="cuda").manual_seed(19)
    at = torch.tensor([-10.0, -15.0, -16.0, -16.6, -16.7, -17.0, -18.0, -20.0, -50.0, -80.0, -86.0, -87.5, -88.0, -88.8, -90.0, -100.0,
                       -200.0, -500.0, -650.0], device="cuda")
    for E, topk, groups in ((64, 8, {}), (130, 9, {}), (512, 10, {}), (256, 8, dict(n_group=8, topk_group=4))):
        lg = torch.randn(40, E, generator=g, device="cuda")
        lg[:19] += at[:, None]
        lg[19] = -100.0
        b = 0.1 * torch.randn(E, generator=g, device="cuda") if bias else None
        for dtype in DTYPES:
            print(f"case route sigmoid far below E={E} bias={bias} {dtype}", flush=True)
            ids, w = _check(lg.to(dtype), topk, scoring="sigmoid", bias=b, scale=2.5, **groups)
            assert torch.allclose(w.sum(-1), torch.full((40,), 2.5, device="cuda"), rtol=1e-5)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_route_masked_experts_and_a_bias(scoring):
    """A logit of -inf leaves the bias alone to compete; a bias of -inf rules the expert out. NaN and +inf with softmax scores and
    a bias: the first experts that compete, weighed by their own logits."""
    lg = torch.full((3, 8), -3.0, device="cuda")
    lg[:, 6] = -math.inf
    bias = torch.zeros(8, device="cuda")
    bias[6] = 2.0
    ids, w = _check(lg, 2, scoring=scoring, bias=bias)
    assert ids.tolist() == [[6, 0]] * 3 and w.tolist() == [[0.0, 1.0]] * 3
    bias[6] = -math.inf
    ids, w = _check(lg, 2, scoring=scoring, bias=bias)
    assert ids.tolist() == [[0, 1]] * 3 and w.tolist() == [[0.5, 0.5]] * 3
    lg[1, 7], lg[2, 7] = math.nan, math.inf
    ids, w = _router(2, scoring=scoring, bias=bias)(lg)
    torch.cuda.synchronize()
    if scoring == "softmax":
        assert ids.tolist() == [[0, 1]] * 3 and w.tolist() == [[0.5, 0.5]] * 3
        assert _router(2, bias=bias, renormalize=False)(lg)[1][1:].isnan().all()
    else:
        assert ids.tolist() == [[0, 1], [7, 0], [7, 0]] and w[1].isnan().all() and w[2].isfinite().all()
