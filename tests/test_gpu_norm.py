"""The norm (torch.ops.exl3xpu_C.rms_norm, exl3xpu.norm) against its definition in 64 bits, where it can go wrong: sizes around
the blocks and the rows that one wave, one workgroup or two passes hold, strides, odd addresses, zero, tiny, huge, infinite and
NaN rows, one row and none, streams and graphs.

The held sum has to be equal, bit for bit (a fp32 addition and a rounding). The sum of squares and all that follows is in 64 bits, where
its roundings (2^-53 each, at most 8 ceil(k / 8,192) + 50 of them) are below 2^-44: y is within 2^-24 (the rounding to 32 bits) and
2^-44 of itself, and half a step of its type. Quantised outputs are those of some value in that range (e4m3's scale and quotient with
one rounding each)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
EPS = 1e-6


def _norm():
    from exl3xpu.norm import RmsNorm
    return RmsNorm


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _odd(t):
    """The same values at an odd element of their storage."""
    store = torch.zeros(t.numel() + 3, dtype=t.dtype, device=t.device)
    v = store[1:1 + t.numel()].view(t.shape)
    v.copy_(t)
    return v


def _units(k):
    return 1 + 2.0 ** -20                                    # in 2^-24


def _ref(h, weight, eps=EPS):
    y = h.double() / torch.sqrt(h.double().square().mean(-1, keepdim=True) + eps)
    return y if weight is None else y * weight.double()


def _held(x, residual):
    return (x.float() + residual.float()).to(residual.dtype)


def _check_rows(y, ref, k):
    half = torch.finfo(y.dtype).eps / 2
    tol = _units(k) * 2.0 ** -24 * ref.abs()
    tol = tol + half * (ref.abs() + tol) + torch.finfo(y.dtype).smallest_normal * torch.finfo(y.dtype).eps
    bad = ~((y.double() - ref).abs() <= tol)
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist(), float(((y.double() - ref).abs() / tol).max()))


def _e4m3(v):
    a = v.abs().clamp_min(2.0 ** -6)
    step = torch.exp2(torch.floor(torch.log2(a)).clamp(-6, 8) - 3)
    return torch.round(v / step) * step


def _check_fp8(q, s, ref, k):
    M = ref.size(0)
    p = torch.nn.functional.pad(ref, (0, -k % 128)).reshape(M, -1, 128)
    rs = (p.abs().amax(-1) / 448).clamp_min(2.0 ** -80)
    u = _units(k) * 2.0 ** -24
    assert q.dtype == torch.float8_e4m3fn and q.shape == (M, p.size(1) * 128) and s.shape == rs.shape
    assert ((s.double() - rs).abs() <= (u + 2.0 ** -24) * rs).all()
    quo = (p / rs[..., None]).reshape(M, -1)
    off = 2 * u + 2 * 2.0 ** -24
    lo, hi = _e4m3(quo.abs() * (1 - off)), _e4m3((quo.abs() * (1 + off)).clamp_max(448.0))
    got = q.double()
    assert ((got.abs() >= lo) & (got.abs() <= hi) & ((got == 0) | (got.sign() == quo.sign()))).all()
    assert not q.view(torch.uint8)[:, k:].any()


def _check_fp4(q, s, ref, k):
    M, cols = ref.size(0), -(-k // 128) * 128
    u = _units(k) * 2.0 ** -24
    p = torch.nn.functional.pad(ref, (0, cols - k)).reshape(M, -1, 32)
    top = p.abs().amax(-1)

    def exponent(v):
        return torch.where(v > 0, (torch.frexp(v).exponent - 3).clamp_min(-126) + 127, 1)
    got_s = s.reshape(M, -1)
    blocks = -(-k // 32)
    assert q.shape == (M, cols // 2) and s.shape == (M, -(-k // 256), 8) and not got_s[:, blocks:].any()
    e = got_s[:, :blocks].int()
    assert ((e >= exponent(top * (1 - u))[:, :blocks]) & (e <= exponent(top * (1 + u))[:, :blocks])).all()
    quo = (p[:, :blocks] * torch.exp2(127 - e.double())[..., None])
    v = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=q.device)
    codes = torch.stack([q & 15, q >> 4], -1).view(M, -1, 32)
    assert not codes[:, blocks:].any() and not codes.view(M, -1)[:, k:].any()
    codes = codes[:, :blocks].long()
    mid = (v[1:] + v[:-1]) / 2
    lo = torch.bucketize(quo.abs() * (1 - u) * (1 - 1e-12), mid, right=False)
    hi = torch.bucketize(quo.abs() * (1 + u) * (1 + 1e-12), mid, right=True)
    got = codes % 8
    assert ((got >= lo) & (got <= hi) & ((got == 0) | ((codes >= 8) == (quo < 0)))).all()


KS = [1, 7, 8, 31, 64, 127, 128, 129, 250, 256, 264, 500, 640, 1000, 2048, 2056, 4096, 5001, 8192, 8200, 20000, 32768, 32776, 40001]


@pytest.mark.parametrize("k", KS)
def test_norm(k):
    g = _gen(k)
    for dtype in DTYPES:
        for M in (1, 2, 5, 33) if k < 6000 else (1, 3):
            for with_weight in (True, False):
                x = (torch.randn(M, k, generator=g, device="cuda") * torch.exp(2 * torch.randn(M, 1, generator=g, device="cuda"))).to(dtype)
                if M > 2:
                    x[1] = 0
                weight = torch.randn(k, generator=g, device="cuda") + 1 if with_weight else None
                norm = _norm()(weight, EPS)
                print(f"case norm k={k} M={M} {dtype} weight={with_weight}", flush=True)
                y = norm(x)
                torch.cuda.synchronize()
                assert y.dtype == dtype and y.shape == x.shape
                ref = _ref(x, weight)
                _check_rows(y, ref, k)
                assert torch.equal(norm(_odd(x)), y)
                q, s = norm.quant(x)
                _check_fp8(q, s, ref, k)
                q4, s4 = norm.quant(x, form="fp4")
                _check_fp4(q4, s4, ref, k)
                for form, want in (("fp8", (q, s)), ("fp4", (q4, s4))):
                    got = norm.quant(_odd(x), None, form, rows=True)
                    assert all(torch.equal(a.view(torch.uint8) if a.dtype != torch.float32 else a, b.view(torch.uint8) if b.dtype != torch.float32 else b) for a, b in zip(got, want))
                    assert len(got) == 3 and torch.equal(got[2], y)
                for rtype in {dtype, torch.float32}:
                    res = 2 * torch.randn(M, k, generator=g, device="cuda").to(rtype)
                    y2, h = norm(x, res)
                    torch.cuda.synchronize()
                    assert h.dtype == rtype and torch.equal(h, _held(x, res))
                    ref2 = _ref(h, weight)
                    _check_rows(y2, ref2, k)
                    if rtype == dtype:
                        assert torch.equal(norm(h), y2)              # the norm of what is held
                    q, s, y3, h3 = norm.quant(x, _odd(res), "fp8", rows=True)
                    _check_fp8(q, s, ref2, k)
                    assert torch.equal(y3, y2) and torch.equal(h3, h)
                    q, s, h3 = norm.quant(x, res, "fp4")
                    _check_fp4(q, s, ref2, k)
                    assert torch.equal(h3, h)


def test_fp4_outputs_are_those_of_the_norm():
    """4-bit rows of the norm in fp32: dividing by a power of two is exact, so quantising its rows afterwards is the same."""
    from exl3xpu import fp4
    g = _gen(3)
    for M, k in ((1, 128), (40, 2048), (7, 1000), (300, 4096), (2, 12288)):
        norm = _norm()(torch.randn(k, generator=g, device="cuda"), EPS)
        x = torch.randn(M, k, generator=g, device="cuda") * 3
        got, want = norm.quant(x, None, "fp4"), fp4.quant(norm(x))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_fp8_outputs_next_to_a_border():
    """Of 4 million values none is on the wrong side of a border between two of e4m3's: the norm is computed in 64 bits, and only
    its scale and its quotient are rounded to 32, as the definition says."""
    g = _gen(4)
    for k in (128, 500, 2048, 4096):
        M = 4_000_000 // k
        norm = _norm()(torch.randn(k, generator=g, device="cuda") + 1, EPS)
        x = torch.randn(M, k, generator=g, device="cuda").bfloat16()
        q, s = norm.quant(x)
        p = torch.nn.functional.pad(_ref(x, norm.weight, float(torch.tensor(EPS))), (0, -k % 128)).reshape(M, -1, 128)
        rs = (p.abs().amax(-1) / 448).float().double().clamp_min(2.0 ** -80)
        want = _e4m3((p / rs[..., None]).float().double()).copysign(p).reshape(M, -1)
        assert int((s.double() != rs).sum()) == 0 and int((q.double() != want).sum()) == 0


@pytest.mark.parametrize("k", [64, 96, 128, 200, 256, 512])
def test_heads_inside_wider_rows(k):
    g = _gen(k)
    for dtype in DTYPES:
        for tokens, heads, wide in ((1, 1, 1), (1, 4, 6), (5, 1, 3), (37, 16, 20), (300, 3, 5)):
            print(f"case norm heads k={k} {tokens} x {heads} {dtype}", flush=True)
            rows = torch.randn(tokens, wide * k + 24, generator=g, device="cuda").to(dtype)
            norm = _norm()(torch.randn(k, generator=g, device="cuda"), EPS)
            for first in (0, 8, 3):
                x = rows[:, first:first + heads * k].view(tokens, heads, k)
                y = norm(x)
                torch.cuda.synchronize()
                assert torch.equal(y, norm(x.contiguous())) and y.is_contiguous()
                _check_rows(y.view(-1, k), _ref(x, norm.weight).view(-1, k), k)
                for form in ("fp8", "fp4"):
                    for a, b in zip(norm.quant(x, None, form), norm.quant(x.contiguous(), None, form)):
                        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
                res = torch.randn(tokens, heads, k, generator=g, device="cuda").to(dtype)
                assert all(torch.equal(a, b) for a, b in zip(norm(x, res), norm(x.contiguous(), res)))
    # other orders of the sizes and strides are copied first
    x = torch.randn(4, 6, 5, k, generator=g, device="cuda")
    for v in (x, x.transpose(0, 2), x[:, ::2], x[:, :, :, ::2], x[:1].expand(4, 6, 5, k), x[0].transpose(0, 1), x[0, :, :1].expand(6, 5, k)):
        norm = _norm()(torch.randn(v.size(-1), generator=g, device="cuda"), EPS)
        assert torch.equal(norm(v), norm(v.contiguous()))
        assert all(torch.equal(a, b) for a, b in zip(norm(v, v), norm(v.contiguous(), v.contiguous())))


def test_infinities_nan_and_extremes():
    for k in (200, 2048, 6000, 20000, 40000):
        x = torch.randn(8, k, generator=_gen(5), device="cuda")
        x[0, 5] = math.inf
        x[1, k - 1] = -math.inf
        x[2, 100] = math.nan
        x[3] *= 1e37                                         # squares past fp32, which 64 bits hold
        x[4] *= 1e-30
        x[5] = 0
        x[6, 150] = 1e18
        norm = _norm()(None, EPS)
        y = norm(x)
        torch.cuda.synchronize()
        assert y[0, 5].isnan() and not y[0, 6:].any() and y[1, -1].isnan() and not y[1, :-1].any()
        assert y[2].isnan().all() and not y[5].any()
        _check_rows(y[[3, 4, 6, 7]], _ref(x[[3, 4, 6, 7]], None), k)
        q, s = norm.quant(x)
        assert s[0, 0].isnan() and s[2].isnan().all() and s[3:].isfinite().all() and s[0, 1:].isfinite().all()
        q, s = norm.quant(x, None, "fp4")
        flat = s.reshape(8, -1)[:, :-(-k // 32)]
        assert flat[0, 0] == 255 and (flat[0, 1:] == 1).all() and (flat[2] == 255).all() and (flat[3:] < 255).all()
        # a weight of infinity makes its column infinite and nothing behind the row
        w = torch.ones(k, device="cuda")
        w[3] = math.inf
        y = _norm()(w, EPS)(x[7:])
        assert y[0, 3].isinf() and y[0, 4:].isfinite().all()
        for form in ("fp8", "fp4"):
            q, s = _norm()(w, EPS).quant(x[7:], None, form)
            assert not q.view(torch.uint8)[:, k if form == "fp8" else -(-k // 2):].any()


def test_large_and_small_eps():
    x = torch.randn(3, 700, generator=_gen(6), device="cuda") * 1e-3
    for eps in (2.0 ** -126, 1e-12, 1e-5, 1.0, 1e30):
        _check_rows(_norm()(None, eps)(x), _ref(x, None, eps), 700)


def test_empty_and_one_row():
    norm = _norm()(torch.ones(300, device="cuda"), EPS)
    x = torch.randn(3, 300, generator=_gen(7), device="cuda").bfloat16()
    assert norm(x[:0]).shape == (0, 300) and norm(x.view(1, 3, 300)[:, :0]).shape == (1, 0, 300)
    q, s, y, h = norm.quant(x[:0], x[:0], "fp4", rows=True)
    assert q.shape == (0, 192) and s.shape == (0, 2, 8) and y.shape == h.shape == (0, 300)
    assert torch.equal(norm(x[0]), norm(x)[0]) and torch.equal(norm.quant(x[0], None, "fp4")[1], norm.quant(x, None, "fp4")[1][0])


def test_c_abi_in_place_and_what_is_behind():
    """held may be the residual itself; rows behind the last one and a wider scale stage are left as they were."""
    from exl3xpu import capi
    L, st = capi.lib(), torch.cuda.current_stream().cuda_stream
    g = _gen(8)
    for k in (96, 1000, 2048, 9000, 40000):
        M = 5
        x = torch.randn(M, k + 8, generator=g, device="cuda").bfloat16()
        res = torch.randn(M + 1, k, generator=g, device="cuda")
        norm = _norm()(torch.randn(k, generator=g, device="cuda"), EPS)
        want = norm.quant(x[:, :k], res[:M], "fp4", rows=True)
        y = torch.full((M + 1, k), 7.0, dtype=torch.bfloat16, device="cuda")
        q = torch.full((M + 1, -(-k // 128) * 64), 99, dtype=torch.uint8, device="cuda")
        s = torch.full((-(-k // 256), M + 3, 8), 99, dtype=torch.uint8, device="cuda")
        last = res[M].clone()
        print(f"case norm c-abi k={k}", flush=True)
        capi.check(L.exl3_rms_norm(x.data_ptr(), 1, k + 8, 1, 0, res.data_ptr(), 2, k, res.data_ptr(), norm.weight.data_ptr(), 0,
                                   EPS, M, k, y.data_ptr(), 2, q.data_ptr(), s.data_ptr(), 8 * (M + 3), st))
        torch.cuda.synchronize()
        assert torch.equal(q[:M], want[0]) and torch.equal(s[:, :M].movedim(0, 1), want[1]) and torch.equal(y[:M], want[2])
        assert torch.equal(res[:M], want[3]) and torch.equal(res[M], last)
        assert (y[M:] == 7).all() and (q[M:] == 99).all() and (s[:, M:] == 99).all()


@pytest.mark.parametrize("k", [100, 128, 1000, 2048, 2049, 5000, 9000, 40000])
def test_unit_offset(k):
    """1 + weight is not rounded: fp32 rows are off by their own rounding, 2^-24, and 2^-44; and no e4m3 value is on the wrong side
    of a border that the norm rounded to 32 bits and its quotient do not come within 2^-40 of."""
    g = _gen(31 * k)
    for M in (1, 600):
        x = torch.randn(M, k, generator=g, device="cuda")
        weight = 0.2 * torch.randn(k, generator=g, device="cuda")
        norm = _norm()(weight, EPS, unit_offset=True)
        print(f"case norm unit_offset k={k} M={M}", flush=True)
        y = norm(x)
        q, s, h = norm.quant(x.bfloat16(), x)
        torch.cuda.synchronize()
        ref = _ref(x, 1 + weight.double())
        assert ((y.double() - ref).abs() <= _units(k) * 2.0 ** -24 * ref.abs() + 2.0 ** -149).all()
        ref = _ref(h, 1 + weight.double())
        _check_fp8(q, s, ref, k)
        quo = (torch.nn.functional.pad(ref, (0, -k % 128)).view(M, -1, 128) / s.double()[..., None]).view(M, -1)
        lo, hi = (_e4m3((quo * f).float().double()) for f in (1 - 2.0 ** -40, 1 + 2.0 ** -40))
        assert ((q.double() == lo) | (q.double() == hi)).all()


def test_rows_past_32_bits():
    k, M = 4096, 600_000
    x = torch.zeros(M, k, dtype=torch.bfloat16, device="cuda")
    x[-50:] = torch.randn(50, k, generator=_gen(9), device="cuda").bfloat16()
    norm = _norm()(torch.ones(k, device="cuda"), EPS)
    print("case norm rows past 32 bits", flush=True)
    y, h = norm(x, x)
    assert torch.equal(y[-50:], norm(x[-50:], x[-50:])[0]) and torch.equal(h[-50:], (2 * x[-50:])) and not y[:-50].any()
    q, s = norm.quant(x, None, "fp4")
    small = norm.quant(x[-50:], None, "fp4")
    assert torch.equal(q[-50:], small[0]) and torch.equal(s[-50:], small[1])
    del x, y, h, q, s
    far = torch.zeros((1 << 31) + 2000, dtype=torch.bfloat16, device="cuda")       # rows 2^31 elements apart
    v = far.as_strided((2, 3, 200), (1 << 31, 256, 1))
    v.copy_(torch.randn(2, 3, 200, generator=_gen(10), device="cuda"))
    norm = _norm()(None, EPS)
    assert torch.equal(norm(v), norm(v.contiguous()))


def test_many_short_rows():
    g = _gen(11)
    x = torch.randn(1_000_003, 64, generator=g, device="cuda").bfloat16()
    norm = _norm()(torch.randn(64, generator=g, device="cuda"), EPS)
    y = norm(x)
    for a, b in ((0, 1000), (500_000, 501_000), (1_000_003 - 77, 1_000_003)):
        _check_rows(y[a:b], _ref(x[a:b], norm.weight), 64)


def test_refusals():
    x = torch.randn(4, 256, device="cuda").bfloat16()
    norm = _norm()(torch.ones(256, device="cuda"), EPS)
    from exl3xpu.linear import C
    bad = [lambda: norm(x[:, :255]), lambda: norm(x.double()), lambda: norm(x, x[:3]), lambda: norm(x, x.half()), lambda: norm(x, x.cpu()),
           lambda: norm(x.float(), x), lambda: _norm()(torch.ones(256), EPS)(x), lambda: norm(x[:, :0]),
           lambda: C().rms_norm(x, None, None, 1e-6, 0, False), lambda: C().rms_norm(x, None, None, 1e-6, 3, True),
           lambda: C().rms_norm(x, None, None, 0.0, 0, True), lambda: C().rms_norm(x, None, norm.weight.bfloat16(), 1e-6, 0, True),
           lambda: norm(x.clone().requires_grad_()), lambda: norm(x, x.clone().requires_grad_())]
    for i, f in enumerate(bad):
        with pytest.raises((RuntimeError, ValueError)):
            f()
            pytest.fail(f"call {i} was taken")
    with torch.no_grad():
        assert torch.equal(norm(x.clone().requires_grad_()), norm(x))
    with pytest.raises(NotImplementedError):
        _norm()(None, EPS)(x.cpu())


# (as many columns as 16, 64, 256 and 1,024 threads hold in one, two and four chunks of a row, aligned and not)
@pytest.mark.parametrize("k", [128, 250, 1000, 2048, 2047, 4096, 8191, 9000, 9001])
def test_rows_in_a_loop(k):
    """More rows than workgroups, so that one takes several in turn: of magnitudes 2^-30 to 2^30 that differ from row to row, none may
    see anything of the ones before it."""
    M, eps = 5003 if k > 1024 else 40_003, 2.0 ** -40                # (an eps that fp32 holds)
    g = _gen(13 * k)
    norm = _norm()(torch.randn(k, generator=g, device="cuda") + 1, eps)
    for dtype in (torch.float32, torch.bfloat16):
        scale = torch.exp2(torch.randint(-30, 31, (M, 1), generator=g, device="cuda").float())
        x, res = ((torch.randn(M, k, generator=g, device="cuda") * t).to(dtype) for t in (scale, scale.flip(0)))
        print(f"case norm rows in a loop k={k} {dtype}", flush=True)
        outs = [norm.quant(x, res, form, rows=True) for form in ("fp8", "fp4")]
        y = norm(x)
        torch.cuda.synchronize()
        h = _held(x, res)
        for a in range(0, M, 1000):
            at = slice(a, a + 1000)
            _check_rows(y[at], _ref(x[at], norm.weight, eps), k)
            ref = _ref(h[at], norm.weight, eps)
            for (q, s, y2, h2), check in zip(outs, (_check_fp8, _check_fp4)):
                assert torch.equal(h2[at], h[at])
                check(q[at], s[at], ref, k)
                _check_rows(y2[at], ref, k)
