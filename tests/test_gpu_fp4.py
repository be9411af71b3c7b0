"""The 4-bit float linear (torch.ops.exl3xpu_C.fp4_*, exl3xpu.fp4) against its definition in 64 bits, where it can go wrong:
sizes around the blocks of 32, the stages of 256 and the tiles, strides, odd addresses, zero, tiny, huge, infinite and NaN blocks,
one row and none, streams and graphs.

Quantised rows have to be equal, bit for bit: dividing by a power of two is exact and a quotient is rounded once. Behind silu the
value may be 8 units of 2^-24 off, so a code is that of some value within that, and the scale that of some such largest one. A
product's terms are exact; every one of its k + k / 64 additions loses at most 2^-23 of the magnitudes (2^-23: sums that truncate),
half of a step of the output type is added, and as losses of random sign they are below sqrt(k) 2^-23 of the magnitudes' norm."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
VALUES = [0, 0.5, 1, 1.5, 2, 3, 4, 6]


def _fp4():
    from exl3xpu import fp4
    return fp4


def linear_ops():
    from exl3xpu.linear import C
    return C()


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _codes_of(quo):
    """Magnitudes in 64 bits to codes: the nearest value, a half-way one to the even code, 6 at the most."""
    v = torch.tensor(VALUES, dtype=torch.float64, device=quo.device)
    mid = (v[1:] + v[:-1]) / 2
    lo, hi = torch.bucketize(quo, mid, right=False), torch.bucketize(quo, mid, right=True)
    return torch.where(lo % 2 == 0, lo, hi)                  # (they differ only at a half-way value)


def _blocks(x):
    M, k = x.shape
    return torch.nn.functional.pad(x, (0, -k % 128)).reshape(M, -1, 32)


def _exponents(top):
    return torch.where(top > 0, (torch.frexp(top).exponent - 3).clamp_min(-126) + 127, 1)


def _scales_as_held(e, k):
    """Exponent bytes [M, blocks] as [M, stages, 8], 0 behind k."""
    M, blocks, stages = e.size(0), -(-k // 32), -(-k // 256)
    full = torch.zeros(M, stages * 8, dtype=torch.uint8, device=e.device)
    full[:, :blocks] = e[:, :blocks].to(torch.uint8)
    return full.view(M, stages, 8)


def _quant_ref(x):
    """Finite x in 64 bits -> (q, s)."""
    M, k = x.shape
    p = _blocks(x)
    e = _exponents(p.abs().amax(-1))
    codes = _codes_of((p.abs() * torch.exp2(127 - e.double())[..., None])) + 8 * (torch.signbit(p)).long()
    # (a 0 that was filled in is no negative one)
    codes = codes.view(M, -1)
    return (codes[:, ::2] | codes[:, 1::2] << 4).to(torch.uint8), _scales_as_held(e, k)


def _values(q, s, k):
    """What codes and scales stand for, in 64 bits, [M, k]."""
    M = q.size(0)
    v = torch.tensor([*VALUES, *(-a for a in VALUES)], dtype=torch.float64, device=q.device)
    codes = torch.stack([q & 15, q >> 4], -1).view(M, -1)[:, :k].long()
    scale = torch.where(s == 255, math.nan, torch.exp2(s.double() - 127)).reshape(M, -1)
    return v[codes] * scale.repeat_interleave(32, 1)[:, :k]


def _weight(g, n, k):
    """As a checkpoint has it: codes [n, k / 2], scales [n, ceil(k / 32)]; k is even."""
    q, s = _quant_ref(torch.randn(n, k, generator=g, device="cuda").double() * 0.05)
    return q[:, :k // 2].contiguous(), s.reshape(n, -1)[:, :-(-k // 32)].contiguous()


def _linear(w, sw, bias=None):
    return _fp4().Fp4Linear(w, sw, bias)


def _product_ref(xv, w, sw, bias):
    """(the product, the sum of its terms' magnitudes) in 64 bits."""
    n, k = w.size(0), 2 * w.size(1)
    b = _values(w, torch.nn.functional.pad(sw, (0, -sw.size(1) % 8)).view(n, -1, 8), k)
    y, mag = xv @ b.t(), xv.abs() @ b.abs().t()
    return (y, mag) if bias is None else (y + bias.double(), mag + bias.double().abs())


def _check_product(y, xv, w, sw, bias=None):
    ref, mag = _product_ref(xv, w, sw, bias)
    k = xv.size(1)
    half = torch.finfo(y.dtype).eps / 2
    tol = (k + k / 64 + 20) * 2.0 ** -23 * mag
    tol = tol + half * (ref.abs() + tol) + torch.finfo(y.dtype).smallest_normal
    bad = ~((y.double() - ref).abs() <= tol)
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist(), float(((y.double() - ref).abs() / tol).max()))
    if y.numel() > 1000:
        off = float((y.double() - ref).norm())
        assert off <= half * float(ref.norm()) + math.sqrt(k) * 2.0 ** -23 * float(mag.norm()), off


def _odd(t):
    """The same values at an odd element of their storage."""
    store = torch.zeros(t.numel() + 3, dtype=t.dtype, device=t.device)
    v = store[1:1 + t.numel()].view(t.shape)
    v.copy_(t)
    return v


@pytest.mark.parametrize("k", [1, 7, 8, 31, 32, 33, 127, 128, 129, 250, 256, 260, 384, 500, 640, 1000, 2048, 2050])
def test_quant(k):
    g = _gen(k)
    for dtype in DTYPES:
        for M in (1, 2, 7, 8, 9, 130):
            print(f"case fp4 quant k={k} M={M} {dtype}", flush=True)
            x = (torch.randn(M, k, generator=g, device="cuda") * torch.exp(2 * torch.randn(M, 1, generator=g, device="cuda"))).to(dtype)
            if M > 2:
                x[1] = 0
                x[2, k // 2:] = 0
            q, s = _fp4().quant(x)
            torch.cuda.synchronize()
            rq, rs = _quant_ref(x.double())
            assert q.dtype == s.dtype == torch.uint8 and q.shape == rq.shape and s.shape == rs.shape
            assert torch.equal(s, rs) and torch.equal(q, rq)
            for other in (_odd(x), torch.nn.functional.pad(x, (0, 9))[:, :k], x.t().contiguous().t()):
                q2, s2 = _fp4().quant(other)
                assert torch.equal(q2, q) and torch.equal(s2, s)
            for out in DTYPES:
                v = _fp4().dequant(q, s, out, k)
                assert v.shape == x.shape and torch.equal(v, _values(q, s, k).float().to(out))
            assert torch.equal(_fp4().dequant(q, s.contiguous()), _values(q, s, 2 * q.size(1)).float())


def test_quant_every_half_step():
    """Quotients that lie between two values go to the even code, every value comes back as it is, and 6 is the largest."""
    v = torch.tensor(VALUES, device="cuda")
    mid = (v[1:] + v[:-1]) / 2
    x = torch.zeros(6, 32, device="cuda")
    x[0, :8], x[0, 8:16] = v, -v
    x[1, :7], x[1, 7] = mid, 4.0
    x[2, :7], x[2, 7] = -torch.nextafter(mid, mid * 2), 6.0
    x[3, :7], x[3, 7] = torch.nextafter(mid, mid * 0), -6.0
    x[4, :4] = torch.tensor([6.5, 7.0, 7.99, -7.999], device="cuda")
    x[5, :3] = torch.tensor([4.0, 3.9999998, 0.25], device="cuda")
    for scale in (1.0, 2.0 ** -60, 2.0 ** 100, 2.0 ** -120, 2.0 ** -124):
        q, s = _fp4().quant(x * scale)
        rq, rs = _quant_ref((x * scale).double())
        assert torch.equal(s, rs) and torch.equal(q, rq), scale
    q, s = _fp4().quant(x)
    assert torch.equal(_fp4().dequant(q, s, torch.float32, 32)[0], x[0]) and (s[0, 0, 0] == 127).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_quant_every_16_bit_value(dtype):
    """Every finite value of the type, next to block maxima from its own size to 64 times it, and by itself; the same in fp32."""
    v = torch.arange(1 << 16, device="cuda").to(torch.uint16).view(dtype)
    v = v[v.isfinite()]
    for up in (1, 2, 3, 6, 7, 24, 64):
        x = v.view(-1, 16).repeat_interleave(2, 1)
        x[:, 1::2] = (x[:, ::2].float() * up).to(dtype)      # a maximum beside each: some other value's blocks, some its own
        x = torch.cat([x, torch.stack([v, (v.float() * up).to(dtype)], 1).repeat(1, 16)])
        x = x[x.isfinite().all(1)]
        q, s = _fp4().quant(x)
        rq, rs = _quant_ref(x.double())
        assert torch.equal(s, rs) and torch.equal(q, rq)
        q2, s2 = _fp4().quant(x.float())
        assert torch.equal(q2, q) and torch.equal(s2, s)


def test_quant_infinities_nan_and_extremes():
    x = torch.randn(10, 400, generator=_gen(3), device="cuda")
    x[0, 5] = math.inf
    x[1, 200] = -math.inf
    x[2, 300] = math.nan
    x[3, :128] = 3.4e38
    x[4] *= 1e-30
    x[5] *= 1e-42
    x[6, 130:250] = 0
    x[7, 399] = math.nan
    x[8] *= 1e36
    x[9] = 0
    q, s = _fp4().quant(x)
    torch.cuda.synchronize()
    flat = s.reshape(10, -1)
    assert [flat[i].eq(255).nonzero().flatten().tolist() for i in (0, 1, 2, 7)] == [[0], [6], [9], [12]]
    fine = [3, 4, 5, 6, 8, 9]
    rq, rs = _quant_ref(x[fine].double())
    assert torch.equal(q[fine], rq) and torch.equal(s[fine], rs)
    for dtype in (torch.bfloat16, torch.float16):            # (the 16-bit types have a path of their own)
        h = torch.randn(4, 96, generator=_gen(4), device="cuda").to(dtype)
        h[0, 5], h[1, 40], h[2, 95] = math.inf, -math.inf, math.nan
        hs = _fp4().quant(h)[1].reshape(4, -1)
        assert hs.eq(255).nonzero().tolist() == [[0, 0], [1, 1], [2, 2]]
    assert (flat[9, :13] == 1).all() and not flat[:, 13:].any() and not q[9].any()
    back = _fp4().dequant(q, s, torch.float32, 400)
    assert back[0, :32].isnan().all() and back[0, 32:].isfinite().all() and back[7, 384:].isnan().all() and back[7, :384].isfinite().all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_dequant_every_scale(dtype):
    """Every code with every scale, the smallest and the NaN among them."""
    q = torch.tensor([a | b << 4 for a in range(16) for b in range(16)], dtype=torch.uint8, device="cuda")
    q = torch.cat([q, q]).view(1, 512).expand(256, 512).contiguous()
    s = torch.arange(256, dtype=torch.uint8, device="cuda").view(256, 1, 1).expand(256, 4, 8)
    got, want = _fp4().dequant(q, s, dtype), _values(q, s, 1024).float().to(dtype)
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(), want.nan_to_num())


def _check_silu(q, s, gu, k):
    """The rows of silu(gate) * up: codes and scales of some value within 8 units of 2^-24."""
    M, u = gu.size(0), 8 * 2.0 ** -24
    a, b = gu[:, :k].double(), gu[:, k:].double()
    p = _blocks(a / (1 + torch.exp(-a)) * b)
    blocks = -(-k // 32)
    top, e = p.abs().amax(-1), s.reshape(M, -1).int()
    assert not e[:, blocks:].any()
    e = e[:, :blocks]
    assert ((e >= _exponents(top * (1 - u))[:, :blocks]) & (e <= _exponents(top * (1 + u))[:, :blocks])).all()
    quo = p[:, :blocks] * torch.exp2(127 - e.double())[..., None]
    codes = torch.stack([q & 15, q >> 4], -1).view(M, -1, 32)
    assert not codes[:, blocks:].any()
    codes = codes[:, :blocks].long()
    lo, hi = _codes_of(quo.abs() * (1 - u)), _codes_of(quo.abs() * (1 + u))
    got = codes % 8
    assert ((got >= lo) & (got <= hi) & ((got == 0) | ((codes >= 8) == (quo < 0)))).all()


@pytest.mark.parametrize("k", [1, 31, 60, 127, 128, 129, 256, 512, 640, 1001])
def test_silu_mul_quant(k):
    g = _gen(100 + k)
    for dtype in DTYPES:
        for M in (1, 3, 8, 131):
            print(f"case fp4 silu k={k} M={M} {dtype}", flush=True)
            gu = (torch.randn(M, 2 * k, generator=g, device="cuda") * 4).to(dtype)
            if M > 2:
                gu[1, :k] = -95.0
                gu[2] = 0
            q, s = _fp4().silu_mul_quant(gu)
            torch.cuda.synchronize()
            _check_silu(q, s, gu, k)
            for t in (_odd(gu), torch.nn.functional.pad(gu, (0, 5))[:, :2 * k]):
                q2, s2 = _fp4().silu_mul_quant(t)
                assert torch.equal(q2, q) and torch.equal(s2, s)


SIZES = [(1, 128), (5, 2), (16, 130), (17, 640), (31, 32), (127, 1000), (128, 512), (129, 2048), (200, 126), (384, 1152), (1000, 2000)]


@pytest.mark.parametrize("n,k", SIZES)
def test_linear(n, k):
    g = _gen(7 * n + k)
    w, sw = _weight(g, n, k)
    bias = torch.randn(n, generator=g, device="cuda")
    lin, linb = _linear(w, sw), _linear(w, sw, bias)
    for M in (1, 2, 3, 8, 9, 15, 16, 17, 31, 32, 33, 63, 64, 65, 100, 127, 128, 129, 255, 257, 300):
        for dtype in DTYPES:
            print(f"case fp4 linear n={n} k={k} M={M} {dtype}", flush=True)
            x = torch.randn(M, k, generator=g, device="cuda").to(dtype)
            y, yb = lin(x), linb(x)
            torch.cuda.synchronize()
            assert y.dtype == dtype and y.shape == (M, n)
            xv = _values(*_quant_ref(x.double()), k)
            _check_product(y, xv, w, sw)
            _check_product(yb, xv, w, sw, bias)
            assert torch.equal(lin.quantised(*_fp4().quant(x), dtype), y)
            assert torch.equal(lin(_odd(x)), y)


@pytest.mark.parametrize("M,n,k", [(700, 512, 2048), (1025, 640, 384), (2048, 2048, 512), (513, 4096, 130), (64, 8192, 256),
                                   (40, 2048, 4096), (1, 12288, 2048), (4, 1024, 2048), (300, 12288, 512), (2100, 2100, 640),
                                   (1500, 2000, 1100), (4000, 4352, 640), (8192, 2304, 256), (6000, 3000, 384)])
def test_linear_larger(M, n, k):
    g = _gen(M + n)
    w, sw = _weight(g, n, k)
    lin = _linear(w, sw)
    for dtype in DTYPES:
        print(f"case fp4 linear M={M} n={n} k={k} {dtype}", flush=True)
        x = (torch.randn(M, k, generator=g, device="cuda") * torch.exp(torch.randn(M, 1, generator=g, device="cuda"))).to(dtype)
        y = lin(x)
        torch.cuda.synchronize()
        _check_product(y, _values(*_quant_ref(x.double()), k), w, sw)
        assert torch.equal(lin(x), y)                        # the same sums in the same order


@pytest.mark.parametrize("M,n,k", [(2200, 4099, 1100), (4100, 4097, 1030), (8192, 2307, 1024), (600, 2051, 700), (300, 1003, 500),
                                   (40, 2049, 900), (3, 1005, 600)])
def test_outputs_at_any_element(M, n, k):
    """Rows of outputs that start at odd elements, in the kernels of few rows, of tiles and of 256 x 256 ones; nothing outside them
    is written."""
    from exl3xpu import capi
    L, st = capi.lib(), torch.cuda.current_stream().cuda_stream
    g = _gen(M + 3 * n)
    w, sw = _weight(g, n, k)
    bias = torch.randn(n, generator=g, device="cuda")
    for lin in (_linear(w, sw), _linear(w, sw, bias)):
        for code, dtype in ((0, torch.float16), (1, torch.bfloat16), (2, torch.float32)):
            print(f"case fp4 odd outputs M={M} n={n} k={k} {dtype} bias={lin.bias is not None}", flush=True)
            x = torch.randn(M, k, generator=g, device="cuda").to(dtype)
            y = lin(x)
            torch.cuda.synchronize()
            _check_product(y, _values(*_quant_ref(x.double()), k), w, sw, lin.bias)
            q, s = _fp4().quant(x)
            store = torch.full((M * (n + 2) + 5,), 9.0, dtype=dtype, device="cuda")
            out = store[1:1 + M * (n + 2)].view(M, n + 2)
            capi.check(L.exl3_fp4_matmul(q.data_ptr(), s.data_ptr(), 8 * M, M, 2 * q.size(1), n, lin.weight.data_ptr(),
                                         lin.weight_scale.data_ptr(), None if lin.bias is None else lin.bias.data_ptr(),
                                         out.data_ptr(), code, n + 2, st))
            torch.cuda.synchronize()
            assert torch.equal(out[:, :n], y) and (out[:, n:] == 9).all() and store[0] == 9 and (store[-4:] == 9).all()


@pytest.mark.parametrize("n,k,Ms", [(2000, 1300, (33, 40, 47, 64, 90, 100, 127, 300)), (2050, 4000, (17, 64, 97, 128)),
                                    (1990, 640, (770, 1000, 1090, 1500, 2200)), (5000, 2048, (1, 3, 4, 5, 8, 16, 17, 32, 33)),
                                    (1000, 4096, (1, 2, 3, 4, 5, 16, 17, 31)), (1100, 1152, (80, 2030)), (12200, 200, (100, 1100)),
                                    (8300, 640, (14, 16, 20)), (8200, 300, (128, 129)), (520, 8000, (1, 8, 50, 200)), (96, 20000, (1, 33, 300))])
def test_linear_tiles(n, k, Ms):
    """Sizes of every tile, with one workgroup per CU at most and with more, and edges inside a tile."""
    g = _gen(n + k)
    w, sw = _weight(g, n, k)
    bias = torch.randn(n, generator=g, device="cuda")
    lin = _linear(w, sw, bias)
    for M in Ms:
        for dtype in DTYPES:
            print(f"case fp4 linear tiles n={n} k={k} M={M} {dtype}", flush=True)
            x = torch.randn(M, k, generator=g, device="cuda").to(dtype)
            y = lin(x)
            torch.cuda.synchronize()
            _check_product(y, _values(*_quant_ref(x.double()), k), w, sw, bias)
            assert torch.equal(lin(_odd(x)), y)
            assert torch.equal(lin.quantised(*_fp4().quant(x), dtype), y)


def test_linear_rows_do_not_see_each_other():
    """A NaN or an infinity stays in its row, and a NaN weight scale in its column; also where the last stage is half a one."""
    g = _gen(21)
    for k in (384, 512, 126):
        for M in (5, 40, 300, 1100):
            w, sw = _weight(g, 300, k)
            x = torch.randn(M, k, generator=g, device="cuda").bfloat16()
            want = _linear(w, sw)(x)
            x[1, k - 1] = math.nan
            x[3, 0] = math.inf
            sw = sw.clone()
            sw[130, 0] = 255
            y = _linear(w, sw)(x)
            torch.cuda.synchronize()
            assert y[1].isnan().all() and y[3].isnan().all() and y[:, 130].isnan().all()
            rows = [m for m in range(M) if m not in (1, 3)]
            cols = [i for i in range(300) if i != 130]
            assert torch.equal(y[rows][:, cols], want[rows][:, cols])


def test_linear_of_all_sizes_of_scales():
    """Scales from the smallest to the largest: products that fp32 holds come out, others are infinite or 0."""
    g = _gen(22)
    for M in (3, 60, 300):
        w, sw = _weight(g, 140, 256)
        x = torch.randn(M, 256, generator=g, device="cuda")
        for down, up in ((2.0 ** -100, 100), (2.0 ** 100, -100), (2.0 ** -60, 0), (2.0 ** 60, 0), (2.0 ** -40, -20)):
            y = _linear(w, (sw.int() + up).to(torch.uint8))(x * down)
            xv = _values(*_quant_ref((x * down).double()), 256)
            _check_product(y, xv, w, (sw.int() + up).to(torch.uint8))
        y = _linear(w, torch.full_like(sw, 254))(x * 2.0 ** 100)
        assert not y.isfinite().all()
        assert not _linear(w, torch.zeros_like(sw))(x * 2.0 ** -60).any()


def test_columns_behind_the_last_stage_do_not_count():
    """A stage that is half a row's: scales behind the row's columns, NaN ones too, count for nothing."""
    g = _gen(24)
    for M in (4, 40, 300, 1100):
        w, sw = _weight(g, 200, 384)
        lin = _linear(w, sw)
        q, s = _fp4().quant(torch.randn(M, 384, generator=g, device="cuda"))
        want = lin.quantised(q, s, torch.float32)
        for fill in (254, 255):
            s2 = s.clone()
            s2[:, 1, 4:] = fill
            assert torch.equal(lin.quantised(q, s2, torch.float32), want)


def test_linear_shapes_strides_and_empty():
    g = _gen(23)
    w, sw = _weight(g, 260, 300)
    lin = _linear(w, sw)
    x = torch.randn(24, 300, generator=g, device="cuda").bfloat16()
    y = lin(x)
    assert torch.equal(lin(x.view(2, 3, 4, 300)), y.view(2, 3, 4, 260))
    assert torch.equal(lin(x[0]), lin(x[:1])[0])
    assert torch.equal(lin(torch.nn.functional.pad(x, (0, 7))[:, :300]), y)
    assert torch.equal(lin(x.t().contiguous().t()), y)
    assert torch.equal(lin(x[:1].expand(24, 300)), lin(x[:1].expand(24, 300).contiguous()))
    assert lin(x[:0]).shape == (0, 260) and lin(x.view(4, 6, 300)[:, :0]).shape == (4, 0, 260)
    q, s = _fp4().quant(x.view(4, 6, 300))
    assert q.shape == (4, 6, 192) and s.shape == (4, 6, 2, 8)
    assert torch.equal(lin.quantised(q, s, torch.bfloat16), y.view(4, 6, 260))
    assert torch.equal(lin.quantised(q, s.contiguous(), torch.bfloat16), y.view(4, 6, 260))
    assert lin.quantised(q[:, :0], s[:, :0], torch.float16).shape == (4, 0, 260)
    # rows cut out of more, whose scales keep the larger stages' distance
    q, s = _fp4().quant(torch.cat([x, x, x]))
    for a, b in ((24, 48), (31, 40), (71, 72)):
        want = lin.quantised(*_fp4().quant(torch.cat([x, x, x])[a:b]), torch.bfloat16)
        assert torch.equal(lin.quantised(q[a:b], s[a:b], torch.bfloat16), want)
    assert torch.equal(lin.quantised(q[::2], s[::2], torch.bfloat16), lin(torch.cat([x, x, x])[::2]))
    assert torch.equal(_fp4().dequant(q[5:9], s[5:9], torch.float32, 300), _fp4().dequant(q, s, torch.float32, 300)[5:9])


def test_linear_from_quantised_weights():
    g = _gen(26)
    for k in (63, 300, 512):
        w = torch.randn(130, k, generator=g, device="cuda")
        q, s = _fp4().quant(w)
        lin = _fp4().Fp4Linear(q, s, k=k)
        x = torch.randn(20, k, generator=g, device="cuda")
        ref = _values(*_quant_ref(x.double()), k) @ _values(q, s, k).t()
        mag = _values(*_quant_ref(x.double()), k).abs() @ _values(q, s, k).abs().t()
        assert ((lin(x).double() - ref).abs() <= (k + k / 64 + 20) * 2.0 ** -23 * mag).all()


def test_c_abi_leaves_what_is_behind_a_row():
    """Columns behind n and rows behind M of a wider output are left as they were, and a workspace of a larger call does
    for a smaller one."""
    from exl3xpu import capi
    L, st = capi.lib(), torch.cuda.current_stream().cuda_stream
    g = _gen(25)
    for M, n, k in ((1, 130, 256), (20, 200, 384), (200, 257, 512), (700, 600, 640), (1300, 1100, 256)):
        lin = _linear(*_weight(g, n, k))
        x = torch.randn(M, k, generator=g, device="cuda").bfloat16()
        ws = torch.full((L.exl3_fp4_linear_workspace(M + 500, k, n),), 0xFF, dtype=torch.uint8, device="cuda")
        for dt, dtype in ((1, torch.bfloat16), (2, torch.float32)):
            out = torch.full((M + 3, n + 5), 7.0, dtype=dtype, device="cuda")
            print(f"case fp4 c-abi M={M} n={n} k={k} {dtype}", flush=True)
            capi.check(L.exl3_fp4_linear(x.data_ptr(), 1, k, M, k, n, lin.weight.data_ptr(), lin.weight_scale.data_ptr(), None,
                                         out.data_ptr(), dt, n + 5, ws.data_ptr(), ws.numel(), st))
            torch.cuda.synchronize()
            assert torch.equal(out[:M, :n], lin.quantised(*_fp4().quant(x), dtype))
            assert (out[M:] == 7).all() and (out[:, n:] == 7).all()
        q = torch.full((M + 1, -(-k // 128) * 64), 99, dtype=torch.uint8, device="cuda")
        s = torch.full((-(-k // 256), M + 2, 8), 99, dtype=torch.uint8, device="cuda")
        capi.check(L.exl3_fp4_quant(x.data_ptr(), 1, k, M, k, q.data_ptr(), s.data_ptr(), 8 * (M + 2), st))
        want = _fp4().quant(x)
        assert torch.equal(q[:M], want[0]) and torch.equal(s[:, :M].movedim(0, 1), want[1]) and (q[M:] == 99).all() and (s[:, M:] == 99).all()


def test_rows_and_weights_past_32_bits():
    """Rows, quantised rows, weights and outputs whose bytes lie past 2^32."""
    g = _gen(41)
    k, M = 4096, 2_200_000
    x = torch.zeros(M, k, dtype=torch.bfloat16, device="cuda")
    x[-300:] = torch.randn(300, k, generator=g, device="cuda").bfloat16()
    print("case fp4 rows past 32 bits", flush=True)
    q, s = _fp4().quant(x)
    rq, rs = _quant_ref(x[-300:].double())
    assert torch.equal(q[-300:], rq) and torch.equal(s[-300:], rs)
    w, sw = _weight(g, 200, k)
    lin = _linear(w, sw)
    y = lin.quantised(q, s, torch.float16)
    _check_product(y[-300:], _values(rq, rs, k), w, sw)
    assert not y[:1000].any() and not y[M // 2:M // 2 + 1000].any()
    y = _fp4().dequant(q, s, torch.bfloat16)
    assert torch.equal(y[-300:], _values(rq, rs, k).bfloat16()) and not y[:1000].any()
    del x, q, s, y
    n = 2_200_000
    raw = torch.zeros(n, k // 2, dtype=torch.uint8, device="cuda")
    raw[-200:] = w
    scale = torch.full((n, k // 32), 127, dtype=torch.uint8, device="cuda")
    scale[-200:] = sw
    lin = _linear(raw, scale)
    for M in (1, 20, 300):
        print(f"case fp4 weights past 32 bits M={M}", flush=True)
        x = torch.randn(M, k, generator=g, device="cuda").bfloat16()
        y = lin(x)
        _check_product(y[:, -200:], _values(*_quant_ref(x.double()), k), w, sw)
        assert not y[:, :1000].any()
    del raw, scale, lin, y
    far = torch.zeros((1 << 31) + 2000, dtype=torch.bfloat16, device="cuda")      # rows 2^31 elements apart
    x = far.as_strided((2, 1000), (1 << 31, 1))
    x.copy_(torch.randn(2, 1000, generator=g, device="cuda"))
    lin = _linear(*_weight(g, 48, 1000))
    print("case fp4 rows 2^32 bytes apart", flush=True)
    assert torch.equal(lin(x), lin(x.contiguous()))
    assert all(torch.equal(a, b) for a, b in zip(_fp4().quant(x), _fp4().quant(x.contiguous())))


def test_more_small_tiles_than_one_launch_holds():
    """2^26 rows of 128 to 16 columns."""
    g = _gen(37)
    M = 1 << 16
    q, s = _fp4().quant(torch.randn(M, 128, generator=g, device="cuda"))
    lin = _linear(*_weight(g, 16, 128))
    want = lin.quantised(q, s, torch.bfloat16)
    print("case fp4 product of 2^26 rows", flush=True)
    got = lin.quantised(q.repeat(1024, 1), s.repeat(1024, 1, 1), torch.bfloat16)
    assert all(torch.equal(t, want) for t in got.split(M))


def test_refusals():
    g = _gen(27)
    w, sw = _weight(g, 256, 256)
    lin = _linear(w, sw)
    w, sw = lin.weight, lin.weight_scale
    C = linear_ops()
    x = torch.randn(4, 256, generator=g, device="cuda").bfloat16()
    q, s = _fp4().quant(x)
    down = _fp4().Fp4Linear(w[:, :64], sw[:, 0, :4], k=128)
    mlp = _fp4().Fp4Mlp(lin, down)
    bad = [lambda: lin(x[:, :255]), lambda: lin(x.double()), lambda: lin(x.byte()), lambda: C.fp4_linear(x, w.float(), sw, None),
           lambda: C.fp4_linear(x, w.t(), sw, None), lambda: C.fp4_linear(x, w, sw[:1], None), lambda: C.fp4_linear(x, w, sw.int(), None),
           lambda: C.fp4_linear(x, w[:, :64], sw, None), lambda: C.fp4_linear(x, w, torch.cat([sw, sw], 1), None),
           lambda: C.fp4_linear(x, w, sw, torch.zeros(255, device="cuda")), lambda: C.fp4_linear(x, w, sw, torch.zeros(256, device="cuda").half()),
           lambda: C.fp4_linear(x, w.cpu(), sw, None), lambda: C.fp4_linear(x, w, sw.cpu(), None),
           lambda: C.fp4_matmul(q, s[:3], w, sw, None, torch.bfloat16), lambda: C.fp4_matmul(q[:, :100], s, w, sw, None, torch.bfloat16),
           lambda: C.fp4_matmul(q[:, :64], s, w, sw, None, torch.bfloat16), lambda: C.fp4_matmul(q, s, w, sw, None, torch.int32),
           lambda: C.fp4_matmul(q.char(), s, w, sw, None, torch.bfloat16), lambda: C.fp4_matmul(q, s.cpu(), w, sw, None, torch.bfloat16),
           lambda: C.fp4_dequant(q, s, 128, torch.float32), lambda: C.fp4_dequant(q, s, 257, torch.float32),
           lambda: C.fp4_dequant(q, s, 0, torch.float32), lambda: C.fp4_dequant(q, s, 256, torch.int8),
           lambda: C.fp4_mlp(x, 256, w, sw, None, w, sw, None), lambda: C.fp4_mlp(x, 0, w, sw, None, w, sw, None),
           lambda: C.fp4_mlp(x, 128, w, sw, None, w, sw, None), lambda: C.fp4_mlp(x, 128, w[:255], sw[:255], None, down.weight, down.weight_scale, None),
           lambda: mlp(x[:, :200]), lambda: mlp.quantised(q[:, :64], s, torch.float32), lambda: mlp.quantised(q, s, torch.int32),
           lambda: _fp4().quant(x.int()), lambda: _fp4().quant(x[:, :0]), lambda: _fp4().silu_mul_quant(x[:, :255]),
           lambda: _fp4().quant(x.clone().requires_grad_()), lambda: lin(x.clone().requires_grad_()), lambda: mlp(x.clone().requires_grad_()),
           lambda: _fp4().Fp4Mlp(lin, _fp4().Fp4Linear(down.weight.cpu(), down.weight_scale.cpu()))]
    for i, f in enumerate(bad):
        with pytest.raises((RuntimeError, ValueError)):
            f()
            pytest.fail(f"call {i} was taken")
    with pytest.raises(NotImplementedError):
        _fp4().quant(x.cpu())


def _check_mlp(y, x, gu, dn, biases, k, I):  # noqa: E741
    """The MLP against its definition: the rows between are quantised again, so a fp32 rounding may move a value over a border. A
    block's codes and scale are right for some value within (k + k / 64 + 20) 2^-23 of the magnitudes; where no value is so near a
    border the rows are exact, so the reference takes the rows in 64 bits and the tolerance what the near ones could move."""
    xv = _values(*_quant_ref(x.double()), k)
    g, mag = _product_ref(xv, *gu, biases[0])
    a, b = g[:, :I], g[:, I:]
    sig = 1 / (1 + torch.exp(-a))
    h = a * sig * b
    # |d silu(a) / da| is 1.1 at the most, silu's own 8 units
    eps = (k + k / 64 + 20) * 2.0 ** -23
    off = 1.1 * eps * mag[:, :I] * b.abs() + (a * sig).abs() * eps * mag[:, I:] + 8 * 2.0 ** -24 * h.abs()
    lo, hi = (h.abs() - off).clamp_min(0), h.abs() + off

    def quantised(v, e):
        p = _blocks(v)
        return torch.tensor(VALUES, dtype=torch.float64, device=v.device)[_codes_of(p * torch.exp2(127 - e.double())[..., None])] * torch.exp2(e.double() - 127)[..., None]
    tops = [_exponents(_blocks(v).amax(-1)) for v in (lo, hi, h.abs())]
    mid = quantised(h.abs(), tops[2]).view(h.size(0), -1)[:, :I]
    span = torch.zeros_like(h)
    for v in (lo, hi):
        for e in tops[:2]:
            span = torch.maximum(span, (quantised(v, e).view(h.size(0), -1)[:, :I] - mid).abs())
    hv = torch.copysign(mid, h)
    # (the reference's weights have an even k: a column of zeros behind an odd I)
    hv, span = (torch.nn.functional.pad(t, (0, I % 2)) for t in (hv, span))
    ref, mag2 = _product_ref(hv, *dn, biases[1])
    moved = _product_ref(span, *dn, None)[1]
    half = torch.finfo(y.dtype).eps / 2
    tol = (I + I / 64 + 20) * 2.0 ** -23 * mag2 + moved
    tol = tol + half * (ref.abs() + tol) + torch.finfo(y.dtype).smallest_normal
    bad = ~((y.double() - ref).abs() <= tol)
    assert not bad.any(), (int(bad.sum()), float(((y.double() - ref).abs() / tol).max()))
    if y.numel() > 1000:
        assert float((y.double() - ref).norm() / ref.norm()) <= half + 0.01       # (a moved value is one of many)


@pytest.mark.parametrize("M", [1, 4, 16, 37, 300, 1200])
def test_mlp(M):
    g = _gen(31)
    for k, I in ((2048, 512), (512, 640), (300, 200), (128, 30), (256, 1)):  # noqa: E741
        fp4 = _fp4()
        gu = _weight(g, 2 * I, k)
        dn = _weight(g, 260, I + I % 2)
        if I % 2:
            dn = (dn[0] & 15, dn[1])
        for bias in (False, True):
            b = [torch.randn(n, generator=g, device="cuda") if bias else None for n in (2 * I, 260)]
            mlp = fp4.Fp4Mlp(fp4.Fp4Linear(*gu, b[0]), fp4.Fp4Linear(*dn, b[1], k=I))
            for dtype in DTYPES:
                print(f"case fp4 mlp M={M} k={k} I={I} bias={bias} {dtype}", flush=True)
                x = torch.randn(M, k, generator=g, device="cuda").to(dtype)
                y = mlp(x)
                torch.cuda.synchronize()
                assert y.shape == (M, 260) and y.dtype == dtype
                _check_mlp(y, x, gu, dn, b, k, I)
                assert torch.equal(mlp(_odd(x)), y) and torch.equal(mlp(x[None]), y[None])
                assert torch.equal(mlp.quantised(*fp4.quant(x), dtype), y)
                assert mlp(x[:0]).shape == (0, 260)


@pytest.mark.parametrize("M", [1, 4, 37, 300])
def test_mlp_of_large_negative_gates(M):
    """Columns whose gate is far below 0 count for nothing, as those with a gate of 0 do."""
    fp4, g, k, I = _fp4(), _gen(51), 512, 384  # noqa: E741
    w, sw = _weight(g, 2 * I, k)
    w[:I] = 0                                                # (the gates are their biases, exactly)
    down = fp4.Fp4Linear(*_weight(g, k, I))
    gates = torch.randn(I, generator=g, device="cuda").bfloat16().float()
    far = torch.tensor([-91.0, -95.0, -110.0, -128.0, -256.0, -1000.0, -90.0, -200.0], device="cuda")
    biases = []
    for values in (far, torch.zeros_like(far)):
        b = torch.cat([gates, torch.zeros(I, device="cuda")])
        b[3:3 + 40 * 8:8] = values.repeat(5)
        biases.append(b)
    for dtype in DTYPES:
        print(f"case fp4 mlp of large negative gates M={M} {dtype}", flush=True)
        x = torch.randn(M, k, generator=g, device="cuda").to(dtype)
        y, want = (fp4.Fp4Mlp(fp4.Fp4Linear(w, sw, b), down)(x) for b in biases)
        torch.cuda.synchronize()
        assert y.isfinite().all() and torch.equal(y, want)


def test_mlp_rows_do_not_see_each_other():
    fp4, g = _fp4(), _gen(52)
    mlp = fp4.Fp4Mlp(fp4.Fp4Linear(*_weight(g, 400, 384)), fp4.Fp4Linear(*_weight(g, 130, 200)))
    for M in (4, 40, 300, 1200):
        x = torch.randn(M, 384, generator=g, device="cuda").bfloat16()
        want = mlp(x)
        x[1, 380] = math.nan
        x[2, 0] = math.inf
        y = mlp(x)
        rows = [m for m in range(M) if m not in (1, 2)]
        assert y[1:3].isnan().all() and torch.equal(y[rows], want[rows])


def test_a_workspace_of_a_larger_call():
    """One workspace for calls of every size, the largest first, and the smallest: nothing of a call is left in it."""
    from exl3xpu import capi
    L, st = capi.lib(), torch.cuda.current_stream().cuda_stream
    g, fp4 = _gen(45), _fp4()
    k, I, n = 512, 200, 384  # noqa: E741
    mlp = fp4.Fp4Mlp(fp4.Fp4Linear(*_weight(g, 2 * I, k)), fp4.Fp4Linear(*_weight(g, n, I)))
    gu, gs, _, dn, ds, _ = mlp._weights
    ws = torch.full((L.exl3_fp4_mlp_workspace(400, k, I),), 0xFF, dtype=torch.uint8, device="cuda")
    for M in (400, 1, 33, 4, 130, 2, 400):
        x = torch.randn(M, k, generator=g, device="cuda").bfloat16()
        out = torch.full((M, n + 3), 9.0, dtype=torch.bfloat16, device="cuda")
        print(f"case fp4 mlp c-abi M={M}", flush=True)
        capi.check(L.exl3_fp4_mlp(x.data_ptr(), 1, k, M, k, I, n, gu.data_ptr(), gs.data_ptr(), None, dn.data_ptr(), ds.data_ptr(),
                                  None, out.data_ptr(), 1, n + 3, ws.data_ptr(), ws.numel(), st))
        torch.cuda.synchronize()
        assert torch.equal(out[:, :n], mlp(x)) and (out[:, n:] == 9).all()


def _layer(g, M):
    """An MoE layer as a model runs it: the norm with the residual, router, routed experts through the cache, shared expert, and the
    next norm before a projection."""
    from exl3xpu.moe_offload import ExpertStore
    from exl3xpu.norm import RmsNorm
    from exl3xpu.routing import Router
    from exl3xpu.synth import expert_blob
    fp4 = _fp4()
    H, I, E = 256, 128, 16  # noqa: E741
    store = ExpertStore(H, I, 3, E, E, max_layers=1)
    store.add_layer("layer0", torch.stack([expert_blob(5, e, H, I, 3) for e in range(E)]))
    mlp = fp4.Fp4Mlp(fp4.Fp4Linear(*_weight(g, 2 * I, H)), fp4.Fp4Linear(*_weight(g, H, I)))
    proj, wr = _linear(*_weight(g, 600, H)), torch.randn(E, H, generator=g, device="cuda") / 16
    norms = [RmsNorm(0.1 * torch.randn(H, generator=g, device="cuda"), unit_offset=True) for _ in range(2)]
    router = Router(4, scoring="sigmoid", bias=0.05 * torch.randn(E, generator=g, device="cuda"), n_group=4, topk_group=2)

    def forward(x, residual):
        q, s, y, h = norms[0].quant(x, residual, "fp4", rows=True)
        out = store.forward_routed("layer0", y, y.float() @ wr.t(), router) + mlp.quantised(q, s, y.dtype)
        q, s, h = norms[1].quant(out, h, "fp4")
        return proj.quantised(q, s, out.dtype), h

    def plain(x, residual):
        h = (x.float() + residual.float()).to(residual.dtype)
        y = norms[0](h.to(x.dtype)) if residual.dtype == x.dtype else norms[0](h).to(x.dtype)
        q, s = norms[0].quant(h, None, "fp4")
        ids, w = router(y.float() @ wr.t())
        out = store.forward("layer0", y, ids, w) + mlp.quantised(q, s, y.dtype)
        h = (out.float() + h.float()).to(h.dtype)
        return proj.quantised(*norms[1].quant(h, None, "fp4"), out.dtype), h
    return forward, plain


def test_layer_together():
    g = _gen(33)
    for M in (1, 3, 40, 300):
        forward, plain = _layer(g, M)
        for rtype in (torch.bfloat16, torch.float32):
            x = torch.randn(M, 256, generator=g, device="cuda").bfloat16()
            res = torch.randn(M, 256, generator=g, device="cuda").to(rtype)
            got, want = forward(x, res), plain(x, res)
            torch.cuda.synchronize()
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and got[1].dtype == rtype


def test_layer_in_two_graphs_and_on_streams():
    """Two captured layers replayed in turn, eager work between; then the parts on two streams at once."""
    g = _gen(35)
    M = 3
    forward, _ = _layer(g, M)
    xs = [[torch.randn(M, 256, generator=g, device="cuda").bfloat16() for _ in range(2)] for _ in range(3)]
    want = [[t.clone() for t in forward(*x)] for x in xs]
    torch.cuda.synchronize()
    bufs, outs, graphs = [[t.clone() for t in xs[i]] for i in range(2)], [], []
    for b in bufs:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(forward(*b))
        graphs.append(gr)

    def same(a, b):
        return all(torch.equal(x, y) for x, y in zip(a, b))
    for i, j in ((0, 1), (2, 0), (1, 2), (2, 1)):
        for b, x in zip(bufs, (xs[i], xs[j])):
            for t, v in zip(b, x):
                t.copy_(v)
        graphs[0].replay()
        graphs[1].replay()
        assert same(forward(*xs[j]), want[j])
        torch.cuda.synchronize()
        assert same(outs[0], want[i]) and same(outs[1], want[j])
    from exl3xpu.norm import RmsNorm
    fp4 = _fp4()
    mlp = fp4.Fp4Mlp(fp4.Fp4Linear(*_weight(g, 512, 256)), fp4.Fp4Linear(*_weight(g, 256, 256)))
    norm, lin = RmsNorm(torch.ones(256, device="cuda")), _linear(*_weight(g, 1000, 256))

    def parts(x):
        return [mlp(x), lin(x), *norm.quant(x, x, "fp4", rows=True), norm(x), fp4.dequant(*fp4.quant(x))]
    big = [torch.randn(m, 256, generator=g, device="cuda").bfloat16() for m in (1500, 30)]
    alone = [[t.clone() for t in parts(x)] for x in big]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in big], [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(parts(big[i]))
    torch.cuda.synchronize()
    assert all(same(t, alone[i]) for i in range(2) for t in got[i])


@pytest.mark.parametrize("M,n,k", [(3, 200, 512), (40, 200, 512), (300, 256, 1024), (1100, 1000, 384), (2100, 2100, 256)])
def test_products_of_every_code_and_sums_that_cancel(M, n, k):
    """Codes spread evenly, scales over eight powers of two, and products that cancel in pairs."""
    g = _gen(57 + M)
    q, w = (torch.randint(0, 256, (a, k // 2), generator=g, device="cuda").to(torch.uint8) for a in (M, n))
    s, sw = (torch.randint(123, 131, (a, k // 32), generator=g, device="cuda").to(torch.uint8) for a in (M, n))
    for cancel in (False, True):
        if cancel:                                           # (neighbours with the same weight and opposite signs)
            low = q & 15
            q = low | (low ^ 8) << 4
            w = (w & 15) | (w & 15) << 4
        lin = _linear(w, sw)
        held = torch.nn.functional.pad(s, (0, -s.size(1) % 8)).view(M, -1, 8)
        for dtype in DTYPES:
            print(f"case fp4 products of every code M={M} cancel={cancel} {dtype}", flush=True)
            y = lin.quantised(q, held, dtype)
            torch.cuda.synchronize()
            xv = _values(q, held, k)
            ref, mag = _product_ref(xv, w, sw, None)
            half = torch.finfo(dtype).eps / 2
            tol = (k + k / 64 + 20) * 2.0 ** -23 * mag
            tol = tol + half * (ref.abs() + tol)
            fits = ref.abs() + tol < torch.finfo(dtype).max
            assert fits.all() if dtype != torch.float16 else fits.sum() > 50
            assert ((y.double() - ref).abs() <= tol)[fits].all()


# (gate|up in 128 x 128 tiles, one to a CU at most and more; in 256 x 256 ones, one to a workgroup and several; each with an I whose
# last 128 columns are half a stage, one that ends inside a block, ragged rows)
@pytest.mark.parametrize("M,k,I,n", [(2000, 512, 1000, 260), (2000, 1100, 640, 130), (4100, 512, 1000, 260), (8190, 1024, 640, 130),
                                     (8190, 1100, 1000, 260), (16001, 1024, 1000, 260)])
def test_mlp_of_prompts(M, k, I, n):  # noqa: E741
    fp4, g = _fp4(), _gen(61 + M)
    gu, dn = _weight(g, 2 * I, k), _weight(g, n, I)
    for bias in (False, True):
        b = [torch.randn(c, generator=g, device="cuda") if bias else None for c in (2 * I, n)]
        mlp = fp4.Fp4Mlp(fp4.Fp4Linear(*gu, b[0]), fp4.Fp4Linear(*dn, b[1]))
        x = torch.randn(M, k, generator=g, device="cuda").bfloat16()
        for dtype in DTYPES:
            print(f"case fp4 mlp of prompts M={M} k={k} I={I} bias={bias} {dtype}", flush=True)
            y = mlp.quantised(*fp4.quant(x), dtype)
            torch.cuda.synchronize()
            _check_mlp(y, x, gu, dn, b, k, I)
            if dtype == x.dtype:
                assert torch.equal(mlp(x), y)
                want = y
        bad = torch.tensor([0, 31, 32, 130, 255, 256, M // 2, M - 1], device="cuda")
        x[bad[::2], k - 1] = math.nan
        x[bad[1::2], 0] = math.inf
        y = mlp(x)
        rows = torch.ones(M, dtype=torch.bool, device="cuda").index_fill(0, bad, False)
        assert y[bad].isnan().all() and torch.equal(y[rows], want[rows])


# (256 x 256 tiles of one to three stages of k, one to a workgroup and several, the last stage a half one and ending inside a block)
@pytest.mark.parametrize("M,k,n", [(8192, 128, 2048), (8150, 100, 2047), (8150, 256, 2048), (4100, 250, 12287), (8192, 512, 2048),
                                   (8150, 384, 4090), (16001, 300, 2048), (8150, 768, 2047), (2040, 640, 12288)])
def test_products_of_few_stages(M, k, n):
    g = _gen(71 + M + k)
    w = _weight(g, n, k)
    x = torch.randn(M, k, generator=g, device="cuda")
    x[M // 3] = 0
    q, s = _fp4().quant(x)
    xv = _values(q, s, k)
    for bias in (None, torch.randn(n, generator=g, device="cuda")):
        lin = _linear(*w, bias)
        for dtype in DTYPES:
            print(f"case fp4 products of few stages M={M} k={k} n={n} bias={bias is not None} {dtype}", flush=True)
            y = lin.quantised(q, s, dtype)
            torch.cuda.synchronize()
            _check_product(y, xv, *w, bias)
