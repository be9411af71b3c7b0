"""The 8-bit float linear (torch.ops.exl3xpu_C.fp8_*, exl3xpu.fp8) against its definition in 64 bits, where it can go wrong:
sizes around the 128-blocks and the tiles, strides, odd addresses, zero, tiny, huge, infinite and NaN blocks, one row and
none, streams and graphs.

Quantised rows have to be equal, bit for bit: scale and quotient are single roundings. Behind silu the value may be 8 units
of 2^-24 off (exp2 and reciprocal 1 unit each, five roundings), the scale as many and one, so a quotient is at most 18 off
and q the rounding of something within that. A product's error is at most that of its fp32 sums: 128 terms within an MFMA
and three roundings per block, (128 + 3 blocks + 4) 2^-23 of the sum of magnitudes (2^-23: sums that truncate), then half a
step of the output type. With bf16 and fp16 outputs the block sums come from e4m3 MFMAs, which align the products of 8
neighbouring k to the exponent E of their largest and drop what is below 2^(E - 13): at most 7 products of a group lose less
than 2^-13 of the largest each, so less than 7 2^-13 of the group's magnitudes; and as losses of random sign, 2^-13 sqrt(7 /
3) times the root of the group's mean largest square, which for normal values (largest of 8 products: 4 times their own
root mean square at the most) is sqrt(16 groups / 128 terms) 4 sqrt(7 / 3) 2^-13 = 2.6e-4 of the whole product's norm."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _fp8():
    from exl3xpu import fp8
    return fp8


def linear_ops():
    from exl3xpu.linear import C
    return C()


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _e4m3(v):
    """64-bit values to the nearest e4m3 value, halves to even."""
    a = v.abs().clamp_min(2.0 ** -6)
    step = torch.exp2(torch.floor(torch.log2(a)).clamp(-6, 8) - 3)
    return torch.where(v.isfinite(), torch.round(v / step) * step, torch.full_like(v, math.nan))


def _blocks(x):
    M, k = x.shape
    kb = -(-k // 128)
    return torch.nn.functional.pad(x, (0, kb * 128 - k)).reshape(M, kb, 128)


def _quant_ref(x):
    """x in 64 bits -> (q, s), each rounded as the definition says."""
    p = _blocks(x)
    s = (p.abs().amax(-1) / 448).float().double().clamp_min(2.0 ** -80)
    return _e4m3((p / s[..., None]).float().double()).reshape(x.size(0), -1), s


def _weight(g, n, k):
    w = torch.randn(n, k, generator=g, device="cuda") * 0.05
    nb, kb = -(-n // 128), -(-k // 128)
    p = torch.zeros(nb * 128, kb * 128, device="cuda")
    p[:n, :k] = w
    s = (p.view(nb, 128, kb, 128).abs().amax((1, 3)) / 448).clamp_min(1e-12)
    q = (p.view(nb, 128, kb, 128) / s[:, None, :, None]).view(nb * 128, kb * 128)[:n, :k]
    return q.to(torch.float8_e4m3fn), s


def _product_ref(q, s, w, sw, bias):
    """(the product, the sum of its terms' magnitudes) in 64 bits."""
    n, k = w.shape
    a = (q.double().reshape(q.size(0), -1, 128) * s.double()[..., None]).reshape(q.size(0), -1)[:, :k]
    b = w.double() * sw.double().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
    y, mag = a @ b.t(), a.abs() @ b.abs().t()
    return (y, mag) if bias is None else (y + bias.double(), mag + bias.double().abs())


def _check_product(y, q, s, w, sw, bias):
    ref, mag = _product_ref(q, s, w, sw, bias)
    half, loss = torch.finfo(y.dtype).eps / 2, 0.0 if y.dtype == torch.float32 else 7 * 2.0 ** -13
    tol = ((128 + 3 * s.size(-1) + 4) * 2.0 ** -23 + loss) * mag
    tol = tol + half * (ref.abs() + tol) + torch.finfo(y.dtype).smallest_normal
    bad = ~((y.double() - ref).abs() <= tol)
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist(), float(((y.double() - ref).abs() / tol).max()))
    if y.numel() > 1000:
        rel = float((y.double() - ref).norm() / ref.norm())
        assert rel <= half + (2.6e-4 if loss else (128 + 3 * s.size(-1) + 4) * 2.0 ** -23), rel


def _odd(t):
    """The same values at an odd element of their storage."""
    store = torch.zeros(t.numel() + 3, dtype=t.dtype, device=t.device)
    v = store[1:1 + t.numel()].view(t.shape)
    v.copy_(t)
    return v


@pytest.mark.parametrize("k", [1, 7, 8, 127, 128, 129, 500, 640, 1000, 2048, 2050])
def test_quant(k):
    g = _gen(k)
    for dtype in DTYPES:
        for M in (1, 2, 15, 16, 17, 130):
            print(f"case fp8 quant k={k} M={M} {dtype}", flush=True)
            x = (torch.randn(M, k, generator=g, device="cuda") * torch.exp(torch.randn(M, 1, generator=g, device="cuda"))).to(dtype)
            if M > 2:
                x[1] = 0
                x[2, k // 2:] = 0
            q, s = _fp8().quant(x)
            torch.cuda.synchronize()
            rq, rs = _quant_ref(x.double())
            assert q.dtype == torch.float8_e4m3fn and q.shape == rq.shape and s.shape == rs.shape
            assert torch.equal(s.double(), rs) and torch.equal(q.double(), rq)
            for other in (_odd(x), torch.nn.functional.pad(x, (0, 9))[:, :k], x.t().contiguous().t()):
                q2, s2 = _fp8().quant(other)
                assert torch.equal(q2.view(torch.uint8), q.view(torch.uint8)) and torch.equal(s2, s)


def test_quant_every_half_step():
    """Quotients that lie between two e4m3 values go to the even one, and every e4m3 value comes back as it is."""
    vals = torch.arange(127, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn).float()      # 0 .. 448
    mid = (vals[1:] + vals[:-1]) / 2
    x = torch.zeros(4, 128, device="cuda")
    x[0, :127] = vals
    x[1, :126], x[1, 126] = mid, 448
    x[2, :126], x[2, 126] = -torch.nextafter(mid, mid * 2), 448
    x[3, :126], x[3, 126] = torch.nextafter(mid, mid * 0), -448
    for scale in (1.0, 2.0 ** -60, 2.0 ** 90, 3.0, 1 / 3.0):
        q, s = _fp8().quant(x * scale)
        rq, rs = _quant_ref((x * scale).double())
        assert torch.equal(s.double(), rs) and torch.equal(q.double(), rq), scale
    q, s = _fp8().quant(x)
    assert (s == 1).all() and torch.equal(q[0, :127].float(), vals)


def test_quant_infinities_nan_and_extremes():
    x = torch.randn(9, 400, generator=_gen(3), device="cuda")
    x[0, 5] = math.inf
    x[1, 200] = -math.inf
    x[2, 300] = math.nan
    x[3, :128] = 3.4e38
    x[4] *= 1e-30
    x[5] *= 1e-42
    x[6, 130:250] = 0
    x[7, 399] = math.nan
    x[8] *= 1e36
    q, s = _fp8().quant(x)
    torch.cuda.synchronize()
    q, s = q.float(), s.cpu()
    assert s[0, 0] == math.inf and q[0, 5].isnan() and (q[0, [i for i in range(128) if i != 5]] == 0).all()
    assert s[1, 1] == math.inf and s[2, 2].isnan() and q[2, 256:384].isnan().all() and s[7, 3].isnan()
    assert s[[0, 1, 2], [1, 0, 0]].isfinite().all()
    fine = [3, 4, 5, 6, 8]
    rq, rs = _quant_ref(x[fine].double())
    assert torch.equal(q[fine].double(), rq) and torch.equal(s[fine].double(), rs.cpu())
    assert (q[5] == 0).all() and (s[5] == 2.0 ** -80).all()


@pytest.mark.parametrize("k", [1, 60, 127, 128, 129, 512, 640, 1001])
def test_silu_mul_quant(k):
    g = _gen(100 + k)
    for dtype in DTYPES:
        for M in (1, 3, 16, 131):
            print(f"case fp8 silu k={k} M={M} {dtype}", flush=True)
            gu = (torch.randn(M, 2 * k, generator=g, device="cuda") * 4).to(dtype)
            if M > 2:
                gu[1, :k] = -90.0                            # silu far below what fp32 holds comfortably
                gu[2] = 0
            for t in (gu, _odd(gu), torch.nn.functional.pad(gu, (0, 5))[:, :2 * k]):
                q, s = _fp8().silu_mul_quant(t)
                torch.cuda.synchronize()
                a, u = gu[:, :k].double(), gu[:, k:].double()
                v = _blocks(a / (1 + torch.exp(-a)) * u)
                rs = (v.abs().amax(-1) / 448).clamp_min(2.0 ** -80)
                eps = 2.0 ** -24
                assert ((s.double() - rs).abs() <= 9 * eps * rs).all()
                quo = (v / rs[..., None]).reshape(M, -1)
                lo, hi = _e4m3(quo.abs() * (1 - 19 * eps)), _e4m3(quo.abs() * (1 + 19 * eps))
                got = q.double()
                assert ((got.abs() >= lo) & (got.abs() <= hi) & ((got == 0) | (got.sign() == quo.sign()))).all()


def test_silu_infinities_and_nan():
    gu = torch.ones(5, 256, device="cuda")
    gu[0, 3] = math.inf
    gu[1, 3] = -math.inf
    gu[2, 3] = math.nan
    gu[3, 130] = math.inf
    gu[4, 3] = -200.0
    q, s = _fp8().silu_mul_quant(gu)
    torch.cuda.synchronize()
    assert s[0, 0] == math.inf and s[1, 0].isnan() and s[2, 0].isnan() and s[3, 0] == math.inf and s[4, 0].isfinite()
    assert q[4, 3].float() == 0 and (q[0].float().nan_to_num() == 0).all()


SIZES = [(1, 128), (5, 1), (16, 129), (17, 640), (127, 1000), (128, 512), (129, 2048), (200, 127), (384, 1152), (1000, 2000)]


@pytest.mark.parametrize("n,k", SIZES)
def test_linear(n, k):
    g = _gen(7 * n + k)
    w, sw = _weight(g, n, k)
    bias = torch.randn(n, generator=g, device="cuda")
    lin, linb = _fp8().Fp8Linear(w, sw), _fp8().Fp8Linear(w, sw, bias)
    for M in (1, 2, 3, 8, 9, 15, 16, 17, 31, 32, 33, 63, 64, 65, 100, 127, 128, 129, 255, 257, 300):
        for dtype in DTYPES:
            print(f"case fp8 linear n={n} k={k} M={M} {dtype}", flush=True)
            x = torch.randn(M, k, generator=g, device="cuda").to(dtype)
            y, yb = lin(x), linb(x)
            torch.cuda.synchronize()
            assert y.dtype == dtype and y.shape == (M, n)
            q, s = _quant_ref(x.double())
            _check_product(y, q, s, w, sw, None)
            _check_product(yb, q, s, w, sw, bias)
            q, s = _fp8().quant(x)
            assert torch.equal(lin.quantised(q, s, dtype), y)
            assert torch.equal(lin(_odd(x)), y)


@pytest.mark.parametrize("M,n,k", [(700, 512, 2048), (1025, 640, 384), (2048, 2048, 512), (513, 4096, 130), (64, 8192, 256),
                                   (40, 2048, 4096), (1, 12288, 2048), (4, 1024, 2048), (300, 12288, 512)])
def test_linear_larger(M, n, k):
    g = _gen(M + n)
    w, sw = _weight(g, n, k)
    lin = _fp8().Fp8Linear(w, sw)
    for dtype in DTYPES:
        print(f"case fp8 linear M={M} n={n} k={k} {dtype}", flush=True)
        x = (torch.randn(M, k, generator=g, device="cuda") * torch.exp(torch.randn(M, 1, generator=g, device="cuda"))).to(dtype)
        y = lin(x)
        torch.cuda.synchronize()
        _check_product(y, *_quant_ref(x.double()), w, sw, None)
        assert torch.equal(lin(x), y)                        # the same sums in the same order


@pytest.mark.parametrize("n,k,Ms", [(2000, 1300, (33, 40, 47, 64, 90, 100, 127, 300)), (2050, 4000, (64, 97, 128)),
                                    (1990, 640, (770, 1000, 1090, 1500, 2200)), (5000, 2048, (1, 3, 4, 5, 8, 16, 17)), (1000, 4096, (1, 2, 3, 4, 5, 16, 17, 31)),
                                    (1100, 1152, (80, 2030)), (12200, 200, (100, 1100)),
                                    (8300, 640, (14, 16, 20)), (8200, 300, (128, 129))])
def test_linear_tiles(n, k, Ms):
    """Sizes of every tile, with one workgroup per CU at most and with more, and edges inside a tile."""
    g = _gen(n + k)
    w, sw = _weight(g, n, k)
    bias = torch.randn(n, generator=g, device="cuda")
    lin = _fp8().Fp8Linear(w, sw, bias)
    for M in Ms:
        for dtype in DTYPES:
            print(f"case fp8 linear tiles n={n} k={k} M={M} {dtype}", flush=True)
            x = torch.randn(M, k, generator=g, device="cuda").to(dtype)
            y = lin(x)
            torch.cuda.synchronize()
            _check_product(y, *_quant_ref(x.double()), w, sw, bias)
            assert torch.equal(lin(_odd(x)), y)
            assert torch.equal(lin.quantised(*_fp8().quant(x), dtype), y)


def test_linear_rows_do_not_see_each_other():
    """A NaN or an infinity stays in its row, and a NaN weight in its column."""
    g = _gen(21)
    for M in (5, 40, 300):
        w, sw = _weight(g, 300, 384)
        x = torch.randn(M, 384, generator=g, device="cuda").bfloat16()
        want = _fp8().Fp8Linear(w, sw)(x)
        x[1, 200] = math.nan
        x[3, 0] = math.inf
        raw = w.clone().view(torch.uint8)
        raw[130, 5] = 0x7F                                   # e4m3's NaN
        y = _fp8().Fp8Linear(raw.view(torch.float8_e4m3fn), sw)(x)
        torch.cuda.synchronize()
        assert y[1].isnan().all() and y[3].isnan().all() and y[:, 130].isnan().all()
        rows = [m for m in range(M) if m not in (1, 3)]
        cols = [i for i in range(300) if i != 130]
        assert torch.equal(y[rows][:, cols], want[rows][:, cols])


def test_linear_shapes_strides_and_empty():
    g = _gen(23)
    w, sw = _weight(g, 260, 300)
    lin = _fp8().Fp8Linear(w, sw)
    x = torch.randn(24, 300, generator=g, device="cuda").bfloat16()
    y = lin(x)
    assert torch.equal(lin(x.view(2, 3, 4, 300)), y.view(2, 3, 4, 260))
    assert torch.equal(lin(x[0]), lin(x[:1])[0])
    assert torch.equal(lin(torch.nn.functional.pad(x, (0, 7))[:, :300]), y)
    assert torch.equal(lin(x.t().contiguous().t()), y)
    assert torch.equal(lin(x[:1].expand(24, 300)), lin(x[:1]).expand(24, 260))
    assert lin(x[:0]).shape == (0, 260) and lin(x.view(4, 6, 300)[:, :0]).shape == (4, 0, 260)
    q, s = _fp8().quant(x.view(4, 6, 300))
    assert torch.equal(lin.quantised(q, s, torch.bfloat16), y.view(4, 6, 260))
    assert lin.quantised(q[:, :0], s[:, :0], torch.float16).shape == (4, 0, 260)


def test_c_abi_leaves_what_is_behind_a_row():
    """Columns behind n and rows behind M of a wider output are left as they were, and a workspace of a larger call does
    for a smaller one."""
    from exl3xpu import capi
    L, st = capi.lib(), torch.cuda.current_stream().cuda_stream
    g = _gen(25)
    for M, n, k in ((1, 130, 256), (20, 200, 384), (200, 257, 512)):
        w, sw = _weight(g, n, k)
        x = torch.randn(M, k, generator=g, device="cuda").bfloat16()
        out = torch.full((M + 3, n + 5), 7.0, dtype=torch.bfloat16, device="cuda")
        ws = torch.empty(L.exl3_fp8_linear_workspace(M + 500, k, n), dtype=torch.uint8, device="cuda")
        print(f"case fp8 c-abi M={M} n={n} k={k}", flush=True)
        capi.check(L.exl3_fp8_linear(x.data_ptr(), 1, k, M, k, n, w.data_ptr(), sw.data_ptr(), None, out.data_ptr(), 1,
                                     n + 5, ws.data_ptr(), ws.numel(), st))
        torch.cuda.synchronize()
        assert torch.equal(out[:M, :n], _fp8().Fp8Linear(w, sw)(x))
        assert (out[M:] == 7).all() and (out[:, n:] == 7).all()


def test_rows_and_weights_past_32_bits():
    """Rows, quantised rows, weights and outputs whose bytes lie past 2^32."""
    g = _gen(41)
    k, M = 4096, 1_050_000
    x = torch.zeros(M, k, dtype=torch.bfloat16, device="cuda")
    x[-300:] = torch.randn(300, k, generator=g, device="cuda").bfloat16()
    print("case fp8 rows past 32 bits", flush=True)
    q, s = _fp8().quant(x)
    rq, rs = _quant_ref(x[-300:].double())
    assert torch.equal(q[-300:].double(), rq) and torch.equal(s[-300:].double(), rs)
    w, sw = _weight(g, 200, k)
    lin = _fp8().Fp8Linear(w, sw)
    y = lin.quantised(q, s, torch.float16)
    _check_product(y[-300:], rq, rs, w, sw, None)
    assert not y[:1000].any() and not y[M // 2:M // 2 + 1000].any()
    del x, q, s, y
    n = 1_050_000
    raw = torch.zeros(n, k, dtype=torch.uint8, device="cuda")
    raw[-200:] = w.view(torch.uint8)
    sw = torch.ones(-(-n // 128), k // 128, device="cuda")
    lin = _fp8().Fp8Linear(raw.view(torch.float8_e4m3fn), sw)
    for M in (1, 20, 300):
        print(f"case fp8 weights past 32 bits M={M}", flush=True)
        x = torch.randn(M, k, generator=g, device="cuda").bfloat16()
        y = lin(x)
        _check_product(y[:, -200:], *_quant_ref(x.double()), w, torch.ones(2, k // 128, device="cuda"), None)
        assert not y[:, :1000].any()
    far = torch.zeros((1 << 31) + 2000, dtype=torch.bfloat16, device="cuda")      # rows 2^31 elements apart
    x = far.as_strided((2, 1000), (1 << 31, 1))
    x.copy_(torch.randn(2, 1000, generator=g, device="cuda"))
    w, sw = _weight(g, 48, 1000)
    lin = _fp8().Fp8Linear(w, sw)
    print("case fp8 rows 2^32 bytes apart", flush=True)
    assert torch.equal(lin(x), lin(x.contiguous()))
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(_fp8().quant(x), _fp8().quant(x.contiguous())))


def test_more_small_tiles_than_one_launch_holds():
    """2^27 rows of 128 to 16 columns: 16 x 16 tiles, which would be the ones, would take 2^32 threads."""
    g = _gen(37)
    M = 1 << 17
    q, s = _fp8().quant(torch.randn(M, 128, generator=g, device="cuda"))
    lin = _fp8().Fp8Linear(*_weight(g, 16, 128))
    want = lin.quantised(q, s, torch.bfloat16)
    print("case fp8 product of 2^27 rows", flush=True)
    got = lin.quantised(q.view(torch.uint8).repeat(1024, 1).view(q.dtype), s.repeat(1024, 1), torch.bfloat16)
    assert all(torch.equal(t, want) for t in got.split(M))


@pytest.mark.parametrize("k,n", [(128, 64), (384, 40), (2048, 256), (4096, 80), (640, 7000)])
def test_rows_quantised_within_the_product(k, n):
    """The rows up to which the product quantises them itself, and one more, also at strides and odd addresses."""
    g = _gen(43 + k)
    w, sw = _weight(g, n, k)
    lin = _fp8().Fp8Linear(w, sw)
    for M in range(1, 19):
        for dtype in DTYPES:
            print(f"case fp8 own rows k={k} n={n} M={M} {dtype}", flush=True)
            x = (torch.randn(M, k, generator=g, device="cuda") * 3).to(dtype)
            x[M // 2, : k // 2] = 0
            y = lin(x)
            torch.cuda.synchronize()
            _check_product(y, *_quant_ref(x.double()), w, sw, None)
            assert torch.equal(lin(_odd(x)), y) and torch.equal(lin(torch.nn.functional.pad(x, (0, 3))[:, :k]), y)


def test_a_workspace_of_a_larger_call():
    """One workspace for calls of every size, the largest first, and the smallest: nothing of a call is left in it."""
    from exl3xpu import capi
    L, st = capi.lib(), torch.cuda.current_stream().cuda_stream
    g = _gen(45)
    k, I, n = 512, 256, 384  # noqa: E741
    gu, gs = _weight(g, 2 * I, k)
    dn, ds = _weight(g, n, I)
    mlp = _fp8().Fp8Mlp(_fp8().Fp8Linear(gu, gs), _fp8().Fp8Linear(dn, ds))
    ws = torch.full((L.exl3_fp8_mlp_workspace(400, k, I, n, 1),), 0x7F, dtype=torch.uint8, device="cuda")
    for M in (400, 1, 33, 4, 130, 2, 400):
        x = torch.randn(M, k, generator=g, device="cuda").bfloat16()
        out = torch.full((M, n + 3), 9.0, dtype=torch.bfloat16, device="cuda")
        print(f"case fp8 mlp c-abi M={M}", flush=True)
        capi.check(L.exl3_fp8_mlp(x.data_ptr(), 1, k, M, k, I, n, gu.data_ptr(), gs.data_ptr(), None, dn.data_ptr(),
                                  ds.data_ptr(), None, out.data_ptr(), n + 3, ws.data_ptr(), ws.numel(), st))
        torch.cuda.synchronize()
        assert torch.equal(out[:, :n], mlp(x)) and (out[:, n:] == 9).all()


def test_refusals():
    g = _gen(27)
    w, sw = _weight(g, 256, 256)
    lin = _fp8().Fp8Linear(w, sw)
    C = linear_ops()
    x = torch.randn(4, 256, generator=g, device="cuda").bfloat16()
    q, s = _fp8().quant(x)
    bad = [lambda: lin(x[:, :255]), lambda: lin(x.double()), lambda: lin(x.to(torch.float8_e4m3fn)),
           lambda: C.fp8_linear(x, w.float(), sw, None), lambda: C.fp8_linear(x, w.t(), sw, None),
           lambda: C.fp8_linear(x, w, sw[:1], None), lambda: C.fp8_linear(x, w, sw.double(), None),
           lambda: C.fp8_linear(x, w, sw, torch.zeros(255, device="cuda")),
           lambda: C.fp8_linear(x, w, sw, torch.zeros(256, device="cuda").bfloat16()),
           lambda: C.fp8_linear(x, w.cpu(), sw, None), lambda: C.fp8_matmul(q, s[:3], w, sw, None, torch.bfloat16),
           lambda: C.fp8_matmul(q[:, :200], s, w, sw, None, torch.bfloat16),
           lambda: C.fp8_matmul(q, s, w, sw, None, torch.int32),
           lambda: C.fp8_matmul(q.view(torch.float8_e5m2), s, w, sw, None, torch.bfloat16),
           lambda: C.fp8_mlp(x, w, sw, None, w, sw, None), lambda: C.fp8_mlp(x, w[:255], sw, None, w[:, :128], sw[:, :1], None),
           lambda: C.fp8_mlp(x, w, sw, None, w[:, :128].contiguous(), sw[:, :1], None),
           lambda: _fp8().Fp8Mlp(lin, _fp8().Fp8Linear(w[:, :128], sw[:, :1]))(x[:, :200]),
           lambda: _fp8().quant(x.int()), lambda: _fp8().quant(x[:, :0]), lambda: _fp8().silu_mul_quant(x[:, :255])]
    for i, f in enumerate(bad):
        with pytest.raises((RuntimeError, ValueError)):
            f()
            pytest.fail(f"call {i} was taken")
    with pytest.raises(NotImplementedError):
        _fp8().quant(x.cpu())


def _mlp(g, k, I):  # noqa: E741
    fp8 = _fp8()
    return fp8.Fp8Mlp(fp8.Fp8Linear(*_weight(g, 2 * I, k)), fp8.Fp8Linear(*_weight(g, k, I)))


@pytest.mark.parametrize("M", [1, 4, 37, 300])
def test_mlp_is_its_parts(M):
    g = _gen(31)
    for k, I in ((2048, 512), (512, 640), (300, 200)):  # noqa: E741
        fp8 = _fp8()
        for bias in (False, True):
            b = [torch.randn(n, generator=g, device="cuda") if bias else None for n in (2 * I, k)]
            mlp = fp8.Fp8Mlp(fp8.Fp8Linear(*_weight(g, 2 * I, k), b[0]), fp8.Fp8Linear(*_weight(g, k, I), b[1]))
            for dtype in DTYPES:
                print(f"case fp8 mlp M={M} k={k} I={I} bias={bias} {dtype}", flush=True)
                x = torch.randn(M, k, generator=g, device="cuda").to(dtype)
                # gate|up with the sums of fp32 outputs, rounded to the type once
                gu = mlp.gate_up.quantised(*fp8.quant(x), torch.float32).to(dtype)
                want = mlp.down.quantised(*fp8.silu_mul_quant(gu), dtype)
                assert torch.equal(mlp(x), want) and torch.equal(mlp(_odd(x)), want)
                assert mlp(x[:0]).shape == (0, k) and torch.equal(mlp(x[None]), want[None])


def _layer(g, M):
    """An MoE layer as a model runs it: router, routed experts through the cache, shared expert."""
    from exl3xpu.moe_offload import ExpertStore
    from exl3xpu.routing import Router
    from exl3xpu.synth import expert_blob
    H, I, E = 256, 128, 16  # noqa: E741
    store = ExpertStore(H, I, 3, E, E, max_layers=1)
    store.add_layer("layer0", torch.stack([expert_blob(5, e, H, I, 3) for e in range(E)]))
    mlp, wr = _mlp(g, H, I), torch.randn(E, H, generator=g, device="cuda") / 16
    router = Router(4, scoring="sigmoid", bias=0.05 * torch.randn(E, generator=g, device="cuda"), n_group=4, topk_group=2)

    def forward(x):
        return store.forward_routed("layer0", x, x.float() @ wr.t(), router) + mlp(x)
    return store, router, mlp, wr, forward


def test_layer_together():
    g = _gen(33)
    for M in (1, 3, 40):
        store, router, mlp, wr, forward = _layer(g, M)
        x = torch.randn(M, 256, generator=g, device="cuda").bfloat16()
        ids, w = router(x.float() @ wr.t())
        want = store.forward("layer0", x, ids, w) + mlp(x)
        got = forward(x)
        assert torch.equal(got, want)
        assert torch.equal(store.forward_routed("layer0", x, x.float() @ wr.t(), router, cached=False) + mlp(x), want)
        with pytest.raises(ValueError):
            store.forward_routed("layer0", x, (x.float() @ wr.t())[:, :8], router)


def test_layer_in_two_graphs_and_on_streams():
    """Two captured layers replayed in turn, eager work between; then the parts on two streams at once."""
    g = _gen(35)
    M = 3
    store, router, mlp, wr, forward = _layer(g, M)
    xs = [torch.randn(M, 256, generator=g, device="cuda").bfloat16() for _ in range(3)]
    want = [forward(x).clone() for x in xs]
    torch.cuda.synchronize()
    bufs, outs, graphs = [xs[0].clone(), xs[1].clone()], [], []
    for b in bufs:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(forward(b))
        graphs.append(gr)
    for i, j in ((0, 1), (2, 0), (1, 2), (2, 1)):
        bufs[0].copy_(xs[i])
        bufs[1].copy_(xs[j])
        graphs[0].replay()
        graphs[1].replay()
        assert torch.equal(forward(xs[j]), want[j])
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[i]) and torch.equal(outs[1], want[j])
    big = [torch.randn(m, 256, generator=g, device="cuda").bfloat16() for m in (500, 30)]
    alone = [mlp(x).clone() for x in big]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in big], [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(mlp(big[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(t, alone[i]) for i in range(2) for t in got[i])


def _check_silu_gates(gates, ups):
    """silu(gate) * up of single values, each a block of its own, so that its scale shows the value itself: 8 units of 2^-24
    and the scale's own rounding, at every size of the value down to the smallest scale."""
    for up in ups:
        v = gates.double() / (1 + torch.exp(-gates.double())) * up
        fits = v.abs() < 2.0 ** 127
        g, v = gates[fits], v[fits]
        q, s = _fp8().silu_mul_quant(torch.stack([g, torch.full_like(g, up)], 1))
        torch.cuda.synchronize()
        rs = (v.abs() / 448).clamp_min(2.0 ** -80)
        off = (s[:, 0].double() - rs).abs() / rs
        bad = ~(off <= 9 * 2.0 ** -24)
        assert not bad.any(), (up, int(bad.sum()), g[bad][:8].tolist(), s[bad][:8, 0].tolist(), float(off.nan_to_num(9).max()) * 2 ** 24)
        quo, got = v / rs, q[:, 0].double()
        lo, hi = _e4m3(quo.abs() * (1 - 19 * 2.0 ** -24)), _e4m3(quo.abs() * (1 + 19 * 2.0 ** -24))
        assert ((got.abs() >= lo) & (got.abs() <= hi) & ((got == 0) | (got.sign() == quo.sign()))).all()
        assert (q.view(torch.uint8)[:, 1:] == 0).all()


def _finite16(dtype):
    """Every finite value of a 16-bit type."""
    v = torch.arange(1 << 16, device="cuda").to(torch.uint16).view(dtype)
    return v[v.isfinite()]


def test_silu_of_large_negative_gates():
    """Gates at which exp(-gate) passes fp32's largest value, every one of the 16-bit types, with ups of 1 and ups for which the
    product is no zero all the same."""
    for dtype, ups in ((torch.bfloat16, (1.0, 2.0 ** 40, 2.0 ** 90)), (torch.float16, (1.0, 2.0 ** 15))):
        print(f"case fp8 silu of large negative gates {dtype}", flush=True)
        v = _finite16(dtype)
        _check_silu_gates(v[v <= -40], ups)
    steps = torch.cat([torch.linspace(-140, -40, 200_001, device="cuda"), -torch.exp2(torch.arange(6, 128, device="cuda").float()),
                       torch.tensor([-torch.finfo(torch.float32).max], device="cuda")])
    print("case fp8 silu of large negative gates float32", flush=True)
    _check_silu_gates(steps, (1.0, 2.0 ** 40, 2.0 ** 100))


@pytest.mark.parametrize("M", [1, 4, 37, 300])
def test_mlp_of_large_negative_gates(M):
    """Columns whose gate is far below 0 count for nothing, as those with a gate of 0 do, whether the rows are quantised within
    the products or before."""
    fp8, g, k, I = _fp8(), _gen(51), 512, 384  # noqa: E741
    w, sw = _weight(g, 2 * I, k)
    raw = w.view(torch.uint8).clone()
    raw[:I] = 0                                              # (the gates are their biases, exactly)
    down = fp8.Fp8Linear(*_weight(g, k, I))
    gates = torch.randn(I, generator=g, device="cuda").bfloat16().float()
    far = torch.tensor([-91.0, -95.0, -110.0, -128.0, -256.0, -1000.0, -90.0, -200.0], device="cuda")
    biases = []
    for values in (far, torch.zeros_like(far)):
        b = torch.cat([gates, torch.zeros(I, device="cuda")])
        b[3:3 + 40 * 8:8] = values.repeat(5)
        biases.append(b)
    for dtype in DTYPES:
        print(f"case fp8 mlp of large negative gates M={M} {dtype}", flush=True)
        x = torch.randn(M, k, generator=g, device="cuda").to(dtype)
        y, want = (fp8.Fp8Mlp(fp8.Fp8Linear(raw.view(w.dtype), sw, b), down)(x) for b in biases)
        torch.cuda.synchronize()
        assert y.isfinite().all() and torch.equal(y, want)


def test_silu_every_gate():
    """Every finite gate of the 16-bit types and closely spaced ones of fp32, each value by itself."""
    for dtype, ups in ((torch.bfloat16, (1.0, -2.0 ** 40)), (torch.float16, (1.0, -2.0 ** 15))):
        print(f"case fp8 silu of every gate {dtype}", flush=True)
        _check_silu_gates(_finite16(dtype), ups)
    print("case fp8 silu of every gate float32", flush=True)
    _check_silu_gates(torch.linspace(-60, 60, 1_000_001, device="cuda"), (1.0, 3.0))


def test_linear_of_weights_at_odd_addresses():
    g = _gen(53)
    w, sw = _weight(g, 130, 256)
    x = torch.randn(20, 256, generator=g, device="cuda").bfloat16()
    want = _fp8().Fp8Linear(w, sw)(x)
    for at in (1, 8, 15):
        store = torch.zeros(w.numel() + 16, dtype=torch.uint8, device="cuda")
        v = store[at:at + w.numel()].view(w.dtype).view(w.shape)
        v.copy_(w)
        print(f"case fp8 weights at byte {at}", flush=True)
        assert torch.equal(_fp8().Fp8Linear(v, sw)(x), want)


@pytest.mark.parametrize("M,n,k", [(3, 200, 512), (40, 200, 512), (300, 256, 1024), (1100, 1000, 384), (2100, 2100, 256)])
def test_products_of_every_size_and_sums_that_cancel(M, n, k):
    """Operands spread evenly over e4m3's values, from 2^-9 to 448, and products that cancel in pairs: fp16 and bf16 outputs within
    what the e4m3 MFMA may lose, fp32 outputs within fp32 sums; fp32 outputs rounded by the caller have neither loss."""
    g = _gen(57 + M)

    def codes(rows, cols):
        c = torch.randint(0, 127, (rows, cols), generator=g, device="cuda") + 128 * torch.randint(0, 2, (rows, cols), generator=g, device="cuda")
        return c.to(torch.uint8)
    q, w = codes(M, k), codes(n, k)
    s, sw = (torch.rand(a, b, generator=g, device="cuda") + 0.5 for a, b in ((M, k // 128), (-(-n // 128), k // 128)))
    for cancel in (False, True):
        if cancel:                                           # (neighbours with the same weight and opposite signs)
            q[:, 1::2] = q[:, ::2] ^ 128
            w[:, 1::2] = w[:, ::2]
        qv, wv = q.view(torch.float8_e4m3fn), w.view(torch.float8_e4m3fn)
        lin = _fp8().Fp8Linear(wv, sw)
        for dtype in DTYPES:
            print(f"case fp8 products of every size M={M} cancel={cancel} {dtype}", flush=True)
            y = lin.quantised(qv, s, dtype)
            torch.cuda.synchronize()
            ref, mag = _product_ref(qv, s, wv, sw, None)
            half, loss = torch.finfo(dtype).eps / 2, 0.0 if dtype == torch.float32 else 7 * 2.0 ** -13
            tol = ((128 + 3 * s.size(-1) + 4) * 2.0 ** -23 + loss) * mag
            tol = tol + half * (ref.abs() + tol)
            fits = ref.abs() + tol < torch.finfo(dtype).max
            assert fits.sum() > 50 and ((y.double() - ref).abs() <= tol)[fits].all()      # (fp16 cannot hold the others)
