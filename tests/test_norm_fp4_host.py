"""What the norm and the 4-bit float linear refuse, their shapes, layouts and workspace sizes: no GPU."""
import pytest
import torch

from exl3xpu import capi, fp4, norm
from exl3xpu.linear import C

BAD, UNSUPPORTED, WORKSPACE = 1, 2, 4
P = 1 << 20                                     # an address that no refused call reads


def _norm(x=P, dtype=1, stride=256, inner=1, outer=0, res=P, rdt=1, rs=256, held=P, w=P, eps=1e-6, M=2, k=256, y=P, form=0,
          q=None, s=None, stage=0, unit=0):
    return capi.lib().exl3_rms_norm(x, dtype, stride, inner, outer, res, rdt, rs, held, w, unit, eps, M, k, y, form, q, s, stage, None)


@pytest.mark.parametrize("k,code", [
    (dict(k=0), BAD), (dict(M=-1), BAD), (dict(dtype=3), BAD), (dict(dtype=-1), BAD), (dict(x=None), BAD), (dict(x=P + 1), BAD),
    (dict(stride=-1), BAD), (dict(inner=0), BAD), (dict(inner=2, outer=-1), BAD), (dict(rdt=0), BAD), (dict(rdt=3), BAD),
    (dict(res=None), BAD), (dict(held=None), BAD), (dict(rs=255), BAD), (dict(res=P + 1), BAD), (dict(held=P + 1), BAD),
    (dict(rdt=2, held=P + 2), BAD), (dict(w=P + 2), BAD), (dict(eps=0.0), BAD), (dict(eps=-1.0), BAD),
    (dict(eps=float("nan")), BAD), (dict(eps=float("inf")), BAD), (dict(eps=1e-40), BAD), (dict(y=None), BAD), (dict(y=P + 1), BAD),
    (dict(form=3), BAD), (dict(form=-1), BAD), (dict(form=1), BAD), (dict(form=1, q=P, s=None), BAD),
    (dict(form=1, q=P + 8, s=P), BAD), (dict(form=1, q=P, s=P + 2), BAD), (dict(form=2, q=P, s=P + 4, stage=16), BAD),
    (dict(form=2, q=P + 8, s=P, stage=16), BAD), (dict(form=2, q=P, s=P, stage=8), BAD), (dict(form=2, q=P, s=P, stage=20), BAD),
    (dict(k=1 << 23, stride=1 << 23, rs=1 << 23), UNSUPPORTED), (dict(M=1 << 22, k=1 << 14, stride=1 << 14, rs=1 << 14), UNSUPPORTED),
    (dict(M=0, x=None), 0)])
def test_norm_refuses(k, code):
    assert _norm(**k) == code
    assert not code or capi.lib().exl3_last_error()


@pytest.mark.parametrize("size", [2, 4])
def test_norm_refuses_a_held_sum_over_other_elements_of_its_residual(size):
    """Where an element of the held sum lies on another one's residual, it is written while that one is still read: refused, and
    only there, against a search of all pairs of rows. (Every call has an output that is refused later: none is launched.)"""
    k, a = 256, 1 << 30
    seen = set()
    for M in (1, 2, 3, 5):
        for rs in (k, k + 8, k + 1, 2 * k, 3 * k, 8 * k):
            for at in (0, 1, -1, k, -k, k // 2, rs, rs - k, (M - 1) * rs, (M - 1) * rs + k, (M - 1) * rs + k - 1, -M * k, -M * k + 1,
                       1 - rs, rs * M, M * k):
                meet = any(at + m * k < r * rs + k and r * rs < at + m * k + k for m in range(M) for r in range(M))
                bad = meet and not (at == 0 and (M == 1 or rs == k))
                dt = 1 if size == 2 else 2
                assert _norm(dtype=dt, stride=k, res=a, rdt=dt, rs=rs, held=a + at * size, M=M, k=k, y=P + 1) == BAD
                assert (b"held over" in capi.lib().exl3_last_error()) == bad, (M, rs, at)
                seen.add((meet, bad))
    assert seen == {(False, False), (True, False), (True, True)}


def _rows(f, x=P, dtype=1, stride=256, M=2, k=256, q=P, s=P, stage=16):
    return getattr(capi.lib(), f)(x, dtype, stride, M, k, q, s, stage, None)


@pytest.mark.parametrize("k,code", [
    (dict(k=0), BAD), (dict(M=-1), BAD), (dict(dtype=3), BAD), (dict(x=None), BAD), (dict(q=None), BAD), (dict(s=None), BAD),
    (dict(stride=100), BAD), (dict(x=P + 1), BAD), (dict(q=P + 8), BAD), (dict(s=P + 4), BAD), (dict(stage=8), BAD),
    (dict(stage=17), BAD), (dict(k=1 << 29, stride=1 << 30), UNSUPPORTED),
    (dict(M=1 << 30, k=1 << 10, stride=1 << 11, stage=1 << 33), UNSUPPORTED), (dict(M=1 << 27, stage=1 << 30), UNSUPPORTED),
    (dict(M=0, x=None), 0)])
def test_rows_refuse(k, code):
    assert _rows("exl3_fp4_quant", **k) == code
    assert _rows("exl3_fp4_silu_mul_quant", **{"stride": 512 if k.get("k", 0) < 1 << 10 else 1 << 31, **k}) == code
    assert _rows("exl3_fp4_silu_mul_quant", stride=511) == BAD       # gate|up rows are twice as long


def _dequant(q=P, s=P, stage=16, M=2, k=256, out=P, dt=1):
    return capi.lib().exl3_fp4_dequant(q, s, stage, M, k, out, dt, None)


@pytest.mark.parametrize("k,code", [
    (dict(k=0), BAD), (dict(M=-1), BAD), (dict(dt=3), BAD), (dict(q=None), BAD), (dict(s=None), BAD), (dict(out=None), BAD),
    (dict(out=P + 1), BAD), (dict(q=P + 4), BAD), (dict(s=P + 1), BAD), (dict(stage=8), BAD), (dict(k=1 << 23), UNSUPPORTED),
    (dict(M=0, q=None, s=None, out=None), 0)])
def test_dequant_refuses(k, code):
    assert _dequant(**k) == code


def _matmul(q=P, s=P, stage=32, M=4, k=256, n=256, w=P, sw=P, bias=None, out=P, dt=1, stride=256):
    return capi.lib().exl3_fp4_matmul(q, s, stage, M, k, n, w, sw, bias, out, dt, stride, None)


def _linear(x=P, dtype=1, xs=256, M=4, k=256, n=256, w=P, sw=P, bias=None, out=P, dt=1, stride=256, ws=P, size=1 << 40):
    return capi.lib().exl3_fp4_linear(x, dtype, xs, M, k, n, w, sw, bias, out, dt, stride, ws, size, None)


def _mlp(x=P, dtype=1, xs=256, M=4, k=256, I=128, n=256, gu=P, gs=P, gb=None, dn=P, ds=P, db=None, out=P, dt=1, stride=256,  # noqa: E741
         ws=P, size=1 << 40):
    return capi.lib().exl3_fp4_mlp(x, dtype, xs, M, k, I, n, gu, gs, gb, dn, ds, db, out, dt, stride, ws, size, None)


def _mlp_matmul(q=P, s=P, stage=32, M=4, k=256, I=128, n=256, gu=P, gs=P, gb=None, dn=P, ds=P, db=None, out=P, dt=1,  # noqa: E741
                stride=256, ws=P, size=1 << 40):
    return capi.lib().exl3_fp4_mlp_matmul(q, s, stage, M, k, I, n, gu, gs, gb, dn, ds, db, out, dt, stride, ws, size, None)


@pytest.mark.parametrize("k,code", [
    (dict(k=0), BAD), (dict(n=0), BAD), (dict(M=-1), BAD), (dict(dt=3), BAD), (dict(w=None), BAD), (dict(sw=None), BAD),
    (dict(out=None), BAD), (dict(stride=255), BAD), (dict(w=P + 8), BAD), (dict(sw=P + 4), BAD), (dict(bias=P + 2), BAD),
    (dict(out=P + 1), BAD), (dict(n=1 << 29, stride=1 << 29), UNSUPPORTED), (dict(k=1 << 23), UNSUPPORTED),
    (dict(M=1 << 30, n=1 << 12, stride=1 << 12), UNSUPPORTED)])
def test_products_refuse(k, code):
    assert _matmul(**k) == code
    assert _linear(**k) == code


@pytest.mark.parametrize("k,code", [
    (dict(k=0), BAD), (dict(I=0), BAD), (dict(I=(1 << 22) + 1), BAD), (dict(n=0), BAD), (dict(M=-1), BAD), (dict(dt=3), BAD),
    (dict(gu=None), BAD), (dict(gu=P + 8), BAD), (dict(gs=None), BAD), (dict(gb=P + 2), BAD), (dict(dn=None), BAD),
    (dict(dn=P + 4), BAD), (dict(ds=P + 1), BAD), (dict(db=P + 2), BAD), (dict(out=None), BAD), (dict(out=P + 1), BAD),
    (dict(stride=255), BAD), (dict(ws=None), WORKSPACE), (dict(ws=P + 2), WORKSPACE), (dict(size=100), WORKSPACE),
    (dict(k=1 << 23), UNSUPPORTED)])
def test_mlp_refuses(k, code):
    assert _mlp(**k) == code
    assert _mlp_matmul(**k) == code


def test_products_refuse_their_own():
    assert [f(**k) for f in (_matmul, _mlp_matmul) for k in (dict(q=None), dict(s=None), dict(q=P + 8), dict(s=P + 4), dict(stage=24),
                                                             dict(stage=33))] == [BAD] * 12
    assert [f(**k) for f in (_linear, _mlp) for k in (dict(x=None), dict(dtype=3), dict(xs=255), dict(x=P + 1))] == [BAD] * 8
    assert [_linear(M=40, stride=256, ws=None), _linear(M=40, size=16), _linear(M=40, ws=P + 4)] == [WORKSPACE] * 3
    assert _matmul(M=0, q=None, s=None, w=None, sw=None, out=None) == _linear(M=0, x=None, ws=None) == 0
    assert _mlp(M=0, x=None, ws=None) == _mlp_matmul(M=0, q=None, s=None, ws=None) == 0


@pytest.mark.parametrize("k,n", [(1, 1), (128, 128), (2048, 12288), (4096, 2048), (2000, 1000), (512, 2048), (130, 4096)])
def test_workspaces_never_fall_as_the_rows_grow(k, n):
    L = capi.lib()
    for f, least in ((lambda M: L.exl3_fp4_linear_workspace(M, k, n), lambda M: M * k // 2), (lambda M: L.exl3_fp4_mlp_matmul_workspace(M, n), lambda M: M * n // 2),
                     (lambda M: L.exl3_fp4_mlp_workspace(M, k, n), lambda M: M * (k + n) // 2)):
        b = [f(M) for M in [*range(1, 600), 1024, 4096, 8192, 60000]]
        # (few rows are quantised within the product)
        assert all(x <= y for x, y in zip(b, b[1:])) and b[63] >= least(64) and b[-1] >= least(60000)
        assert [f(0), f(-5)] == [0] * 2
    assert [L.exl3_fp4_linear_workspace(4, 0, 8), L.exl3_fp4_linear_workspace(4, 8, -1), L.exl3_fp4_mlp_workspace(4, 0, 8),
            L.exl3_fp4_mlp_workspace(4, 8, 0), L.exl3_fp4_mlp_matmul_workspace(4, 0), L.exl3_fp4_mlp_matmul_workspace(4, 1 << 23)] == [0] * 6


def test_shapes_without_a_device():
    m = torch.device("meta")
    for f, cols in ((C().fp4_quant, 300), (C().fp4_silu_mul_quant, 600)):
        q, s = f(torch.empty(2, 7, cols, device=m, dtype=torch.bfloat16))
        assert q.shape == (2, 7, 192) and s.shape == (2, 7, 2, 8) and s.movedim(-2, 0).is_contiguous()
        assert q.dtype == s.dtype == torch.uint8
    y = C().fp4_dequant(q, s, 300, torch.float16)
    assert y.shape == (2, 7, 300) and y.dtype == torch.float16
    w, sw = torch.empty(130, 192, device=m, dtype=torch.uint8), torch.empty(2, 130, 8, device=m, dtype=torch.uint8).movedim(0, 1)
    y = C().fp4_linear(torch.empty(2, 7, 300, device=m, dtype=torch.float16), w, sw, None)
    assert y.shape == (2, 7, 130) and y.dtype == torch.float16
    y = C().fp4_matmul(q, s, w, sw, None, torch.bfloat16)
    assert y.shape == (2, 7, 130) and y.dtype == torch.bfloat16
    y = C().fp4_mlp(torch.empty(2, 7, 300, device=m), 300, w, sw, None, w, sw, None)
    assert y.shape == (2, 7, 130) and y.dtype == torch.float32
    assert C().fp4_mlp_matmul(q, s, 300, w, sw, None, w, sw, None, torch.float16).shape == (2, 7, 130)
    x, r = torch.empty(2, 7, 300, device=m, dtype=torch.bfloat16), torch.empty(2, 7, 300, device=m)
    assert [(t.shape, t.dtype) for t in C().rms_norm(x, None, None, 1e-6, 0, True)] == [(x.shape, x.dtype)]
    q, s, y, h = C().rms_norm(x, r, None, 1e-6, 1, True)
    assert (q.shape, q.dtype, s.shape, s.dtype) == ((2, 7, 384), torch.float8_e4m3fn, (2, 7, 3), torch.float32)
    assert (y.dtype, h.dtype, h.shape) == (torch.bfloat16, torch.float32, x.shape)
    q, s, h = C().rms_norm(x, x, None, 1e-6, 2, False)
    assert q.shape == (2, 7, 192) and s.shape == (2, 7, 2, 8) and h.dtype == torch.bfloat16


def test_scalars_have_no_rows():
    m = torch.device("meta")
    w, sw, x = torch.empty(130, 192, device=m, dtype=torch.uint8), torch.empty(130, 2, 8, device=m, dtype=torch.uint8), torch.empty((), device=m)
    for f in (lambda: C().fp4_linear(x, w, sw, None), lambda: C().fp4_matmul(x, x, w, sw, None, torch.bfloat16),
              lambda: C().fp4_mlp(x, 300, w, sw, None, w, sw, None), lambda: C().fp4_quant(x), lambda: C().fp4_silu_mul_quant(x),
              lambda: C().fp4_dequant(x, x, 4, torch.float16), lambda: C().rms_norm(x, None, None, 1e-6, 0, True)):
        with pytest.raises((RuntimeError, IndexError)):
            f()


def test_linear_lays_weights_out():
    g = torch.Generator().manual_seed(3)
    for k in (2, 31, 32, 100, 128, 256, 300, 640):
        n, used, blocks = 5, -(-k // 2), -(-k // 32)
        w = torch.randint(0, 256, (n, used), generator=g, dtype=torch.uint8)
        sw = torch.randint(0, 256, (n, blocks), generator=g, dtype=torch.uint8)
        for a, b in ((w, sw), (w.view(torch.float4_e2m1fn_x2), sw.view(torch.float8_e8m0fnu))):
            lin = fp4.Fp4Linear(a, b, k=k if k % 2 else None)
            cols, stages = -(-k // 128) * 128, -(-k // 256)
            assert (lin.n, lin.k) == (n, k) and lin.weight.shape == (n, cols // 2) and lin.weight.data_ptr() % 16 == 0
            full = w.clone()
            full[:, -1] &= 15 if k % 2 else 255
            assert torch.equal(lin.weight[:, :used], full) and not lin.weight[:, used:].any()
            assert lin.weight_scale.shape == (n, stages, 8) and lin.weight_scale.movedim(1, 0).is_contiguous()
            flat = lin.weight_scale.reshape(n, -1)
            assert torch.equal(flat[:, :blocks], sw) and not flat[:, blocks:].any()
        again = fp4.Fp4Linear(lin.weight, lin.weight_scale, k=k)         # the form of quant's rows
        assert torch.equal(again.weight, lin.weight) and torch.equal(again.weight_scale, lin.weight_scale)


def test_weights_at_any_address():
    store = torch.arange(128 * 128 + 16, dtype=torch.int64).remainder(251).to(torch.uint8)
    for at in range(16):
        w = store[at:at + 128 * 128].view(128, 128)
        lin = fp4.Fp4Linear(w, torch.ones(128, 8, dtype=torch.uint8))
        assert lin.weight.data_ptr() % 16 == 0 and torch.equal(lin.weight, w)


@pytest.mark.parametrize("I", [1, 31, 32, 100, 128, 200, 640])  # noqa: E741
def test_mlp_orders_gates_and_ups(I):  # noqa: E741
    k = 64
    w = torch.arange(2 * I).view(-1, 1).remainder(251).to(torch.uint8).expand(2 * I, k // 2).contiguous() + 1
    gu = fp4.Fp4Linear(w, torch.full((2 * I, 2), 120, dtype=torch.uint8), torch.arange(2 * I).float() + 1)
    mlp = fp4.Fp4Mlp(gu, fp4.Fp4Linear(torch.zeros(9, -(-I // 2), dtype=torch.uint8), torch.zeros(9, -(-I // 32), dtype=torch.uint8), k=I))
    weight, scale, bias = mlp._weights[:3]
    Ip = -(-I // 128) * 128
    assert weight.shape == (2 * Ip, 64) and scale.shape == (2 * Ip, 1, 8) and scale.movedim(1, 0).is_contiguous()
    for i in range(Ip):
        for up in (0, 1):
            row = i // 32 * 64 + up * 32 + i % 32
            assert bias[row] == (i + up * I + 1 if i < I else 0)
            assert torch.equal(weight[row], gu.weight[i + up * I] if i < I else torch.zeros_like(weight[row]))
            assert scale[row, 0].tolist() == ([120] * 2 + [0] * 6 if i < I else [0] * 8)


def test_classes_refuse():
    w, s = torch.zeros(256, 150, dtype=torch.uint8), torch.ones(256, 10, dtype=torch.uint8)
    lin = fp4.Fp4Linear(w, s)
    for bad in (lambda: fp4.Fp4Linear(w.float(), s), lambda: fp4.Fp4Linear(w[0], s), lambda: fp4.Fp4Linear(w, s[:1]),
                lambda: fp4.Fp4Linear(w, s[:, :9]), lambda: fp4.Fp4Linear(w, s.float()), lambda: fp4.Fp4Linear(w, s, torch.zeros(255)),
                lambda: fp4.Fp4Linear(w[:0], s[:0]), lambda: fp4.Fp4Linear(w, s, k=298), lambda: fp4.Fp4Linear(w, s, k=0),
                lambda: fp4.Fp4Linear(w, s, k=302), lambda: fp4.Fp4Mlp(lin, lin), lambda: norm.RmsNorm(torch.ones(2, 2)),
                lambda: norm.RmsNorm(torch.ones(0)), lambda: norm.RmsNorm(torch.ones(4), eps=0.0), lambda: norm.RmsNorm(eps=-1.0),
                lambda: norm.RmsNorm(eps=float("nan")), lambda: norm.RmsNorm(eps=1e-45), lambda: norm.RmsNorm(unit_offset=True),
                lambda: norm.RmsNorm(torch.ones(4)).quant(torch.ones(1, 4), form="int8")):
        with pytest.raises(ValueError):
            bad()
    n = norm.RmsNorm(torch.tensor([0.0, 0.5], dtype=torch.bfloat16), unit_offset=True)
    assert n.weight.dtype == torch.float32 and n.weight.tolist() == [0.0, 0.5] and n.unit_offset
    assert _norm(w=None, unit=1) == BAD


def _differentiable():
    """(operator's name, its call, a floating-point input) for every operator and every such input of it."""
    def t(*size, dtype=torch.float32):
        return torch.empty(*size, device="meta", dtype=dtype)
    x, r, w = t(2, 300), t(2, 300), t(300)
    q, s, b = t(2, 192, dtype=torch.uint8), t(2, 2, 8, dtype=torch.uint8), t(130)
    c, sc = t(130, 192, dtype=torch.uint8), t(2, 130, 8, dtype=torch.uint8).movedim(0, 1)
    gu, gs, gb = t(768, 192, dtype=torch.uint8), t(2, 768, 8, dtype=torch.uint8).movedim(0, 1), t(768)
    ops, f32 = C(), torch.float32
    yield from (("rms_norm", lambda v, i=i: ops.rms_norm(*[v if j == i else a for j, a in enumerate((x, r, w))], 1e-6, 2, True), a)
                for i, a in enumerate((x, r, w)))
    yield "fp4_quant", lambda v: ops.fp4_quant(v), x
    yield "fp4_silu_mul_quant", lambda v: ops.fp4_silu_mul_quant(v), x
    yield "fp4_linear", lambda v: ops.fp4_linear(v, c, sc, b), x
    yield "fp4_linear", lambda v: ops.fp4_linear(x, c, sc, v), b
    yield "fp4_matmul", lambda v: ops.fp4_matmul(q, s, c, sc, v, f32), b
    yield "fp4_mlp", lambda v: ops.fp4_mlp(v, 300, gu, gs, gb, c, sc, b), x
    yield "fp4_mlp", lambda v: ops.fp4_mlp(x, 300, gu, gs, v, c, sc, b), gb
    yield "fp4_mlp", lambda v: ops.fp4_mlp(x, 300, gu, gs, gb, c, sc, v), b
    yield "fp4_mlp_matmul", lambda v: ops.fp4_mlp_matmul(q, s, 300, gu, gs, v, c, sc, b, f32), gb
    yield "fp4_mlp_matmul", lambda v: ops.fp4_mlp_matmul(q, s, 300, gu, gs, gb, c, sc, v, f32), b


def test_no_input_loses_its_gradient_or_tangent():
    """Rows, residuals, weights and biases that need a gradient, or carry a tangent, are refused, in torch.func's transforms too; a
    result without them would be taken for a constant."""
    def first(out):
        return out if torch.is_tensor(out) else out[0]
    for name, f, a in _differentiable():
        def refused(call, f=f, name=name):
            with pytest.raises(RuntimeError, match=f"{name}: no gradients"):
                call(f)
        first(f(a))
        refused(lambda f: f(a.clone().requires_grad_()))
        with torch.no_grad():
            first(f(a.clone().requires_grad_()))
        with torch.inference_mode():
            first(f(a))
        with torch.autograd.forward_ad.dual_level():
            refused(lambda f: f(torch.autograd.forward_ad.make_dual(a, torch.ones_like(a))))
            with torch.no_grad():                            # (it stops no tangents)
                refused(lambda f: f(torch.autograd.forward_ad.make_dual(a, torch.ones_like(a))))
            first(f(a))
        refused(lambda f: torch.func.jvp(lambda v: first(f(v)), (a,), (torch.ones_like(a),)))
        refused(lambda f: torch.func.grad(lambda v: first(f(v)).float().sum())(a))
