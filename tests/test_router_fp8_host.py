"""What the router and the 8-bit float linear refuse, their shapes and workspace sizes: no GPU."""
import pytest
import torch

from exl3xpu import capi, fp8, routing
from exl3xpu.linear import C
from exl3xpu.moe_offload import ops

BAD, UNSUPPORTED, WORKSPACE = 1, 2, 4
P = 1 << 20                                     # an address that no refused call reads


def _route(logits=P, dtype=2, stride=64, M=2, E=64, bias=None, topk=4, scoring=0, n_group=1, topk_group=1, ids=P, w=P):
    return capi.lib().exl3_moe_route(logits, dtype, stride, M, E, bias, topk, scoring, n_group, topk_group, 1, 1.0, ids, w,
                                     None)


@pytest.mark.parametrize("k,code", [
    (dict(E=0), BAD), (dict(E=1025, stride=2000), BAD), (dict(M=-1), BAD), (dict(dtype=3), BAD), (dict(dtype=-1), BAD),
    (dict(scoring=2), BAD), (dict(topk=0), BAD), (dict(topk=65, E=128, stride=128), BAD), (dict(topk=9, E=8), BAD),
    (dict(n_group=0), BAD), (dict(n_group=7), BAD), (dict(n_group=8, topk_group=0), BAD), (dict(n_group=8, topk_group=9), BAD),
    (dict(n_group=8, topk_group=1, topk=9), BAD), (dict(E=130, n_group=65, stride=130), BAD), (dict(stride=63), BAD),
    (dict(logits=None), BAD), (dict(ids=None), BAD), (dict(w=None), BAD), (dict(logits=P + 2), BAD), (dict(bias=P + 1), BAD),
    (dict(ids=P + 2), BAD), (dict(M=1 << 30), UNSUPPORTED), (dict(M=0, logits=None), 0)])
def test_route_refuses(k, code):
    assert _route(**k) == code
    assert not code or capi.lib().exl3_last_error()


def _rows(f, x=P, dtype=1, stride=256, M=2, k=256, q=P, s=P):
    return getattr(capi.lib(), f)(x, dtype, stride, M, k, q, s, None)


@pytest.mark.parametrize("k,code", [
    (dict(k=0), BAD), (dict(M=-1), BAD), (dict(dtype=3), BAD), (dict(x=None), BAD), (dict(q=None), BAD), (dict(s=None), BAD),
    (dict(stride=100), BAD), (dict(x=P + 1), BAD), (dict(q=P + 8), BAD), (dict(s=P + 2), BAD),
    (dict(k=1 << 29, stride=1 << 30), UNSUPPORTED), (dict(M=1 << 30, k=1 << 10, stride=1 << 11), UNSUPPORTED),
    (dict(M=0, x=None), 0)])
def test_rows_refuse(k, code):
    assert _rows("exl3_fp8_quant", **k) == code
    assert _rows("exl3_fp8_silu_mul_quant", **{"stride": 512, **k}) == code
    assert _rows("exl3_fp8_silu_mul_quant", stride=511) == BAD       # gate|up rows are twice as long


def _matmul(q=P, s=P, M=4, k=256, n=256, w=P, sw=P, bias=None, out=P, dt=1, stride=256, ws=P, size=1 << 40):
    return capi.lib().exl3_fp8_matmul(q, s, M, k, n, w, sw, bias, out, dt, stride, ws, size, None)


def _linear(x=P, dtype=1, xs=256, M=4, k=256, n=256, w=P, sw=P, bias=None, out=P, dt=1, stride=256, ws=P, size=1 << 40):
    return capi.lib().exl3_fp8_linear(x, dtype, xs, M, k, n, w, sw, bias, out, dt, stride, ws, size, None)


@pytest.mark.parametrize("k,code", [
    (dict(k=0), BAD), (dict(n=0), BAD), (dict(M=-1), BAD), (dict(dt=3), BAD), (dict(w=None), BAD), (dict(sw=None), BAD),
    (dict(out=None), BAD), (dict(stride=255), BAD), (dict(w=P + 8), BAD), (dict(sw=P + 1), BAD), (dict(bias=P + 2), BAD),
    (dict(out=P + 1), BAD), (dict(n=1 << 29, stride=1 << 29), UNSUPPORTED),
    (dict(M=1 << 30, n=1 << 12, stride=1 << 12), UNSUPPORTED)])
def test_products_refuse(k, code):
    assert _matmul(**k) == code
    assert _linear(**k) == code


def _mlp(x=P, dt=1, xs=256, M=4, k=256, I=128, n=256, gu=P, gs=P, gb=None, dn=P, ds=P, db=None, out=P, stride=256, ws=P,  # noqa: E741
         size=1 << 40):
    return capi.lib().exl3_fp8_mlp(x, dt, xs, M, k, I, n, gu, gs, gb, dn, ds, db, out, stride, ws, size, None)


@pytest.mark.parametrize("k,code", [
    (dict(k=0), BAD), (dict(I=0), BAD), (dict(I=1 << 27), BAD), (dict(n=0), BAD), (dict(M=-1), BAD), (dict(dt=3), BAD),
    (dict(dt=-1), BAD), (dict(x=None), BAD), (dict(x=P + 1), BAD), (dict(xs=255), BAD), (dict(gu=None), BAD),
    (dict(gu=P + 8), BAD), (dict(gs=None), BAD), (dict(gb=P + 2), BAD), (dict(dn=None), BAD), (dict(dn=P + 4), BAD),
    (dict(ds=P + 1), BAD), (dict(db=P + 2), BAD), (dict(out=None), BAD), (dict(out=P + 1), BAD), (dict(stride=255), BAD),
    (dict(ws=None), BAD), (dict(ws=P + 2), WORKSPACE), (dict(size=100), WORKSPACE), (dict(k=1 << 23, xs=1 << 23), UNSUPPORTED),
    (dict(M=0, x=None, ws=None), 0)])
def test_mlp_refuses(k, code):
    assert _mlp(**k) == code


def test_products_refuse_their_own():
    assert [_matmul(q=None), _matmul(s=None), _matmul(q=P + 8), _matmul(s=P + 2)] == [BAD] * 4
    assert [_linear(x=None), _linear(dtype=3), _linear(xs=255), _linear(x=P + 1)] == [BAD] * 4
    assert [_linear(ws=None), _linear(size=16), _linear(ws=P + 4)] == [WORKSPACE] * 3
    assert _matmul(M=0, q=None, s=None, w=None, sw=None, out=None) == _linear(M=0, x=None, ws=None) == 0


@pytest.mark.parametrize("k,n", [(1, 1), (128, 128), (2048, 12288), (4096, 2048), (2000, 1000), (512, 2048), (130, 4096)])
def test_workspaces_never_fall_as_the_rows_grow(k, n):
    L = capi.lib()
    for f, least in ((L.exl3_fp8_matmul_workspace, lambda M: 0), (L.exl3_fp8_linear_workspace, lambda M: M * k)):
        b = [f(M, k, n) for M in [*range(1, 600), 1024, 4096, 8192, 60000]]
        assert all(x <= y for x, y in zip(b, b[1:])) and b[0] >= least(1) and b[-1] >= least(60000)
        assert [f(0, k, n), f(-5, k, n), f(4, 0, n), f(4, k, -1)] == [0] * 4


def test_mlp_workspace():
    f = capi.lib().exl3_fp8_mlp_workspace
    for dt in (0, 1, 2):
        b = [f(M, 2048, 512, 2048, dt) for M in [*range(1, 300), 1024, 60000]]
        assert all(x <= y for x, y in zip(b, b[1:])) and b[0] >= 1024 * (4 if dt == 2 else 2)
    assert [f(0, 8, 8, 8, 0), f(1, 0, 8, 8, 0), f(1, 8, -1, 8, 0), f(1, 8, 8, 0, 0), f(1, 8, 8, 8, 5), f(1, 8, 1 << 27, 8, 0)] == [0] * 6


def test_shapes_without_a_device():
    m = torch.device("meta")
    ids, w = ops().moe_route(torch.empty(3, 5, 64, device=m), None, 6, "softmax", 1, 1, True, 1.0)
    assert ids.shape == w.shape == (3, 5, 6) and (ids.dtype, w.dtype) == (torch.int32, torch.float32)
    for f, cols in ((C().fp8_quant, 300), (C().fp8_silu_mul_quant, 600)):
        q, s = f(torch.empty(2, 7, cols, device=m, dtype=torch.bfloat16))
        assert q.shape == (2, 7, 384) and s.shape == (2, 7, 3)
        assert (q.dtype, s.dtype) == (torch.float8_e4m3fn, torch.float32)
    w8, sw = torch.empty(130, 384, device=m, dtype=torch.float8_e4m3fn), torch.empty(2, 3, device=m)
    y = C().fp8_linear(torch.empty(2, 7, 300, device=m, dtype=torch.float16), w8, sw, None)
    assert y.shape == (2, 7, 130) and y.dtype == torch.float16
    m = C().fp8_mlp(torch.empty(2, 7, 300, device=m), w8, sw, None, torch.empty(90, 128, device=m, dtype=w8.dtype),
                    torch.empty(1, 1, device=m), None)
    assert m.shape == (2, 7, 90) and m.dtype == torch.float32
    y = C().fp8_matmul(q, s, w8, sw, None, torch.bfloat16)
    assert y.shape == (2, 7, 130) and y.dtype == torch.bfloat16


def test_scalars_have_no_rows():
    m = torch.device("meta")
    w8, sw, x = torch.empty(130, 384, device=m, dtype=torch.float8_e4m3fn), torch.empty(2, 3, device=m), torch.empty((), device=m)
    for f in (lambda: ops().moe_route(x, None, 1, "softmax", 1, 1, True, 1.0), lambda: C().fp8_linear(x, w8, sw, None),
              lambda: C().fp8_matmul(x, x, w8, sw, None, torch.bfloat16), lambda: C().fp8_mlp(x, w8, sw, None, w8, sw, None),
              lambda: C().fp8_quant(x), lambda: C().fp8_silu_mul_quant(x)):
        with pytest.raises((RuntimeError, IndexError)):
            f()


@pytest.mark.parametrize("M,k", [(1 << 28, 128), (1 << 27, 200), (1 << 24, 2048), (1 << 16, 1 << 21)])
def test_rows_of_one_launch(M, k):
    """16 lanes a block of 128, rounded up to whole workgroups: 2^32 threads and more are refused."""
    assert _rows("exl3_fp8_quant", M=M, k=k, stride=k) == UNSUPPORTED


def test_classes_refuse():
    w, s = torch.zeros(256, 300).to(torch.float8_e4m3fn), torch.ones(2, 3)
    lin = fp8.Fp8Linear(w, s)
    assert lin.weight.shape == (256, 384) and (lin.n, lin.k) == (256, 300)
    assert (lin.weight.view(torch.uint8)[:, 300:] == 0).all()
    for bad in (lambda: fp8.Fp8Linear(w.float(), s), lambda: fp8.Fp8Linear(w[0], s), lambda: fp8.Fp8Linear(w, s[:1]),
                lambda: fp8.Fp8Linear(w, s.t()), lambda: fp8.Fp8Linear(w, s, torch.zeros(255)),
                lambda: fp8.Fp8Linear(w[:0], s[:0]), lambda: fp8.Fp8Mlp(lin, lin), lambda: routing.Router(0),
                lambda: routing.Router(65), lambda: routing.Router(4, scoring="none"), lambda: routing.Router(4, n_group=0),
                lambda: routing.Router(4, n_group=4, topk_group=5), lambda: routing.Router(4, n_group=65),
                lambda: routing.Router(4, bias=torch.zeros(2, 4)), lambda: routing.Router(4, bias=torch.zeros(9), n_group=2)):
        with pytest.raises(ValueError):
            bad()
    assert routing.Router(2, bias=torch.zeros(8, dtype=torch.bfloat16)).bias.dtype == torch.float32


def test_weights_at_any_address():
    """Weights cut out of a larger buffer, as a checkpoint's file is one, are moved to an address that the kernels take."""
    store = torch.arange(128 * 256 + 16, dtype=torch.int64).remainder(126).to(torch.uint8)
    for at in range(16):
        w = store[at:at + 128 * 256].view(torch.float8_e4m3fn).view(128, 256)
        lin = fp8.Fp8Linear(w, torch.ones(1, 2))
        assert lin.weight.data_ptr() % 16 == 0 and torch.equal(lin.weight.view(torch.uint8), w.view(torch.uint8))
