"""Refusals of the layer-norm, dropout and MXFP4 entry points, on the host: the C ABI returns a negative status
before any HIP call, the Python layer raises ValueError."""

import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def L(pkg):
    return pkg._lib


P, Q, R_, S, T_ = (ctypes.c_void_p(0x10000 * i) for i in range(1, 6))


def _drop(L, **kw):
    d = dict(keep=32768, seed=1, offset=0, state=None)
    d.update(kw)
    return ctypes.byref(L.LrqDropout(d["keep"], d["seed"], d["offset"], d["state"]))


@pytest.mark.parametrize("change,code", [
    (dict(d=None), "NULL"), (dict(x=None), "NULL"), (dict(out=None), "NULL"), (dict(dt=3), "UNSUPPORTED"),
    (dict(dt=-1), "UNSUPPORTED"), (dict(rows=-1), "SHAPE"), (dict(n=-1), "SHAPE"), (dict(ldx=7), "SHAPE"),
    (dict(ldo=7), "SHAPE"), (dict(ldr=7), "SHAPE"), (dict(x=ctypes.c_void_p(0x10001)), "ALIGN"),
    (dict(dt=2, x=ctypes.c_void_p(0x10002)), "ALIGN"), (dict(keep=65537), "SHAPE"), (dict(state=0x10004), "ALIGN"),
    (dict(rows=1 << 31), "SHAPE"),
])
def test_dropout_arguments(L, change, code):
    a = dict(x=P, ldx=8, res=Q, ldr=8, dt=0, rows=4, n=8, out=R_, ldo=8)
    d = change.get("d", _drop(L, **{k: v for k, v in change.items() if k in ("keep", "state")}))
    a.update({k: v for k, v in change.items() if k in a})
    st = L.call_raw("lrq_dropout_add", d, a["x"], a["ldx"], a["res"], a["ldr"], a["dt"], a["rows"], a["n"], a["out"],
                    a["ldo"], None)
    assert st == getattr(L, "LRQ_ERR_" + code)


def _fwd(L, **kw):
    a = dict(drop=None, x=P, ldx=8, res=None, ldr=0, dt=0, w=Q, b=Q, wdt=0, rows=4, n=8, eps=1e-5, h=None, ldh=0, y=R_,
             ldy=8, mean=S, rstd=T_)
    a.update(kw)
    return L.call_raw("lrq_layer_norm_fwd", *a.values(), None)


@pytest.mark.parametrize("change,code", [
    (dict(x=None), "NULL"), (dict(y=None), "NULL"), (dict(mean=None), "NULL"), (dict(rstd=None), "NULL"),
    (dict(dt=3), "UNSUPPORTED"), (dict(wdt=7), "UNSUPPORTED"), (dict(rows=-1), "SHAPE"), (dict(n=0), "SHAPE"),
    (dict(ldx=7), "SHAPE"), (dict(ldy=7), "SHAPE"), (dict(res=Q, ldr=8), "NULL"),  # a residual needs h
    (dict(h=Q, ldh=7), "SHAPE"), (dict(h=Q, ldh=8, res=Q, ldr=7), "SHAPE"), (dict(w=ctypes.c_void_p(0x10001)), "ALIGN"),
    (dict(dt=2, y=ctypes.c_void_p(0x10002)), "ALIGN"), (dict(mean=ctypes.c_void_p(0x10002)), "ALIGN"),
])
def test_layer_norm_forward_arguments(L, change, code):
    assert _fwd(L, **change) == getattr(L, "LRQ_ERR_" + code)


def test_layer_norm_forward_dropout_needs_h(L):
    assert _fwd(L, drop=_drop(L)) == L.LRQ_ERR_NULL
    assert _fwd(L, drop=_drop(L, keep=70000), h=Q, ldh=8) == L.LRQ_ERR_SHAPE


def _bwd(L, **kw):
    a = dict(drop=None, dy=P, lddy=8, dh=None, lddh=0, h=Q, ldh=8, dt=0, w=Q, wdt=0, mean=S, rstd=T_, rows=4, n=8, dx=R_,
             lddx=8, dres=None, lddr=0, dw=P, db=P, ws=S, wsb=1 << 20)
    a.update(kw)
    return L.call_raw("lrq_layer_norm_bwd", *a.values(), None)


@pytest.mark.parametrize("change,code", [
    (dict(dy=None), "NULL"), (dict(h=None), "NULL"), (dict(mean=None), "NULL"), (dict(dx=None), "NULL"),
    (dict(dw=None), "NULL"), (dict(db=None), "NULL"), (dict(ws=None), "NULL"), (dict(wsb=8), "WORKSPACE"),
    (dict(dt=9), "UNSUPPORTED"), (dict(n=0), "SHAPE"), (dict(lddy=7), "SHAPE"), (dict(ldh=7), "SHAPE"),
    (dict(lddx=7), "SHAPE"), (dict(dh=P, lddh=7), "SHAPE"), (dict(dres=P, lddr=7), "SHAPE"),
    (dict(dy=ctypes.c_void_p(0x10001)), "ALIGN"), (dict(ws=ctypes.c_void_p(0x10002)), "ALIGN"),
    (dict(dw=ctypes.c_void_p(0x10001)), "ALIGN"),
])
def test_layer_norm_backward_arguments(L, change, code):
    assert _bwd(L, **change) == getattr(L, "LRQ_ERR_" + code)


def test_layer_norm_workspace(L):
    for rows, n in ((1, 1), (16384, 4096), (100, 20000), (1 << 20, 64)):
        b = L.call_raw("lrq_layer_norm_bwd_workspace", rows, n)
        assert 8 * n <= b <= 1024 * 8 * n
    assert L.call_raw("lrq_layer_norm_bwd_workspace", 0, 8) == 0
    assert L.call_raw("lrq_layer_norm_bwd_workspace", 4, 0) == L.LRQ_ERR_SHAPE
    assert L.call_raw("lrq_layer_norm_bwd_workspace", -1, 8) == L.LRQ_ERR_SHAPE


def _mx(L, **kw):
    a = dict(codes=0x10000, ld_codes=128, scales=0x20000, ld_scales=8, rows=16, cols=256)
    a.update(kw)
    return L.LrqMxfp4(*a.values())


BAD_MX = [(dict(codes=None), "NULL"), (dict(scales=None), "NULL"), (dict(rows=-1), "SHAPE"), (dict(cols=0), "SHAPE"),
          (dict(ld_codes=112), "SHAPE"), (dict(ld_scales=4), "SHAPE"), (dict(ld_codes=136), "ALIGN"),
          (dict(ld_scales=10), "ALIGN"), (dict(codes=0x10008), "ALIGN"), (dict(scales=0x20002), "ALIGN")]


@pytest.mark.parametrize("change,code", BAD_MX)
def test_mxfp4_descriptors(L, change, code):
    bad, good = _mx(L, **change), _mx(L)
    want = getattr(L, "LRQ_ERR_" + code)
    b, g = ctypes.byref(bad), ctypes.byref(good)
    assert L.call_raw("lrq_mxfp4_quantize", P, 256, 0, b, None) == want
    assert L.call_raw("lrq_mxfp4_dequantize", b, P, 256, 0, None) == want
    assert L.call_raw("lrq_mxfp4_gemm", b, g, P, 16, 0, None, 0, None) == want
    assert L.call_raw("lrq_mxfp4_gemm", g, b, P, 16, 0, None, 0, None) == want
    assert L.call_raw("lrq_mxfp4_linear", P, 256, 4, b, Q, 16, 0, None, 0, None) == want
    assert L.call_raw("lrq_mxfp4_linear_t", P, 16, 4, b, Q, 256, 0, None, 0, None) == want
    assert L.call_raw("lrq_mxfp4_linear_workspace", 4, b, 0) == want


def test_mxfp4_arguments(L):
    g = ctypes.byref(_mx(L))
    other = ctypes.byref(_mx(L, cols=255))
    assert L.call_raw("lrq_mxfp4_gemm", g, other, P, 16, 0, None, 0, None) == L.LRQ_ERR_SHAPE
    assert L.call_raw("lrq_mxfp4_gemm", g, g, None, 16, 0, None, 0, None) == L.LRQ_ERR_NULL
    assert L.call_raw("lrq_mxfp4_gemm", g, g, P, 15, 0, None, 0, None) == L.LRQ_ERR_SHAPE
    assert L.call_raw("lrq_mxfp4_gemm", g, g, ctypes.c_void_p(0x10002), 16, 1, None, 0, None) == L.LRQ_ERR_ALIGN
    assert L.call_raw("lrq_mxfp4_linear", None, 256, 4, g, Q, 16, 0, None, 0, None) == L.LRQ_ERR_NULL
    assert L.call_raw("lrq_mxfp4_linear", P, 255, 4, g, Q, 16, 0, None, 0, None) == L.LRQ_ERR_SHAPE
    assert L.call_raw("lrq_mxfp4_linear", P, 256, -4, g, Q, 16, 0, None, 0, None) == L.LRQ_ERR_SHAPE
    assert L.call_raw("lrq_mxfp4_linear", ctypes.c_void_p(0x10001), 256, 4, g, Q, 16, 0, None, 0, None) == L.LRQ_ERR_ALIGN
    assert L.call_raw("lrq_mxfp4_linear", P, 256, 4, g, Q, 15, 0, None, 0, None) == L.LRQ_ERR_SHAPE
    assert L.call_raw("lrq_mxfp4_linear_t", P, 8, 4, g, Q, 256, 0, None, 0, None) == L.LRQ_ERR_SHAPE
    assert L.call_raw("lrq_mxfp4_linear_t", P, 16, 4, g, Q, 255, 0, None, 0, None) == L.LRQ_ERR_SHAPE
    assert L.call_raw("lrq_mxfp4_linear", ctypes.c_void_p(0x10008), 256, 4, g, Q, 16, 0, None, 0, None) == L.LRQ_ERR_ALIGN
    assert L.call_raw("lrq_mxfp4_linear", P, 260, 4, g, Q, 16, 0, None, 0, None) == L.LRQ_ERR_ALIGN
    # a product split over workgroups needs its workspace
    big = ctypes.byref(_mx(L, rows=1024, cols=8192, ld_codes=4096, ld_scales=256))
    need = L.call_raw("lrq_mxfp4_linear_workspace", 256, big, 0)
    assert need > 0 and need % (256 * 1024 * 4) == 0
    args = (P, 8192, 256, big, Q, 1024, 0)
    assert L.call_raw("lrq_mxfp4_linear", *args, None, need, None) == L.LRQ_ERR_NULL
    assert L.call_raw("lrq_mxfp4_linear", *args, R_, need - 1, None) == L.LRQ_ERR_WORKSPACE
    assert L.call_raw("lrq_mxfp4_linear", *args, ctypes.c_void_p(0x30004), need, None) == L.LRQ_ERR_ALIGN
    assert L.call_raw("lrq_mxfp4_linear_workspace", 1, big, 0) == 0
    need = L.call_raw("lrq_mxfp4_gemm_workspace", big, big)
    assert need > 0 and need % (1024 * 1024 * 4) == 0
    assert L.call_raw("lrq_mxfp4_gemm", big, big, P, 1024, 0, None, need, None) == L.LRQ_ERR_NULL
    assert L.call_raw("lrq_mxfp4_gemm", big, big, P, 1024, 0, Q, need - 4, None) == L.LRQ_ERR_WORKSPACE
    assert L.call_raw("lrq_mxfp4_gemm_workspace", big, g) == L.LRQ_ERR_SHAPE
    assert L.call_raw("lrq_mxfp4_linear_workspace", -1, big, 0) == L.LRQ_ERR_SHAPE
    empty = ctypes.byref(_mx(L, rows=0))
    assert L.call_raw("lrq_mxfp4_linear_t", P, 8, 4, empty, Q, 256, 0, None, 0, None) == L.LRQ_ERR_SHAPE
    assert L.call_raw("lrq_mxfp4_quantize", P, 255, 0, g, None) == L.LRQ_ERR_SHAPE
    assert L.call_raw("lrq_mxfp4_quantize", P, 256, 5, g, None) == L.LRQ_ERR_UNSUPPORTED
    assert L.call_raw("lrq_mxfp4_dequantize", g, P, 256, 5, None) == L.LRQ_ERR_UNSUPPORTED


def test_structures_match_the_header(L):
    assert ctypes.sizeof(L.LrqDropout) == 32 and ctypes.sizeof(L.LrqMxfp4) == 48
    assert L.LrqDropout.seed.offset == 8 and L.LrqDropout.state.offset == 24


def test_host_tensors_are_refused(pkg):
    x = torch.zeros(4, 8, dtype=torch.bfloat16)
    q = pkg.MXFP4Tensor(torch.zeros(4, 64, dtype=torch.uint8), torch.zeros(4, 4, dtype=torch.uint8), (4, 8))
    m = torch.zeros(4)
    for f in (lambda: pkg.layer_norm_forward(x), lambda: pkg.layer_norm_backward(x, x, None, m, m),
              lambda: pkg.dropout(x, 0.1, 1), lambda: pkg.dropout_add_layer_norm_forward(x, x, None, None, 0.1, 1),
              lambda: pkg.mxfp4_quantize(x), lambda: pkg.mxfp4_dequantize(q), lambda: pkg.mxfp4_gemm(q, q),
              lambda: pkg.mxfp4_linear(x, q), lambda: pkg.mxfp4_linear_backward(x, q)):
        with pytest.raises(ValueError, match="device tensors only"):
            f()


def test_dropout_probability_and_seed(pkg):
    N = pkg.norm
    assert N._keep(0.0) == 65536 and N._keep(1.0) == 0 and N._keep(0.5) == 32768
    assert N._keep(1e-9) == 65535 and N._keep(1 - 1e-9) == 1
    for p in (-0.1, 1.1, float("nan")):
        with pytest.raises(ValueError):
            N._keep(p)
    dev = torch.device("cpu")
    d, s = N._drop(0.25, (-1, 1 << 40), dev)
    assert d.seed == 2 ** 64 - 1 and d.offset == 1 << 40 and s is None
    for bad in (None, 1.5, "1", (1,), (1, 2, 3), (1, 2.0), True, torch.zeros(3, dtype=torch.int64),
                torch.zeros(2, dtype=torch.int32), torch.zeros(4, dtype=torch.int64)[::2]):
        with pytest.raises(ValueError):
            N._drop(0.25, bad, dev)


def test_no_dropout_needs_no_seed(pkg):
    N, dev = pkg.norm, torch.device("cpu")
    d, s = N._drop(0.0, None, dev)
    assert d.keep == 65536 and d.state is None and s is None
    for p in (1e-9, 0.5, 1.0):
        with pytest.raises(ValueError):
            N._drop(p, None, dev)


@pytest.mark.gpu
def test_no_dropout_needs_no_seed_on_the_device(pkg, dev):
    """p = 0 without a seed: dropout is the identity (plus the residual), its gradient too, in every form."""
    AG = pkg.autograd
    x, r = (torch.randn(5, 40, device=dev).requires_grad_() for _ in range(2))
    assert torch.equal(pkg.dropout(x.detach(), 0.0, None), x)
    dy = torch.randn(5, 40, device=dev)
    y = AG.dropout(x, 0.0, None, residual=r)
    y.backward(dy)
    assert torch.equal(y, r + x) and torch.equal(x.grad, dy) and torch.equal(r.grad, dy)
    want = AG.dropout_add_layer_norm(x, r, None, None, 0.0, 7)
    for got, e in zip(AG.dropout_add_layer_norm(x, r, None, None, 0.0, None), want):
        assert torch.equal(got, e)
    y, h, mean, rstd = pkg.dropout_add_layer_norm_forward(x.detach(), r.detach(), None, None, 0.0, None)
    assert torch.equal(y, want[0]) and torch.equal(h, want[1])
    got = pkg.dropout_add_layer_norm_backward(dy, None, h, None, mean, rstd, 0.0, None)
    assert torch.equal(got[0], pkg.dropout_add_layer_norm_backward(dy, None, h, None, mean, rstd, 0.0, 7)[0])


@pytest.mark.gpu
def test_python_refusals(pkg, dev):
    x = torch.zeros(4, 8, dtype=torch.bfloat16, device=dev)
    w = torch.ones(8, device=dev)
    y, mean, rstd = pkg.layer_norm_forward(x, w, w)
    q = pkg.mxfp4_quantize(x)
    bad = [
        lambda: pkg.layer_norm_forward(x.double()), lambda: pkg.layer_norm_forward(x, w[:7]),
        lambda: pkg.layer_norm_forward(x, w, w.half()), lambda: pkg.layer_norm_forward(x, w.double()),
        lambda: pkg.layer_norm_forward(x[:, :0]), lambda: pkg.layer_norm_forward(x[0, 0]),
        lambda: pkg.layer_norm_backward(x.float(), x, w, mean, rstd),
        lambda: pkg.layer_norm_backward(x[:3], x, w, mean, rstd),
        lambda: pkg.layer_norm_backward(x, x, w, mean[:3], rstd),
        lambda: pkg.layer_norm_backward(x, x, w, mean, rstd.double()),
        lambda: pkg.layer_norm_backward(x, x, w.cpu(), mean, rstd),
        lambda: pkg.dropout(x, 1.5, 1), lambda: pkg.dropout(x, 0.5, None), lambda: pkg.dropout(x.int(), 0.5, 1),
        lambda: pkg.dropout(x, 0.5, 1, residual=x[:1]), lambda: pkg.dropout(x, 0.5, 1, residual=x.float()),
        lambda: pkg.dropout(x, 0.5, torch.zeros(2, dtype=torch.int64)),
        lambda: pkg.dropout_add_layer_norm_forward(x, x[:2], w, w, 0.1, 1),
        lambda: pkg.dropout_add_layer_norm_backward(x, x.float(), x, w, mean, rstd, 0.1, 1),
        lambda: pkg.mxfp4_quantize(x.int()), lambda: pkg.mxfp4_quantize(x[:, :0]),
        lambda: pkg.mxfp4_dequantize(q, torch.float64), lambda: pkg.mxfp4_gemm(q, q, torch.float16),
        lambda: pkg.mxfp4_gemm(q, pkg.mxfp4_quantize(x.reshape(2, 2, 8))),
        lambda: pkg.mxfp4_gemm(q, pkg.mxfp4_quantize(x[:, :7])),
        lambda: pkg.mxfp4_linear(x.float(), q), lambda: pkg.mxfp4_linear(x[:, :7], q),
        lambda: pkg.mxfp4_linear_backward(x, q), lambda: pkg.mxfp4_linear(x, pkg.mxfp4_quantize(x.reshape(1, 4, 8))),
        lambda: pkg.mxfp4_linear(x, pkg.MXFP4Tensor(q.codes, q.scales, (4, 200))),
        lambda: pkg.mxfp4_linear(x, pkg.MXFP4Tensor(q.codes[:3], q.scales, (4, 8))),
        lambda: pkg.mxfp4_linear(x, pkg.MXFP4Tensor(q.codes, q.scales.int(), (4, 8))),
        lambda: pkg.mxfp4_linear(x, pkg.MXFP4Tensor(q.codes, q.scales.cpu(), (4, 8))),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"call {i} was accepted")
    AG = pkg.autograd
    with pytest.raises(ValueError):
        AG.lora_linear_compressed(x, torch.zeros(8, 8, dtype=torch.bfloat16, device=dev), x[:, :2], x[:2], dropout_p=0.1)
