"""Refusals of the 8-bit and root-mean-square norm entry points, on the host: the C ABI returns a negative status before
any HIP call, the Python layer raises ValueError."""

import ctypes
import importlib

import pytest
import torch


@pytest.fixture(scope="module")
def L(pkg):
    return pkg._lib


P, Q, R_, S, T_ = (ctypes.c_void_p(0x10000 * i) for i in range(1, 6))


def _t(L, **kw):
    a = dict(codes=0x10000, ld_codes=256, scales=0x20000, ld_scales=4, rows=16, cols=256, block=1)
    a.update(kw)
    return L.LrqFp8(*a.values())


BAD = [(dict(codes=None), "NULL"), (dict(scales=None), "NULL"), (dict(rows=-1), "SHAPE"), (dict(rows=1 << 31), "SHAPE"),
       (dict(cols=0), "SHAPE"), (dict(cols=257), "SHAPE"), (dict(ld_codes=240), "SHAPE"), (dict(ld_scales=0), "SHAPE"),
       (dict(ld_codes=264), "ALIGN"), (dict(ld_scales=6), "ALIGN"), (dict(codes=0x10008), "ALIGN"),
       (dict(scales=0x20002), "ALIGN"), (dict(block=64), "UNSUPPORTED"), (dict(block=0), "UNSUPPORTED")]


@pytest.mark.parametrize("change,code", BAD)
def test_descriptors(L, change, code):
    b, g = ctypes.byref(_t(L, **change)), ctypes.byref(_t(L, block=128))
    want = getattr(L, "LRQ_ERR_" + code)
    assert L.call_raw("lrq_fp8_quantize", P, 512, 0, b, 0, None) == want
    assert L.call_raw("lrq_fp8_dequantize", b, P, 512, 0, None) == want
    assert L.call_raw("lrq_fp8_linear", P, 512, 0, 4, b, P, 16, 0, None) == want
    for name in ("lrq_fp8_gemm", "lrq_fp8_gemm_nn"):
        assert L.call_raw(name, b, g, P, 512, 0, None, 0, None) == want
        assert L.call_raw(name, g, b, P, 512, 0, None, 0, None) == want
    for nn in (0, 1):
        assert L.call_raw("lrq_fp8_gemm_workspace", b, g, nn) == want
        assert L.call_raw("lrq_fp8_gemm_workspace", g, b, nn) == want
    assert L.call_raw("lrq_rms_norm_fwd", P, 256, None, 0, 0, Q, 0, 16, 256, 1e-6, None, 0, None, 0, b, R_, None) == want


def test_no_descriptor(L):
    g = ctypes.byref(_t(L, block=128))
    assert L.call_raw("lrq_fp8_quantize", P, 512, 0, None, 0, None) == L.LRQ_ERR_NULL
    assert L.call_raw("lrq_fp8_gemm", None, g, P, 512, 0, None, 0, None) == L.LRQ_ERR_NULL
    assert L.call_raw("lrq_fp8_gemm", g, None, P, 512, 0, None, 0, None) == L.LRQ_ERR_NULL


@pytest.mark.parametrize("change,code", [
    (dict(x=None), "NULL"), (dict(dt=3), "UNSUPPORTED"), (dict(dt=-1), "UNSUPPORTED"), (dict(ldx=255), "SHAPE"),
    (dict(x=ctypes.c_void_p(0x10001)), "ALIGN"), (dict(dt=2, x=ctypes.c_void_p(0x10002)), "ALIGN"),
    (dict(tr=1, block=128), "UNSUPPORTED"), (dict(tr=1, ldx=15), "SHAPE"),
])
def test_quantize_arguments(L, change, code):
    a = dict(x=P, ldx=256, dt=0, tr=0, block=1)
    a.update(change)
    t = _t(L, block=a["block"])
    assert L.call_raw("lrq_fp8_quantize", a["x"], a["ldx"], a["dt"], ctypes.byref(t), a["tr"], None) == getattr(L, "LRQ_ERR_" + code)


@pytest.mark.parametrize("change,code", [
    (dict(out=None), "NULL"), (dict(ldo=15), "SHAPE"), (dict(dt=3), "UNSUPPORTED"), (dict(dt=-1), "UNSUPPORTED"),
    (dict(out=ctypes.c_void_p(0x10001)), "ALIGN"), (dict(dt=2, out=ctypes.c_void_p(0x10002)), "ALIGN"),
])
def test_product_outputs(L, change, code):
    a = dict(out=P, ldo=256, dt=0)
    a.update(change)
    want = getattr(L, "LRQ_ERR_" + code)
    x, w = _t(L), _t(L, block=128, rows=256)
    ldo = 255 if "ldo" in change else 256
    assert L.call_raw("lrq_fp8_gemm", ctypes.byref(x), ctypes.byref(w), a["out"], ldo, a["dt"], None, 0, None) == want
    assert L.call_raw("lrq_fp8_gemm_nn", ctypes.byref(x), ctypes.byref(w), a["out"], ldo, a["dt"], None, 0, None) == want
    assert L.call_raw("lrq_fp8_linear", Q, 256, 0, 4, ctypes.byref(w), a["out"], ldo, a["dt"], None) == want


def test_products_that_do_not_fit(L):
    x, w = _t(L), _t(L, block=128)
    b = ctypes.byref
    assert L.call_raw("lrq_fp8_gemm", b(x), b(_t(L, cols=250)), P, 512, 0, None, 0, None) == L.LRQ_ERR_SHAPE
    assert L.call_raw("lrq_fp8_gemm_nn", b(x), b(w), P, 512, 0, None, 0, None) == L.LRQ_ERR_SHAPE  # 256 columns, 16 rows
    assert L.call_raw("lrq_fp8_gemm_nn", b(x), b(_t(L, rows=256)), P, 512, 0, None, 0, None) == L.LRQ_ERR_UNSUPPORTED  # block 1
    wide = _t(L, ld_codes=1 << 24)
    assert L.call_raw("lrq_fp8_gemm", b(wide), b(w), P, 512, 0, None, 0, None) == L.LRQ_ERR_SHAPE
    far = _t(L, rows=1 << 20, ld_scales=1 << 16)
    assert L.call_raw("lrq_fp8_gemm", b(far), b(w), P, 512, 0, None, 0, None) == L.LRQ_ERR_SHAPE
    for name, args in (("rows", (P, 256, 0, 5)), ("rows", (P, 256, 0, -1)), ("ldx", (P, 255, 0, 4))):
        assert L.call_raw("lrq_fp8_linear", *args, b(w), P, 512, 0, None) == L.LRQ_ERR_SHAPE, name
    assert L.call_raw("lrq_fp8_linear", P, 256, 2, 4, b(w), P, 512, 0, None) == L.LRQ_ERR_UNSUPPORTED
    assert L.call_raw("lrq_fp8_linear", None, 256, 0, 4, b(w), P, 512, 0, None) == L.LRQ_ERR_NULL
    assert L.call_raw("lrq_fp8_linear", ctypes.c_void_p(0x10001), 256, 0, 4, b(w), P, 512, 0, None) == L.LRQ_ERR_ALIGN
    odd = _t(L, cols=252, block=128)
    assert L.call_raw("lrq_fp8_linear", P, 256, 0, 4, b(odd), P, 512, 0, None) == L.LRQ_ERR_SHAPE


def test_workspace(L):
    """Split products ask for their parts, and refuse less; few rows and whole grids ask for none."""
    b = ctypes.byref
    a, w = _t(L, rows=100, cols=16384, ld_codes=16384, ld_scales=128), _t(L, rows=64, cols=16384, ld_codes=16384, ld_scales=128)
    n = L.call_raw("lrq_fp8_gemm_workspace", b(a), b(w), 0)
    assert n > 0 and n % (100 * 64 * 4) == 0
    assert L.call_raw("lrq_fp8_gemm", b(a), b(w), P, 64, 0, None, n, None) == L.LRQ_ERR_NULL
    assert L.call_raw("lrq_fp8_gemm", b(a), b(w), P, 64, 0, Q, n - 1, None) == L.LRQ_ERR_WORKSPACE
    assert L.call_raw("lrq_fp8_gemm", b(a), b(w), P, 64, 0, ctypes.c_void_p(0x20008), n, None) == L.LRQ_ERR_ALIGN
    few = _t(L, rows=16, cols=16384, ld_codes=16384, ld_scales=128)
    assert L.call_raw("lrq_fp8_gemm_workspace", b(few), b(w), 0) == 0
    big = _t(L, rows=4096, cols=4096, ld_codes=4096, ld_scales=32)
    assert L.call_raw("lrq_fp8_gemm_workspace", b(big), b(big), 0) == 0


@pytest.mark.parametrize("change,code", [
    (dict(x=None), "NULL"), (dict(dt=3), "UNSUPPORTED"), (dict(ldx=255), "SHAPE"), (dict(x=ctypes.c_void_p(0x10001)), "ALIGN"),
    (dict(t=dict(block=128)), "UNSUPPORTED"), (dict(tt=dict(block=128)), "UNSUPPORTED"), (dict(t=dict(rows=17)), "SHAPE"),
    (dict(tt=dict(rows=255)), "SHAPE"), (dict(t=dict(codes=None)), "NULL"), (dict(tt=dict(scales=None)), "NULL"),
    (dict(tt=dict(ld_codes=120)), "SHAPE"), (dict(t=dict(rows=0), tt=dict(cols=0)), "SHAPE"),
])
def test_quantize_both(L, change, code):
    a = dict(x=P, ldx=256, dt=0, t={}, tt={})
    a.update(change)
    t, tt = _t(L, **a["t"]), _t(L, **{**dict(rows=256, cols=16), **a["tt"]})
    got = L.call_raw("lrq_fp8_quantize_both", a["x"], a["ldx"], a["dt"], ctypes.byref(t), ctypes.byref(tt), None)
    assert got == getattr(L, "LRQ_ERR_" + code)


@pytest.mark.parametrize("nn", [0, 1])
def test_quantize_gemm(L, nn):
    b = ctypes.byref
    w = _t(L, rows=384, block=128)
    depth, cols = (384, 256) if nn else (256, 384)
    n = L.call_raw("lrq_fp8_quantize_gemm_workspace", 20, b(w), nn)
    assert n >= 20 * (depth + 4)

    def go(**kw):
        a = dict(x=P, ldx=depth, dt=0, rows=20, w=b(w), nn=nn, out=Q, ldo=cols, odt=0, ws=R_, n=n)
        a.update(kw)
        return L.call_raw("lrq_fp8_quantize_gemm", *a.values(), None)
    for kw, code in ((dict(x=None), "NULL"), (dict(out=None), "NULL"), (dict(ws=None), "NULL"), (dict(w=None), "NULL"),
                     (dict(ldx=depth - 1), "SHAPE"), (dict(ldo=cols - 1), "SHAPE"), (dict(rows=-1), "SHAPE"),
                     (dict(rows=1 << 31), "SHAPE"), (dict(dt=3), "UNSUPPORTED"), (dict(odt=3), "UNSUPPORTED"),
                     (dict(x=ctypes.c_void_p(0x10001)), "ALIGN"), (dict(ws=ctypes.c_void_p(0x20008)), "ALIGN"),
                     (dict(n=n - 1), "WORKSPACE"), (dict(w=b(_t(L, rows=384, block=128, ld_codes=1 << 24))), "SHAPE")):
        assert go(**kw) == getattr(L, "LRQ_ERR_" + code), kw
    assert go(rows=0, ws=None) == 0
    assert L.call_raw("lrq_fp8_quantize_gemm_workspace", 0, b(w), nn) == 0
    rows = b(_t(L, rows=384))
    assert L.call_raw("lrq_fp8_quantize_gemm_workspace", 4, rows, 1) == L.LRQ_ERR_UNSUPPORTED
    none = b(_t(L, rows=0, block=128))
    assert L.call_raw("lrq_fp8_quantize_gemm_workspace", 4, none, 1) == L.LRQ_ERR_SHAPE
    assert L.call_raw("lrq_fp8_quantize_gemm_workspace", 4, none, 0) == 4 * (256 + 4)
    deep = _t(L, rows=64, cols=16384, ld_codes=16384, ld_scales=128, block=128)
    parts = L.call_raw("lrq_fp8_gemm_workspace", b(_t(L, rows=100, cols=16384, ld_codes=16384, ld_scales=128)), b(deep), 0)
    assert L.call_raw("lrq_fp8_quantize_gemm_workspace", 100, b(deep), 0) == parts + 100 * (16384 + 128) > 100 * (16384 + 128)


def _fwd(L, **kw):
    a = dict(x=P, ldx=8, res=None, ldr=0, dt=0, w=Q, wdt=0, rows=4, n=8, eps=1e-6, h=None, ldh=0, y=R_, ldy=8, q=None, rstd=T_)
    a.update(kw)
    return L.call_raw("lrq_rms_norm_fwd", *a.values(), None)


@pytest.mark.parametrize("change,code", [
    (dict(x=None), "NULL"), (dict(y=None), "NULL"), (dict(rstd=None), "NULL"), (dict(dt=3), "UNSUPPORTED"),
    (dict(wdt=7), "UNSUPPORTED"), (dict(rows=-1), "SHAPE"), (dict(n=0), "SHAPE"), (dict(ldx=7), "SHAPE"),
    (dict(ldy=7), "SHAPE"), (dict(res=Q, ldr=8), "NULL"),  # a residual needs h
    (dict(h=Q, ldh=7), "SHAPE"), (dict(h=Q, ldh=8, res=Q, ldr=7), "SHAPE"), (dict(w=ctypes.c_void_p(0x10001)), "ALIGN"),
    (dict(dt=2, y=ctypes.c_void_p(0x10002)), "ALIGN"), (dict(rstd=ctypes.c_void_p(0x10002)), "ALIGN"),
])
def test_rms_forward_arguments(L, change, code):
    assert _fwd(L, **change) == getattr(L, "LRQ_ERR_" + code)


def test_rms_forward_outputs(L):
    q = _t(L, rows=4, cols=8)
    assert _fwd(L, q=ctypes.byref(q)) == L.LRQ_ERR_UNSUPPORTED  # y or q
    assert _fwd(L, y=None, q=ctypes.byref(_t(L, rows=4, cols=8, block=128))) == L.LRQ_ERR_UNSUPPORTED
    assert _fwd(L, y=None, q=ctypes.byref(_t(L, rows=5, cols=8))) == L.LRQ_ERR_SHAPE
    assert _fwd(L, y=None, q=ctypes.byref(_t(L, rows=4, cols=9))) == L.LRQ_ERR_SHAPE


def _bwd(L, **kw):
    a = dict(dy=P, lddy=8, dh=None, lddh=0, h=Q, ldh=8, dt=0, w=Q, wdt=0, rstd=T_, rows=4, n=8, dx=R_, lddx=8, dw=P, ws=S,
             wsb=1 << 20)
    a.update(kw)
    return L.call_raw("lrq_rms_norm_bwd", *a.values(), None)


@pytest.mark.parametrize("change,code", [
    (dict(dy=None), "NULL"), (dict(h=None), "NULL"), (dict(rstd=None), "NULL"), (dict(dx=None), "NULL"),
    (dict(ws=None), "NULL"), (dict(wsb=8), "WORKSPACE"), (dict(dt=9), "UNSUPPORTED"), (dict(n=0), "SHAPE"),
    (dict(rows=1 << 31), "SHAPE"), (dict(lddy=7), "SHAPE"), (dict(ldh=7), "SHAPE"), (dict(lddx=7), "SHAPE"),
    (dict(dh=P, lddh=7), "SHAPE"), (dict(dy=ctypes.c_void_p(0x10001)), "ALIGN"), (dict(ws=ctypes.c_void_p(0x10002)), "ALIGN"),
    (dict(dw=ctypes.c_void_p(0x10001)), "ALIGN"),
])
def test_rms_backward_arguments(L, change, code):
    assert _bwd(L, **change) == getattr(L, "LRQ_ERR_" + code)


def test_rms_workspace(L):
    for rows, n in ((1, 1), (16384, 4096), (100, 20000), (1 << 20, 64)):
        b = L.call_raw("lrq_rms_norm_bwd_workspace", rows, n)
        assert 4 * n <= b <= 1024 * 4 * n
    assert L.call_raw("lrq_rms_norm_bwd_workspace", 0, 8) == 0
    assert L.call_raw("lrq_rms_norm_bwd_workspace", 4, 0) == L.LRQ_ERR_SHAPE
    assert L.call_raw("lrq_rms_norm_bwd_workspace", -1, 8) == L.LRQ_ERR_SHAPE


def test_python_refusals(pkg):
    x = torch.zeros(4, 256, dtype=torch.bfloat16)
    q = pkg.FP8Tensor(torch.zeros(256, 256, dtype=torch.uint8), torch.zeros(2, 4, dtype=torch.uint8), (256, 256), 128)
    for f in (lambda: pkg.fp8_quantize(x), lambda: pkg.fp8_quantize_both(x), lambda: pkg.fp8_dequantize(q), lambda: pkg.fp8_linear(x, q),
              lambda: pkg.fp8_linear_backward(x, q), lambda: pkg.fp8_weight_gradient(x, x), lambda: pkg.fp8_gemm(q, q),
              lambda: pkg.rms_norm_forward(x), lambda: pkg.add_rms_norm_forward(x, x),
              lambda: pkg.rms_norm_backward(x, x, None, torch.zeros(4)),
              lambda: pkg.fp8_from_parts(q.codes, q.scales[:, :2], 128)):
        with pytest.raises(ValueError, match="device tensors only"):
            f()
    with pytest.raises(ValueError, match="needs a residual"):
        pkg.add_rms_norm_forward(x, None)
    with pytest.raises(ValueError, match="FP8Tensor"):
        pkg.fp8_linear(x, x)
    with pytest.raises(ValueError, match="1 or 128 rows"):
        pkg.FP8Tensor(q.codes, q.scales, (256, 256), 64).descriptor()
    with pytest.raises(ValueError, match="at least one element"):
        pkg.FP8Tensor(q.codes, q.scales, (256, 0)).descriptor()


def test_autograd_refusals(pkg):
    """A weight whose gradient would be refused in the backward pass is refused in the call."""
    AG = importlib.import_module("triton-kernel-test_amd.autograd")
    x, a = torch.zeros(4, 256, dtype=torch.bfloat16), torch.zeros(256, 16, dtype=torch.bfloat16)
    rows = pkg.FP8Tensor(torch.zeros(256, 256, dtype=torch.uint8), torch.zeros(256, 4, dtype=torch.uint8), (256, 256), 1)
    for f in (lambda: AG.fp8_linear(x, rows), lambda: AG.rms_norm_linear(x, None, rows),
              lambda: AG.rms_norm_linear(x, None, [rows, rows], residual=x),
              lambda: AG.lora_linear_compressed(x, rows, a, a.mT.contiguous())):
        with pytest.raises(ValueError, match="128 x 128"):
            f()
    for f in (lambda: AG.fp8_linear(rows, x), lambda: AG.fp8_linear(x[0, 0], x)):
        with pytest.raises(ValueError, match="at least one dimension"):
            f()
    for w in ([], [x], x, (rows, None)):
        with pytest.raises(ValueError, match="must be FP8Tensors"):
            AG.rms_norm_linear(x, None, w)
    for w in (None, x[0]):
        with pytest.raises(ValueError, match="FP8Tensor or a dense matrix"):
            AG.fp8_linear(x, w)


def test_tensor_attributes(pkg):
    c, s = torch.zeros(6, 128, dtype=torch.uint8), torch.zeros(6, 4, dtype=torch.uint8)
    q = pkg.FP8Tensor(c, s, [2, 3, 100])
    assert q.rows == 6 and q.cols == 100 and q.shape == (2, 3, 100) and q.block == 1 and q.codes is c and q.scales is s
    assert q.nbytes() == 6 * 132 and "FP8Tensor" in repr(q)
    q.scales = s + 1
    assert q.codes is c and q.scales.eq(1).all()
