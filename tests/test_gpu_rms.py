"""Root-mean-square norm, forward and backward, in its types and with its 8-bit output, against 64-bit forms."""

import importlib

import pytest
import torch

import opref8 as R
from opref import assert_within

pytestmark = pytest.mark.gpu
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32
EPS = 1e-6


def _r(rows, n, dtype, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(7000 * rows + n + seed)
    return (scale * torch.randn(rows, n, generator=g)).to(dtype).cuda()


def _w(n, dtype, seed=9):
    return (1.0 + 0.1 * torch.randn(n, generator=torch.Generator().manual_seed(n + seed))).to(dtype).cuda()


# rows in 16 lanes, a wave, several waves; one and two chunks a thread (four backward); rows that end inside a chunk; wide rows
SIZES = [(1, 1), (5, 7), (33, 64), (70, 128), (3, 200), (9, 512), (300, 513), (4, 1000), (1030, 1024), (5, 4096), (2, 5003),
         (7, 8200), (3, 12000), (2, 16384), (3, 16390), (2, 20003)]


@pytest.mark.parametrize("rows,n", SIZES)
@pytest.mark.parametrize("dtype,wdtype", [(BF, BF), (F16, F16), (F32, F32), (BF, F32), (F32, BF)],
                         ids=["bf16", "fp16", "fp32", "bf16-w32", "fp32-wb"])
def test_norm(pkg, rows, n, dtype, wdtype):
    x, res, w = _r(rows, n, dtype), _r(rows, n, dtype, 1), _w(n, wdtype)
    dy, dh = _r(rows, n, dtype, 2), _r(rows, n, dtype, 3)
    y, rstd = pkg.rms_norm_forward(x, w, EPS)
    ref = R.Rms64(x, w, EPS)
    assert_within(y, ref.y, ref.bound_y(dtype), "y")
    assert_within(rstd, ref.rstd[:, 0], ref.r_rstd * ref.rstd[:, 0], "rstd")
    (dx, dw), (bx, bw) = ref.grads(dy, dtype, wdtype)
    gx, gw = pkg.rms_norm_backward(dy, x, w, rstd)
    assert_within(gx, dx, bx, "dx")
    assert_within(gw, dw, bw, "dw")
    y, h, rstd = pkg.add_rms_norm_forward(x, res, w, EPS)
    assert torch.equal(h, (x.float() + res.float()).to(dtype))
    ref = R.Rms64(h, w, EPS)
    assert_within(y, ref.y, ref.bound_y(dtype), "y of the sum")
    (dx, dw), (bx, bw) = ref.grads(dy, dtype, wdtype, dh)
    gx, gw = pkg.rms_norm_backward(dy, h, w, rstd, dh)
    assert_within(gx, dx, bx, "dx of the sum")
    assert_within(gw, dw, bw, "dw of the sum")
    assert torch.equal(pkg.rms_norm_backward(dy, h, w, rstd, dh, weight_grad=False)[0], gx)


@pytest.mark.parametrize("rows,n", SIZES)
@pytest.mark.parametrize("dtype", [BF, F16, F32], ids=["bf16", "fp16", "fp32"])
def test_norm_in_8_bits(pkg, rows, n, dtype):
    """The codes are those of y's fp32 values: each within y's own error of a rounding of the exact y, under a scale that the
    block's largest magnitude allows."""
    x, res, w = _r(rows, n, dtype), _r(rows, n, dtype, 1), _w(n, dtype)
    for add in (False, True):
        if add:
            q, h, rstd = pkg.add_rms_norm_forward(x, res, w, EPS, fp8=True)
            _, h2, r2 = pkg.add_rms_norm_forward(x, res, w, EPS)
            assert torch.equal(h, h2)
        else:
            h = x
            q, rstd = pkg.rms_norm_forward(x, w, EPS, fp8=True)
            _, r2 = pkg.rms_norm_forward(x, w, EPS)
        assert torch.equal(rstd, r2) and q.shape == x.shape and q.block == 1
        ref = R.Rms64(h, w, EPS)
        steps = -(-n // 128)
        s = q.scales.cpu().long()[:, :steps]
        e = ref.e_y()
        top, slack = R.blocks(ref.y, 1).abs().amax((1, 3)), R.blocks(e, 1).amax((1, 3))
        scale = torch.exp2(s.double() - 127)
        assert (top - slack <= 448 * scale).all() and ((top + slack > 224 * scale) | (s == 0)).all()
        got = R.tensor_values(q)
        unit = scale.repeat_interleave(128, 1)[:, :n]
        # half a step of 2^-3 in its binade, or of the subnormal codes
        half = torch.maximum((ref.y.abs() + e) * 2.0 ** -4, 2.0 ** -10 * unit)
        assert_within(got, ref.y, half + e, "values")
        assert (q.codes.view(torch.uint8)[:, n:] == 0).all()


def test_strides_and_shapes(pkg):
    base, res = _r(60, 1200, BF), _r(60, 1200, BF, 1)
    w = _w(1000, BF)
    for x, r in ((base[::2, 3:1003], res[::2, :1000]), (base[:, 5:1005], res[:, 7:1007]), (base[:1, :1000].expand(9, 1000), res[:9, :1000]),
                 (base[:, :1000].reshape(5, 12, 1000), res[:, :1000].reshape(5, 12, 1000))):
        y, h, rstd = pkg.add_rms_norm_forward(x, r, w, EPS)
        y2, h2, rstd2 = pkg.add_rms_norm_forward(x.contiguous(), r.contiguous(), w, EPS)
        assert torch.equal(y, y2) and torch.equal(h, h2) and torch.equal(rstd, rstd2) and rstd.shape == x.shape[:-1]
        q, _, _ = pkg.add_rms_norm_forward(x, r, w, EPS, fp8=True)
        q2, _, _ = pkg.add_rms_norm_forward(x.contiguous(), r.contiguous(), w, EPS, fp8=True)
        assert torch.equal(q.codes.view(torch.uint8), q2.codes.view(torch.uint8)) and q.shape == x.shape
        steps = 8
        assert torch.equal(q.scales[:, :steps], q2.scales[:, :steps])
        dx, dw = pkg.rms_norm_backward(x, h, w, rstd, r)
        dx2, dw2 = pkg.rms_norm_backward(x.contiguous(), h, w, rstd, r.contiguous())
        assert torch.equal(dx, dx2) and torch.equal(dw, dw2)
    one = base[0, :1000]
    assert torch.equal(pkg.rms_norm_forward(one, w, EPS)[0], pkg.rms_norm_forward(one.reshape(1, -1), w, EPS)[0][0])


def test_what_lies_behind_a_row_does_not_matter(pkg):
    """Rows that end inside a chunk are read whole: NaN in the gap between rows stays there."""
    for n in (13, 203, 1003, 5003):
        wide = torch.full((9, n + 8), float("nan"), dtype=BF, device="cuda")
        x = _r(9, n, BF)
        wide[:, :n] = x
        w = _w(n, BF)
        y, rstd = pkg.rms_norm_forward(x, w, EPS)
        y2, rstd2 = pkg.rms_norm_forward(wide[:, :n], w, EPS)
        assert torch.equal(y, y2) and torch.equal(rstd, rstd2)
        for a, b in zip(pkg.rms_norm_backward(x, x, w, rstd), pkg.rms_norm_backward(wide[:, :n], wide[:, :n], w, rstd, None)):
            assert torch.equal(a, b)
        for a, b in zip(pkg.rms_norm_backward(x, x, w, rstd, x), pkg.rms_norm_backward(wide[:, :n], wide[:, :n], w, rstd, wide[:, :n])):
            assert torch.equal(a, b)


def test_special_values(pkg):
    """NaN and infinity stay in their row, rows of zeros give zeros, no rows give zeros of the weight's gradient."""
    x = _r(6, 300, BF)
    x[1, 3], x[2, 299], x[3] = float("nan"), float("inf"), 0.0
    w = _w(300, BF)
    y, rstd = pkg.rms_norm_forward(x, w, EPS)
    assert torch.isnan(y[1]).all() and torch.isnan(y[2, 299]) and y[3].eq(0).all() and torch.isfinite(y[[0, 4, 5]]).all()
    q, _ = pkg.rms_norm_forward(x, w, EPS, fp8=True)
    s = q.scales[:, :3].cpu()
    assert s[1].eq(255).all() and s[2, 2] == 255 and s[3].eq(0).all() and s[[0, 4, 5]].ne(255).all()
    dx, dw = pkg.rms_norm_backward(x[:0], x[:0], w, rstd[:0])
    assert dx.shape == (0, 300) and dw.eq(0).all()
    y, rstd = pkg.rms_norm_forward(x[:0], None, EPS)
    assert y.shape == (0, 300) and pkg.rms_norm_forward(x[:0], None, EPS, fp8=True)[0].rows == 0
    y, rstd = pkg.rms_norm_forward(x[4:], None, EPS)
    assert torch.equal(y, pkg.rms_norm_forward(x[4:], torch.ones(300, device="cuda"), EPS)[0])
    assert pkg.rms_norm_backward(x[4:], x[4:], None, rstd)[1].dtype == F32


def test_offsets_past_32_bits(pkg):
    n, rows = 4096, (1 << 20) + 37
    x = torch.zeros(rows, n, dtype=BF, device="cuda")
    tail = _r(37, n, BF)
    x[-37:] = tail
    w = _w(n, BF)
    y, rstd = pkg.rms_norm_forward(x, w, EPS)
    y2, r2 = pkg.rms_norm_forward(tail, w, EPS)
    assert torch.equal(y[-37:], y2) and torch.equal(rstd[-37:], r2)
    del y
    dx, _ = pkg.rms_norm_backward(x, x, w, rstd)
    assert torch.equal(dx[-37:], pkg.rms_norm_backward(tail, tail, w, r2)[0])


def test_streams_and_graphs(pkg):
    """Steps on several streams at once, and a captured step replayed on new inputs between eager ones."""
    w = _w(1000, BF)

    def step(x):
        y, h, rstd = pkg.add_rms_norm_forward(x, x, w, EPS)
        q, _, _ = pkg.add_rms_norm_forward(x, x, w, EPS, fp8=True)
        return (y, h, q.codes.view(torch.uint8), *pkg.rms_norm_backward(y, h, w, rstd, x))
    xs = [_r(m, 1000, BF, m) for m in (3, 200, 700)]
    want = [step(x) for x in xs]
    torch.cuda.synchronize()
    got = []
    for x in xs:
        with torch.cuda.stream(torch.cuda.Stream()):
            got.append(step(x))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(u, v) for u, v in zip(a, b))
    static = _r(200, 1000, BF, 5)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(static)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(static)
    for i in range(3):
        static.copy_(_r(200, 1000, BF, 60 + i))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(u, v) for u, v in zip(out, step(static)))


# ---------------------------------------------------------------- autograd
@pytest.fixture(scope="module")
def AG(pkg):
    return importlib.import_module("triton-kernel-test_amd.autograd")


@pytest.mark.parametrize("n", [40, 700])
def test_gradients_are_differences(pkg, AG, n):
    """The gradient along a direction against the difference quotient of the 64-bit norm."""
    x, res, w = _r(6, n, F32).requires_grad_(), _r(6, n, F32, 1).requires_grad_(), _w(n, F32).requires_grad_()
    cy, ch = _r(6, n, F32, 2), _r(6, n, F32, 3)
    y, h = AG.add_rms_norm(x, res, w, EPS)
    ((y * cy).sum() + (h * ch).sum()).backward()
    assert torch.equal(x.grad, res.grad)

    def loss(x, res, w):
        h = (x + res).double().cpu()
        z = h / torch.sqrt((h * h).mean(-1, keepdim=True) + EPS) * w.double().cpu()
        return float((z * cy.double().cpu()).sum() + (h * ch.double().cpu()).sum())
    t = 1e-4
    for p, g in ((x, x.grad), (res, res.grad), (w, w.grad)):
        d = torch.randn(p.shape, generator=torch.Generator().manual_seed(n), dtype=torch.float64).cuda()
        args = lambda k: [(q.detach().double() + (k * t * d if q is p else 0)) for q in (x, res, w)]  # noqa: E731
        diff = (loss(*args(1)) - loss(*args(-1))) / (2 * t)
        # central differences are off by t^2 / 6 times the third derivative, and the fp32 gradients by their rounding
        assert abs(diff - float((g.double() * d).sum())) <= 1e-4 * float((g.double() * d).abs().sum()) + 1e-4


def test_autograd_calls(pkg, AG):
    x, w = _r(30, 300, BF).requires_grad_(), _w(300, BF).requires_grad_()
    dy = _r(30, 300, BF, 2)
    y = AG.rms_norm(x, w, EPS)
    y.backward(dy)
    yf, rstd = pkg.rms_norm_forward(x.detach(), w.detach(), EPS)
    dx, dw = pkg.rms_norm_backward(dy, x.detach(), w.detach(), rstd)
    assert torch.equal(y, yf) and torch.equal(x.grad, dx) and torch.equal(w.grad, dw)
    frozen = AG.rms_norm(x, w.detach(), EPS)
    x.grad = None
    frozen.backward(dy)
    assert torch.equal(x.grad, dx)
    # only one of the two outputs used
    res = _r(30, 300, BF, 1).requires_grad_()
    x.grad = None
    _, h = AG.add_rms_norm(x, res, w, EPS)
    h.backward(dy)
    assert torch.equal(x.grad, dy) and torch.equal(res.grad, dy)
    x.grad = res.grad = None
    y, _ = AG.add_rms_norm(x, res, w, EPS)
    y.backward(dy)
    assert torch.equal(x.grad, res.grad)


@pytest.mark.parametrize("rows", [4, 100])
def test_norm_and_products_together(pkg, AG, rows):
    """A pre-norm layer as it is used: residual, norm in 8 bits, query, key and value products, and all gradients."""
    x, res = _r(rows, 512, BF).requires_grad_(), _r(rows, 512, BF, 1).requires_grad_()
    w = _w(512, BF).requires_grad_()
    ws = [pkg.fp8_quantize(_r(n, 512, BF, n, 0.05), 128) for n in (512, 128, 130)]
    *ys, h = AG.rms_norm_linear(x, w, ws, residual=res)
    dys, dh = [_r(rows, q.rows, BF, q.rows + 1) for q in ws], _r(rows, 512, BF, 3)
    torch.autograd.backward([*ys, h], [*dys, dh])
    q, h2, rstd = pkg.add_rms_norm_forward(x.detach(), res.detach(), w.detach(), fp8=True)
    assert torch.equal(h, h2)
    for y, t in zip(ys, ws):
        assert torch.equal(y, pkg.fp8_gemm(q, t))
    parts = [pkg.fp8_linear_backward(d, t, F32) for d, t in zip(dys, ws)]
    dn = (parts[0] + parts[1] + parts[2]).to(BF)
    dx, dw = pkg.rms_norm_backward(dn, h2, w.detach(), rstd, dh)
    assert torch.equal(x.grad, dx) and torch.equal(res.grad, dx) and torch.equal(w.grad, dw)
    # one weight, no residual; a product whose output goes unused
    x2 = x.detach().clone().requires_grad_()
    y = AG.rms_norm_linear(x2, w.detach(), ws[0])
    y.backward(dys[0])
    _, r2 = pkg.rms_norm_forward(x2.detach(), w.detach())
    dn = pkg.fp8_linear_backward(dys[0], ws[0])
    assert torch.equal(x2.grad, pkg.rms_norm_backward(dn, x2.detach(), w.detach(), r2)[0])
    x3 = x.detach().clone().requires_grad_()
    a, b = AG.rms_norm_linear(x3, w.detach(), ws[:2])
    b.sum().backward()
    assert torch.isfinite(x3.grad).all()


def test_no_rows(pkg, AG):
    none, w = _r(4, 512, BF)[:0].requires_grad_(), _w(512, BF).requires_grad_()
    q = pkg.fp8_quantize(_r(256, 512, BF, 1, 0.05), 128)
    y, h = AG.rms_norm_linear(none, w, q, residual=none.detach())
    (y.sum() + h.sum()).backward()
    assert y.shape == (0, 256) and none.grad.shape == (0, 512) and w.grad.eq(0).all()


def test_captured_step(pkg, AG):
    """A layer's forward and backward pass in one graph, with a trained and a frozen product: every replay gives the eager
    results of its inputs, with eager work between."""
    frozen = pkg.fp8_quantize(_r(512, 512, BF, 1, 0.05), 128)
    wn, wt = _w(512, BF).requires_grad_(), _r(384, 512, BF, 2, 0.05).requires_grad_()
    x, res, dy = _r(300, 512, BF), _r(300, 512, BF, 1), _r(300, 384, BF, 4)

    def step(x, res, dy):
        x, res = x.detach().requires_grad_(), res.detach().requires_grad_()
        y, h = AG.rms_norm_linear(x, wn, frozen, residual=res)
        z = AG.fp8_linear(y, wt)
        gx, gr, gn, gt = torch.autograd.grad([z, h], [x, res, wn, wt], [dy, h.detach()])
        return z.detach(), gx, gr, gn, gt

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x, res, dy)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(x, res, dy)
    for seed in range(4):
        x.copy_(_r(300, 512, BF, 10 + seed))
        dy.copy_(_r(300, 384, BF, 20 + seed))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        for a, b in zip(got, step(x, res, dy)):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("n", [100, 512, 5003, 9000, 20000])
def test_outputs_over_inputs(pkg, n, dtype):
    """Through the C ABI h may take the place of x or the residual, and dx that of dy or dh."""
    L = importlib.import_module("triton-kernel-test_amd._lib")
    rows, dt = 70, {BF: L.LRQ_BF16, F32: L.LRQ_F32}[dtype]
    x, res, w, dh, dy = _r(rows, n, dtype), _r(rows, n, dtype, 1), _w(n, BF), _r(rows, n, dtype, 2), _r(rows, n, dtype, 3)
    y, h, rstd = pkg.add_rms_norm_forward(x, res, w, EPS)
    dx, dw = pkg.rms_norm_backward(dy, h, w, rstd, dh)
    stream = torch.cuda.current_stream().cuda_stream
    for over in range(2):
        a, b, y2, r2 = x.clone(), res.clone(), torch.empty_like(x), torch.empty_like(rstd)
        h2 = (a, b)[over]
        L.call("lrq_rms_norm_fwd", a.data_ptr(), n, b.data_ptr(), n, dt, w.data_ptr(), L.LRQ_BF16, rows, n, EPS, h2.data_ptr(),
               n, y2.data_ptr(), n, None, r2.data_ptr(), stream)
        assert torch.equal(h2, h) and torch.equal(y2, y) and torch.equal(r2, rstd)
        a, b, dw2 = dy.clone(), dh.clone(), torch.empty_like(dw)
        size = L.call_raw("lrq_rms_norm_bwd_workspace", rows, n)
        ws = torch.empty(size // 4, device="cuda")
        dx2 = (a, b)[over]
        L.call("lrq_rms_norm_bwd", a.data_ptr(), n, b.data_ptr(), n, h.data_ptr(), n, dt, w.data_ptr(), L.LRQ_BF16,
               rstd.data_ptr(), rows, n, dx2.data_ptr(), n, dw2.data_ptr(), ws.data_ptr(), size, stream)
        assert torch.equal(dx2, dx) and torch.equal(dw2, dw)


def test_under_compressed_saved_tensors(pkg, AG):
    """A norm's rows are kept compressed and decoded for its gradients; a trained product keeps its own 8 bits of x."""
    def kept(t):
        return pkg.decode(pkg.encode(t.detach(), None, bits=8, group_size=64))

    x, w, dy = _r(64, 512, BF).requires_grad_(), _w(512, BF).requires_grad_(), _r(64, 512, BF, 2)
    hooks = AG.compressed_saved_tensors(bits=8, group=64, min_numel=1)
    with hooks:
        y = AG.rms_norm(x * 1, w, EPS)
    assert hooks.stats["compressed"] == 1
    y.backward(dy)
    _, rstd = pkg.rms_norm_forward(x.detach(), w.detach(), EPS)
    for got, want in zip((x.grad, w.grad), pkg.rms_norm_backward(dy, kept(x), w.detach(), rstd)):
        assert torch.equal(got, want)
    q, wt = pkg.fp8_quantize(_r(256, 512, BF, 3, 0.05), 128), _r(128, 256, BF, 4, 0.05).requires_grad_()
    x.grad = w.grad = None
    hooks = AG.compressed_saved_tensors(bits=8, group=64, min_numel=1)
    with hooks:
        y, h = AG.rms_norm_linear(x, w, q, residual=x.detach(), eps=EPS)
        z = AG.fp8_linear(y, wt)
    assert hooks.stats["compressed"] == 1  # h
    dz = _r(64, 128, BF, 5)
    torch.autograd.backward([z, h], [dz, dy])
    n8, hh, rstd = pkg.add_rms_norm_forward(x.detach(), x.detach(), w.detach(), EPS, fp8=True)
    wq = pkg.fp8_quantize(wt.detach(), 128)
    dn = pkg.fp8_linear_backward(pkg.fp8_linear_backward(dz, wq), q)
    dx, dw = pkg.rms_norm_backward(dn, kept(hh), w.detach(), rstd, dy)
    assert torch.equal(x.grad, dx) and torch.equal(w.grad, dw)
    assert torch.equal(wt.grad, pkg.fp8_weight_gradient(dz, pkg.fp8_linear(n8, q)))
