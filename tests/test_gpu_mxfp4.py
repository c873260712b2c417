"""MXFP4 on the HIP kernels: quantisation bit for bit against a search for the nearest code, products against
64-bit products of the decoded operands within their rounding bounds (opref.py)."""

import importlib

import pytest
import torch

import opref as R

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _check_quantized(pkg, x):
    q = pkg.mxfp4_quantize(x)
    x2 = x.reshape(-1, x.shape[-1])
    codes, scales = R.mx_quantize(x2)
    assert torch.equal(q.scales.cpu().long(), scales), "scales"
    got = R.mx_nibbles(q.codes)
    assert torch.equal(got, codes), f"codes differ at {(got != codes).nonzero()[:4].tolist()}"
    back = pkg.mxfp4_dequantize(q, x.dtype)
    want = R.mx_values(codes, scales, x.shape[-1]).reshape(x.shape)
    nan = (scales == 255).repeat_interleave(32, dim=1)[:, :x.shape[-1]].reshape(x.shape)
    assert torch.isnan(back.cpu()[nan]).all()
    assert torch.equal(back.cpu()[~nan], want[~nan].to(x.dtype))
    return q


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("rows,k", [(1, 1), (3, 7), (5, 32), (2, 33), (4, 127), (4, 128), (7, 129), (9, 1000), (64, 4096)])
def test_quantize(pkg, dev, rows, k, dtype):
    g = _gen(rows * 1000 + k)
    # magnitudes over many binades from block to block, zeros and both signs
    x = torch.randn(rows, k, generator=g) * torch.exp2(torch.randint(-12, 12, (rows, 1), generator=g).float())
    x[torch.rand(rows, k, generator=g) < 0.05] = 0.0
    _check_quantized(pkg, x.to(DT[dtype]).to(dev))


def test_quantize_every_rounding(pkg, dev):
    """Blocks whose largest element pins the scale, swept over every bf16 value of five binades below it (all ties
    and their neighbours), at scales over the whole range of the exponent."""
    mant = torch.arange(128).float() / 128 + 1
    vals = torch.cat([mant * 2.0 ** e for e in range(-3, 3)] + [torch.zeros(1), -mant * 0.5])
    for top in (4.0, 7.0, 7.96875):
        n = -(-vals.numel() // 31)
        block = torch.nn.functional.pad(vals, (0, 31 * n - vals.numel())).reshape(n, 31)
        block = torch.cat([block, torch.full((n, 1), top)], 1)
        block = torch.where(block.abs() > top, torch.zeros(()), block)
        for e in (-125, -100, -24, -1, 0, 5, 60, 125):
            _check_quantized(pkg, (block * 2.0 ** e).to(torch.float32).to(dev))
            _check_quantized(pkg, (block * 2.0 ** e).to(torch.bfloat16).to(dev))


def test_quantize_extremes(pkg, dev):
    x = torch.zeros(8, 64, dtype=torch.float32)
    x[0, 3] = 2.0 ** -126           # the smallest normal number
    x[1, 3], x[1, 4] = 2.0 ** -130, -(2.0 ** -128)  # subnormal
    x[2, 3], x[2, 40] = float("inf"), 1.0
    x[3, 3], x[3, 40] = float("nan"), -2.0
    x[4] = torch.finfo(torch.float32).max
    x[5, 0] = 2.0 ** -124
    x[6, :] = -0.0
    _check_quantized(pkg, x.to(dev))
    _check_quantized(pkg, x.to(torch.bfloat16).to(dev))


def test_quantize_strides_shapes_and_empty(pkg, dev):
    base = torch.randn(30, 300, generator=_gen(5)).to(torch.bfloat16).to(dev)
    q1, q2 = pkg.mxfp4_quantize(base[2:19, 7:200]), pkg.mxfp4_quantize(base[2:19, 7:200].contiguous())
    assert torch.equal(q1.codes, q2.codes) and torch.equal(q1.scales, q2.scales)
    q3 = pkg.mxfp4_quantize(base.reshape(5, 6, 300))
    assert q3.shape == (5, 6, 300) and pkg.mxfp4_dequantize(q3).shape == (5, 6, 300)
    assert pkg.mxfp4_dequantize(pkg.mxfp4_quantize(base[:0])).shape == (0, 300)
    assert q3.nbytes() == 30 * (3 * 64 + 3 * 4)


def _operands(pkg, dev, m, n, k, seed):
    g = _gen(seed)
    x = torch.randn(m, k, generator=g)
    x[:, ::37] *= 15
    w = torch.randn(n, k, generator=g) * 0.05 * torch.exp2(torch.randint(-3, 3, (n, 1), generator=g).float())
    w = pkg.mxfp4_quantize(w.to(dev))
    w64 = R.mx_values(R.mx_nibbles(w.codes), w.scales.cpu().long(), k)
    return x.to(torch.bfloat16).to(dev), w, w64


# one row to several tiles; widths that end inside a block, a step and a tile
SIZES = [(1, 1, 1), (1, 16, 32), (2, 17, 33), (1, 300, 4096), (5, 129, 1000), (16, 256, 128), (17, 100, 520), (33, 64, 96),
         (64, 512, 2048), (65, 257, 136), (130, 1, 257), (128, 128, 128), (129, 260, 640), (300, 513, 1111),
         (512, 768, 1024), (1, 5000, 8), (700, 40, 72), (4096, 4096, 160), (200, 13000, 288), (40, 13000, 264), (300, 500, 6000)]


@pytest.mark.parametrize("m,n,k", SIZES)
def test_linear_and_gradient(pkg, dev, m, n, k):
    print(f"[mx] linear {m} {n} {k}", flush=True)
    x, w, w64 = _operands(pkg, dev, m, n, k, m + n + k)
    dy = torch.randn(m, n, generator=_gen(1)).to(torch.bfloat16).to(dev)
    x64, dy64 = x.double().cpu(), dy.double().cpu()
    for dt in (torch.bfloat16, torch.float32):
        ref, bound = R.product_bound(x64, w64.T, dt)
        R.assert_within(pkg.mxfp4_linear(x, w, dt), ref, bound, f"y {dt}")
        ref, bound = R.product_bound(dy64, w64, dt)
        R.assert_within(pkg.mxfp4_linear_backward(dy, w, dt), ref, bound, f"dx {dt}")


@pytest.mark.parametrize("m,n,k", SIZES)
def test_gemm(pkg, dev, m, n, k):
    print(f"[mx] gemm {m} {n} {k}", flush=True)
    x, w, w64 = _operands(pkg, dev, m, n, k, m * n + k)
    a = pkg.mxfp4_quantize(x)
    a64 = R.mx_values(R.mx_nibbles(a.codes), a.scales.cpu().long(), k)
    for dt in (torch.bfloat16, torch.float32):
        ref, bound = R.product_bound(a64, w64.T, dt)
        R.assert_within(pkg.mxfp4_gemm(a, w, dt), ref, bound, f"{dt}")


def _grid(shape, dev, seed, values=(0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)):
    g = torch.Generator(device=dev).manual_seed(seed)
    v = torch.tensor(values, device=dev)[torch.randint(len(values), shape, generator=g, device=dev)]
    return v * (2 * torch.randint(2, shape, generator=g, device=dev) - 1).to(v.dtype)


# (m, n, k, which product, whether the contraction is split over workgroups): each height of each kernel, both ways
PLANS = [(100, 200, 72, "linear", False), (40, 100, 1200, "linear", True), (4100, 260, 72, "linear", False),
         (2050, 100, 3300, "linear", True), (600, 6500, 72, "linear", False), (4100, 100, 13000, "linear", True),
         (3, 40, 9000, "linear", False), (9, 8300, 300, "linear", False), (4, 8200, 1000, "linear", False),
         (16, 300, 5000, "linear", False), (40, 100, 72, "back", False), (40, 1300, 72, "back", True),
         (4100, 100, 300, "back", False), (2050, 4100, 72, "back", True), (2050, 100, 2000, "back", False),
         (4100, 4100, 72, "back", True), (40, 100, 72, "gemm", False), (40, 100, 2000, "gemm", True),
         (600, 6500, 72, "gemm", False), (4100, 100, 9000, "gemm", True), (2050, 4100, 72, "gemm", False),
         (2048, 4096, 49152, "gemm", True)]


@pytest.mark.parametrize("m,n,k,which,split", PLANS)
def test_every_plan_is_exact_on_small_numbers(pkg, dev, m, n, k, which, split):
    """Multiples of 1/2 (1/4 for two MXFP4 operands) whose sums stay below 2^22: fp32 holds every partial sum exactly in
    any order, so the outputs are those of 64 bits, rounded once in bf16; a block left out or taken twice shows."""
    import ctypes
    L = importlib.import_module("triton-kernel-test_amd._lib")
    print(f"[mx] plan {which} {m} {n} {k}", flush=True)
    w = _grid((n, k), dev, 1)
    wq = pkg.mxfp4_quantize(w)
    assert torch.equal(pkg.mxfp4_dequantize(wq, torch.float32), w)
    if which == "gemm":
        x = _grid((m, k), dev, 2)
        xq = pkg.mxfp4_quantize(x)
        ref = x.double() @ w.double().T
        run = lambda dt: pkg.mxfp4_gemm(xq, wq, dt)
        ws = L.call_raw("lrq_mxfp4_gemm_workspace", ctypes.byref(xq.descriptor()), ctypes.byref(wq.descriptor()))
    else:
        x = _grid((m, k if which == "linear" else n), dev, 2, (0.0, 1.0, 2.0))
        ref = x.double() @ (w.double().T if which == "linear" else w.double())
        xb = x.to(torch.bfloat16)
        run = lambda dt: (pkg.mxfp4_linear if which == "linear" else pkg.mxfp4_linear_backward)(xb, wq, dt)
        ws = L.call_raw("lrq_mxfp4_linear_workspace", m, ctypes.byref(wq.descriptor()), int(which == "back"))
    assert (ws > 0) == split
    assert float(ref.abs().max()) < 2 ** 22
    assert torch.equal(run(torch.float32).double(), ref)
    assert torch.equal(run(torch.bfloat16), ref.to(torch.float32).to(torch.bfloat16))


def test_products_over_the_range_of_scales(pkg, dev):
    """Every scale from 2^-127 (elements below the smallest normal number) to 2^125, picked out by one-hot operands."""
    n, k = 64, 256
    codes = torch.randint(0, 256, (n, 128), generator=_gen(5), dtype=torch.uint8)
    scales = (torch.arange(n * 8) % 253).to(torch.uint8).reshape(n, 8)
    w = pkg.MXFP4Tensor(codes.to(dev), scales.to(dev), (n, k))
    w64 = R.mx_values(R.mx_nibbles(codes), scales.long(), k)
    eye, eye_n = (torch.eye(i, dtype=torch.bfloat16, device=dev) for i in (k, n))
    assert torch.equal(pkg.mxfp4_dequantize(w, torch.float32).cpu().double(), w64)
    assert torch.equal(pkg.mxfp4_linear(eye, w, torch.float32).cpu().double(), w64.T)
    assert torch.equal(pkg.mxfp4_linear(eye[:9], w, torch.float32).cpu().double(), w64.T[:9])
    assert torch.equal(pkg.mxfp4_linear_backward(eye_n, w, torch.float32).cpu().double(), w64)
    assert torch.equal(pkg.mxfp4_gemm(pkg.mxfp4_quantize(eye), w, torch.float32).cpu().double(), w64.T)


def test_past_32_bits(pkg, dev):
    """An activation of more than 2^32 bytes: its last rows, quantised and multiplied, are those of the rows alone."""
    rows, k, n = 524300, 4104, 40
    x = torch.zeros(rows, k, dtype=torch.bfloat16, device=dev)
    tail = _grid((3, k), dev, 3).to(torch.bfloat16)
    x[-3:] = tail
    q, qt = pkg.mxfp4_quantize(x), pkg.mxfp4_quantize(tail)
    assert torch.equal(q.codes[-3:], qt.codes) and torch.equal(q.scales[-3:], qt.scales)
    assert torch.equal(pkg.mxfp4_dequantize(q)[-3:], tail)
    w = _grid((n, k), dev, 4)
    wq = pkg.mxfp4_quantize(w)
    ref = tail.double() @ w.double().T  # exact in fp32, as above
    for y in (pkg.mxfp4_linear(x, wq, torch.float32), pkg.mxfp4_gemm(q, wq, torch.float32)):
        assert torch.equal(y[-3:].double(), ref) and not y[:-3].any()
    # and as the output of the gradient
    dy = torch.zeros(rows, n, dtype=torch.bfloat16, device=dev)
    dy[-3:] = tail[:, :n]
    dx = pkg.mxfp4_linear_backward(dy, wq)
    assert torch.equal(dx[-3:].float(), (tail[:, :n].double() @ w.double()).float().to(torch.bfloat16).float())
    assert not dx[:-3].any()
    del x, q, dx


def test_two_graphs_with_split_products(pkg, dev):
    """Two captured graphs and eager calls, each with workspaces of its own, replayed in turn."""
    x, w, _ = _operands(pkg, dev, 40, 100, 2048, 11)
    x2 = x.flip(0).contiguous()
    a, a2 = pkg.mxfp4_quantize(x), pkg.mxfp4_quantize(x2)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for xx, aa in ((x, a), (x2, a2)):
        g = torch.cuda.CUDAGraph()
        print("[mx] capture", flush=True)
        with torch.cuda.graph(g):
            outs.append((pkg.mxfp4_linear(xx, w), pkg.mxfp4_gemm(aa, w)))
        graphs.append(g)
    want = [(pkg.mxfp4_linear(xx, w), pkg.mxfp4_gemm(aa, w)) for xx, aa in ((x, a), (x2, a2))]
    for _ in range(3):
        for g in graphs:
            g.replay()
        again = pkg.mxfp4_linear(x, w)
        torch.cuda.synchronize()
        assert torch.equal(again, want[0][0])
        for out, exp in zip(outs, want):
            assert torch.equal(out[0], exp[0]) and torch.equal(out[1], exp[1])


def test_products_map_every_element(pkg, dev):
    """One-hot operands pick single elements of the weight: any swap of rows, columns, nibbles or scales shows."""
    n, k = 150, 300
    _, w, w64 = _operands(pkg, dev, 1, n, k, 9)
    eye = torch.eye(k, dtype=torch.bfloat16, device=dev)
    assert torch.equal(pkg.mxfp4_linear(eye, w, torch.float32).cpu().double(), w64.T)
    assert torch.equal(pkg.mxfp4_gemm(pkg.mxfp4_quantize(eye), w, torch.float32).cpu().double(), w64.T)
    assert torch.equal(pkg.mxfp4_linear_backward(torch.eye(n, dtype=torch.bfloat16, device=dev), w,
                                                 torch.float32).cpu().double(), w64)


def test_products_strides_and_leading_dims(pkg, dev):
    x, w, _ = _operands(pkg, dev, 24, 96, 256, 3)
    wide = torch.randn(24, 300, generator=_gen(4)).to(torch.bfloat16).to(dev)
    wide[:, 8:264] = x
    y = pkg.mxfp4_linear(x, w)
    assert torch.equal(pkg.mxfp4_linear(wide[:, 8:264], w), y)
    assert torch.equal(pkg.mxfp4_linear(x.reshape(2, 3, 4, 256), w).reshape(24, 96), y)
    dy = torch.randn(24, 96, generator=_gen(6)).to(torch.bfloat16).to(dev)
    d = pkg.mxfp4_linear_backward(dy, w)
    wide[:, 16:112] = dy
    assert torch.equal(pkg.mxfp4_linear_backward(wide[:, 16:112], w), d)
    assert torch.equal(pkg.mxfp4_linear_backward(dy.T.contiguous().T, w), d)
    row = dy[:1].expand(24, 96)
    assert torch.equal(pkg.mxfp4_linear_backward(row, w), pkg.mxfp4_linear_backward(row.contiguous(), w))
    # codes and scales with wider rows than needed, at rows of a larger buffer
    codes = torch.full((100, 256), 0xAB, dtype=torch.uint8, device=dev)
    scales = torch.full((100, 16), 99, dtype=torch.uint8, device=dev)
    codes[2:98, :128], scales[2:98, :8] = w.codes, w.scales
    w2 = pkg.MXFP4Tensor(codes[2:98], scales[2:98], (96, 256))
    assert torch.equal(pkg.mxfp4_linear(x, w2), y) and torch.equal(pkg.mxfp4_linear_backward(dy, w2), d)
    a = pkg.mxfp4_quantize(x.reshape(4, 6, 256))
    assert torch.equal(pkg.mxfp4_gemm(a, w2), pkg.mxfp4_gemm(a, w)) and pkg.mxfp4_gemm(a, w).shape == (4, 6, 96)


def test_products_empty(pkg, dev):
    x, w, _ = _operands(pkg, dev, 4, 32, 64, 3)
    none = pkg.mxfp4_quantize(torch.empty(0, 64, device=dev))
    assert pkg.mxfp4_linear(x[:0], w).shape == (0, 32) and pkg.mxfp4_linear(x, none).shape == (4, 0)
    dx = pkg.mxfp4_linear_backward(torch.empty(4, 0, dtype=torch.bfloat16, device=dev), none)
    assert dx.shape == (4, 64) and not dx.any()
    assert pkg.mxfp4_gemm(none, w).shape == (0, 32) and pkg.mxfp4_gemm(pkg.mxfp4_quantize(x), none).shape == (4, 0)


def test_not_finite_values_stay_in_their_rows(pkg, dev):
    x, w, _ = _operands(pkg, dev, 40, 64, 256, 8)
    clean, clean_g = pkg.mxfp4_linear(x, w), pkg.mxfp4_gemm(pkg.mxfp4_quantize(x), w)
    x[7, 100] = float("nan")
    x[30, 255] = float("inf")
    y, yg = pkg.mxfp4_linear(x, w), pkg.mxfp4_gemm(pkg.mxfp4_quantize(x), w)
    rows = [i for i in range(40) if i not in (7, 30)]
    assert torch.equal(y[rows], clean[rows]) and torch.equal(yg[rows], clean_g[rows])
    assert torch.isnan(y[7]).all() and torch.isnan(yg[7]).all() and torch.isnan(yg[30]).all()
    assert not torch.isfinite(y[30]).any()
    # a NaN block of the weight: its output column, and its 32 columns of the gradient
    scales = w.scales.clone()
    scales[5, 1] = 255
    bad = pkg.MXFP4Tensor(w.codes, scales, w.shape)
    x2 = torch.ones(3, 256, dtype=torch.bfloat16, device=dev)
    for y in (pkg.mxfp4_linear(x2, bad), pkg.mxfp4_gemm(pkg.mxfp4_quantize(x2), bad)):
        assert torch.isnan(y[:, 5]).all() and torch.isfinite(y[:, :5]).all() and torch.isfinite(y[:, 6:]).all()
    dx = pkg.mxfp4_linear_backward(torch.ones(3, 64, dtype=torch.bfloat16, device=dev), bad)
    assert torch.isnan(dx[:, 32:64]).all() and torch.isfinite(dx[:, :32]).all() and torch.isfinite(dx[:, 64:]).all()


def test_deterministic_and_captured(pkg, dev):
    x, w, _ = _operands(pkg, dev, 48, 512, 2048, 10)
    dy = torch.randn(48, 512, generator=_gen(2)).to(torch.bfloat16).to(dev)

    def step():
        return (pkg.mxfp4_linear(x, w), pkg.mxfp4_linear(x[:1], w), pkg.mxfp4_linear_backward(dy, w),
                pkg.mxfp4_gemm(pkg.mxfp4_quantize(x), w))

    want = step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    print("[mx] capture", flush=True)
    with torch.cuda.graph(graph):
        outs = step()
    for _ in range(3):
        graph.replay()
        again = step()
        torch.cuda.synchronize()
        for a, b, c in zip(want, outs, again):
            assert torch.equal(a, b) and torch.equal(a, c)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        side = step()
    s.synchronize()
    for a, b in zip(want, side):
        assert torch.equal(a, b)


def test_one_dimensional_rows_and_two_streams(pkg, dev):
    x, w, _ = _operands(pkg, dev, 40, 300, 2048, 15)
    assert torch.equal(pkg.mxfp4_linear(x[5], w), pkg.mxfp4_linear(x[5:6], w)[0])
    q1, q2 = pkg.mxfp4_quantize(x[5]), pkg.mxfp4_quantize(x[5:6])
    assert q1.shape == (2048,) and torch.equal(q1.codes, q2.codes)
    assert torch.equal(pkg.mxfp4_dequantize(q1), pkg.mxfp4_dequantize(q2)[0])
    assert torch.equal(pkg.mxfp4_gemm(q1, w), pkg.mxfp4_gemm(q2, w)[0])
    dy = torch.randn(40, 300, generator=_gen(16)).to(torch.bfloat16).to(dev)
    assert torch.equal(pkg.mxfp4_linear_backward(dy[5], w), pkg.mxfp4_linear_backward(dy[5:6], w)[0])
    xs = [x, x.flip(0).contiguous()]
    qs = [pkg.mxfp4_quantize(t) for t in xs]

    def step(i):
        return pkg.mxfp4_linear(xs[i], w), pkg.mxfp4_gemm(qs[i], w), pkg.mxfp4_linear_backward(dy, w)

    want = [step(0), step(1)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(step(i))
    torch.cuda.synchronize()
    for i in range(2):
        for g in got[i]:
            for a, e in zip(g, want[i]):
                assert torch.equal(a, e)


def test_autograd_linear(pkg, dev):
    AG = importlib.import_module("triton-kernel-test_amd.autograd")
    x, w, w64 = _operands(pkg, dev, 12, 96, 256, 12)
    x = x.reshape(3, 4, 256).requires_grad_()
    y = AG.mxfp4_linear(x, w)
    dy = torch.randn(3, 4, 96, generator=_gen(3)).to(torch.bfloat16).to(dev)
    y.backward(dy)
    assert torch.equal(y, pkg.mxfp4_linear(x.detach(), w)) and torch.equal(x.grad, pkg.mxfp4_linear_backward(dy, w))
    # against differences: the product is linear, so any step is exact up to rounding
    v = torch.randn(3, 4, 256, generator=_gen(4)).double()
    diff = float((((x.detach().double().cpu() + v) @ w64.T - x.detach().double().cpu() @ w64.T) * dy.double().cpu()).sum())
    got = float((x.grad.double().cpu() * v).sum())
    bound = float((((dy.double().cpu().abs() @ w64.abs()) * (96 * R.U + R.half_step(torch.bfloat16))) * v.abs()).sum())
    assert abs(got - diff) <= bound + 1e-9 * abs(diff)


@pytest.mark.parametrize("p", [0.0, 0.1])
@pytest.mark.parametrize("mx", [False, True])
def test_lora_layer_with_dropout_and_mxfp4_base(pkg, dev, mx, p):
    """lora_linear_compressed with LoRA dropout and / or an MXFP4 base weight, behind dropout + add + layer norm, as a
    block would use them: outputs and gradients against float64 autograd of the same formulas."""
    AG = importlib.import_module("triton-kernel-test_amd.autograd")
    g = _gen(13)
    rows, d1, d2, r = 96, 512, 768, 16
    bf = torch.bfloat16
    x0, res = (torch.randn(rows, d1, generator=g).to(bf).to(dev).requires_grad_() for _ in range(2))
    lw, lb = ((1 + 0.1 * torch.randn(d1, generator=g)).to(bf).to(dev).requires_grad_() for _ in range(2))
    a = (torch.randn(d1, r, generator=g) / d1 ** 0.5).to(bf).to(dev).requires_grad_()
    b = (torch.randn(r, d2, generator=g) * 0.1).to(bf).to(dev).requires_grad_()
    w = (torch.randn(d2, d1, generator=g) / d1 ** 0.5).to(bf).to(dev)
    q = pkg.mxfp4_quantize(w)
    base = q if mx else w
    w64 = (pkg.mxfp4_dequantize(q) if mx else w).double().cpu()
    x, h = AG.dropout_add_layer_norm(x0, res, lw, lb, 0.1, 5)
    x.retain_grad()
    y = AG.lora_linear_compressed(x, base, a, b, bits=8, group=64, dropout_p=p, seed=(21, 3))
    dy = torch.randn(rows, d2, generator=g).to(bf).to(dev)
    dh = torch.randn(rows, d1, generator=g).to(bf).to(dev)
    torch.autograd.backward([y, h], [dy, dh])

    # the layer alone: its input as stored in bf16; its factor gradients see the decoded activation
    xh = pkg.decode(pkg.encode(x.detach(), None, bits=8, group_size=64)).double().cpu()
    dr, mask = R.drop64(x.detach(), p, 21, 3)
    a64, b64, dy64 = a.detach().double().cpu(), b.detach().double().cpu(), dy.double().cpu()
    y64 = x.detach().double().cpu() @ w64.T + (dr @ a64) @ b64
    g64 = dy64 @ b64.T
    dx64 = dy64 @ w64 + (g64 @ a64.T) * mask
    da64 = (xh * mask).T @ g64
    db64 = (xh * mask @ a64).T @ dy64

    def rel(got, ref):
        return float((got.detach().double().cpu() - ref).norm() / ref.norm())

    # each is a product of bf16 operands, some rounded once to bf16 on the way (2^-8 each in the worst case, at most
    # three in sequence: the intermediate factor, the sum, the output); in the 2-norm a rounding is a third of its worst
    bound = 3 * 2.0 ** -8
    rep = {"y": rel(y, y64), "dx": rel(x.grad, dx64), "dA": rel(a.grad, da64), "dB": rel(b.grad, db64)}
    print(f"[lora] mx={mx} p={p}: {rep}", flush=True)
    assert all(v <= bound for v in rep.values()), rep
    # and the block's input gradients are those of the fused norm for this dx
    _, hh, mean, rstd = pkg.dropout_add_layer_norm_forward(x0.detach(), res.detach(), lw.detach(), lb.detach(), 0.1, 5)
    dx, dres, dw, db = pkg.dropout_add_layer_norm_backward(x.grad, dh, hh, lw.detach(), mean, rstd, 0.1, 5)
    for got, want in ((x0.grad, dx), (res.grad, dres), (lw.grad, dw), (lb.grad, db)):
        assert torch.equal(got, want)


@pytest.mark.parametrize("layer", ["linear", "lora"])
@pytest.mark.parametrize("part", ["codes", "scales"])
def test_weight_changed_before_backward_is_refused(pkg, dev, layer, part):
    """A weight that was changed in place after the forward pass would give the gradient of another one."""
    AG = importlib.import_module("triton-kernel-test_amd.autograd")
    q = pkg.mxfp4_quantize(torch.randn(96, 256, generator=_gen(401)).to(torch.bfloat16).to(dev))
    x = torch.randn(24, 256, generator=_gen(402)).to(torch.bfloat16).to(dev).requires_grad_()
    a, b = (torch.randn(s, generator=_gen(403)).to(torch.bfloat16).to(dev) for s in ((256, 16), (16, 96)))

    def forward():
        return AG.mxfp4_linear(x, q) if layer == "linear" else AG.lora_linear_compressed(x, q, a, b)

    y = forward()
    getattr(q, part).add_(0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    y = forward()
    y.backward(torch.ones_like(y))
    assert torch.isfinite(x.grad).all()


def test_weight_quantised_in_inference_mode(pkg, dev):
    """Such tensors carry no version and cannot be saved; the layer takes them all the same."""
    AG = importlib.import_module("triton-kernel-test_amd.autograd")
    w = torch.randn(96, 256, generator=_gen(411)).to(torch.bfloat16).to(dev)
    with torch.inference_mode():
        qi = pkg.mxfp4_quantize(w)
    q = pkg.mxfp4_quantize(w)
    x = torch.randn(24, 256, generator=_gen(412)).to(torch.bfloat16).to(dev).requires_grad_()
    a, b = (torch.randn(s, generator=_gen(413)).to(torch.bfloat16).to(dev) for s in ((256, 16), (16, 96)))
    for f in (lambda w4: AG.mxfp4_linear(x, w4), lambda w4: AG.lora_linear_compressed(x, w4, a, b)):
        got, want = (torch.autograd.grad(f(w4).float().sum(), x)[0] for w4 in (qi, q))
        assert torch.equal(got, want)
