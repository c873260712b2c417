"""Layer norm, dropout and dropout + add + layer norm on the HIP kernels against 64-bit forms, within bounds
counted from the roundings the kernels make (opref.py)."""

import importlib

import pytest
import torch

import opref as R

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-5
SEED, OFFSET = 0x1234_5678_9ABC_DEF1, 0x2_0000_0003


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _x(shape, dtype, dev, seed, offset=0.3):
    g = _gen(seed)
    x = torch.randn(shape, generator=g) + offset
    x[..., ::64] *= 10
    return x.to(dtype).to(dev)


def _w(n, dtype, dev, seed):
    g = _gen(seed)
    return (1 + 0.2 * torch.randn(n, generator=g)).to(dtype).to(dev), (0.2 * torch.randn(n, generator=g)).to(dtype).to(dev)


def _bits(t):
    return t.view(torch.int16 if t.element_size() == 2 else torch.int32)


# row widths: one element, inside a chunk, one chunk, the limits of each register geometry (16 lanes, a wave or several whole
# waves a row, of one, two or four chunks a thread) and past the last one; odd widths start rows off every alignment
WIDTHS = [1, 3, 8, 77, 128, 129, 512, 1000, 1024, 1025, 2048, 2050, 4096, 4099, 5120, 6144, 6145, 8192, 8200, 16384,
          16385, 20011]


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("n", WIDTHS)
def test_layer_norm(pkg, dev, n, dtype):
    dt = DT[dtype]
    for rows in (1, 37):
        print(f"[norm] rows={rows} n={n} {dtype}", flush=True)
        x = _x((rows, n), dt, dev, n)
        w, b = _w(n, dt, dev, n + 1)
        dy = _x((rows, n), dt, dev, n + 2, 0.0)
        y, mean, rstd = pkg.layer_norm_forward(x, w, b, EPS)
        dx, dw, db = pkg.layer_norm_backward(dy, x, w, mean, rstd)
        dx2, none_w, none_b = pkg.layer_norm_backward(dy, x, w, mean, rstd, weight_grad=False)
        torch.cuda.synchronize()
        ref = R.Norm64(x, w, b, EPS)
        R.assert_within(y, ref.y, ref.bound_y(dt), "y")
        R.assert_within(mean, ref.mean[:, 0], (ref.e_mean + R.U * ref.mean.abs())[:, 0], "mean")
        R.assert_within(rstd, ref.rstd[:, 0], ref.e_rstd[:, 0], "rstd")
        (rdx, rdw, rdb), (bx, bw, bb), _ = ref.grads(dy, dt, dt)
        R.assert_within(dx, rdx, bx, "dx")
        R.assert_within(dw, rdw, bw, "dw")
        R.assert_within(db, rdb, bb, "db")
        assert torch.equal(_bits(dx2), _bits(dx)) and none_w is None and none_b is None


@pytest.mark.parametrize("rows,n", [(5000, 64), (3000, 512), (2111, 1024), (1500, 4096), (1100, 8192), (300, 17000)])
def test_layer_norm_many_rows(pkg, dev, rows, n):
    """More rows than row groups run at once: each group walks several; the weight gradients' parts add up, and
    twice the same call gives the same bits."""
    x = _x((rows, n), torch.bfloat16, dev, 5)
    w, b = _w(n, torch.float32, dev, 6)
    dy = _x((rows, n), torch.bfloat16, dev, 7, 0.01)
    y, mean, rstd = pkg.layer_norm_forward(x, w, b, EPS)
    first = pkg.layer_norm_backward(dy, x, w, mean, rstd)
    again = pkg.layer_norm_backward(dy, x, w, mean, rstd)
    torch.cuda.synchronize()
    ref = R.Norm64(x, w, b, EPS)
    R.assert_within(y, ref.y, ref.bound_y(torch.bfloat16), "y")
    refs, bounds, _ = ref.grads(dy, torch.bfloat16, torch.float32)
    for got, g2, r, bound, name in zip(first, again, refs, bounds, ("dx", "dw", "db")):
        R.assert_within(got, r, bound, name)
        assert torch.equal(_bits(got), _bits(g2)), name


# (rows, columns) whose row groups walk several rows each: 16 lanes, a wave and several waves a row, rows of whole chunks and
# rows that end inside one, wave counts that do and do not divide a workgroup's sixteen, one group a workgroup and several
GEOMETRIES = [(17000, 96), (17000, 100), (17000, 5), (5000, 512), (5000, 333), (3000, 1000), (3000, 1003), (2700, 1300),
              (2700, 1304), (1500, 2000), (1500, 2003), (1700, 2500), (1700, 2504), (1100, 2900), (1100, 2904), (1100, 3500),
              (1100, 3504), (1030, 4096), (530, 4500), (530, 4504), (1003, 5003), (600, 5120), (530, 8000), (530, 8190),
              (520, 9001), (520, 9008), (530, 16390)]


def _backward_plan(rows, n, fp32):
    """The backward pass's launch (csrc/lrq_norm_bwd.hip, csrc/lrq_norm.h): kind of rows, lanes and chunks a thread, groups of
    a workgroup, workgroups, parts of the weight gradients."""
    nc = -(-n // 8)
    if n > (8192 if fp32 else 16384):
        return "wide", 0, 0, 1, min(rows, 512), min(-(-rows // 4), 64)
    chunks = 1 if nc <= 1024 else 4
    lanes = 16 if nc <= 16 else 64 if nc <= 64 * chunks else 0
    waves = -(-nc // (64 * chunks))
    most = 64 * (8 if chunks == 4 else 16) // lanes if lanes else max(1, (8 if chunks == 4 else 16) // waves)
    groups = min(most, max(1, 4 * -(-rows // 1024) if lanes == 16 else -(-rows // 256)))
    grid = min(-(-rows // groups), 256)
    kind = "plain" if chunks > 1 or n < 8 or n % 8 == 0 else "odd"
    return kind, lanes, chunks, groups, grid, grid


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("rows,n", GEOMETRIES)
def test_layer_norm_of_every_geometry(pkg, dev, rows, n, dtype):
    """Plain and fused, both ways, with dh and the weights' gradients, against 64 bits."""
    dt, p, seed = DT[dtype], 0.2, (SEED, 9)
    print(f"[norm] geometry rows={rows} n={n} {dtype}", flush=True)
    x, res, dy, dh = (_x((rows, n), dt, dev, 400 + i, 0.1) for i in range(4))
    w, b = _w(n, dt, dev, 404)
    y, mean, rstd = pkg.layer_norm_forward(x, w, b, EPS)
    plain = pkg.layer_norm_backward(dy, x, w, mean, rstd)
    y2, h, mean2, rstd2 = pkg.dropout_add_layer_norm_forward(x, res, w, b, p, seed, EPS)
    fused = pkg.dropout_add_layer_norm_backward(dy, dh, h, w, mean2, rstd2, p, seed)
    torch.cuda.synchronize()
    ref = R.Norm64(x, w, b, EPS)
    R.assert_within(y, ref.y, ref.bound_y(dt), "y")
    refs, bounds, _ = ref.grads(dy, dt, dt)
    for got, r, bound, name in zip(plain, refs, bounds, ("dx", "dw", "db")):
        R.assert_within(got, r, bound, name)
    d64, mask = R.drop64(x, p, *seed)
    h64 = res.double().cpu() + d64
    e = 3 * R.U * (d64.abs() + res.double().cpu().abs())
    R.assert_within(h, h64, R.half_step(dt) * (h64.abs() + e) + e + R.smallest(dt), "h")
    ref = R.Norm64(h, w, b, EPS)
    R.assert_within(y2, ref.y, ref.bound_y(dt), "fused y")
    (rd, rdw, rdb), (bd, bw, bb), e_d = ref.grads(dy, dt, dt, dh=dh)
    R.assert_within(fused[1], rd, bd, "dresidual")
    rdx = rd * mask
    e = e_d * mask + 2 * R.U * rdx.abs()
    R.assert_within(fused[0], rdx, R.half_step(dt) * (rdx.abs() + e) + e + R.smallest(dt), "fused dx")
    R.assert_within(fused[2], rdw, bw, "fused dw")
    R.assert_within(fused[3], rdb, bb, "fused db")


def test_layer_norm_without_weights_and_mixed_types(pkg, dev):
    x = _x((9, 300), torch.float16, dev, 11)
    dy = _x((9, 300), torch.float16, dev, 12, 0.0)
    w, b = _w(300, torch.bfloat16, dev, 13)
    for ww, bb in ((None, None), (w, None), (None, b), (w, b)):
        y, mean, rstd = pkg.layer_norm_forward(x, ww, bb, EPS)
        dx, dw, db = pkg.layer_norm_backward(dy, x, ww, mean, rstd)
        ref = R.Norm64(x, ww, bb, EPS)
        R.assert_within(y, ref.y, ref.bound_y(torch.float16), "y")
        wt = torch.float32 if ww is None else torch.bfloat16
        assert dw.dtype == wt and db.dtype == wt
        refs, bounds, _ = ref.grads(dy, torch.float16, wt)
        for got, r, bound in zip((dx, dw, db), refs, bounds):
            R.assert_within(got, r, bound, "grad")


def test_layer_norm_variance_of_a_large_offset(pkg, dev):
    """Rows of 1000 + noise in fp32: a variance from the difference of squared sums would lose all digits."""
    x = (1000 + torch.randn(7, 4096, generator=_gen(1))).to(dev)
    y, mean, rstd = pkg.layer_norm_forward(x, None, None, EPS)
    ref = R.Norm64(x, None, None, EPS)
    R.assert_within(y, ref.y, ref.bound_y(torch.float32), "y")
    # a constant row: deviations are zero or the mean's rounding, y is at most that over sqrt(eps)
    y, _, rstd = pkg.layer_norm_forward(torch.full((3, 1000), 7.0, device=dev), None, None, EPS)
    assert float(y.abs().max()) <= 64 * R.U * 7 / EPS ** 0.5
    assert torch.isfinite(rstd).all()


def test_layer_norm_not_finite_rows_stay_apart(pkg, dev):
    x = _x((6, 500), torch.float32, dev, 3)
    clean, _, _ = pkg.layer_norm_forward(x, None, None, EPS)
    x[1, 7] = float("nan")
    x[4, 499] = float("inf")
    y, _, _ = pkg.layer_norm_forward(x, None, None, EPS)
    assert torch.isnan(y[1]).all() and torch.isnan(y[4]).all()
    keep = [0, 2, 3, 5]
    assert torch.equal(y[keep], clean[keep])


def test_layer_norm_strides_and_empty(pkg, dev):
    base = _x((40, 1000), torch.bfloat16, dev, 21)
    w, b = _w(333, torch.bfloat16, dev, 22)
    x = base[3:, 5:338]  # rows 1000 apart, starting off alignment
    y, mean, rstd = pkg.layer_norm_forward(x, w, b, EPS)
    y2, mean2, rstd2 = pkg.layer_norm_forward(x.contiguous(), w, b, EPS)
    assert torch.equal(_bits(y), _bits(y2)) and torch.equal(mean, mean2)
    # a broadcast gradient (stride 0 over the rows, over everything) and a transposed one
    for dy in (base[0, 5:338].expand(37, 333), torch.ones((), dtype=torch.bfloat16, device=dev).expand(37, 333),
               base[:333, :37].T if base.shape[0] >= 333 else _x((333, 37), torch.bfloat16, dev, 23).T):
        got = pkg.layer_norm_backward(dy, x, w, mean, rstd)
        exp = pkg.layer_norm_backward(dy.contiguous(), x.contiguous(), w, mean, rstd)
        for g, e in zip(got, exp):
            assert torch.equal(_bits(g), _bits(e))
    # 3-D, and the neighbours of a strided view stay as they are
    x3 = _x((4, 5, 96), torch.float32, dev, 24)
    y3, m3, r3 = pkg.layer_norm_forward(x3.transpose(0, 1), None, None, EPS)
    assert y3.shape == (5, 4, 96) and m3.shape == (5, 4) and y3.is_contiguous()
    R.assert_within(y3, R.Norm64(x3.transpose(0, 1), None, None, EPS).y,
                    R.Norm64(x3.transpose(0, 1), None, None, EPS).bound_y(torch.float32), "y3")
    e = torch.empty(0, 333, dtype=torch.bfloat16, device=dev)
    y, mean, rstd = pkg.layer_norm_forward(e, w, b, EPS)
    dx, dw, db = pkg.layer_norm_backward(e, e, w, mean, rstd)
    assert y.shape == (0, 333) and dx.shape == (0, 333) and not dw.any() and not db.any()


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("n", [1, 5, 9, 77, 333, 1001, 5003, 9001])
def test_rows_of_a_buffer_of_nans(pkg, dev, n, dtype):
    """Rows that end inside a chunk, with NaN and infinity right behind them (and behind the last): nothing of it shows."""
    dt = DT[dtype]
    print(f"[norm] nans n={n} {dtype}", flush=True)

    def view(seed, pad):
        buf = torch.full((20, n + pad), float("nan"), dtype=dt, device=dev)
        buf[:, n:] = torch.tensor([float("inf"), float("nan"), float("-inf")] * 5, dtype=dt, device=dev)[:pad]
        buf[1:18, :n] = _x((17, n), dt, dev, seed)
        return buf, buf[1:18, :n]

    (bx, x), (br, res), (by, dy), (bh, dh) = (view(200 + i, p) for i, p in enumerate((1, 3, 7, 13)))
    kept = [t.clone() for t in (bx, br, by, bh)]
    w, b = _w(n, dt, dev, 205)
    c = [t.contiguous() for t in (x, res, dy, dh)]

    def run(x, res, dy, dh):
        y, mean, rstd = pkg.layer_norm_forward(x, w, b)
        y2, h, m2, r2 = pkg.dropout_add_layer_norm_forward(x, res, w, b, 0.2, (SEED, 1))
        return (y, mean, rstd, *pkg.layer_norm_backward(dy, x, w, mean, rstd), y2, h, m2, r2,
                *pkg.dropout_add_layer_norm_backward(dy, dh, h, w, m2, r2, 0.2, (SEED, 1)),
                pkg.dropout(x, 0.2, 3), pkg.dropout(x, 0.2, 3, residual=res), pkg.mxfp4_quantize(x).codes)

    for got, want in zip(run(x, res, dy, dh), run(*c)):
        assert torch.isfinite(got.float()).all() and torch.equal(got, want)
    # the same where h, whose rows the backward pass reads, is such a view
    _, mean, rstd = pkg.layer_norm_forward(x, w, b)
    for got, want in zip(pkg.dropout_add_layer_norm_backward(dy, dh, x, w, mean, rstd, 0.2, 9),
                         pkg.dropout_add_layer_norm_backward(c[2], c[3], c[0], w, mean, rstd, 0.2, 9)):
        assert torch.equal(got, want)
    for t, k in zip((bx, br, by, bh), kept):
        assert torch.equal(_bits(t), _bits(k))


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("n", [4, 12, 256, 300, 1000, 1003, 5003, 9001, 16387])
def test_layer_norm_backward_of_large_means(pkg, dev, n, dtype):
    """Rows of 2^96 with a mean of that and a reciprocal deviation of 2^33: every z is 0, while (0 - mean) rstd of a place
    past the row's end overflows.  dx = rstd (g - mean(g)), dw = 0."""
    dt = DT[dtype]
    print(f"[norm] large means n={n} {dtype}", flush=True)
    rows = 5
    x = torch.full((rows, n), 2.0 ** 96, dtype=dt, device=dev)
    dy = _x((rows, n), dt, dev, 300 + n, 0.1)
    mean, rstd = torch.full((rows,), 2.0 ** 96, device=dev), torch.full((rows,), 2.0 ** 33, device=dev)
    g = dy.double().cpu()
    ref = 2.0 ** 33 * (g - g.mean(-1, keepdim=True))
    # the sum's roundings and the division's, the two terms' difference; the factor is a power of two
    adds = R.Norm64(x[:1], None, None, EPS).adds
    e = 2.0 ** 33 * R.U * ((adds + 4) * g.abs().mean(-1, keepdim=True) + 4 * g.abs())
    bound = R.half_step(dt) * (ref.abs() + e) + e
    dx, dw, db = pkg.layer_norm_backward(dy, x, None, mean, rstd)
    R.assert_within(dx, ref, bound, "dx")
    assert not dw.any()
    R.assert_within(db, g.sum(0), (rows + 8) * R.U * g.abs().sum(0), "db")
    dx2, dres, dw, _ = pkg.dropout_add_layer_norm_backward(dy, None, x, None, mean, rstd, 0.0, 0)
    R.assert_within(dres, ref, bound, "dresidual")
    assert not dw.any()


# ---------------------------------------------------------------- dropout
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("shape", [(1, 1), (1, 7), (5, 8), (3, 9), (33, 1001), (2, 3, 77), (7, 4096), (2, 20000)])
def test_dropout(pkg, dev, shape, dtype):
    dt = DT[dtype]
    x, res = _x(shape, dt, dev, 31), _x(shape, dt, dev, 32)
    for p in (0.0, 0.1, 0.5, 1.0):
        y = pkg.dropout(x, p, (SEED, OFFSET))
        yr = pkg.dropout(x, p, (SEED, OFFSET), residual=res)
        ref, _ = R.drop64(x, p, SEED, OFFSET)
        # one rounding of the product in fp32, one of the scale, the output's
        e = 2 * R.U * ref.abs()
        R.assert_within(y, ref, R.half_step(dt) * ref.abs() * (1 + 2 * R.U) + e + R.smallest(dt), f"p={p}")
        assert torch.equal(y.cpu() == 0, (ref == 0)), "mask"
        r64 = res.double().cpu() + ref
        e = e + R.U * (ref.abs() + res.double().cpu().abs())
        R.assert_within(yr, r64, R.half_step(dt) * (r64.abs() + e) + e + R.smallest(dt), f"p={p} residual")


def test_dropout_generator_is_the_published_one():
    """The oracle's generator gives the published known answers of Philox4x32-10 (counter and key all zeros, all ones)."""
    zero = R.philox([[0]] * 4, (0, 0))
    assert [int(w[0]) for w in zero] == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    ones = R.philox([[0xFFFFFFFF]] * 4, (0xFFFFFFFF, 0xFFFFFFFF))
    assert [int(w[0]) for w in ones] == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]


def test_dropout_rate_and_independence(pkg, dev):
    """The kept share of 2^22 draws is within 6 standard deviations; other seeds and offsets give other masks, which
    agree as often as independent ones do."""
    x = torch.ones(1024, 4096, device=dev)
    n = x.numel()
    keep = 1 - round(65536 * 0.1) / 65536
    masks = [pkg.dropout(x, 0.1, s) != 0 for s in (1, 2, (1, 1), (1, 1 << 32), 1 << 32)]
    for m in masks:
        assert abs(float(m.double().mean()) - keep) <= 6 * (keep * (1 - keep) / n) ** 0.5
    agree = keep * keep + (1 - keep) ** 2
    for i in range(len(masks)):
        for j in range(i):
            share = float((masks[i] == masks[j]).double().mean())
            assert abs(share - agree) <= 6 * (agree * (1 - agree) / n) ** 0.5, (i, j, share)


def test_dropout_drops_what_is_not_finite(pkg, dev):
    x = torch.full((64, 64), float("nan"), device=dev)
    x[::2] = float("inf")
    y = pkg.dropout(x, 0.5, SEED)
    k = R.kept(64, 64, 32768, SEED, 0).to(dev)
    assert not y[~k].any() and not torch.isfinite(y[k]).any()
    assert not pkg.dropout(x, 1.0, SEED).any()


def test_dropout_strides_offsets_and_tensor_seed(pkg, dev):
    base = _x((20, 700), torch.bfloat16, dev, 41)
    x = base[1:18, 3:500]
    want = pkg.dropout(x.contiguous(), 0.2, (SEED, 5))
    assert torch.equal(_bits(pkg.dropout(x, 0.2, (SEED, 5))), _bits(want))
    state = torch.tensor([SEED, 2], dtype=torch.int64, device=dev)
    assert torch.equal(_bits(pkg.dropout(x, 0.2, (state, 3))), _bits(want))
    state[1] = 5
    assert torch.equal(_bits(pkg.dropout(x, 0.2, state)), _bits(want))
    # negative seeds are the same 64 bits
    assert torch.equal(pkg.dropout(x, 0.2, -1), pkg.dropout(x, 0.2, (1 << 64) - 1))
    assert pkg.dropout(x[:0], 0.2, 1).shape == (0, 497)
    assert pkg.dropout(x[:, :0], 0.2, 1).shape == (17, 0)


def test_dropout_past_32_bits(pkg, dev):
    """2^31 + elements (offsets past 2^32 bytes): the last rows against the oracle."""
    rows, n = 524300, 4104
    x = torch.ones(rows, n, dtype=torch.bfloat16, device=dev)
    y = pkg.dropout(x, 0.5, (SEED, OFFSET))
    for first in (0, rows // 2, rows - 3):
        k = R.kept(3, n, 32768, SEED, OFFSET, first)
        assert torch.equal(y[first:first + 3].cpu() != 0, k)
    del x, y


# ---------------------------------------------------------------- dropout + add + norm
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("rows,n", [(1, 1), (3, 13), (65, 1000), (130, 1024), (19, 4096), (40, 5120), (6, 9001), (3, 18000)])
def test_dropout_add_layer_norm(pkg, dev, rows, n, dtype):
    dt = DT[dtype]
    p = 0.1
    print(f"[add_norm] rows={rows} n={n} {dtype}", flush=True)
    x, res = _x((rows, n), dt, dev, 51), _x((rows, n), dt, dev, 52)
    w, b = _w(n, dt, dev, 53)
    dy, dh = _x((rows, n), dt, dev, 54, 0.0), _x((rows, n), dt, dev, 55, 0.0)
    y, h, mean, rstd = pkg.dropout_add_layer_norm_forward(x, res, w, b, p, (SEED, OFFSET), EPS)
    dx, dres, dw, db = pkg.dropout_add_layer_norm_backward(dy, dh, h, w, mean, rstd, p, (SEED, OFFSET))
    torch.cuda.synchronize()
    d64, mask = R.drop64(x, p, SEED, OFFSET)
    h64 = res.double().cpu() + d64
    e = 3 * R.U * (d64.abs() + res.double().cpu().abs())
    R.assert_within(h, h64, R.half_step(dt) * (h64.abs() + e) + e + R.smallest(dt), "h")
    ref = R.Norm64(h, w, b, EPS)  # the norm is that of h as stored
    R.assert_within(y, ref.y, ref.bound_y(dt), "y")
    (rd, rdw, rdb), (bd, bw, bb), e_d = ref.grads(dy, dt, dt, dh=dh)
    R.assert_within(dres, rd, bd, "dresidual")
    rdx = rd * mask
    e = e_d * mask + 2 * R.U * rdx.abs()
    R.assert_within(dx, rdx, R.half_step(dt) * (rdx.abs() + e) + e + R.smallest(dt), "dx")
    assert torch.equal((dx.cpu() == 0) | (rdx == 0), dx.cpu() == 0), "dropped gradients are zero"
    R.assert_within(dw, rdw, bw, "dw")
    R.assert_within(db, rdb, bb, "db")
    # without dh, without dropout, without a residual
    dx0, dres0, _, _ = pkg.dropout_add_layer_norm_backward(dy, None, h, w, mean, rstd, 0.0, 0)
    plain, _, _ = pkg.layer_norm_backward(dy, h, w, mean, rstd)
    assert dx0 is dres0 and torch.equal(_bits(dx0), _bits(plain))
    y1, h1, _, _ = pkg.dropout_add_layer_norm_forward(x, None, w, b, 0.0, 0, EPS)
    yp, _, _ = pkg.layer_norm_forward(x, w, b, EPS)
    assert torch.equal(_bits(h1), _bits(x)) and torch.equal(_bits(y1), _bits(yp))


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("rows,n", [(5000, 100), (2100, 512), (3000, 1000), (1100, 5120), (600, 9001), (520, 12000), (530, 17000)])
def test_dropout_add_layer_norm_many_rows(pkg, dev, rows, n, dtype):
    """More rows than row groups run at once, with dropout, dh and the weights' gradients, which the groups' sums must
    make up whole; twice the same call gives the same bits."""
    dt, p, seed = DT[dtype], 0.2, (SEED, 7)
    print(f"[add_norm] rows={rows} n={n} {dtype}", flush=True)
    x, res, dy, dh = (_x((rows, n), dt, dev, 100 + i, 0.1) for i in range(4))
    w, b = _w(n, torch.float32, dev, 104)
    y, h, mean, rstd = pkg.dropout_add_layer_norm_forward(x, res, w, b, p, seed, EPS)
    got = pkg.dropout_add_layer_norm_backward(dy, dh, h, w, mean, rstd, p, seed)
    again = pkg.dropout_add_layer_norm_backward(dy, dh, h, w, mean, rstd, p, seed)
    torch.cuda.synchronize()
    for g, e in zip(got, again):
        assert torch.equal(_bits(g), _bits(e))
    ref = R.Norm64(h, w, b, EPS)
    R.assert_within(y, ref.y, ref.bound_y(dt), "y")
    (rd, rdw, rdb), (bd, bw, bb), e_d = ref.grads(dy, dt, torch.float32, dh=dh)
    _, mask = R.drop64(x, p, *seed)
    R.assert_within(got[1], rd, bd, "dresidual")
    rdx = rd * mask
    e = e_d * mask + 2 * R.U * rdx.abs()
    R.assert_within(got[0], rdx, R.half_step(dt) * (rdx.abs() + e) + e + R.smallest(dt), "dx")
    R.assert_within(got[2], rdw, bw, "dw")
    R.assert_within(got[3], rdb, bb, "db")


def test_layer_norm_past_32_bits(pkg, dev):
    """2^31 + elements (offsets past 2^32 bytes): the last rows are those of the same rows alone, both ways."""
    rows, n = 524300, 4104
    x = torch.zeros(rows, n, dtype=torch.bfloat16, device=dev)
    tail = _x((3, n), torch.bfloat16, dev, 131)
    x[-3:] = tail
    w, b = _w(n, torch.bfloat16, dev, 132)
    y, mean, rstd = pkg.layer_norm_forward(x, w, b, EPS)
    yt, mt, rt = pkg.layer_norm_forward(tail, w, b, EPS)
    assert torch.equal(_bits(y[-3:]), _bits(yt)) and torch.equal(mean[-3:], mt) and torch.equal(rstd[-3:], rt)
    dx, dw, db = pkg.layer_norm_backward(y, x, w, mean, rstd)
    dt, _, _ = pkg.layer_norm_backward(yt, tail, w, mt, rt)
    assert torch.equal(_bits(dx[-3:]), _bits(dt)) and torch.isfinite(dw).all() and torch.isfinite(db).all()
    del x, y, dx


def test_dropout_in_place(pkg, dev):
    """out may be x or the residual."""
    import ctypes
    L = importlib.import_module("triton-kernel-test_amd._lib")
    x, res = _x((70, 1001), torch.bfloat16, dev, 141), _x((70, 1001), torch.bfloat16, dev, 142)
    want = pkg.dropout(x, 0.25, SEED, residual=res)
    drop = L.LrqDropout(49152, SEED, 0, None)
    stream = torch.cuda.current_stream().cuda_stream
    for over in (0, 1):
        a, r = x.clone(), res.clone()
        out = (a, r)[over]
        L.call("lrq_dropout_add", ctypes.byref(drop), a.data_ptr(), 1001, r.data_ptr(), 1001, L.LRQ_BF16, 70, 1001,
               out.data_ptr(), 1001, stream)
        assert torch.equal(_bits(out), _bits(want))


def test_layer_norm_under_compressed_saved_tensors(pkg, dev):
    """The layer's input is kept compressed and decoded for its gradients."""
    AG = importlib.import_module("triton-kernel-test_amd.autograd")
    x = _x((64, 512), torch.bfloat16, dev, 151).requires_grad_()
    w, b = (t.requires_grad_() for t in _w(512, torch.float32, dev, 152))
    dy = _x((64, 512), torch.bfloat16, dev, 153, 0.0)
    hooks = AG.compressed_saved_tensors(bits=8, group=64, min_numel=1)
    with hooks:
        y = AG.layer_norm(x * 1, w, b)  # (leaves are kept as they are)
    assert hooks.stats["compressed"] == 1
    y.backward(dy)
    _, mean, rstd = pkg.layer_norm_forward(x.detach(), w.detach(), b.detach())

    def kept(t):
        return pkg.decode(pkg.encode(t.detach(), None, bits=8, group_size=64))

    for got, want in zip((x.grad, w.grad, b.grad), pkg.layer_norm_backward(dy, kept(x), w.detach(), mean, rstd)):
        assert torch.equal(got, want)
    # the fused form keeps h, one of its outputs
    x.grad = w.grad = b.grad = None
    hooks = AG.compressed_saved_tensors(bits=8, group=64, min_numel=1)
    with hooks:
        y, h = AG.dropout_add_layer_norm(x, x.detach(), w, b, 0.3, 8)
    assert hooks.stats["compressed"] == 1
    torch.autograd.backward([y, h], [dy, dy])
    _, hh, mean, rstd = pkg.dropout_add_layer_norm_forward(x.detach(), x.detach(), w.detach(), b.detach(), 0.3, 8)
    dx, _, dw, db = pkg.dropout_add_layer_norm_backward(dy, dy, kept(hh), w.detach(), mean, rstd, 0.3, 8)
    for got, want in zip((x.grad, w.grad, b.grad), (dx, dw, db)):
        assert torch.equal(got, want)


def test_gradients_against_differences(pkg, dev):
    """The gradient of sum(dy y + dh h) along random directions, against central differences of the oracle's 64-bit
    forward pass (the mask fixed): truncation is O(step^2), the rest is the fp32 kernel's."""
    AG = importlib.import_module("triton-kernel-test_amd.autograd")
    g = _gen(61)
    rows, n, p = 5, 40, 0.25
    x, res = (torch.randn(rows, n, generator=g).to(dev).requires_grad_() for _ in range(2))
    w, b = (t.requires_grad_() for t in _w(n, torch.float32, dev, 62))
    cy, ch = torch.randn(rows, n, generator=g).double(), torch.randn(rows, n, generator=g).double()
    y, h = AG.dropout_add_layer_norm(x, res, w, b, p, 77, EPS)
    (y * cy.float().to(dev) + h * ch.float().to(dev)).sum().backward()

    def loss(x_, r_, w_, b_):
        d, _ = R.drop64(x_, p, 77)
        h_ = r_ + d
        m = h_.mean(-1, keepdim=True)
        z = (h_ - m) / torch.sqrt(((h_ - m) ** 2).mean(-1, keepdim=True) + EPS)
        return float(((z * w_ + b_) * cy + h_ * ch).sum())

    at = [t.detach().double().cpu() for t in (x, res, w, b)]
    for i, t in enumerate((x, res, w, b)):
        for _ in range(3):
            v = torch.randn(at[i].shape, generator=g).double()
            step = 1e-5
            up = [a + (step * v if k == i else 0) for k, a in enumerate(at)]
            dn = [a - (step * v if k == i else 0) for k, a in enumerate(at)]
            diff = (loss(*up) - loss(*dn)) / (2 * step)
            got = float((t.grad.double().cpu() * v).sum())
            scale = float((t.grad.double().cpu().abs() * v.abs()).sum())
            # 1e-5 of the terms: fp32 gradients (about 200 U), differences (1e-16 * loss / 1e-5, and step^2)
            assert abs(got - diff) <= 2e-5 * scale, (i, got, diff)


# ---------------------------------------------------------------- autograd, streams, graphs
def test_autograd_layer_norm_and_dropout(pkg, dev):
    AG = importlib.import_module("triton-kernel-test_amd.autograd")
    x = _x((4, 6, 256), torch.bfloat16, dev, 71).requires_grad_()
    w, b = (t.requires_grad_() for t in _w(256, torch.bfloat16, dev, 72))
    y = AG.layer_norm(x, w, b)
    z = AG.dropout(y, 0.3, (9, 1), residual=x)
    z.float().sum().backward()  # a broadcast gradient
    dz = torch.ones_like(z)
    dyd = pkg.dropout(dz, 0.3, (9, 1))
    _, mean, rstd = pkg.layer_norm_forward(x.detach(), w.detach(), b.detach())
    dx, dw, db = pkg.layer_norm_backward(dyd, x.detach(), w.detach(), mean, rstd)
    assert torch.equal(w.grad, dw) and torch.equal(b.grad, db)
    assert torch.equal(x.grad, dx + dz)
    # frozen weights, no bias
    x2 = x.detach().requires_grad_()
    AG.layer_norm(x2, w.detach(), None).backward(torch.ones_like(x2))
    assert x2.grad is not None
    # evaluation: dropout is the identity plus the residual
    assert AG.dropout(y, 0.3, 9, training=False) is y
    with pytest.raises(RuntimeError):
        gx, = torch.autograd.grad(AG.layer_norm(x2, None, None).sum(), x2, create_graph=True)
        gx.sum().backward()


def test_autograd_state_changed_before_backward_is_refused(pkg, dev):
    AG = importlib.import_module("triton-kernel-test_amd.autograd")
    state = torch.tensor([3, 0], dtype=torch.int64, device=dev)
    x = _x((8, 64), torch.float32, dev, 73).requires_grad_()
    y = AG.dropout(x, 0.5, state)
    state[1] += 1
    with pytest.raises(RuntimeError):
        y.sum().backward()


def test_side_stream(pkg, dev):
    x = _x((300, 1024), torch.bfloat16, dev, 81)
    w, b = _w(1024, torch.bfloat16, dev, 82)
    want = pkg.layer_norm_forward(x, w, b)
    grads = pkg.layer_norm_backward(x, x, w, want[1], want[2])
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = pkg.layer_norm_forward(x, w, b)
        g2 = pkg.layer_norm_backward(x, x, w, got[1], got[2])
        d = pkg.dropout(x, 0.5, 4)
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    for a, e in zip((*got, *g2, d), (*want, *grads, pkg.dropout(x, 0.5, 4))):
        assert torch.equal(a, e)


def test_captured_graphs_draw_new_masks(pkg, dev):
    """Two captured graphs of the fused pass over one seed tensor, replayed in turn with eager work between: every
    replay equals the eager call at the tensor's value."""
    x, res = _x((70, 1000), torch.bfloat16, dev, 91), _x((70, 1000), torch.bfloat16, dev, 92)
    w, b = _w(1000, torch.bfloat16, dev, 93)
    state = torch.tensor([11, 0], dtype=torch.int64, device=dev)

    def step(offset):
        y, h, mean, rstd = pkg.dropout_add_layer_norm_forward(x, res, w, b, 0.2, (state, offset))
        return (y, h, *pkg.dropout_add_layer_norm_backward(x, res, h, w, mean, rstd, 0.2, (state, offset)))

    step(0)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for offset in (0, 100):
        g = torch.cuda.CUDAGraph()
        print("[norm] capture", flush=True)
        with torch.cuda.graph(g):
            outs.append(step(offset))
        graphs.append(g)
    seen = []
    for i in range(3):
        state[1] = i
        for k, offset in enumerate((0, 100)):
            graphs[k].replay()
        torch.cuda.synchronize()
        for k, offset in enumerate((0, 100)):
            for got, want in zip(outs[k], step(offset)):
                assert torch.equal(_bits(got), _bits(want)), (i, k)
            seen.append(outs[k][1].clone())
    for i in range(len(seen)):
        for j in range(i):
            assert not torch.equal(seen[i], seen[j])


def test_fused_norm_without_weights_and_one_dimensional(pkg, dev):
    """The fused pass normalises h as the plain one does, whatever weights there are; one-dimensional operands."""
    x, res = _x((21, 700), torch.bfloat16, dev, 161), _x((21, 700), torch.bfloat16, dev, 162)
    dy = _x((21, 700), torch.bfloat16, dev, 163, 0.0)
    for wdt in (torch.bfloat16, torch.float16):
        w, b = _w(700, wdt, dev, 164)
        for ww, bb in ((None, None), (w, None), (None, b), (w, b)):
            y, h, mean, rstd = pkg.dropout_add_layer_norm_forward(x, res, ww, bb, 0.3, 5)
            yp, mp, rp = pkg.layer_norm_forward(h, ww, bb)
            assert torch.equal(_bits(y), _bits(yp)) and torch.equal(mean, mp) and torch.equal(rstd, rp)
            got = pkg.dropout_add_layer_norm_backward(dy, None, h, ww, mean, rstd, 0.3, 5)
            want = pkg.layer_norm_backward(dy, h, ww, mean, rstd)
            for g, e in zip(got[1:], want):
                assert torch.equal(g, e)
    y1, m1, r1 = pkg.layer_norm_forward(x[3], None, None)
    y2, m2, r2 = pkg.layer_norm_forward(x[3:4], None, None)
    assert m1.shape == () and torch.equal(y1, y2[0]) and torch.equal(m1, m2[0])
    dx, dw, db = pkg.layer_norm_backward(dy[3], x[3], None, m1, r1)
    assert torch.equal(dx, pkg.layer_norm_backward(dy[3:4], x[3:4], None, m2, r2)[0][0]) and dw.shape == (700,)
    assert torch.equal(pkg.dropout(x[3], 0.3, 9), pkg.dropout(x[3:4], 0.3, 9)[0])
    assert pkg.dropout(x[3, 3], 1.0, 9).shape == () and not pkg.dropout(x[3, 3], 1.0, 9).any()


def test_two_streams_at_once(pkg, dev):
    x = [_x((3000, 1024), torch.bfloat16, dev, 171 + i) for i in range(2)]
    w, b = _w(1024, torch.bfloat16, dev, 173)

    def step(i):
        y, h, mean, rstd = pkg.dropout_add_layer_norm_forward(x[i], x[1 - i], w, b, 0.1, (6, i))
        return (y, *pkg.dropout_add_layer_norm_backward(x[i], h, h, w, mean, rstd, 0.1, (6, i)))

    want = [step(0), step(1)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(step(i))
    torch.cuda.synchronize()
    for i in range(2):
        for g in got[i]:
            for a, e in zip(g, want[i]):
                assert torch.equal(a, e)


def test_captured_training_step(pkg, dev):
    """Forward and backward of the block captured whole: every replay equals the eager step at the seed tensor's value."""
    AG = importlib.import_module("triton-kernel-test_amd.autograd")
    x, res = (_x((70, 256), torch.bfloat16, dev, 181 + i).requires_grad_() for i in range(2))
    w, b = (t.requires_grad_() for t in _w(256, torch.bfloat16, dev, 183))
    q = pkg.mxfp4_quantize(_x((128, 256), torch.bfloat16, dev, 184))
    dy, dh = _x((70, 128), torch.bfloat16, dev, 185, 0.0), _x((70, 256), torch.bfloat16, dev, 186, 0.0)
    state = torch.tensor([3, 0], dtype=torch.int64, device=dev)
    leaves = (x, res, w, b)

    def step():
        y, h = AG.dropout_add_layer_norm(x, res, w, b, 0.2, (state, 1))
        return torch.autograd.grad([AG.mxfp4_linear(y, q), h], leaves, [dy, dh])

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    print("[norm] capture", flush=True)
    with torch.cuda.graph(graph):
        outs = step()
    for i in range(3):
        state[1] = i
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in outs]
        y, h, mean, rstd = pkg.dropout_add_layer_norm_forward(x.detach(), res.detach(), w.detach(), b.detach(), 0.2,
                                                              (state, 1))
        g = pkg.mxfp4_linear_backward(dy, q)
        want = pkg.dropout_add_layer_norm_backward(g, dh, h, w.detach(), mean, rstd, 0.2, (state, 1))
        for a, e in zip(got, want):
            assert torch.equal(a, e), i
