"""The root-mean-square norm where its row groups walk several rows each: the next row's loads under the last one's sums, the two
places of the waves' sums, and the weight gradient's addition over rounds, against 64-bit forms."""

import pytest
import torch

import opref8 as R
from opref import assert_within

pytestmark = pytest.mark.gpu
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32
EPS = 1e-6

# rows, columns.  tests/test_rms_plan.py holds that every form takes three rounds of rows or more on some workgroup: 16 lanes, a
# wave and several waves a row, one, two and four chunks a thread, rows of whole chunks and rows that end inside one, several
# groups a workgroup and one, rows past the registers
SHAPES = [(33000, 100), (33000, 104), (8300, 333), (8300, 512), (8300, 1000), (8300, 1003), (4200, 1304), (4200, 1300), (4200, 2003),
          (4200, 2000), (2100, 4096), (1600, 5003), (1600, 5120), (1100, 8190), (1030, 9001), (1030, 9008), (1030, 16390)]


def _r(rows, n, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(7000 * rows + n + seed)
    return torch.randn(rows, n, generator=g, device="cuda").to(dtype)


def _w(n, dtype):
    return (1.0 + 0.1 * torch.randn(n, generator=torch.Generator().manual_seed(n + 9))).to(dtype).cuda()


def _twice(f):
    """What f returns; the same bits the second time."""
    one, two = f(), f()
    for a, b in zip(one, two):
        assert (a is None and b is None) or torch.equal(a, b)
    return one


@pytest.mark.parametrize("dtype", [BF, F16, F32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("rows,n", SHAPES)
def test_rounds(pkg, rows, n, dtype):
    x, res, dy, dh = (_r(rows, n, dtype, i) for i in range(4))
    w = _w(n, dtype)
    y, rstd = _twice(lambda: pkg.rms_norm_forward(x, w, EPS))
    ref = R.Rms64(x, w, EPS)
    assert_within(y, ref.y, ref.bound_y(dtype), "y")
    assert_within(rstd, ref.rstd[:, 0], ref.r_rstd * ref.rstd[:, 0], "rstd")
    (dx, dw), (bx, bw) = ref.grads(dy, dtype, dtype)
    gx, gw = _twice(lambda: pkg.rms_norm_backward(dy, x, w, rstd))
    assert_within(gx, dx, bx, "dx")
    assert_within(gw, dw, bw, "dw")
    y, h, rstd = _twice(lambda: pkg.add_rms_norm_forward(x, res, w, EPS))
    assert torch.equal(h, (x.float() + res.float()).to(dtype))
    ref = R.Rms64(h, w, EPS)
    assert_within(y, ref.y, ref.bound_y(dtype), "y of the sum")
    (dx, dw), (bx, bw) = ref.grads(dy, dtype, dtype, dh)
    gx, gw = _twice(lambda: pkg.rms_norm_backward(dy, h, w, rstd, dh))
    assert_within(gx, dx, bx, "dx of the sum")
    assert_within(gw, dw, bw, "dw of the sum")


@pytest.mark.parametrize("dtype", [BF, F16, F32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("rows,n", SHAPES)
def test_rounds_in_8_bits(pkg, rows, n, dtype):
    """The codes and scales of the same rows in parts of 37, which are one round each."""
    x, res, w = _r(rows, n, dtype, 0), _r(rows, n, dtype, 1), _w(n, dtype)
    steps = -(-n // 128)
    for add in (False, True):
        f = (lambda s: pkg.add_rms_norm_forward(x[s], res[s], w, EPS, fp8=True)) if add else \
            (lambda s: pkg.rms_norm_forward(x[s], w, EPS, fp8=True))
        q, *rest = f(slice(None))
        codes, scales = q.codes.view(torch.uint8), q.scales[:, :steps]
        for at in sorted({37 * i for i in range(0, rows // 37, max(1, rows // 37 // 40))} | {rows - 37}):
            s = slice(at, at + 37)
            part, *others = f(s)
            assert torch.equal(codes[s], part.codes.view(torch.uint8)) and torch.equal(scales[s], part.scales[:, :steps])
            assert all(torch.equal(a[s], b) for a, b in zip(rest, others))
        ref = R.Rms64(rest[0] if add else x, w, EPS)
        got = R.tensor_values(q)
        unit = torch.exp2(scales.cpu().double() - 127).repeat_interleave(128, 1)[:, :n]
        e = ref.e_y()
        # half a step of 2^-3 in its binade, or of the subnormal codes
        assert_within(got, ref.y, torch.maximum((ref.y.abs() + e) * 2.0 ** -4, 2.0 ** -10 * unit) + e, "values")
