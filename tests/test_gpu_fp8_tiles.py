"""The 8-bit products' kernels at the lengths that they are used at: every tile over a contraction that its ring of steps, both
places of the scales and its splits go round in, the few-row kernel in all its widths, and every output type of each."""

import pytest
import torch

import opref8 as R
from opref import assert_within

pytestmark = pytest.mark.gpu
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32
F8 = torch.float8_e4m3fn

# tile (64 rows by 64 columns times these), whether its contraction is split, rows, depth, columns: ragged in all three.
# tests/test_fp8_plan.py holds that each comes to its tile, either way, and how many steps a split has.
TILES = [((1, 1), False, 60, 1283, 201), ((1, 1), True, 60, 6001, 201), ((1, 2), False, 1003, 1283, 1031),
         ((1, 2), True, 130, 12001, 2049), ((1, 4), False, 260, 1283, 11003), ((1, 4), True, 130, 7001, 3001),
         ((2, 2), False, 1003, 1283, 2049), ((2, 2), True, 1003, 6001, 1031), ((2, 4), False, 1031, 1283, 4101),
         ((2, 4), True, 1301, 9001, 1501), ((3, 4), False, 1301, 1283, 6001), ((3, 4), True, 1301, 20001, 1501),
         ((4, 4), False, 1003, 1283, 11003), ((4, 4), True, 1003, 12001, 4101)]
NAMES = [f"{64 * t[0]}x{64 * t[1]}{'-split' if s else ''}" for t, s, *_ in TILES]
# rows of e4m3, depth, weight rows of the few-row kernel: one and two tiles of weight rows a wave in workgroups of 16 waves, two in
# workgroups of 8, one and two tiles of rows; fewer steps than waves, and several for each
FEW = [(1, 300, 4090), (16, 5000, 4100), (3, 9000, 8190), (1, 1411, 8200), (16, 4700, 14341), (5, 1411, 33001), (17, 1411, 4090),
       (32, 5000, 4090), (21, 1411, 4100), (32, 5100, 8190)]
# the same of 16-bit rows, which are whole 16-byte pieces
FEW_16 = [(1, 1408, 4090), (4, 1408, 4100), (3, 9000, 8190), (1, 1408, 8200), (4, 4704, 14341), (2, 1408, 33001)]


def _integers(pkg, rows, cols, block, seed, deep):
    """Whole numbers of -3 to 3, no block's scale like its neighbours': 2^-2 to 2^2 (2^-1 to 2^1 in deep contractions)."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    steps, wide = -(-cols // 128), 1 if deep else 2
    c = torch.zeros(rows, 128 * steps, device="cuda")
    c[:, :cols] = torch.randint(-3, 4, (rows, cols), generator=g, device="cuda").float()
    s = torch.randint(127 - wide, 128 + wide, (-(-rows // block), -(-steps // 4) * 4), generator=g, device="cuda")
    return pkg.FP8Tensor(c.to(F8), s.to(torch.uint8), (rows, cols), block)


def _values(q):
    """On the device; finite operands alone."""
    rows, cols = q.shape
    f = torch.exp2(q.scales.view(torch.uint8).double() - 127).repeat_interleave(q.block, 0)[:rows].repeat_interleave(128, 1)[:, :cols]
    return q.codes.view(F8)[:, :cols].double() * f


def _exact(a, b, deep):
    """a b^T of ``_integers``, in fp32: all its sums are multiples of 2^-4 (2^-2), at most 9 * 2^4 (2^2) of a product, and
    fewer than 2^24 such steps, so exact in any order."""
    assert a.shape[1] * 9 * (16 if deep else 256) < 1 << 24
    return a.float() @ b.float().T.contiguous()


def _random(pkg, rows, cols, block, seed):
    """Normal numbers, block scales apart by up to 2^8."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, cols, generator=g, device="cuda")
    for part in x.split(128, 1):
        part *= torch.exp2(torch.randint(-4, 5, (rows, 1), generator=g, device="cuda").float())
    return pkg.fp8_quantize(x, block)


def _check_exact(f, a, b, va, vb, deep):
    """f(a, b) against va vb^T: to the bit in fp32, and rounded once to the others."""
    want = _exact(va, vb, deep)
    for dtype in (F32, BF, F16):
        got = f(a, b, dtype)
        assert torch.equal(got, want.to(dtype)), (dtype, (got != want.to(dtype)).nonzero()[:5].tolist())


@pytest.mark.parametrize("nn", [False, True], ids=["xw", "dyw"])
@pytest.mark.parametrize("tile,split,m,depth,cols", TILES, ids=NAMES)
def test_every_step_meets_its_own(pkg, tile, split, m, depth, cols, nn):
    """Exact sums: each code and scale, of every step and split, has met its own partner, and every output its rounding."""
    deep = depth > 7000
    a = _integers(pkg, m, depth, 1, m, deep)
    b = _integers(pkg, *((depth, cols) if nn else (cols, depth)), 128, cols, deep)
    vb = _values(b)
    _check_exact(pkg.fp8_linear_backward if nn else pkg.fp8_gemm, a, b, _values(a), vb.T.contiguous() if nn else vb, deep)


@pytest.mark.parametrize("m,depth,cols", FEW)
def test_few_rows(pkg, m, depth, cols):
    """The same of the few-row kernel; random rows within the bound, and the same bits each time."""
    deep = depth > 7000
    a, b = _integers(pkg, m, depth, 1, m, deep), _integers(pkg, cols, depth, 128, cols, deep)
    _check_exact(pkg.fp8_gemm, a, b, _values(a), _values(b), deep)
    _check_random(pkg, pkg.fp8_gemm, _random(pkg, m, depth, 1, m), _random(pkg, cols, depth, 128, cols), False)


@pytest.mark.parametrize("dtype", [BF, F16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("m,depth,cols", FEW_16)
def test_few_16_bit_rows(pkg, m, depth, cols, dtype):
    """Quantised inside the few-row kernel: exact sums, and on random rows the bits of two calls."""
    deep = depth > 7000
    b = _integers(pkg, cols, depth, 128, cols, deep)
    x = _values(_integers(pkg, m, depth, 1, m, deep)).to(dtype)
    _check_exact(pkg.fp8_linear, x, b, x, _values(b), deep)
    g = torch.Generator(device="cuda").manual_seed(depth)
    x = torch.randn(m, depth, generator=g, device="cuda")
    x *= torch.exp2(torch.randint(-6, 7, (m, depth), generator=g, device="cuda").float())
    x, w = x.to(dtype), _random(pkg, cols, depth, 128, cols)
    for out in (F32, BF, F16):
        assert torch.equal(pkg.fp8_linear(x, w, out), pkg.fp8_gemm(pkg.fp8_quantize(x), w, out))


def _check_random(pkg, f, a, b, nn):
    outs = {t: f(a, b, t) for t in (F32, BF, F16)}
    for t, got in outs.items():
        for _ in range(2):
            assert torch.equal(f(a, b, t), got)
    ref, bound = R.product(_values(a), _values(b) if nn else _values(b).T, F32)
    assert_within(outs[F32], ref, bound, "fp32")
    for t in (BF, F16):  # the same sums, rounded once more
        assert torch.equal(outs[t], outs[F32].to(t))


@pytest.mark.parametrize("nn", [False, True], ids=["xw", "dyw"])
@pytest.mark.parametrize("tile,split,m,depth,cols", TILES, ids=NAMES)
def test_random_operands(pkg, tile, split, m, depth, cols, nn):
    """Within the bound of the instruction's window and the additions, and the same bits each time."""
    a, b = _random(pkg, m, depth, 1, m), _random(pkg, *((depth, cols) if nn else (cols, depth)), 128, cols)
    _check_random(pkg, pkg.fp8_linear_backward if nn else pkg.fp8_gemm, a, b, nn)


@pytest.mark.parametrize("m", [5, 64, 300])
def test_one_signed_operands(pkg, m):
    """Where all products have one sign, what the window cuts off adds up: still within its bound."""
    g = torch.Generator(device="cuda").manual_seed(m)
    a = pkg.fp8_quantize(torch.rand(m, 4096, generator=g, device="cuda") + 0.01)
    w = torch.rand(1000, 4096, generator=g, device="cuda") + 0.01
    _check_random(pkg, pkg.fp8_gemm, a, pkg.fp8_quantize(w, 128), False)
    _check_random(pkg, pkg.fp8_linear_backward, a, pkg.fp8_quantize(w.T, 128), True)
