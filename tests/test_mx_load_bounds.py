"""The direct global-to-LDS loads of the MXFP4 products, replayed in numpy from the launch arithmetic of
csrc/lrq_mxgemm.hip: every read lies in its operand, every LDS write in the part of the allocation it belongs to, and no two
loads of a step write the same bytes."""

import numpy as np
import pytest

LANE, WAVE = np.arange(64), np.arange(8)[:, None]  # [waves, lanes] below


def _plan(rows, cols, depth, per_row, times, fixed, least_steps):
    """The tile height's index and the splits that the host's cost model picks."""
    steps = -(-depth // 128)
    best = None
    for i, t in enumerate(times):
        tiles = -(-rows // (per_row << i)) * -(-cols // 256)
        for s in range(1, min(16, max(1, steps // least_steps)) + 1):
            cost = -(-tiles * s // 256) * fixed(-(-steps // s), t) + (4 + 2e-6 * s * rows * cols if s > 1 else 0)
            if best is None or cost < best[0]:
                best = (cost, 1 << i, s)
    return best[1], best[2]


def _inside(at, size, limit, what):
    assert at.min() >= 0 and at.max() + size <= limit, (what, int(at.min()), int(at.max()) + size, limit)


def _lds(dests, low, high, what):
    """Each load instruction of a wave writes 64 lanes' bytes from one base: bases and their size."""
    spans = sorted((int(b), int(b) + n) for b, n in dests)
    assert spans[0][0] >= low and spans[-1][1] <= high, what
    assert all(a[1] <= b[0] for a, b in zip(spans, spans[1:])), f"{what}: two loads write the same bytes"


def _tiles(rows, per_m, cols):
    """First and last tiles, which hold the clamps."""
    tm, tn = -(-rows // per_m), -(-cols // 256)
    return {(m * per_m, n * 256) for m in {0, tm // 2, tm - 1} for n in {0, tn // 2, tn - 1}}


def _runs(steps, splits):
    return {(steps * z // splits, steps * (z + 1) // splits) for z in {0, splits // 2, splits - 1}}


def _scale_base(step, steps):
    return max(0, min(step, steps - 4))


def _b_row(n0, r, rows):
    return np.minimum(n0 + (r & ~63) + 2 * (r & 31) + (r >> 5 & 1), rows - 1)


SIZES = [(1, 1, 1), (17, 100, 520), (65, 257, 136), (129, 260, 640), (300, 513, 1111), (700, 40, 72), (200, 13000, 288),
         (40, 13000, 264), (300, 500, 6000), (2050, 4100, 72), (4100, 100, 300), (600, 1300, 13000), (512, 14336, 4096)]


@pytest.mark.parametrize("m,n,k", SIZES)
def test_gemm(m, n, k):
    mt, splits = _plan(m, n, k, 64, (0.35, 0.4, 0.6), lambda s, t: (s + 3) * t, 4)
    steps = -(-k // 128)
    ldc, lds = 64 * steps, 4 * steps
    ka, stage, deep = 64 * mt * 64, 64 * mt * 64 + 16384, 4
    la = mt // 2 if mt >= 2 else 1
    total = deep * stage + 2 * (64 * mt + 256) * 16
    assert total <= 160 * 1024
    for m0, n0 in _tiles(m, 64 * mt, n):
        for first, last in _runs(steps, splits):
            dest = []
            for i in range(la):
                inst = la * WAVE + i if mt >= 2 else WAVE & 3
                r = 16 * inst + (LANE >> 2)
                base = np.minimum(m0 + r, m - 1) * ldc + 16 * ((LANE & 3) ^ (r >> 2 & 3))
                _inside(base + 64 * first, 16, m * ldc, "A codes")
                _inside(base + 64 * (last - 1), 16, m * ldc, "A codes")
                dest += [(1024 * x, 1024) for x in np.unique(inst)]
            _lds(dest, 0, ka, "A")
            dest = []
            for i in range(2):
                r = 16 * (2 * WAVE + i) + (LANE >> 2)
                base = _b_row(n0, r, n) * ldc + 16 * ((LANE & 3) ^ (r >> 2 & 3))
                _inside(base + 64 * first, 16, n * ldc, "B codes")
                _inside(base + 64 * (last - 1), 16, n * ldc, "B codes")
                dest += [(ka + 1024 * x, 1024) for x in np.unique(2 * WAVE + i)]
            _lds(dest, ka, stage, "B")
            ring = deep * stage
            for part in range(mt + 4):
                rows = np.minimum(m0 + 64 * part + LANE, m - 1) if part < mt else _b_row(n0, 64 * (part - mt) + LANE, n)
                limit = (m if part < mt else n) * lds
                if steps >= 4:
                    for step in {first, *range(first + 4, last + 4, 4)}:
                        _inside(rows * lds + 4 * _scale_base(step, steps), 16, limit, "scales")
                else:
                    _inside(rows * lds, 4 * steps, limit, "scales")
            _lds([(ring + 1024 * p, 1024) for p in range(mt + 4)], ring, ring + (64 * mt + 256) * 16, "scales")
            # a step's scale is read inside the group that was loaded for it
            for step in range(first, last):
                phase = (step - first) & 3
                assert not steps >= 4 or 0 <= step - _scale_base(step - phase, steps) < 4


@pytest.mark.parametrize("trans", [False, True])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_tile(m, n, k, trans):
    cols, depth = (k, n) if trans else (n, k)
    mt, splits = _plan(m, cols, depth, 32, (0.6, 1.0, 1.6) if trans else (0.53, 0.72, 1.4), lambda s, t: s * t + 9, 2)
    steps, wsteps = -(-depth // 128), -(-k // 128)
    ldc, lds, chunks = 64 * wsteps, 4 * wsteps, -(-depth // 8)
    ldx = 8 * chunks
    ka, stage = 32 * mt * 256, 32 * mt * 256 + 16384 + (3 * 1024 if trans else 0)
    loop = 3 * stage + (0 if trans else 8192)
    assert max(loop, (4 * mt if mt >= 2 else 4) * 8192) <= 160 * 1024
    for m0, n0 in _tiles(m, 32 * mt, cols):
        for first, last in _runs(steps, splits):
            dest = []
            for i in range(mt):
                r = 4 * (mt * WAVE + i) + (LANE >> 4)
                q = (LANE & 15) ^ (r & 15)
                row = np.minimum(m0 + r, m - 1) * ldx
                for step in {first, last - 1}:
                    at = (row + 8 * q + 128 * step)[16 * step + q < chunks]  # (the others read zeros elsewhere)
                    if at.size:
                        _inside(2 * at, 16, 2 * m * ldx, "x")
                dest += [(1024 * x, 1024) for x in np.unique(mt * WAVE + i)]
            _lds(dest, 0, ka, "x")
            dest = []
            for i in range(2):
                inst = 2 * WAVE + i
                if not trans:
                    r = 16 * inst + (LANE >> 2)
                    base = _b_row(n0, r, n) * ldc + 16 * ((LANE & 3) ^ (r >> 2 & 3))
                    for step in {first, last - 1}:
                        _inside(base + 64 * step, 16, n * ldc, "codes")
                else:
                    r = 8 * inst + (LANE >> 3)
                    col = np.minimum(n0 // 2 + 16 * ((LANE & 7) ^ (r >> 1 & 3)), 64 * wsteps - 16)
                    for step in {first, last - 1}:
                        _inside(np.minimum(128 * step + r, n - 1) * ldc + col, 16, n * ldc, "codes")
                dest += [(ka + 1024 * x, 1024) for x in np.unique(inst)]
            _lds(dest, ka, ka + 16384, "codes")
            if trans:
                w4 = np.arange(4)[:, None]
                r = (64 * w4 + LANE) >> 1
                col = np.minimum(n0 // 32 + 4 * (LANE & 1), 4 * wsteps - 4)
                for step in {first, last - 1}:
                    _inside(np.minimum(128 * step + r, n - 1) * lds + col, 4, n * lds, "scales")
                _lds([(ka + 16384 + 256 * x, 256) for x in range(4)], ka + 16384, ka + 16384 + 1024, "scales")
            else:
                r = 64 * np.arange(4)[:, None] + LANE
                rows = _b_row(n0, r, n)
                if steps >= 4:
                    for step in {first, *range(first + 4, last + 4, 4)}:
                        _inside(rows * lds + 4 * _scale_base(step, steps), 16, n * lds, "scales")
                else:
                    _inside(rows * lds, 4 * steps, n * lds, "scales")
                _lds([(3 * stage + 1024 * x, 1024) for x in range(4)], 3 * stage, 3 * stage + 4096, "scales")
                for step in range(first, last):
                    phase = (step - first) & 3
                    assert not steps >= 4 or 0 <= step - _scale_base(step - phase, steps) < 4


@pytest.mark.parametrize("rows,n,k", [(1, 1, 1), (1, 16, 32), (2, 17, 33), (4, 300, 4096), (5, 129, 1000), (16, 256, 128),
                                      (3, 40, 9000), (9, 8300, 300), (16, 300, 5000), (1, 14336, 4096), (7, 14336, 4096)])
def test_token(rows, n, k):
    steps, cap = -(-k // 128), 4 if rows <= 4 else 16
    tiles = -(-n // 16)
    waves = (4 if tiles >= 512 or steps <= 64 else 8) if rows <= 4 else (4 if tiles >= 512 else 8)
    cols = 2 if rows > 4 and tiles >= 512 else 1
    wgs = -(-tiles // cols)
    depth = 8 if cap == 4 else 4
    krow, ldc, lds, ldx = 256 * depth, 64 * steps, 4 * steps, -(-k // 8) * 8
    assert waves * cap * krow + waves * cols * 1024 <= 160 * 1024
    per = -(-steps // waves)
    j, g = LANE & 15, LANE >> 4
    for wave in range(waves):
        first, last = min(wave * per, steps), min(min(wave * per, steps) + per, steps)
        for s0 in range(first, last, depth):
            for r in range(rows):
                for i in range(krow // 1024):
                    at = 128 * s0 + 512 * i + 8 * (LANE ^ r)
                    at = at[at < k]
                    if at.size:
                        _inside(2 * (r * ldx + at), 16, 2 * rows * ldx, "x")
                    assert ((wave * cap + r) * krow + 1024 * i) + 1024 <= waves * cap * krow
            for n0 in {16 * cols * wg + 16 * t for wg in (0, wgs - 1) for t in range(cols)}:
                w = np.minimum(n0 + j, n - 1)
                for u in range(depth):
                    _inside(w * ldc + 16 * g + 64 * min(s0 + u, last - 1), 16, n * ldc, "codes")
                if s0 + depth <= steps:
                    for u in range(0, depth, 4):
                        _inside(w * lds + 4 * (s0 + u), 16, n * lds, "scales")
                else:
                    for u in range(depth):
                        _inside(w * lds + 4 * min(s0 + u, last - 1), 4, n * lds, "scales")


def _matrix(pkg, rows, cols):
    steps = -(-cols // 128)
    return pkg._lib.LrqMxfp4(0x10000, 64 * steps, 0x20000, 4 * steps, rows, cols)


@pytest.mark.parametrize("m,n,k", SIZES)
def test_the_plans_are_the_librarys(pkg, m, n, k):
    """The splits that the replays above take are those whose parts the library asks a workspace for."""
    import ctypes

    def want(splits, rows, cols):
        return splits * rows * (-(-cols // 4) * 4) * 4 if splits > 1 else 0

    a, w = ctypes.byref(_matrix(pkg, m, k)), ctypes.byref(_matrix(pkg, n, k))
    _, splits = _plan(m, n, k, 64, (0.35, 0.4, 0.6), lambda s, t: (s + 3) * t, 4)
    assert pkg._lib.call_raw("lrq_mxfp4_gemm_workspace", a, w) == want(splits, m, n)
    for trans in (0, 1):
        cols, depth = (k, n) if trans else (n, k)
        _, splits = _plan(m, cols, depth, 32, (0.6, 1.0, 1.6) if trans else (0.53, 0.72, 1.4), lambda s, t: s * t + 9, 2)
        if not trans and m <= 16:
            splits = 1  # the few-row kernel
        assert pkg._lib.call_raw("lrq_mxfp4_linear_workspace", m, w, trans) == want(splits, m, cols)


def _distinct(inst, count, what):
    """Every (wave, load) pair's kilobyte, all pairs counted: each of `count` once."""
    flat = np.concatenate([np.broadcast_to(i, (8, 1)).ravel() for i in inst])
    assert flat.size == count and sorted(flat.tolist()) == list(range(count)), what


@pytest.mark.parametrize("mt", [1, 2, 4])
def test_no_two_waves_load_to_the_same_place(mt):
    if mt >= 2:
        _distinct([mt // 2 * WAVE + i for i in range(mt // 2)], 4 * mt, "both operands: A")
    else:  # the upper four waves load the same again: from the same rows to the same place
        inst = (WAVE & 3).ravel()
        assert inst[:4].tolist() == inst[4:].tolist() == [0, 1, 2, 3]
    _distinct([2 * WAVE + i for i in range(2)], 16, "both operands: B")
    _distinct([mt * WAVE + i for i in range(mt)], 8 * mt, "x")
    _distinct([2 * WAVE + i for i in range(2)], 16, "codes")
