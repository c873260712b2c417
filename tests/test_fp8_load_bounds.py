"""The loads of the 8-bit products, replayed in numpy from the launch arithmetic of csrc/lrq_fp8gemm.hip for every tile
and split the host may choose: every read lies in its operand, every LDS write in the part of the allocation it belongs to,
no two loads of a step write the same bytes, and the transposing and plain LDS reads find the element they are meant to."""

import numpy as np
import pytest

LANE, WAVE = np.arange(64), np.arange(4)[:, None]  # [waves, lanes] below


def _inside(at, size, limit, what):
    at = np.asarray(at)
    assert at.min() >= 0 and at.max() + size <= limit, (what, int(at.min()), int(at.max()) + size, limit)


def _lds(dests, low, high, what):
    spans = sorted((int(b), int(b) + n) for b, n in dests)
    assert spans[0][0] >= low and spans[-1][1] <= high, what
    assert all(a[1] <= b[0] for a, b in zip(spans, spans[1:])), f"{what}: two loads write the same bytes"


TILES = [(1, 1), (1, 2), (1, 4), (2, 2), (2, 4), (3, 4), (4, 4)]  # 64 mt rows by 64 nb columns


def _deep(mt, nb):
    return min(4, (160 * 1024 - 2 * 2048) // (64 * (mt + nb) * 128))


def _turn(r, nb):
    return (r ^ (r >> 2 & 1)) & 3 if nb == 1 else r & 7


def _runs(steps, splits):
    groups = (steps + 3) // 4
    for z in sorted({0, splits // 2, splits - 1}):
        yield 4 * (groups * z // splits), min(4 * (groups * (z + 1) // splits), steps)


SIZES = [(1, 1, 1), (17, 100, 520), (65, 257, 136), (129, 260, 640), (300, 513, 1111), (700, 40, 72), (200, 13000, 288),
         (40, 1300, 2640), (300, 500, 6000), (2050, 4100, 72), (600, 1300, 13000), (512, 14336, 4096)]


def _lds_sizes(mt, nb):
    kx, kw = 64 * mt * 128, 64 * nb * 128
    stage = kx + kw
    ring = _deep(mt, nb) * stage
    assert _deep(mt, nb) >= 2
    loop = ring + 2 * 2048
    assert loop <= 160 * 1024 and 4 * 32 * 144 <= loop
    return kx, stage, ring


@pytest.mark.parametrize("nn", [False, True])
@pytest.mark.parametrize("mt,nb", TILES)
@pytest.mark.parametrize("m,n,k", SIZES)
def test_tile(m, n, k, mt, nb, nn):
    """x [m, depth], w [n, k]: depth = k, output columns n; NN: depth = n, output columns k."""
    depth, cols = (n, k) if nn else (k, n)
    steps, wsteps = -(-depth // 128), -(-k // 128)
    ldx, ldw, ldsx, ldsw = 128 * steps, 128 * wsteps, -(-steps // 4) * 4, -(-wsteps // 4) * 4
    kx, stage, ring = _lds_sizes(mt, nb)
    klx, klw = 2 * mt, 2 * nb
    lanes, even = 4 * nb, 1 if nb <= 2 else 2
    each = 64 // lanes
    wrows = -(-n // 128)
    for splits in {min(wanted, max(1, steps // 4)) for wanted in (1, 2, 3, 16)}:  # none without a step
        for m0 in {0, (m - 1) // (64 * mt) * 64 * mt}:
            for n0 in {0, (cols - 1) // (64 * nb) * 64 * nb}:
                for first, last in _runs(steps, splits):
                    assert 0 <= first < last <= steps and first % 4 == 0
                    # X
                    dest = []
                    mx = min(64 * mt, m - m0) - 1
                    for i in range(klx):
                        r = 8 * (klx * WAVE + i) + (LANE >> 3)
                        piece = (LANE & 7) ^ (r >> 1 & 7)
                        ox = np.minimum(r, mx) * ldx + 16 * piece
                        for step in (first, last - 1):
                            _inside(m0 * ldx + 128 * step + ox, 16, m * ldx, "X codes")
                        dest += [(1024 * v, 1024) for v in np.unique(klx * WAVE + i)]
                    _lds(dest, 0, kx, "X")
                    # W
                    dest = []
                    for i in range(klw):
                        if not nn:
                            r = 8 * (klw * WAVE + i) + (LANE >> 3)
                            ow = np.minimum(r, min(64 * nb, n - n0) - 1) * ldw + 16 * ((LANE & 7) ^ (r >> 1 & 7))
                            for step in (first, last - 1):
                                _inside(n0 * ldw + 128 * step + ow, 16, n * ldw, "W codes")
                        else:
                            r = 32 * WAVE + each * i + LANE // lanes
                            ow = np.minimum(16 * ((LANE % lanes) ^ _turn(r, nb)), min(64 * nb, 128 * wsteps - n0) - 16)
                            # offset i % even serves
                            assert (_turn(32 * WAVE + each * (i % even) + LANE // lanes, nb) == _turn(r, nb)).all()
                            for step in (first, last - 1):
                                row = np.minimum(r, n - 1 - 128 * step)
                                _inside((128 * step + row) * ldw + n0 + ow, 16, n * ldw, "W codes")
                        dest += [(kx + 1024 * v, 1024) for v in np.unique(klw * WAVE + i)]
                    _lds(dest, kx, stage, "W")
                    # scales: group g in slot (g - first / 4) % 2
                    part = np.minimum(WAVE, mt - 1)
                    wpart = WAVE if nn else np.minimum(WAVE, nb - 1)
                    dest = [(ring + 256 * v, 256) for v in np.unique(part)] + [(ring + 1024 + 256 * v, 256) for v in np.unique(wpart)]
                    _lds(dest, ring, ring + 2048, "scales")
                    for g in {first // 4, (last - 1) // 4}:
                        for shift in (0, 7):
                            tall = -(-m // (1 << shift))
                            row = np.minimum(m0 + 64 * part + LANE, m - 1) >> shift
                            _inside(row * ldsx + 4 * g, 4, tall * ldsx, "X scales")
                        if not nn:
                            for shift in (0, 7):
                                tall = -(-n // (1 << shift))
                                row = np.minimum(n0 + 64 * wpart + LANE, n - 1) >> shift
                                _inside(row * ldsw + 4 * g, 4, tall * ldsw, "W scales")
                        else:
                            block = np.minimum((n0 + 32 * nb * (WAVE & 1)) // 128, wsteps - 1)
                            row = np.minimum(4 * g + (LANE & 3), steps - 1)
                            _inside(row * ldsw + (block & ~3), 4, wrows * ldsw, "W scales")


@pytest.mark.parametrize("mt,nb", TILES)
@pytest.mark.parametrize("first,steps", [(0, n) for n in (1, 2, 3, 4, 5, 6, 7, 8, 9, 12, 13, 17, 32, 112)] + [(8, 40), (12, 37)])
def test_order(first, steps, mt, nb):
    """What is read from LDS has come, and nothing is written over that is still to be read: a wave's loads in their order (they
    come in in that order), its waits, which leave the newest so many under way, and its reads of each step."""
    deep, loads = _deep(mt, nb), 2 * (mt + nb)
    early, last = 3 * loads // 8, steps
    issued, place, come = [], {}, {}  # loads in order; what a place holds or will hold; which loads are in

    def issue(key, where):
        issued.append((key, where))
        place[where] = key

    def wait(newest):
        for i, (key, where) in enumerate(issued[:len(issued) - newest] if newest else issued):
            come[where] = key

    def scales(group, slot):
        for operand in range(2):
            issue(("scales", group, operand), ("slot", slot, operand))

    def step_in(step, buf):
        return all(come.get(("buf", buf, i)) == ("step", step, i) == place[("buf", buf, i)] for i in range(loads))

    def scales_in(step, slot):
        want = [("scales", step // 4, o) for o in range(2)]
        return all(come.get(("slot", slot, o)) == want[o] == place[("slot", slot, o)] for o in range(2))

    scales(first // 4, 0)
    for d in range(deep):
        for i in range(loads):
            issue(("step", min(first + d, last - 1), i), ("buf", d, i))
    wait((deep - 1) * loads)
    assert step_in(first, 0) and scales_in(first, 0)  # half 0's operands are read here
    buf = slot = 0
    for step in range(first, last):
        ahead = min(step + deep, last - 1)
        assert step_in(step, buf)  # half 1's operands
        for i in range(early):
            issue(("step", ahead, i), ("buf", buf, i))
        wait((deep - 2) * loads + early)
        following = (buf + 1) % deep
        if step % 4 == 0 and step + 4 < last:
            scales(step // 4 + 1, slot ^ 1)
        for i in range(early, loads):
            issue(("step", ahead, i), ("buf", buf, i))
        if step + 1 < last:
            assert step_in(step + 1, following)  # half 0 of the next step
        slot ^= step % 4 == 3
        if step + 1 < last:
            assert scales_in(step + 1, slot)
        buf = following


def _loads_x(mt):
    """What LDS holds of X after a step's loads: [byte] = (row, byte of the row)."""
    image = np.full((64 * mt * 128, 2), -1)
    for wave in range(4):
        for i in range(2 * mt):
            r = 8 * (2 * mt * wave + i) + (LANE >> 3)
            for b in range(16):
                at = 1024 * (2 * mt * wave + i) + 16 * LANE + b
                image[at] = np.stack([r, 16 * ((LANE & 7) ^ (r >> 1 & 7)) + b], 1)
    assert (image >= 0).all()
    return image


@pytest.mark.parametrize("mt", [1, 2, 3, 4])
def test_reads_of_rows(mt):
    """Lane (c, h) of half Q finds bytes 64 Q + 32 h .. + 31 of its row; 16 neighbouring lanes read all banks."""
    image = _loads_x(mt)
    c, h = LANE & 31, LANE >> 5
    for half in range(2):
        for q in range(2):
            for tile in range(2 * mt):
                r = 32 * tile + c
                at = 128 * r + 16 * ((4 * half + 2 * h + q) ^ (r >> 1 & 7))
                for b in range(16):
                    got = image[at + b]
                    assert (got[:, 0] == r).all() and (got[:, 1] == 64 * half + 32 * h + 16 * q + b).all()
                banks = (at // 16) % 16
                assert all(len(set(banks[16 * g:16 * g + 16])) == 16 for g in range(4))


@pytest.mark.parametrize("nb", [1, 2, 4])
def test_reads_of_columns(nb):
    """NN: the transposing read of lane (c, h), half Q, piece q, gives bytes of column 32 t + c in rows 64 Q + 32 h + 16 q ..
    + 15, in the order in which X's operand has them."""
    lanes = 4 * nb
    image = np.full((128 * 64 * nb, 2), -1)  # (row of the step, column of the tile)
    for wave in range(4):
        for i in range(2 * nb):
            r = 32 * wave + 64 // lanes * i + LANE // lanes
            for b in range(16):
                image[1024 * (2 * nb * wave + i) + 16 * LANE + b] = np.stack([r, 16 * ((LANE % lanes) ^ _turn(r, nb)) + b], 1)
    assert (image >= 0).all()
    for wn in range(2):
        for t in range(nb):
            for half in range(2):
                for q in range(2):
                    r = 64 * half + 32 * (LANE >> 5) + 16 * q + (LANE >> 1 & 7)
                    piece = 2 * nb * wn + 2 * t + (LANE >> 4 & 1)
                    p = 64 * nb * r + 16 * (piece ^ _turn(r, nb)) + 8 * (LANE & 1)
                    for second in range(2):
                        at = p + 8 * 64 * nb * second
                        for lane in range(64):
                            group, i = lane & ~15, lane & 15
                            # 16 lanes read 8 rows of 16 bytes, two lanes a row; lane i is given byte i of each
                            for e in range(8):
                                src = at[group + 2 * e + i // 8] + i % 8
                                row, col = image[src]
                                assert col == 32 * nb * wn + 32 * t + (lane & 31)
                                assert row == 64 * half + 32 * (lane >> 5) + 16 * q + 8 * second + e


def _rows_of(n, tn, wgs):
    own = min(16 * tn, (-(-n // wgs) + 3) // 4 * 4)
    return own, -(-n // own)


@pytest.mark.parametrize("rows,xt", [(1, "fp8"), (4, "16"), (16, "fp8"), (17, "fp8"), (32, "fp8")])
@pytest.mark.parametrize("n,k", [(1, 1), (5, 128), (100, 1000), (4096, 4096), (4097, 640), (8190, 130), (14336, 4096), (40000, 256)])
def test_few_rows(n, k, rows, xt):
    if xt == "16" and k % 8:
        pytest.skip("16-bit rows are whole 16-byte pieces")
    tm = 1 if rows <= 16 else 2
    if tm == 2 and (n > 8192 or k > 40 * 128):
        pytest.skip("in tiles")
    if n <= 4096:
        tn, waves, d, wgs = 1, 16, 4 // tm, 256
    elif n <= 8192:
        tn, waves, d, wgs = 2, 16, 4 // tm, 256
    else:
        tn, waves, d, wgs = 2, 8, 4, 512 * -(-n // 16384)
    own, grid = _rows_of(n, tn, wgs)
    assert own <= 16 * tn and (grid - 1) * own < n <= grid * own
    steps = -(-k // 128)
    ldc, sw4 = 128 * steps, -(-steps // 4) * 4
    j, g = LANE & 15, LANE >> 4
    # LDS: the waves' sums and, of 16-bit rows, their codes
    assert waves * tm * tn * 64 * 16 + (waves * 512 if xt == "16" else 0) <= 64 * 1024
    seen = np.zeros(steps, dtype=int)
    for wave in range(waves):
        first, last = steps * wave // waves, steps * (wave + 1) // waves
        for s0 in range(first, last, d):
            count = min(d, last - s0)
            base = min(s0, sw4 - 4)
            _inside(base, 4, sw4, "scales of a row")
            for u in range(count):
                seen[s0 + u] += 1
                assert 0 <= s0 + u - base < 4
                for wg in {0, grid - 1}:
                    n0, n1 = wg * own, min(wg * own + own, n)
                    for t in range(tn):
                        r = np.minimum(n0 + 16 * t + j, n1 - 1)
                        assert (r >= n0).all()
                        _inside(r * ldc + 16 * g + 128 * (s0 + u) + 64, 16, n * ldc, "W codes")
                if xt == "16":
                    at = 128 * (s0 + u) + 8 * j
                    take = at < k
                    if take.any():
                        _inside((np.minimum(g, rows - 1) * k + at)[take], 8, rows * k, "X")
                else:
                    for i in range(tm):
                        _inside(np.minimum(16 * i + j, rows - 1) * ldc + 16 * g + 128 * (s0 + u) + 64, 16, rows * ldc, "X codes")
    assert (seen == 1).all()
