"""The shapes that the root-mean-square norm's tests run reach every form of it with several rows a row group (no GPU)."""

import importlib

import pytest

T = importlib.import_module("test_gpu_rms_rounds")
MANY = [(1, 1), (7, 129), (37, 4096), (1003, 5003), (2048, 2560), (16384, 4096), (100, 20000), (1 << 20, 64), (4096, 14336)]


def _groups(nc, lanes, waves, rows, most):
    most = 64 * most // lanes if lanes else max(1, most // waves)
    return min(most, max(1, 4 * -(-rows // 1024) if lanes == 16 else -(-rows // 256)))


def _even(most, rows, each):
    """The most groups that leave the fullest CU with as few rows as any number does."""
    load = {g: -(-rows // (256 * each(g) * g)) * each(g) * g for g in range(1, most + 1)}
    return max(g for g in load if load[g] == min(load.values()))


def _shape(n, one, more):
    nc = -(-n // 8)
    if nc <= 64:
        return nc, 16 if nc <= 16 else 64, 1, 1
    chunks = 1 if nc <= one else more
    return nc, 64 if nc <= 64 * chunks else 0, chunks, -(-nc // (64 * chunks))


def forward(rows, n):
    """Lanes and chunks a thread, waves of a row, groups of a workgroup, rounds of rows (csrc/lrq_rms.hip: rms_fwd)."""
    if n > 16384:
        return "wide", 0, 0, 1, -(-rows // 512)
    nc, lanes, chunks, waves = _shape(n, 64, 2)
    groups = _groups(nc, lanes, waves, rows, 16)
    if not lanes:
        groups = _even(groups, rows, lambda g: 16 // (waves * g))
    threads = max(64, (lanes or 64 * waves) * groups)
    return lanes, chunks, waves, groups, -(-rows // (groups * min(-(-rows // groups), 256 * (1024 // threads))))


def backward(rows, n, fp32):
    """The same of rms_plan, and the parts of the weight gradient."""
    if n > (8192 if fp32 else 16384):
        return "wide", 0, 0, 1, -(-rows // min(rows, 512)), min(-(-rows // 4), 64)
    nc, lanes, chunks, waves = _shape(n, 1024, 4)
    groups = _groups(nc, lanes, waves, rows, 8 if chunks == 4 else 16)
    if not lanes:
        groups = _even(groups, rows, lambda g: 1)
    grid = min(-(-rows // groups), 256)
    return lanes, chunks, waves, groups, -(-rows // (groups * grid)), grid


@pytest.mark.parametrize("rows,n", T.SHAPES + MANY)
def test_the_plan_is_the_librarys(pkg, rows, n):
    """The workspace is that of the larger of the two types' parts."""
    parts = max(backward(rows, n, fp32)[-1] for fp32 in (False, True))
    assert pkg._lib.call_raw("lrq_rms_norm_bwd_workspace", rows, n) == parts * n * 4


def test_every_form_takes_three_rounds():
    seen, one = set(), set()
    for rows, n in T.SHAPES:
        end = "odd" if n % 8 else "whole"
        lanes, chunks, waves, groups, rounds = forward(rows, n)
        assert rounds >= 3, (rows, n, rounds)
        seen.add(("forward", lanes, chunks, end))
        one.add(("forward", groups > 1))
        for fp32 in (False, True):
            lanes, chunks, waves, groups, rounds, _ = backward(rows, n, fp32)
            assert rounds >= 3, (rows, n, fp32, rounds)
            seen.add(("backward", fp32, lanes, chunks, end))
            one.add(("backward", groups > 1))
    want = {("forward", lanes, chunks, end) for lanes, chunks in ((16, 1), (64, 1), (64, 2), (0, 2)) for end in ("odd", "whole")}
    want |= {("backward", fp32, lanes, 1, end) for fp32 in (False, True) for lanes in (16, 64, 0) for end in ("odd", "whole")}
    want |= {("backward", False, 0, 4, "odd"), ("backward", False, 0, 4, "whole"), ("forward", "wide", 0, "odd"),
             ("backward", False, "wide", 0, "odd"), ("backward", True, "wide", 0, "odd"), ("backward", True, "wide", 0, "whole")}
    assert want <= seen, want - seen
    assert one == {(way, several) for way in ("forward", "backward") for several in (False, True)}
