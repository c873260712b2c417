"""The 8-bit products' plans, from the library's own source compiled for the host (tests/fp8_plan.cpp): the tests on the GPU run
the tiles, splits and steps that they are there for (no GPU)."""

import ctypes
import importlib
import shutil
import subprocess
from pathlib import Path

import pytest

HERE = Path(__file__).resolve().parent
TILES = {(1, 1), (1, 2), (1, 4), (2, 2), (2, 4), (3, 4), (4, 4)}  # 64 mt rows by 64 nb columns


@pytest.fixture(scope="module")
def plans(tmp_path_factory):
    """[(rows, cols, depth, nn)] -> [(mt, nb, splits, steps)]"""
    if shutil.which("g++") is None:
        pytest.skip("needs g++")
    exe = tmp_path_factory.mktemp("plan") / "fp8_plan"
    subprocess.run(["g++", "-O1", "-std=c++17", "-o", str(exe), str(HERE / "fp8_plan.cpp")], check=True)

    def ask(shapes):
        lines = "".join(f"{m} {n} {k} {int(nn)}\n" for m, n, k, nn in shapes)
        out = subprocess.run([str(exe)], input=lines, capture_output=True, text=True, check=True, timeout=60).stdout
        return [tuple(map(int, line.split())) for line in out.splitlines()]
    return ask


def _parameters(test):
    """What a test's first mark of three names is parametrised by."""
    return next(m.args[1] for m in test.pytestmark if m.name == "parametrize" and m.args[0].count(",") == 2)


def test_the_plans_are_the_librarys(pkg, plans):
    """The workspace is that of the plan's splits."""
    shapes = [(m, n, k, nn) for m in (1, 16, 17, 32, 33, 100, 300, 512, 2048) for n in (1, 64, 130, 4096, 5120, 14300)
              for k in (1, 128, 700, 4096, 9000, 14336) for nn in (False, True)]
    for (m, n, k, nn), (_, _, splits, _) in zip(shapes, plans(shapes)):
        def t(rows, cols, block):
            ld = -(-cols // 128) * 128
            return pkg._lib.LrqFp8(0x10000, ld, 0x20000, -(-ld // 512) * 4, rows, cols, block)
        a, b = t(m, k, 1), t(*((k, n) if nn else (n, k)), 128)
        want = splits * m * -(-n // 4) * 16 if splits > 1 else 0
        assert pkg._lib.call_raw("lrq_fp8_gemm_workspace", ctypes.byref(a), ctypes.byref(b), int(nn)) == want, (m, n, k, nn)


def test_every_tile_is_run(plans):
    """``test_every_tile`` comes to each, either way."""
    T = importlib.import_module("test_gpu_fp8")
    for nn in (False, True):
        got = plans([(m, cols, depth, nn) for m, depth, cols in _parameters(T.test_every_tile)])
        assert {p[:2] for p in got} - {(0, 0)} == TILES
        assert any(p[2] > 1 for p in got) and any(p[2] == 1 for p in got)


def test_the_tiles_run_round(plans):
    """``test_gpu_fp8_tiles``: each tile, whole and split, either way, takes more steps than its ring holds (4 at most), in one
    piece also more than the two groups of four whose scales LDS holds; the last group is not whole."""
    T = importlib.import_module("test_gpu_fp8_tiles")
    assert {(t, s) for t, s, *_ in T.TILES} == {(t, s) for t in TILES for s in (False, True)}
    for nn in (False, True):
        for (tile, split, *_), (mt, nb, splits, steps) in zip(T.TILES, plans([(m, n, k, nn) for _, _, m, k, n in T.TILES])):
            assert (mt, nb) == tile and (splits > 1) == split
            groups = -(-steps // 4)
            runs = [min(4 * (groups * (z + 1) // splits), steps) - 4 * (groups * z // splits) for z in range(splits)]
            assert sum(runs) == steps and min(runs) > 4 and (split or steps > 8) and steps % 4 != 0, runs


def test_the_few_row_kernel_is_run(plans):
    """All its widths: tiles of rows, tiles of weight rows, waves."""
    T = importlib.import_module("test_gpu_fp8_tiles")
    assert all(p[0] == 0 for p in plans([(m, n, k, False) for m, k, n in T.FEW]))

    def forms(shapes):
        return {(1 if m <= 16 else 2, 1 if n <= 4096 else 2, 16 if n <= 8192 else 8) for m, _, n in shapes}
    assert forms(T.FEW) == {(1, 1, 16), (1, 2, 16), (1, 2, 8), (2, 1, 16), (2, 2, 16)}
    assert forms(T.FEW_16) == {(1, 1, 16), (1, 2, 16), (1, 2, 8)} and all(m <= 4 and k % 8 == 0 for m, k, _ in T.FEW_16)
