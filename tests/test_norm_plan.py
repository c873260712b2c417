"""The shapes that the layer norm's tests run reach every form of its backward pass with several rows a row group (no GPU)."""

import importlib

import pytest

T = importlib.import_module("test_gpu_norm")


@pytest.mark.parametrize("rows,n", T.GEOMETRIES + [(1, 1), (7, 129), (16384, 4096), (100, 20000), (1 << 20, 64)])
def test_the_plan_is_the_librarys(pkg, rows, n):
    """The sums' workspace is that of the larger of the two plans' parts."""
    parts = max(T._backward_plan(rows, n, fp32)[-1] for fp32 in (False, True))
    assert pkg._lib.call_raw("lrq_layer_norm_bwd_workspace", rows, n) == parts * 2 * n * 4


def test_every_form_walks_rows():
    forms, waves = {}, set()
    for rows, n in T.GEOMETRIES:
        for fp32 in (False, True):
            kind, lanes, chunks, groups, grid, _ = T._backward_plan(rows, n, fp32)
            steps = -(-rows // (groups * grid))
            key = (kind, lanes, chunks, fp32, groups > 1)
            forms[key] = max(forms.get(key, 0), steps)
            if chunks == 1 and lanes == 0 and steps > 1:
                waves.add((kind, -(-n // 512), groups))
    for fp32 in (False, True):
        for kind in ("plain", "odd"):
            for lanes in (16, 64, 0):
                assert forms[kind, lanes, 1, fp32, True] >= 2, (kind, lanes, fp32)
            assert forms[kind, 0, 1, fp32, False] >= 2, (kind, fp32)
        assert forms["wide", 0, 0, fp32, False] >= 2
    assert forms["plain", 0, 4, False, False] >= 2
    for kind in ("plain", "odd"):
        for w in range(2, 8):
            assert any(k == kind and v == w and g == 16 // w for k, v, g in waves), (kind, w)
