"""The arithmetic each source is compiled with."""

import importlib

import pytest

FINITE_ONLY = ("-fno-honor-nans", "-mno-amdgpu-ieee", "-ffinite-math-only", "-ffast-math", "-fno-honor-infinities",
               "-Ofast")


@pytest.fixture(scope="module")
def build():
    return importlib.import_module("triton-kernel-test_amd.build")


def _commands(build, monkeypatch):
    """The compiler's command line for every source."""
    seen = {}

    class Done:
        returncode, stderr = 0, ""

    def run(cmd, **kw):
        seen[cmd[cmd.index("-c") + 1]] = cmd
        return Done

    monkeypatch.setattr(build.subprocess, "run", run)
    for src in sorted(build.CSRC.glob("*.hip")):
        build._compile(src)
    return {s.rsplit("/", 1)[1]: c for s, c in seen.items()}


def test_kernels_that_carry_nan_are_compiled_to(build, monkeypatch):
    """Layer norm, dropout and MXFP4 promise to carry NaN and infinity: no option may let the compiler assume there are
    none."""
    cmds = _commands(build, monkeypatch)
    for name in ("lrq_dropout.hip", "lrq_mx.hip", "lrq_mxgemm.hip", "lrq_norm_bwd.hip", "lrq_norm_fwd.hip"):
        assert not set(FINITE_ONLY) & set(cmds[name]), name


def test_options_of_every_source(build, monkeypatch):
    for name, cmd in _commands(build, monkeypatch).items():
        assert "--offload-arch=gfx950" in cmd and "-ffp-contract=off" in cmd, name
        assert cmd[cmd.index("-packed-fp32-ops") - 1] == "-Xclang", name
        assert cmd[cmd.index("-amdgpu-remove-redundant-endcf=0") - 1] == "-mllvm", name
