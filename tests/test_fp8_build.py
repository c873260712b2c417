"""The root-mean-square norm and 8-bit kernels as built: none spills registers or uses scratch memory, none is compiled as if
there were no NaN, and the tiles' LDS fits a CU."""

import importlib
import re
import shutil
import subprocess
from pathlib import Path

import pytest

from test_build_flags import FINITE_ONLY, _commands
from test_registers import _code_objects


def test_kernels_that_carry_nan_are_compiled_to(monkeypatch):
    cmds = _commands(importlib.import_module("triton-kernel-test_amd.build"), monkeypatch)
    for name in ("lrq_fp8.hip", "lrq_fp8gemm.hip", "lrq_rms.hip"):
        assert not set(FINITE_ONLY) & set(cmds[name]), name


def test_products_keep_their_sums_in_accumulation_registers(monkeypatch):
    cmds = _commands(importlib.import_module("triton-kernel-test_amd.build"), monkeypatch)
    form = "-amdgpu-mfma-vgpr-form"
    assert [n for n, c in cmds.items() if form not in c] == ["lrq_fp8gemm.hip"]


def test_no_kernel_spills(tmp_path):
    L = importlib.import_module("triton-kernel-test_amd._lib")
    readelf = Path("/opt/rocm/llvm/bin/llvm-readelf")
    readelf = str(readelf) if readelf.exists() else shutil.which("llvm-readelf")
    if not L.LIB_PATH.exists() or readelf is None:
        pytest.skip("needs the built library and llvm-readelf")
    seen = {}
    for i, obj in enumerate(_code_objects(L.LIB_PATH.read_bytes())):
        f = tmp_path / f"{i}.elf"
        f.write_bytes(obj)
        notes = subprocess.run([readelf, "--notes", str(f)], capture_output=True, text=True, check=True).stdout
        for kernel in notes.split("\n  - .agpr_count:")[1:]:
            get = lambda key: int(re.search(rf"\.{key}:\s+(\d+)", kernel).group(1))
            name = re.search(r"\.symbol:\s+'?(\S+?)\.kd", kernel).group(1)
            if re.search(r"k_(rms|fp8)_", name):
                seen[name] = (get("vgpr_spill_count"), get("sgpr_spill_count"), get("private_segment_fixed_size"))
    for stem, least in (("k_rms_fwd", 54), ("k_rms_bwd", 26), ("k_fp8_tile", 42), ("k_fp8_token", 11), ("k_fp8_rows", 3)):
        assert sum(stem in n for n in seen) >= least, (stem, sum(stem in n for n in seen))
    bad = {n: v for n, v in seen.items() if v != (0, 0, 0)}
    assert not bad, bad


def test_loads_to_lds_set_their_own_base(tmp_path):
    """The tiles' loads to LDS are written in assembly with the move to m0 that each needs in the same statement: in the
    built kernels every one is preceded by its move, nothing else touches m0, and no other load from memory is in flight
    whose arrival the compiler would count among theirs."""
    L = importlib.import_module("triton-kernel-test_amd._lib")
    tool = Path("/opt/rocm/llvm/bin/llvm-objdump")
    tool = str(tool) if tool.exists() else shutil.which("llvm-objdump")
    if not L.LIB_PATH.exists() or tool is None:
        pytest.skip("needs the built library and llvm-objdump")
    kernels = loads = 0
    for i, obj in enumerate(_code_objects(L.LIB_PATH.read_bytes())):
        if b"k_fp8_tile" not in obj:
            continue
        f = tmp_path / f"{i}.elf"
        f.write_bytes(obj)
        listing = subprocess.run([tool, "-d", "--no-show-raw-insn", str(f)], capture_output=True, text=True, check=True).stdout
        name, code = None, {}
        for line in listing.splitlines():
            m = re.match(r"^[0-9a-f]+ <(\S+)>:", line)
            if m:
                name = m.group(1)
                code[name] = []
            elif name and line.startswith("\t"):
                code[name].append(line.split("//")[0].strip())
        for name, ins in code.items():
            if "k_fp8_tile" not in name:
                continue
            kernels += 1
            for k, text in enumerate(ins):
                if "global_load_lds" in text:
                    loads += 1
                    assert ins[k - 1] == "s_nop 0" and re.match(r"s_mov_b32 m0, s\d+$", ins[k - 2]), (name, ins[k - 2:k + 1])
                elif re.search(r"\bm0\b", text):
                    assert "global_load_lds" in ins[k + 2], (name, ins[k:k + 3])
                else:
                    assert not re.match(r"(global|flat|scratch|buffer)_load", text), (name, text)
    assert kernels >= 24 and loads > 1000, (kernels, loads)
