"""The norm, dropout and MXFP4 kernels as built: none spills vector registers or uses scratch memory."""

import importlib
import re
import shutil
import struct
import subprocess
from pathlib import Path

import pytest

_MAGIC = b"__CLANG_OFFLOAD_BUNDLE__"


def _code_objects(data):
    """The gfx950 code objects of a library's offload bundles."""
    at = data.find(_MAGIC)
    while at >= 0:
        pos = at + len(_MAGIC)
        count, = struct.unpack_from("<Q", data, pos)
        pos += 8
        for _ in range(count):
            offset, size, name = struct.unpack_from("<QQQ", data, pos)
            triple = data[pos + 24:pos + 24 + name]
            pos += 24 + name
            if b"gfx950" in triple and size:
                yield data[at + offset:at + offset + size]
        at = data.find(_MAGIC, at + 1)


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
            seen[name] = (get("vgpr_spill_count"), get("private_segment_fixed_size"))
    mine = {n: v for n, v in seen.items() if re.search(r"k_(norm|dropout|mx)_?", n)}
    for stem, least in (("k_norm_fwd", 18), ("k_norm_bwd", 22), ("k_dropout", 6), ("k_mx_gemm", 6), ("k_mx_tile", 12),
                        ("k_mx_token", 8)):
        assert sum(stem in n for n in mine) >= least, stem
    bad = {n: v for n, v in mine.items() if v != (0, 0)}
    assert not bad, bad


def test_no_kernel_spills_scalars(tmp_path):
    """Nor do they spill scalar registers (to lanes of a vector register, which a kernel short of those then lacks)."""
    L = importlib.import_module("triton-kernel-test_amd._lib")
    readelf = Path("/opt/rocm/llvm/bin/llvm-readelf")
    readelf = str(readelf) if readelf.exists() else shutil.which("llvm-readelf")
    if not L.LIB_PATH.exists() or readelf is None:
        pytest.skip("needs the built library and llvm-readelf")
    bad, count = {}, 0
    for i, obj in enumerate(_code_objects(L.LIB_PATH.read_bytes())):
        f = tmp_path / f"{i}.elf"
        f.write_bytes(obj)
        notes = subprocess.run([readelf, "--notes", str(f)], capture_output=True, text=True, check=True).stdout
        for kernel in notes.split("\n  - .agpr_count:")[1:]:
            name = re.search(r"\.symbol:\s+'?(\S+?)\.kd", kernel).group(1)
            if re.search(r"k_(norm|dropout|mx)_?", name):
                count += 1
                spilled = int(re.search(r"\.sgpr_spill_count:\s+(\d+)", kernel).group(1))
                if spilled:
                    bad[name] = spilled
    assert count >= 100 and not bad, (count, bad)
