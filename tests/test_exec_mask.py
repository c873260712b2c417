"""Vector instructions between the end of a masked region and the restore of its mask, in the built kernels.

Lanes whose condition is false skip a region with their bit of the execution mask cleared; where the region ends, the mask is
restored.  For two regions that end together the compiler may leave out the inner restore, and its register allocator has
then put reloads of spilled registers between the two ends, where the skipped lanes do not take part: they go on with whatever
the register held.  (A row loop's step that was reloaded so let lanes without columns add 0 to their row for ever.)  The build
turns the omission off; this looks for its trace in what was built."""

import importlib
import re
import shutil
import subprocess
from pathlib import Path

import pytest

from test_registers import _code_objects

_INSTR = re.compile(r"^\s+(\S.*?)\s*// ([0-9A-F]+):")
_TARGET = re.compile(r"<(\S+?)(?:\+0x([0-9a-f]+))?>\s*$")
_LANES = re.compile(r"(v_|ds_|global_|scratch_|buffer_|flat_)(?!readlane|writelane|readfirstlane)")
_ENDS = re.compile(r"s_(endpgm|branch|setpc|swappc|cbranch)")


def _functions(listing):
    """(name, [(address, text, the branch's target or None)]) of a disassembly."""
    name, start, code, starts = None, 0, [], {}
    for line in listing.splitlines():
        m = re.match(r"^([0-9a-f]+) <(\S+)>:", line)
        if m:
            if code:
                yield name, code
            name, start, code = m.group(2), int(m.group(1), 16), []
            starts[name] = start
            continue
        m = _INSTR.match(line)
        if m:
            t = _TARGET.search(line) if m.group(1).startswith("s_cbranch_exec") else None
            to = starts.get(t.group(1), -1) + int(t.group(2) or "0", 16) if t else None
            code.append((int(m.group(2), 16), m.group(1), to))
    if code:
        yield name, code


def _masked(code):
    """[(address, instruction)] that only the lanes of a region that has ended execute, ahead of its restore."""
    index = {a: i for i, (a, _, _) in enumerate(code)}
    joins = set()
    for i, (_, text, to) in enumerate(code):
        if text.startswith("s_cbranch_execz") and to in index:
            joins.add(index[to])
        if text.startswith("s_cbranch_execnz"):
            joins.add(i + 1)
    found = []
    for i in sorted(joins):
        lanes = []
        for a, text, _ in code[i:]:
            if "exec" in text.split("//")[0] and not text.startswith("s_cbranch"):
                if lanes and re.match(r"s_or_b64 exec, exec,", text):
                    found += lanes
                break
            if _ENDS.match(text):
                break
            if _LANES.match(text):
                lanes.append((a, text))
    return found


# the end of a row loop as it was once built: v[78:79] is the loop's step
_LISTING = """
0000000000001000 <k>:
	s_and_saveexec_b64 s[42:43], s[38:39]                      // 000000001000: BEAA2026
	s_cbranch_execz 6                                          // 000000001004: BF880006 <k+0x20>
	s_and_b64 exec, exec, s[20:21]                             // 000000001008: 86FE147E
	s_cbranch_execz 2                                          // 00000000100C: BF880002 <k+0x18>
	v_mad_u64_u32 v[78:79], s[8:9], v58, s67, 0                // 000000001010: D1E8084E 0000013A
	scratch_load_dwordx2 v[78:79], off, off offset:44          // 000000001018: DC54402C 4E7F0000
	s_or_b64 exec, exec, s[42:43]                              // 000000001020: 87FE2A7E
	v_lshl_add_u64 v[68:69], v[68:69], 0, v[78:79]             // 000000001024: D2080044 04390144
	s_endpgm                                                   // 00000000102C: BF810000
"""


def test_the_trace_is_recognised():
    (_, code), = _functions(_LISTING)
    assert [t for _, t in _masked(code)] == ["scratch_load_dwordx2 v[78:79], off, off offset:44"]
    good = _LISTING.replace("	scratch_load_dwordx2 v[78:79], off, off offset:44 ", "	s_or_b64 exec, exec, s[38:39] ")
    (_, code), = _functions(good)
    assert not _masked(code)


def test_every_region_restores_its_own_mask():
    build = importlib.import_module("triton-kernel-test_amd.build")
    at = build.HIPFLAGS.index("-amdgpu-remove-redundant-endcf=0")
    assert build.HIPFLAGS[at - 1] == "-mllvm"


def test_no_lane_is_left_out_in_the_built_kernels(tmp_path):
    L = importlib.import_module("triton-kernel-test_amd._lib")
    tool = Path("/opt/rocm/llvm/bin/llvm-objdump")
    tool = str(tool) if tool.exists() else shutil.which("llvm-objdump")
    if not L.LIB_PATH.exists() or tool is None:
        pytest.skip("needs the built library and llvm-objdump")
    bad, kernels = {}, 0
    for i, obj in enumerate(_code_objects(L.LIB_PATH.read_bytes())):
        f = tmp_path / f"{i}.elf"
        f.write_bytes(obj)
        listing = subprocess.run([tool, "-d", "--no-show-raw-insn", str(f)], capture_output=True, text=True, check=True).stdout
        for name, code in _functions(listing):
            kernels += 1
            found = _masked(code)
            if found:
                bad[name] = found[:4]
    assert kernels > 1000 and not bad, bad
