"""Values that a compiled kernel would lose where lanes part (CPU tier).

Where registers are short the compiler splits a value's live range with a copy to
another register or to memory. Placed at the head of the block in which lanes meet again,
before the instruction that brings those back which had skipped the branch, such a copy
leaves their part of the new place as an earlier kernel left it. Results then depend on
what ran before, and most tests of them pass. So the built device code is read here:
a block that an empty EXEC branches to writes no lane's registers or memory before EXEC is widened.
"""

import re
import shutil
import struct
import subprocess
from pathlib import Path

import pytest

BUILD = Path(__file__).resolve().parents[1] / "open-pacho_amd" / "_build"
UNITS = sorted(path.stem for path in (BUILD.parent / "csrc").glob("*.hip"))
PER_LANE = ("v_", "ds_", "global_", "scratch_", "buffer_", "flat_")
WHOLE_WAVE = ("v_readlane", "v_writelane", "v_readfirstlane")  # whatever EXEC is


def lost_copies(lines):
    """(kernel, label, instructions) of every block as above in a disassembly with labels for its branches."""
    lines = [line.split("//")[0].strip() for line in lines]
    heads = [(n, m.group(1)) for n, line in enumerate(lines) if line.endswith(">:") for m in [re.search(r"<(\S+)>:$", line)]]
    labels = {n: name for n, name in heads if re.fullmatch(r"L\d+", name)}
    kernels = [(n, name) for n, name in heads if n not in labels] + [(len(lines), None)]
    found = []
    for (start, kernel), (end, _) in zip(kernels, kernels[1:]):
        joins = {line.split()[1] for line in lines[start:end] if line.startswith("s_cbranch_execz")}  # labels are a kernel's own
        for at in range(start, end):
            if labels.get(at) not in joins:
                continue
            early = []
            for line in lines[at + 1 : end]:
                if line.startswith("s_or_b64 exec, exec,"):
                    if early:
                        found.append((kernel, labels[at], early))
                    break
                if line.startswith(("s_cbranch", "s_branch", "s_endpgm")) or "exec" in line or line.endswith(">:"):
                    break
                if line.startswith(PER_LANE) and not line.startswith(WHOLE_WAVE):
                    early.append(line)
    return found


def disassembly(unit, tmp_path):
    """Of the unit's gfx950 code, which the object file bundles with the host's."""
    data = (BUILD / f"{unit}.o").read_bytes()
    start = data.find(b"__CLANG_OFFLOAD_BUNDLE__")
    if start < 0:
        return []
    (count,), at = struct.unpack_from("<Q", data, start + 24), start + 32
    for _ in range(count):
        offset, size, length = struct.unpack_from("<QQQ", data, at)
        name = data[at + 24 : at + 24 + length]
        at += 24 + length
        if name.endswith(b"gfx950"):
            code = tmp_path / "code"
            code.write_bytes(data[start + offset : start + offset + size])
            tool = shutil.which("llvm-objdump") or "/opt/rocm/llvm/bin/llvm-objdump"
            command = [tool, "-d", "--symbolize-operands", "--no-show-raw-insn", "--no-leading-addr", str(code)]
            return subprocess.run(command, capture_output=True, text=True, check=True).stdout.splitlines()
    return []


@pytest.mark.parametrize("unit", UNITS)
def test_no_copy_is_lost_where_lanes_meet(unit, tmp_path):
    if not (BUILD / f"{unit}.o").exists():
        pytest.skip("library not built in this tree (open-pacho_amd/build.py)")
    lines = disassembly(unit, tmp_path)
    assert any("s_endpgm" in line for line in lines) or unit in ("runtime", "gemm", "gemm_edges"), "no device code found"
    assert not lost_copies(lines)


PLANTED = """
<kernel>:
\ts_and_saveexec_b64 s[24:25], s[26:27]                      // 0000
\ts_cbranch_execz L0                                         // 0004
\tv_mov_b32_e32 v1, v2                                       // 0008
<L0>:
%s
\ts_or_b64 exec, exec, s[24:25]                              // 0010
\ts_endpgm                                                   // 0014
"""


def test_a_planted_copy_is_found():
    assert lost_copies((PLANTED % "\tv_accvgpr_write_b32 a2, v98").splitlines()) == [("kernel", "L0", ["v_accvgpr_write_b32 a2, v98"])]
    assert lost_copies((PLANTED % "\tscratch_store_dword off, v98, off").splitlines())
    assert not lost_copies((PLANTED % "\ts_mov_b32 s64, s53\n\tv_readlane_b32 s3, v255, 4").splitlines())
