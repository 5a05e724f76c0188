"""Wait states in front of loads that an asm block issues straight into LDS: the compiler, which keeps them everywhere else, does not look into such a block.
On gfx9 a load into LDS needs one wait state behind a scalar write of M0, and any vector memory instruction five behind a vector instruction's write of a scalar
register that it reads. Each source with such a load is built to assembly, and every load in it is looked at."""
import os
import re
import subprocess

import pytest

from onnx_genai_amd import build

SOURCES = sorted(s for s in build.HIP_SOURCES if re.search(r"buffer_load_\w+ [^\"]* lds\"", open(os.path.join(build.CSRC, s)).read()))


def registers(operands):
    """The scalar registers that a text of operands names."""
    found = set()
    for first, last, one, name in re.findall(r"\bs\[(\d+):(\d+)\]|\bs(\d+)\b|\b(vcc|m0)\b", operands):
        found |= set(range(int(first), int(last) + 1)) if first else {int(one)} if one else {name}
    return found


def waits_missing(instructions):
    """(loads into LDS, those of them that come too early)"""
    loads, early = 0, []
    for at, text in enumerate(instructions):
        if not re.match(r"(buffer|global)_load_.* lds$", text):
            continue
        loads += 1
        reads = registers(text)
        states = 0
        for before in reversed(instructions[max(at - 5, 0):at]):
            nop = re.match(r"s_nop (\w+)$", before)
            if nop:
                states += int(nop.group(1), 0) + 1
                continue
            written = registers(before.split(None, 1)[-1].split(",")[0])
            if (before.startswith("s_") and "m0" in written and states < 1) or (before.startswith("v_") and written & reads and states < 5):
                early.append((before, text))
            states += 1
    return loads, early


def test_rules_find_what_comes_too_early():
    load = "buffer_load_dwordx4 v6, s[0:3], 0 offen lds"
    assert waits_missing(["s_mov_b32 m0, s14", load]) == (1, [("s_mov_b32 m0, s14", load)])
    assert waits_missing(["s_mov_b32 m0, s14", "s_nop 0", load]) == (1, [])
    assert waits_missing(["v_readfirstlane_b32 s2, v1", "s_mov_b32 m0, s14", "s_nop 0", load])[1] == [("v_readfirstlane_b32 s2, v1", load)]
    assert waits_missing(["v_readfirstlane_b32 s2, v1", "s_nop 4", "s_mov_b32 m0, s14", "s_nop 0", load]) == (1, [])
    assert waits_missing(["v_readfirstlane_b32 s4, v1", "s_mov_b32 m0, s14", "s_nop 0", load]) == (1, [])


@pytest.mark.parametrize("source", SOURCES)
def test_loads_into_lds_wait(source, tmp_path):
    assembly = tmp_path / "kernels.s"
    built = subprocess.run([build.HIPCC, *build.DEVICE_FLAGS, "-S", "--cuda-device-only", os.path.join(build.CSRC, source), "-o", str(assembly)], capture_output=True, text=True)
    assert built.returncode == 0, built.stderr
    lines = (line.split(";")[0].strip() for line in assembly.read_text().splitlines())
    loads, early = waits_missing([line for line in lines if line and not line.startswith(".") and not line.endswith(":")])
    assert loads > 0 and not early, (len(early), loads, early[:3])


def test_sources_with_such_loads_are_found():
    assert "kernels/int8_gemm.hip" in SOURCES and "hip_ffi.hip" in SOURCES
