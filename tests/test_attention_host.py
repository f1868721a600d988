"""Host checks of the paged cache's operators: how a step is divided, what their inline assembly holds."""
from __future__ import annotations

import glob
import os
import re
import subprocess

from voxwerk_amd import build

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_step_plans(tmp_path):
    exe = tmp_path / "step_plan"
    subprocess.run(["g++", "-std=c++17", "-O2", "-D__HIP_PLATFORM_AMD__", "-I", os.path.join(build.ROCM, "include"),
                    os.path.join(REPO, "tests", "step_plan.cpp"), "-o", str(exe)], check=True)
    p = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert p.returncode == 0, p.stdout


def assembly():
    """(place, instructions, the rest: operands and what is clobbered) of each inline assembly statement of the attention kernels."""
    for path in sorted(glob.glob(os.path.join(build.CSRC, "vxs_attn*")) + [os.path.join(build.CSRC, "vxs_append.hip")]):
        text = open(path, encoding="utf-8").read()
        for m in re.finditer(r"\basm\b(?:\s+volatile)?\s*\(\s*\"([^\"]*)\"([^;]*);", text):
            lines = [x.strip() for x in m.group(1).replace("\\t", " ").split("\\n")]
            yield f"{os.path.basename(path)}:{text.count(chr(10), 0, m.start()) + 1}", [x for x in lines if x], m.group(2)


def test_assembly_has_no_vector_arithmetic():
    """The compiler keeps the wait states between a matrix product (or a vector instruction before a swap of lanes) and the next
    instruction that reads its result only where it knows that instruction: none of them may be inline assembly."""
    found = list(assembly())
    assert len(found) >= 5
    for place, lines, _ in found:
        assert not [x for x in lines if x.startswith("v_")], f"{place}: {lines}"


def test_assembly_keeps_what_a_store_reads():
    """The registers of a store of more than 8 bytes may be written again two wait states after it; the compiler counts none of
    them for a store that is inline assembly, so they are part of it."""
    stores = [(place, lines) for place, lines, _ in assembly() if any(re.match(r"global_store_dwordx[34]", x) for x in lines)]
    assert stores
    for place, lines in stores:
        assert re.match(r"global_store_dwordx[34]", lines[-2]) and lines[-1] == "s_nop 1", f"{place}: {lines}"


def test_assembly_of_loads_into_lds():
    """A load into LDS that is inline assembly names m0, which it overwrites, and holds the five wait states between a vector
    instruction's writing a scalar register and a load's reading it."""
    loads = [x for x in assembly() if any(i.startswith("global_load_lds") for i in x[1])]
    assert loads
    for place, lines, rest in loads:
        waits = 0
        for x in lines[:lines.index(next(i for i in lines if i.startswith("global_load_lds")))]:
            waits += int(x.split()[1]) + 1 if x.startswith("s_nop") else 1
        assert lines[0].startswith("s_mov_b32 m0") and waits >= 5, f"{place}: {lines}"
        assert '"m0"' in rest, f"{place}: {rest}"
