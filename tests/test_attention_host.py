"""Host checks of the paged cache's operators: how a step is divided."""
from __future__ import annotations

import os
import subprocess

from voxwerk_amd import build

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_step_plans(tmp_path):
    exe = tmp_path / "step_plan"
    subprocess.run(["g++", "-std=c++17", "-O2", "-D__HIP_PLATFORM_AMD__", "-I", os.path.join(build.ROCM, "include"),
                    os.path.join(REPO, "tests", "step_plan.cpp"), "-o", str(exe)], check=True)
    p = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert p.returncode == 0, p.stdout
