"""Host check of how an 8-bit append's launch is divided."""
from __future__ import annotations

import os
import subprocess

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_append_plans(tmp_path):
    exe = tmp_path / "append_plan"
    subprocess.run(["g++", "-std=c++17", "-O2", os.path.join(REPO, "tests", "append_plan.cpp"), "-o", str(exe)], check=True)
    p = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert p.returncode == 0, p.stdout
