"""The plans of a batch's steps (wick_amd/csrc/batch_plan.h) fit what a handle allocates and
what a captured call launches: a plan that did not would be refused, or a replay's rows NaN."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_plans_fit_their_handles(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not available")
    exe = str(tmp_path / "check")
    subprocess.run([gxx, "-std=c++17", "-O2", "-Wall", "-Wextra", "-Werror", "-I", os.path.join(ROOT, "wick_amd", "csrc"),
                    os.path.join(ROOT, "tests", "batch_bounds_check.cpp"), "-o", exe], check=True)
    r = subprocess.run([exe, "60000", "1"], stdout=subprocess.PIPE, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout
