"""The cut of a batch's step into workgroups (wick_amd/csrc/batch_plan.h): every key a row
sees is taken once, and partial states are joined from where they were written."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_plan_covers_every_key_once(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not available")
    exe = str(tmp_path / "check")
    subprocess.run([gxx, "-std=c++17", "-O2", "-D_GLIBCXX_ASSERTIONS", "-Wall", "-Wextra", "-Werror", "-I",
                    os.path.join(ROOT, "wick_amd", "csrc"), os.path.join(ROOT, "tests", "batch_plan_check.cpp"), "-o",
                    exe], check=True)
    r = subprocess.run([exe], stdout=subprocess.PIPE, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout
