"""Compiles tests/paged_plan_check.cpp (the paged kernels' own index arithmetic, csrc/fa_paged_plan.h, built with g++)."""
import os
import subprocess
import tempfile

from conftest import ROOT


def test_every_visible_key_belongs_to_one_piece():
    exe = os.path.join(tempfile.mkdtemp(prefix="fa_paged_"), "paged_plan_check")
    subprocess.run(["g++", "-O2", "-std=c++17", "-Wall", os.path.join(ROOT, "tests", "paged_plan_check.cpp"), "-o", exe], check=True)
    out = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stdout + out.stderr
    assert out.stdout.startswith("OK "), out.stdout
    assert int(out.stdout.split()[1]) > 20000
