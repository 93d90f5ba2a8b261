"""Compiles tests/paged_few_check.cpp: split calls that use fewer parts than their workspace has room for."""
import os
import subprocess
import tempfile

from conftest import ROOT


def test_few_of_the_parts():
    exe = os.path.join(tempfile.mkdtemp(prefix="fa_paged_few_"), "paged_few_check")
    subprocess.run(["g++", "-O2", "-std=c++17", "-Wall", os.path.join(ROOT, "tests", "paged_few_check.cpp"), "-o", exe], check=True)
    out = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stdout + out.stderr
    assert out.stdout.startswith("OK 20000"), out.stdout
