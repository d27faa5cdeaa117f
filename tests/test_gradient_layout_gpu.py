"""Gradients that come back with strides (attention lays its own out as (B, T, H, D); a permuted view) and are then added to by operators that
walk over them row by row."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
pytestmark = pytest.mark.gpu


def test_a_gradient_with_strides_is_added_to(tmp_path):
    exe, pkg = str(tmp_path / "gradient_layout_check"), os.path.join(ROOT, "gradcraft_b200")
    cmd = ["g++", "-std=c++20", "-O1", "-I", pkg, "-I/usr/local/cuda/include", os.path.join(ROOT, "tests", "gradient_layout_check.cpp"), "-o", exe, "-L" + pkg, "-lgradc_b200",
           "-L/usr/local/cuda/lib64", "-lcudart", "-pthread", "-Wl,-rpath," + pkg, "-Wl,-rpath,/usr/local/cuda/lib64"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-3000:]
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr[-2000:] + r.stdout
    lines = [l.split() for l in r.stdout.splitlines()]
    assert len(lines) == 120 and all(v == "0" for _, v in lines), [l for l in lines if l[1] != "0"]
