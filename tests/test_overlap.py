"""Whether two strided tensors share memory (csrc/overlap.h; no GPU): against a list of every byte, for random layouts, and for the
views of a fused projection's rows."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_layouts_that_share_memory_are_always_seen(tmp_path):
    exe = str(tmp_path / "overlap_check")
    subprocess.check_call(["g++", "-O2", "-std=c++17", "-Wall", "-Werror", "-I", os.path.join(ROOT, "onebitsparsemul_b200", "csrc"),
                           os.path.join(ROOT, "tests", "host", "overlap_check.cpp"), "-o", exe])
    out = subprocess.run([exe, "300000"], capture_output=True, text=True)
    assert out.returncode == 0, out.stdout + out.stderr
    wrong, overlapping, told_apart, taken_to_meet = map(int, out.stdout.split())
    assert wrong == 0 and overlapping > 1000 and told_apart > 5 * taken_to_meet
