"""A wait that gave up and a batch that named a bad page are both reported, the wait first (csrc/device_status.h; no GPU)."""
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "onebitsparsemul_b200", "csrc")


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_a_bad_batch_does_not_hide_a_wait_that_gave_up(tmp_path):
    exe = str(tmp_path / "device_status_check")
    subprocess.check_call(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-I", CSRC, os.path.join(ROOT, "tests", "host", "device_status_check.cpp"), "-o", exe])
    out = subprocess.run([exe], capture_output=True, text=True)
    assert out.returncode == 0 and out.stdout.split() == ["0"], out.stdout + out.stderr


@pytest.mark.parametrize("name", ["cache_attend.cu", "cache_attend_sm100.cu"])
def test_waits_and_bad_batches_have_words_of_their_own(name):
    with open(os.path.join(CSRC, name)) as f:
        code = f.read()
    waits = set(re.findall(r"budget, &(\w+), \d+\)", code))
    marks = set(re.findall(r"note_bad_batch\(&(\w+)\)", code))
    assert len(waits) == 1 and len(marks) == 1 and not waits & marks
    assert not re.search(r"atomic\w+\(&(?:%s)\b" % "|".join(waits | marks), code)
