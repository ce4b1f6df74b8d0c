"""The phases by which a CTA that gave up waits for its copies (bk_ring.h), against a model of the barriers: no GPU."""
import os
import shutil
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


def test_a_ring_of_copies_is_waited_for_to_the_last(tmp_path):
    if not shutil.which("g++"):
        pytest.skip("needs g++")
    exe = str(tmp_path / "ring")
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-Wall", os.path.join(HERE, "ring_host.cpp"), "-o", exe])
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and r.stdout.strip() == "0", r.stdout
