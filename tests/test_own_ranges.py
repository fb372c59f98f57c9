"""The token ranges that the waves of a shared-prefix decode take of a sequence's
own tokens: nothing of a sequence whose length and block counts the cache cannot
hold, and ranges inside the sequence otherwise (own_ranges_check.cpp, on the
host, from the kernel's own header)."""
import shutil
import subprocess
from pathlib import Path

import pytest

HERE = Path(__file__).resolve().parent


def test_ranges_stay_inside_the_sequence(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not available")
    exe = tmp_path / "own_ranges_check"
    subprocess.run([gxx, "-std=c++17", "-O1", "-Wall", "-o", str(exe), str(HERE / "own_ranges_check.cpp")], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr
    assert " 0 faults" in r.stdout
