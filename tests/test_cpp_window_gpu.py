"""The C++ mirror's windowed attention (tests/cpp/test_window.cpp)."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.gpu
def test_windowed_forward_through_the_mirror():
    res = subprocess.run([os.path.join(ROOT, "tests", "cpp", "test_window")], capture_output=True, text=True, timeout=300)
    print(res.stdout)
    assert res.returncode == 0 and "test_window: ok" in res.stdout, res.stdout + res.stderr
