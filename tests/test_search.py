"""The searches for borders in rows of logits, on the host: right, and with a bound on their steps."""

import os
import shutil
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(os.path.dirname(HERE), "mlxturbo_b200", "csrc")


@pytest.fixture(scope="module")
def check(tmp_path_factory):
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("needs a C++ compiler")
    exe = str(tmp_path_factory.mktemp("search") / "check")
    subprocess.run([cxx, "-O2", "-std=c++17", "-I", CSRC, os.path.join(HERE, "search_check.cpp"), "-o", exe],
                   check=True)

    def run(*args):
        out = subprocess.run([exe, *args], check=True, capture_output=True, text=True).stdout.splitlines()
        return [int(x) for x in out[-1].split()], out[:-1]

    return run


def test_borders(check):
    """min-p's border where a largest logit of 0, min_p = 1 or a huge temperature puts 1e9 keys between it and where
    its formula says, and in ordinary rows; the number of equal weights that a mass takes, down to weights that the
    sum does not feel."""
    (bad, most), lines = check()
    assert bad == 0, lines[:5]
    assert most <= 66


def test_walking_key_by_key_does_not_end(check):
    """What the bound is for: from the formula's guess the same borders are more than a million keys away."""
    (bad, most), lines = check("walk")
    assert bad > 0 and most >= 1000000 and any(line.startswith("max 0 T 1 min-p 1:") for line in lines)
    assert any(line.startswith("above 1 w 1e-22") for line in lines)
