"""The few-row mxfp4 kernel's ring of k-blocks, run as a model on the host over the kernel's own rules."""

import os
import shutil
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(os.path.dirname(HERE), "mlxturbo_b200", "csrc")


@pytest.fixture(scope="module")
def model(tmp_path_factory):
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("needs a C++ compiler")
    exe = str(tmp_path_factory.mktemp("ring") / "ring_model")
    subprocess.run([cxx, "-O2", "-std=c++17", "-I", CSRC, os.path.join(HERE, "mx_ring_model.cpp"), "-o", exe],
                   check=True)

    def run(early):
        out = subprocess.run([exe, "4000", "0", str(early)], check=True, capture_output=True, text=True).stdout
        lines = out.splitlines()
        return int(lines[-1].split()[0]), lines[:-1]

    return run


def test_planes_are_those_of_the_block_read(model):
    """No planes are overwritten before the tensor core has read them, however far it trails, and nothing stops."""
    bad, lines = model(0)
    assert bad == 0, lines[:5]


def test_model_sees_a_slot_taken_one_block_early(model):
    """A warp that looks at its slot when one k-block fewer has begun overwrites planes still to be read."""
    bad, lines = model(1)
    assert bad > 0 and any("wrong planes" in line for line in lines)
