"""The attention kernels' rings: the waits before a block ends, after one that ran out too, are for each stage's last fill, so
that no copy is in flight then and none of them waits in vain (csrc/ring.cuh, compiled for the host)."""
import ctypes
import os
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(os.path.dirname(HERE), "nemotron-3.5-bolt-tensorfold-dgx-spark_b200", "csrc")


@pytest.fixture(scope="module")
def ring(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("ring") / "ring_harness.so")
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-I", CSRC, os.path.join(HERE, "ring_harness.cpp"), "-o", out], check=True)
    return ctypes.CDLL(out)


@pytest.mark.parametrize("stages", [2, 4, 24, 48])
def test_fills_without_a_gap(ring, stages):
    for issued in range(5 * stages):
        assert ring.ring_plain(stages, issued) == 0, issued


@pytest.mark.parametrize("stages", [24, 48])
def test_fills_of_which_some_of_eight_lanes_made_theirs(ring, stages):
    for base in range(4 * stages):
        for mask in range(256):
            assert ring.ring_gap(stages, base, mask) == 0, (base, mask)
