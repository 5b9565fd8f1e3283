"""The cache operators' plain C++ parts, compiled into host programs with the kernels' own headers."""
import os
import re
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(os.path.dirname(HERE), "daisychain-infer_b200", "csrc")


def source(name):
    return open(os.path.join(CSRC, name)).read()


@pytest.fixture
def run(tmp_path):
    def go(name):
        exe = str(tmp_path / name)
        subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-I", CSRC, "-o", exe,
                        os.path.join(HERE, "host", name + ".cpp")], check=True)
        got = subprocess.run([exe], capture_output=True, text=True, timeout=120)
        assert got.returncode == 0, got.stdout + got.stderr
    return go


def test_checks_of_strided_buffers(run):
    run("span")


def test_drained_rings_have_nothing_in_flight(run):
    run("ring")


@pytest.mark.parametrize("name, copiers, own", [("dc_prefix.cu", 1, 1), ("dc_weights.cu", 2, 0)])
def test_kernels_drain_before_they_end(name, copiers, own):
    """Each copying lane drains its ring in any case, each issuing warp waits for its products, and no
    kernel has a drain of its own making."""
    src = source(name)
    assert len(re.findall(r"\bdcr::drain<", src)) == copiers and len(re.findall(r"\bdcr::drain_own<", src)) == own
    assert len(re.findall(r"commit\(idle\);\s*__syncwarp\(\);\s*dcu::warp_wait\(idle, 0, a\.status\);", src)) == copiers
    assert not re.search(r"if \(issued < ", src)


@pytest.mark.parametrize("name, waits", [("dc_prefix.cu", 1), ("dc_weights.cu", 2)])
def test_lanes_that_wait_for_different_barriers_are_ordered(name, waits):
    """A vote tells a warp that all its waits are met but orders no memory between its lanes: waits whose
    lanes look at different barriers end in __syncwarp."""
    src = source(name)
    assert len(re.findall(r"\bwarp_wait_each\(odd \?", src)) == waits and not re.search(r"\bwarp_wait\(odd \?", src)
    body = re.search(r"bool warp_wait_each\(.*?\n}", source("dc_umma.cuh"), re.S).group(0)
    assert re.search(r"warp_wait\(bar, parity, status\);\s*__syncwarp\(\);\s*return", body)
