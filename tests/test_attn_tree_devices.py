"""The tree attention called on several devices of one process, without a GPU: its host side over a
CUDA runtime that keeps count of shared-memory limits and launches."""
import os
import subprocess

import pytest

from conftest import ROOT


@pytest.fixture(scope="module")
def lines(tmp_path_factory):
    lib = os.path.join(ROOT, "slate_b200")
    objs = [os.path.join(lib, "_build", f) for f in ("attn_tree.o", "attn_tree_tc.o", "rope.o")]
    if not all(os.path.exists(o) for o in objs):
        subprocess.run(["make", "-C", os.path.join(lib, "csrc"), "-j8"], check=True, stdout=subprocess.DEVNULL)
    exe = str(tmp_path_factory.mktemp("devices") / "attn_tree_devices")
    cuda = os.environ.get("CUDA", "/usr/local/cuda")
    subprocess.run(["g++", "-std=c++17", "-O1", f"-I{cuda}/include", f"-I{ROOT}/include", "-o", exe,
                    os.path.join(ROOT, "tests", "attn_tree_devices.cpp"), *objs, "-lm"], check=True)
    return subprocess.run([exe], check=True, capture_output=True, text=True, timeout=60).stdout.splitlines()


def test_every_device_is_given_its_limits(lines):
    for i in range(2):
        assert lines[i].startswith(f"pass 0 device {i}: 0 failed") and not lines[i].endswith(" 0 set")


def test_limits_are_set_once_a_device(lines):
    assert lines[2:4] == ["pass 1 device 0: 0 failed, 0 set", "pass 1 device 1: 0 failed, 0 set"]


def test_a_failure_is_not_remembered(lines):
    assert lines[4] == "device 2: -5 then 0"


def test_a_device_beyond_the_known_ordinals(lines):
    assert lines[5] == "device 70: 0 0"


def test_an_error_of_another_call_is_not_this_ones(lines):
    assert lines[6] == "after an error of another call: 0 0"
