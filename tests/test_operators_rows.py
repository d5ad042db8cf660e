"""What the operators refuse, without a device: rows that lie over each other (against the bytes of all small layouts), values that f32 does not hold."""
import os
import subprocess

import pytest

from conftest import ROOT, package

CSRC = os.path.join(ROOT, "pjrt-ocl_b200", "csrc")


def test_rows_over_each_other(tmp_path):
    exe = str(tmp_path / "rows_probe")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-I" + CSRC, os.path.join(ROOT, "tests", "adapter", "rows_probe.cc"),
                    os.path.join(CSRC, "operators_check.cc"), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr


def test_a_magnitude_that_f32_does_not_hold():
    """It is multiplied in f32: an infinity there would make sines of 0 a NaN."""
    vm = package()
    for magnitude in (1e39, -1e300, float("nan"), float("inf")):
        with pytest.raises(vm.InvalidArgument, match="magnitude"):
            vm.Rope.Create(None, 64, 1, 1, "bf16", magnitude=magnitude)
    with pytest.raises(vm.InvalidArgument, match="null runtime"):
        vm.Rope.Create(None, 64, 1, 1, "bf16", magnitude=3e38)
