"""Which rows lie over each other, without a device: the operators' checks against the bytes of all small layouts."""
import os
import subprocess

from conftest import ROOT

CSRC = os.path.join(ROOT, "pjrt-ocl_b200", "csrc")


def test_rows_over_each_other(tmp_path):
    exe = str(tmp_path / "rows_probe")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-I" + CSRC, os.path.join(ROOT, "tests", "adapter", "rows_probe.cc"),
                    os.path.join(CSRC, "operators_check.cc"), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr
