"""The operators beside the programs without a device: refusals, the arithmetic that host and kernels share, frequencies."""
import ctypes
import math
import os
import subprocess

import pytest

from conftest import ROOT, package

CSRC = os.path.join(ROOT, "pjrt-ocl_b200", "csrc")


def test_checks_and_shared_arithmetic(tmp_path):
    exe = str(tmp_path / "operators_probe")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-I" + CSRC, os.path.join(ROOT, "tests", "adapter", "operators_probe.cc"),
                    os.path.join(CSRC, "operators_check.cc"), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr


@pytest.mark.parametrize("rot, base, scaling, factor", [(2, 10000.0, "plain", 1.0), (64, 10000.0, "linear", 8.0), (128, 500000.0, "stretch", 4.0), (96, 10000.0, "parts", 8.0)])
def test_frequencies_are_the_formulas(rot, base, scaling, factor):
    f = package().RopeFrequencies(rot, base, scaling, factor, 4096.0, 1.0, 32.0)
    assert len(f) == rot // 2
    for i, got in enumerate(f):
        b = base * factor ** (rot / (rot - 2)) if scaling == "stretch" else base
        want = b ** (-2.0 * i / rot)
        if scaling == "linear":
            want /= factor
        if scaling == "parts":                           # turns over the original length: fast ones stay, slow ones are divided
            turns = 4096.0 * want / (2.0 * math.pi)
            keep = min(1.0, max(0.0, (turns - 1.0) / (32.0 - 1.0)))
            want = want * keep + want / factor * (1.0 - keep)
        assert abs(got - want) <= 1e-13 * want           # (a power and a few products, 2^-53 each)


def test_refusals_before_a_device_is_asked_for():
    vm = package()
    for bad in (dict(rot_dim=7), dict(rot_dim=258), dict(base=0.0, rot_dim=8), dict(rot_dim=8, scaling="bent"), dict(rot_dim=8, scaling="linear", factor=0.0),
                dict(rot_dim=8, scaling="parts", factor=2.0), dict(rot_dim=8, scaling="parts", factor=2.0, original_length=4096.0, slow=32.0, fast=1.0)):
        with pytest.raises(vm.InvalidArgument):
            vm.RopeFrequencies(**bad)
    with pytest.raises(vm.InvalidArgument, match="frequencies, want"):
        vm.Rope.Create(None, 64, 1, 1, "bf16", frequencies=[1.0])
    with pytest.raises(vm.InvalidArgument, match="unknown type"):
        vm.Rope.Create(None, 64, 1, 1, "f64")
    with pytest.raises(vm.InvalidArgument, match="head_dim"):
        vm.Rope.Create(None, 63, 1, 1, "bf16", rot_dim=0)
    with pytest.raises(vm.InvalidArgument, match="null runtime"):
        vm.Rope.Create(None, 64, 1, 1, "bf16")
    good = dict(dtype="bf16", row_dtype="bf16", heads=2, head_dim=64, page_size=16, n_pages=4, k_pages=4096, v_pages=8192)
    with pytest.raises(vm.InvalidArgument, match="null runtime"):
        vm.PagedCache.Create(None, **good)
    for change, part in ((dict(head_dim=40), "head_dim"), (dict(dtype="e4m3"), "need scales"), (dict(k_pages=0), "null pages"), (dict(q_heads=3), "multiple"),
                         (dict(dtype="f16"), "own type"), (dict(k_pages=4104), "aligned")):
        with pytest.raises(vm.InvalidArgument, match=part):
            vm.PagedCache.Create(None, **{**good, **change})
    with pytest.raises(vm.InvalidArgument, match="out of range"):
        vm.Batch(-1, 0, 0, 0, 0, 0)
    lib, err = vm.runtime.lib(), ctypes.create_string_buffer(256)
    for name, args in (("b2_rope_apply", (None, 0, None) + (None,) * 6 + (None,)), ("b2_cache_write", (None,) * 5), ("b2_cache_read", (None,) * 5),
                       ("b2_cache_attend", (None, None, None, None, 1.0, 1, 0, None, None, None)), ("b2_cache_status", (None, None)),
                       ("b2_scratch_create", (None, None)), ("b2_rope_create", (None, None, None)), ("b2_cache_create", (None, None, None))):
        assert getattr(lib, name)(*args, err, 256) != 0 and b"null" in err.value, name
    for name in ("b2_rope_destroy", "b2_cache_destroy", "b2_scratch_destroy"):
        getattr(lib, name)(None)
    # without room for a message
    assert lib.b2_cache_write(None, None, None, None, None, None, 0) != 0
