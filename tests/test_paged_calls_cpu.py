"""Calls on a paged cache that have to be refused, each for its own reason, without a device."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ not available")
def test_overlapping_caches_are_told_from_others(tmp_path):
    """Builds tests/native/overlap_check.cpp with g++ against flexkv_amd/csrc/kv_overlap.h."""
    exe = tmp_path / "overlap_check"
    cmd = ["g++", "-std=c++17", "-O1", "-Wall", "-I", os.path.join(ROOT, "flexkv_amd", "csrc"),
           os.path.join(ROOT, "tests", "native", "overlap_check.cpp"), "-o", str(exe)]
    build = subprocess.run(cmd, capture_output=True, text=True)
    assert build.returncode == 0, build.stderr
    res = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert res.returncode == 0 and "FAIL" not in res.stdout, res.stdout + res.stderr
    assert res.stdout.count("ok:") == 20
