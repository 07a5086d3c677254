"""Host check of the counts kept per device (tensorrs_b200/csrc/device_cache.h),
which the launch sizes of most kernels come from."""
from __future__ import annotations

import subprocess
from pathlib import Path

from conftest import ROOT

SRC = ROOT / "tests" / "cpp" / "device_cache_check.cpp"
BIN = ROOT / "tests" / "cpp" / "_build" / "device_cache_check"


def test_counts_are_kept_per_device_and_failures_not_at_all():
    BIN.parent.mkdir(exist_ok=True)
    cxx = "/usr/bin/g++" if Path("/usr/bin/g++").exists() else "g++"
    cmd = [cxx, "-std=c++17", "-O1", "-Wall", "-Wextra", "-pthread", "-I", str(ROOT / "tensorrs_b200" / "csrc"), str(SRC),
           "-o", str(BIN)]
    subprocess.run(cmd, check=True, capture_output=True, text=True)
    r = subprocess.run([str(BIN)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and r.stdout == "ok\n", r.stdout
