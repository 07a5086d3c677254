"""Host check of the attention layer's overlap test (tensorrs_b200/csrc/heads.h):
tests/cpp/heads_check.cpp compares it with the bytes that random small views
reach.  A shared byte is never missed, and slices of one buffer along any of
its dimensions are never taken for overlapping."""
from __future__ import annotations

import subprocess
from pathlib import Path

from conftest import ROOT

SRC = ROOT / "tests" / "cpp" / "heads_check.cpp"
BIN = ROOT / "tests" / "cpp" / "_build" / "heads_check"


def test_overlaps_are_those_of_the_bytes():
    BIN.parent.mkdir(exist_ok=True)
    cxx = "/usr/bin/g++" if Path("/usr/bin/g++").exists() else "g++"
    csrc = ROOT / "tensorrs_b200" / "csrc"
    cmd = [cxx, "-std=c++17", "-O2", "-Wall", "-Wextra", "-I", str(csrc), str(SRC), str(csrc / "plan.cpp"), "-o", str(BIN)]
    subprocess.run(cmd, check=True, capture_output=True, text=True)
    out = subprocess.run([str(BIN)], check=True, capture_output=True, text=True, timeout=300).stdout.split("\n")
    _, pairs, share, missed, apart = out[0].split()
    assert int(share) > 10000 and int(missed) == 0 and int(apart) > 10000
    _, cases, refused = out[1].split()
    assert int(cases) == 120 and int(refused) == 0
