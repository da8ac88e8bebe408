"""The cluster-size rule of the few-rows tensor-core kernel (xvram_b200/csrc/split_rule.hpp): its
table of cluster capacities belongs to one kernel and keeps no failed query, and an input whose
quantised rows fit no size is told apart from an error."""
from __future__ import annotations

import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_split_rule(tmp_path):
    exe = tmp_path / "split_rule"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Wextra", "-Werror", "-I",
                    str(ROOT / "xvram_b200" / "csrc"), str(ROOT / "tests" / "split_rule.cpp"), "-o",
                    str(exe), "-lpthread"], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout


def test_each_kernel_has_its_own_table():
    """One table inside the function that is instantiated per kernel, none keyed by a pointer's
    type (which all instantiations share)."""
    text = (ROOT / "xvram_b200" / "csrc" / "feed_split.cuh").read_text()
    assert "template <Kind K, Epilogue E, class T>\ncudaError_t choose_split" in text
    assert text.count("CapacityTable") == 1 and "static CapacityTable table;" in text
