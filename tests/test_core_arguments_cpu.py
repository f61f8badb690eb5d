"""Combinations of the block core's arguments, without a GPU."""

from __future__ import annotations

import os
import re
import shutil
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


def test_arguments_under_the_sanitizers():
    """tests/sanitize/arguments: calls that are refused, with a message, beside ones that are not."""
    if not os.path.exists("/opt/rocm/llvm/bin/clang++") or shutil.which("make") is None:
        pytest.skip("ROCm clang++ or make not available")
    d = os.path.join(HERE, "sanitize", "arguments")
    r = subprocess.run(["make", "-s", "-C", d], capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stdout + r.stderr
    env = dict(os.environ, ASAN_OPTIONS="detect_leaks=1:abort_on_error=1",
               UBSAN_OPTIONS="print_stacktrace=1:halt_on_error=1")
    r = subprocess.run([os.path.join(d, "_build", "core_arguments")], capture_output=True, text=True,
                       timeout=300, env=env)
    assert r.returncode == 0, r.stdout + r.stderr
    assert int(re.search(r"core_arguments: (\d+) checks", r.stdout).group(1)) > 3000
