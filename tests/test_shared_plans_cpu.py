"""The plans of ``attention_shared`` on 256 CUs: both sides of its rules, and for many sizes that
ranges and tiles cover keys and rows (no GPU)."""

import os
import re
import shutil
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
DIR = os.path.join(HERE, "sanitize", "shared_plans")


def test_plans():
    if not os.path.exists("/opt/rocm/llvm/bin/clang++") or shutil.which("make") is None:
        pytest.skip("ROCm clang++ or make not available")
    r = subprocess.run(["make", "-s", "-C", DIR], capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stdout + r.stderr
    env = dict(os.environ, ASAN_OPTIONS="detect_leaks=1:abort_on_error=1",
               UBSAN_OPTIONS="print_stacktrace=1:halt_on_error=1")
    r = subprocess.run([os.path.join(DIR, "_build", "shared_plans")], capture_output=True, text=True,
                       timeout=120, env=env)
    assert r.returncode == 0, r.stdout + r.stderr
    assert int(re.search(r"shared_plans: (\d+) checks", r.stdout).group(1)) > 50000
