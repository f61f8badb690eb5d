"""imq_qmm_lora_plan and factors by rank without a GPU, under the sanitizers (tests/sanitize/lora_plan)."""

from __future__ import annotations

import os
import re
import shutil
import subprocess

import pytest

DIR = os.path.join(os.path.dirname(os.path.abspath(__file__)), "sanitize", "lora_plan")


def test_plan_and_refusals():
    if not os.path.exists("/opt/rocm/llvm/bin/clang++") or shutil.which("make") is None:
        pytest.skip("ROCm clang++ or make not available")
    r = subprocess.run(["make", "-s", "-C", DIR], capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stdout + r.stderr
    env = dict(os.environ, ASAN_OPTIONS="detect_leaks=1:abort_on_error=1",
               UBSAN_OPTIONS="print_stacktrace=1:halt_on_error=1")
    r = subprocess.run([os.path.join(DIR, "_build", "lora_plan_refusals")], capture_output=True, text=True,
                       timeout=300, env=env)
    assert r.returncode == 0, r.stdout + r.stderr
    assert int(re.search(r"lora_plan_refusals: (\d+) checks", r.stdout).group(1)) > 35
