"""Calls from several host threads on a host-only build (no GPU): a call's two kernels, which meet
in the workspace of their stream, follow each other."""

import os
import re
import shutil
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
DIR = os.path.join(HERE, "sanitize", "threads")


def test_split_calls_of_several_threads():
    if not os.path.exists("/opt/rocm/llvm/bin/clang++") or shutil.which("make") is None:
        pytest.skip("ROCm clang++ or make not available")
    r = subprocess.run(["make", "-s", "-C", DIR], capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stdout + r.stderr
    run = [os.path.join(DIR, "_build", "stream_threads")]
    r = subprocess.run(run, capture_output=True, text=True, timeout=120)
    if "unexpected memory mapping" in r.stderr:  # addresses too random for the sanitizer's shadow
        r = subprocess.run(["setarch", "-R", *run], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "ThreadSanitizer" not in r.stderr, r.stdout + r.stderr[-4000:]
    assert int(re.search(r"stream_threads: (\d+) calls", r.stdout).group(1)) == 6 * 40 + 2 + 4
