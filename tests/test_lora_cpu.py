"""Adapters without a GPU: the C entry points' refusals under the sanitizers, the struct that
Python passes."""

from __future__ import annotations

import os
import re
import shutil
import subprocess

import pytest
import torch

import aestrix_amd as imq
from aestrix_amd import _lib

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)


def test_refusals_under_the_sanitizers():
    """tests/sanitize/lora: refused arguments with their status and a message, and calls that
    reach the device (which is not there)."""
    if not os.path.exists("/opt/rocm/llvm/bin/clang++") or shutil.which("make") is None:
        pytest.skip("ROCm clang++ or make not available")
    d = os.path.join(HERE, "sanitize", "lora")
    r = subprocess.run(["make", "-s", "-C", d], capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stdout + r.stderr
    env = dict(os.environ, ASAN_OPTIONS="detect_leaks=1:abort_on_error=1",
               UBSAN_OPTIONS="print_stacktrace=1:halt_on_error=1")
    r = subprocess.run([os.path.join(d, "_build", "lora_refusals")], capture_output=True, text=True,
                       timeout=300, env=env)
    assert r.returncode == 0, r.stdout + r.stderr
    assert int(re.search(r"lora_refusals: (\d+) checks", r.stdout).group(1)) > 70


def test_struct_matches_the_header(tmp_path):
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    src = tmp_path / "s.c"
    prints = "\n".join(f'printf("%zu ", offsetof(imq_lora, {f}));' for f, _ in _lib.Lora._fields_)
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "imq_lora.h"\n'
                   f'int main(void) {{ {prints} printf("%zu", sizeof(imq_lora)); return 0; }}')
    subprocess.run([cc, "-I", os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "s")], check=True)
    offsets = [int(x) for x in subprocess.run([str(tmp_path / "s")], capture_output=True, text=True).stdout.split()]
    import ctypes
    assert offsets.pop() == ctypes.sizeof(_lib.Lora)
    assert offsets == [getattr(_lib.Lora, f).offset for f, _ in _lib.Lora._fields_]


def test_host_tensors_are_refused():
    a, b = torch.zeros(8, 128, dtype=torch.bfloat16), torch.zeros(96, 8, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        imq.LoraAdapters([(a, b)])
    with pytest.raises(ValueError):
        imq.LoraAdapters([])
