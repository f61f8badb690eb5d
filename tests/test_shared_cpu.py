"""attention_shared without a GPU: the C entry point's refusals under the sanitizers, the
struct that Python packs."""

from __future__ import annotations

import os
import re
import shutil
import subprocess

import pytest
import torch

import aestrix_amd as imq
from aestrix_amd import core

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)


def test_refusals_under_the_sanitizers():
    """tests/sanitize/shared: refused arguments with their status and a message, and calls that
    reach the device (which is not there)."""
    if not os.path.exists("/opt/rocm/llvm/bin/clang++") or shutil.which("make") is None:
        pytest.skip("ROCm clang++ or make not available")
    d = os.path.join(HERE, "sanitize", "shared")
    r = subprocess.run(["make", "-s", "-C", d], capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stdout + r.stderr
    env = dict(os.environ, ASAN_OPTIONS="detect_leaks=1:abort_on_error=1",
               UBSAN_OPTIONS="print_stacktrace=1:halt_on_error=1")
    r = subprocess.run([os.path.join(d, "_build", "shared_refusals")], capture_output=True, text=True,
                       timeout=300, env=env)
    assert r.returncode == 0, r.stdout + r.stderr
    assert int(re.search(r"shared_refusals: (\d+) checks", r.stdout).group(1)) > 25


def test_packed_struct_matches_the_header(tmp_path):
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    fields = ["k", "v", "k_row", "k_head", "v_row", "v_head", "rows"]
    src = tmp_path / "s.c"
    prints = "\n".join(f'printf("%zu ", offsetof(imq_shared_keys, {m}));' for m in fields)
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "imq_core.h"\n'
                   f'int main(void) {{ {prints} printf("%zu", sizeof(imq_shared_keys)); return 0; }}')
    subprocess.run([cc, "-I", os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "s")], check=True)
    offsets = [int(x) for x in subprocess.run([str(tmp_path / "s")], capture_output=True, text=True).stdout.split()]
    assert offsets.pop() == core._SHARED_KEYS.size
    for i, at in enumerate(offsets):
        values = [0] * len(fields)
        values[i] = 0x11
        raw = core._SHARED_KEYS.pack(*values)
        assert raw[at] == 0x11 and sum(raw) == 0x11, fields[i]


def test_host_tensors_are_refused():
    z = torch.zeros(2, 3, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        imq.attention_shared(z, z, z, z, z)
