"""The block core without a GPU: the C entry points' refusals under the sanitizers, the
structs that Python packs, the frequencies of ``rope``."""

from __future__ import annotations

import math
import os
import re
import shutil
import struct
import subprocess

import pytest
import torch

import aestrix_amd as imq
from aestrix_amd import core

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)


def test_refusals_under_the_sanitizers():
    """tests/sanitize/core: every argument that the checks refuse, with its status and a
    message, and every call that they let through reaches the device (which is not there)."""
    if not os.path.exists("/opt/rocm/llvm/bin/clang++") or shutil.which("make") is None:
        pytest.skip("ROCm clang++ or make not available")
    d = os.path.join(HERE, "sanitize", "core")
    r = subprocess.run(["make", "-s", "-C", d], capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stdout + r.stderr
    env = dict(os.environ, ASAN_OPTIONS="detect_leaks=1:abort_on_error=1",
               UBSAN_OPTIONS="print_stacktrace=1:halt_on_error=1")
    r = subprocess.run([os.path.join(d, "_build", "core_refusals")], capture_output=True, text=True,
                       timeout=300, env=env)
    assert r.returncode == 0, r.stdout + r.stderr
    assert int(re.search(r"core_refusals: (\d+) checks", r.stdout).group(1)) > 150


def test_packed_structs_match_the_header(tmp_path):
    """Offsets of every field, from the C compiler."""
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "imq_core.h")).read(), flags=re.S)
    for name, fields in (("imq_rope_heads", core._ROPE_HEADS), ("imq_attention_args", core._ATTENTION_ARGS)):
        body = re.search(r"typedef struct %s \{(.*?)\}" % name, text, re.S).group(1)
        members = [re.sub(r".*[ *]", "", m.strip()) for line in body.split(";")
                   for m in line.split(",") if m.strip()]
        src = tmp_path / f"{name}.c"
        prints = "\n".join(f'printf("%zu ", offsetof({name}, {m}));' for m in members)
        src.write_text(f'#include <stdio.h>\n#include <stddef.h>\n#include "imq_core.h"\n'
                       f'int main(void) {{ {prints} printf("%zu", sizeof({name})); return 0; }}')
        exe = tmp_path / name
        subprocess.run([cc, "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
        offsets = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True).stdout.split()]
        assert offsets.pop() == fields.size
        # One value at a time: its bytes stand where the field does.
        codes = [c for n, c in re.findall(r"(\d*)([Pqif])", fields.format.replace("4x", "")) for _ in range(int(n or 1))]
        assert len(codes) == len(members)
        for i, c in enumerate(codes):
            values = [0] * len(codes)
            values[i] = 1.5 if c == "f" else 0x11
            raw = fields.pack(*values)
            assert raw.index(struct.pack("@" + c, values[i]).strip(b"\0")[:1]) >= offsets[i]
            assert struct.unpack_from("@" + c, raw, offsets[i])[0] == values[i], members[i]


def test_frequencies():
    f, a = imq.rope_frequencies(128, 1e4)
    assert f.dtype == torch.float64 and a == 1.0
    want = torch.tensor([1e4 ** (-2.0 * j / 128) for j in range(64)], dtype=torch.float64)
    assert torch.allclose(f, want, rtol=1e-14, atol=0)
    g, a = imq.rope_frequencies(128, 1e4, scaling="linear", factor=4.0)
    assert a == 1.0 and torch.allclose(g, want / 4, rtol=1e-14, atol=0)
    g, a = imq.rope_frequencies(128, 1e4, scaling="ntk", factor=4.0)
    assert a == 1.0 and g[0] == 1.0 and abs(float(g[-1] * 4 / want[-1]) - 1) < 1e-12
    assert bool((g[1:] < want[1:]).all() and (g[1:] > want[1:] / 4 - 1e-18).all())


@pytest.mark.parametrize("rot,base,factor,old", [(128, 1e6, 4.0, 32768), (64, 1e4, 32.0, 4096), (32, 500.0, 8.0, 64)])
def test_yarn_frequencies(rot, base, factor, old):
    """Fast pairs kept, slow ones divided, a ramp between whose ends are the pairs that turn
    32 times and once over the trained length."""
    f, a = imq.rope_frequencies(rot, base, scaling="yarn", factor=factor, original_len=old)
    plain, _ = imq.rope_frequencies(rot, base)
    assert a == pytest.approx(0.1 * math.log(factor) + 1.0, rel=1e-15)
    turns = old * plain / (2 * math.pi)
    r = f / plain
    assert bool(((r <= 1 + 1e-12) & (r >= 1 / factor - 1e-12)).all())
    assert bool((r[1:] <= r[:-1] + 1e-12).all()), "monotone"
    step = base ** (2.0 / rot)  # a pair's turns against the next one's: the ends are whole pairs
    assert bool((r[turns > 32 * step] == 1).all())
    assert torch.allclose(r[turns < 1 / step], torch.tensor(1 / factor, dtype=torch.float64), rtol=1e-12)


def test_frequency_refusals():
    for kw in (dict(rot_dim=0), dict(rot_dim=63), dict(rot_dim=64, base=1.0), dict(rot_dim=64, factor=0.5),
               dict(rot_dim=64, scaling="cubic"), dict(rot_dim=2, scaling="ntk", factor=2.0),
               dict(rot_dim=64, scaling="yarn", beta_fast=1.0), dict(rot_dim=64, scaling="yarn", original_len=0)):
        with pytest.raises(ValueError):
            imq.rope_frequencies(**kw)


def test_host_tensors_are_refused():
    z = torch.zeros(2, 3, 64, dtype=torch.bfloat16)
    pos, f = torch.zeros(2, dtype=torch.int32), imq.rope_frequencies(64)[0]
    with pytest.raises(ValueError):
        imq.attention(z, z, z)
    with pytest.raises(ValueError):
        imq.rope(z, positions=pos, inv_freq=f)
    with pytest.raises(ValueError):
        imq.ln_mod(z, torch.zeros(64), torch.zeros(64))


def test_rows_past_32_bits_are_refused():
    """They would be passed on modulo 2^32."""
    from aestrix_amd.core import _int32
    assert _int32((1 << 31) - 1, "rows") == (1 << 31) - 1 and _int32(0, "rows") == 0
    with pytest.raises(ValueError, match="2147483648 rows"):
        _int32(1 << 31, "rows")
