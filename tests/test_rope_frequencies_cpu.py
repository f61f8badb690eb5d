"""The YaRN frequencies of ``rope_frequencies``, pair by pair from their description."""

import math

import pytest

import aestrix_amd as imq


def described(rot, base, factor, old, fast, slow):
    """The share of its frequency that each pair keeps: 1 where it turns more than `fast` times over
    `old` positions, 1 / factor under `slow`, a line over the pair's index between the last pair that
    is kept (the first one, if none is) and the first that is divided, wherever that would be."""
    log = lambda turns: rot / 2 * math.log(old / (2 * math.pi * turns), base)  # the index that turns so often
    a, b = max(math.floor(log(fast)), 0), math.ceil(log(slow))
    out = []
    for j in range(rot // 2):
        turns = old * base ** (-2 * j / rot) / (2 * math.pi)
        divided = 1.0 if turns < slow else 0.0 if turns > fast or j <= a else min((j - a) / (b - a), 1.0)
        out.append(1.0 - divided + divided / factor)
    return out


@pytest.mark.parametrize("rot,base,factor,old,fast,slow", [
    (128, 1e4, 4.0, 131072, 32.0, 1.0),   # the slowest pair turns 2.4 times: none is divided whole
    (128, 1e4, 8.0, 1 << 20, 32.0, 1.0),  # nor nearly
    (64, 1e6, 4.0, 32768, 32.0, 1.0), (128, 1e6, 16.0, 8192, 32.0, 1.0), (32, 500.0, 8.0, 64, 32.0, 1.0),
    (64, 1e4, 4.0, 4, 32.0, 1.0),         # every pair turns less than once: all are divided whole
    (96, 5e5, 2.0, 40000, 16.0, 4.0), (2, 1e4, 4.0, 4096, 32.0, 1.0), (2, 1e4, 4.0, 3, 32.0, 1.0)])
def test_yarn_keeps_divides_and_ramps(rot, base, factor, old, fast, slow):
    f, amplitude = imq.rope_frequencies(rot, base, scaling="yarn", factor=factor, original_len=old, beta_fast=fast,
                                        beta_slow=slow)
    plain, _ = imq.rope_frequencies(rot, base)
    assert amplitude == pytest.approx(0.1 * math.log(factor) + 1.0, rel=1e-15)
    assert (f / plain).tolist() == pytest.approx(described(rot, base, factor, old, fast, slow), rel=1e-9)


def test_yarn_past_the_last_pair():
    """128 elements, base 1e4, trained on 131072 positions, 4 times that: the ramp goes from pair 45 to
    pair 70, and the last pair, 63, keeps 1 - 18 / 25 * 3 / 4 of its frequency."""
    f, _ = imq.rope_frequencies(128, 1e4, scaling="yarn", factor=4.0, original_len=131072)
    plain, _ = imq.rope_frequencies(128, 1e4)
    assert float(f[63] / plain[63]) == pytest.approx(1 - 18 / 25 * 0.75, rel=1e-12)
