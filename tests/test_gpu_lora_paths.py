"""LoraAdapters and quantized_matmul_lora where other tests do not go."""

from __future__ import annotations

import gc
import weakref

import pytest
import torch

import aestrix_amd as imq

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _need_gpu(request):
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")
    print(request.node.name, flush=True)


@pytest.mark.parametrize("t", [torch.bfloat16, torch.float16])
def test_a_set_of_parameters_is_a_copy(t):
    """Adapters that are trained elsewhere: no part of a graph, and nothing of them is kept."""
    ab = [tuple(torch.nn.Parameter(torch.ones(s, dtype=t, device="cuda")) for s in ((8, 64), (100, 8))) for _ in range(2)]
    left = [weakref.ref(p) for pair in ab for p in pair]
    ad = imq.LoraAdapters(ab, 0.5)
    assert not (ad.a.requires_grad or ad.b.requires_grad or ad.scale.requires_grad)
    del ab
    gc.collect()
    assert all(r() is None for r in left)
