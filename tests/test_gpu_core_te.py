"""``TextEncoderLayers.attn_core``: what it refuses, and the epsilon it takes."""

from __future__ import annotations

import pytest
import torch

import aestrix_amd as imq
from aestrix_amd.te import TextEncoderLayers, random_te_layers
from core_reference import check, rope

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


@pytest.fixture(autouse=True)
def _need_gpu(request):
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")
    print(request.node.name, flush=True)


def encoder(**kw):
    layers = random_te_layers(1, dtype=BF16, seed=4, hidden=512, nq=1024, nkv=256, inter=768)
    g = torch.Generator(device="cuda").manual_seed(4)
    for l in layers:
        l.norm_q, l.norm_k = (1 + 0.1 * torch.randn(128, generator=g, device="cuda") for _ in range(2))
    return TextEncoderLayers(layers, max_rows=64, **kw)


def test_a_refused_call_leaves_qkv_alone():
    """q and k are turned in place before the attention runs: nothing may be refused after that."""
    plan = encoder()
    g = torch.Generator(device="cuda").manual_seed(5)
    qkv = torch.randn(48, plan.nq + 2 * plan.nkv, generator=g, device="cuda").to(BF16)
    keep = qkv.clone()
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
    bad = [dict(lens=i32(24, 24).long()), dict(lens=i32(24)), dict(lens=i32(24, 24).cpu()), dict(lens=i32(24, 0, 24, 0)[::2]),
           dict(lens=i32(24, 24).view(2, 1)), dict(positions=i32(*range(47))), dict(positions=torch.arange(48, device="cuda")),
           dict(out=torch.empty((47, plan.nq), dtype=BF16, device="cuda")), dict(out=qkv.flatten()[:48 * plan.nq].view(48, plan.nq)),
           dict(out=qkv.flatten()[-48 * plan.nq:].view(48, plan.nq))]
    for kw in bad:
        with pytest.raises(ValueError):
            plan.attn_core(0, qkv, 2, **kw)
        torch.cuda.synchronize()
        assert torch.equal(qkv, keep), kw.keys()


@pytest.mark.parametrize("eps", [1e-6, 0.5])
def test_the_head_norms_take_the_encoders_epsilon(eps):
    plan = encoder(eps=eps)
    g = torch.Generator(device="cuda").manual_seed(6)
    qkv = torch.randn(20, plan.nq + 2 * plan.nkv, generator=g, device="cuda").to(BF16)
    keep = qkv.clone()
    plan.attn_core(0, qkv)
    f, _ = imq.rope_frequencies(128, 1e6, device="cuda")
    pos = torch.arange(20, dtype=torch.int32, device="cuda")
    want, bound = rope(keep[:, :plan.nq].unflatten(1, (-1, 128)), pos, f, None, False, 1.0, plan.layers[0].norm_q, eps)
    check(qkv[:, :plan.nq].unflatten(1, (-1, 128)), want, bound, f"q, epsilon {eps}")
