"""Attention where one key outweighs all others: what the small weights add up to is kept."""

from __future__ import annotations

import pytest
import torch

import aestrix_amd as imq
from core_reference import U32, check, half_step, least

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def _need_gpu(request):
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")
    print(request.node.name, flush=True)


# Half of f16's smallest step against a weight of 2^11, the most that the row's largest has
# when it is the newest: what a weight's rounding can cost at least.  (2^-25 would be that of
# weights of 1, and lose the whole sum of 2^17 weights of 2^-25.1.)
LEAST_WEIGHT = {F16: 2.0 ** -36, BF16: 0.0}


def exact(q, k, v, scale, causal, softcap, slopes):
    """(o, bound) of one sequence from the definition in 64 bits.  Every bound is worst case:
    the dot products' and the sums' roundings as many as there are terms, a weight half a
    step of T or LEAST_WEIGHT, the result half a step of T."""
    nq, h, d = q.shape
    nk, hk = k.shape[:2]
    o = torch.empty((nq, h, d), dtype=torch.float64, device=q.device)
    bound = torch.empty_like(o)
    away = (torch.arange(nq, device=q.device)[:, None] + nk - nq - torch.arange(nk, device=q.device)).double()
    for i in range(h):
        qi, ki, vi = q[:, i].double(), k[:, i * hk // h].double(), v[:, i * hk // h].double()
        e = scale * (qi @ ki.T.contiguous())
        err = (d + 8) * U32 * scale * (qi.abs() @ ki.abs().T.contiguous())
        if softcap:
            e = softcap * torch.tanh(e / softcap)
            err = err + 8 * U32 * softcap
        if slopes is not None:
            e = e - slopes[i].double() * away.abs()
            err = err + 4 * U32 * slopes[i].double() * away.abs()
        if causal:
            e = e.masked_fill(away < 0, -torch.inf)
        w = torch.exp(e - e.amax(-1, keepdim=True))
        p = w / w.sum(-1, keepdim=True)
        err = (err + 4 * U32 * (e - e.amax(-1, keepdim=True)).abs()).nan_to_num(posinf=0.0)
        n = (w > 0).sum(-1, keepdim=True)
        av = vi.abs()
        small = LEAST_WEIGHT[q.dtype] / w.sum(-1, keepdim=True)
        # The sum is of the same rounded weights: its error is divided by all of them.
        lost = ((p * err).sum(-1, keepdim=True) + (half_step(q.dtype) + (2 * n + 32) * U32) + small * n) * (p @ av)
        o[:, i] = p @ vi
        bound[:, i] = half_step(q.dtype) * o[:, i].abs() + 1.02 * (
            (p * (err * 1.01 + half_step(q.dtype))) @ av + small * ((w > 0).double() @ av) + lost) + least(q.dtype)
    return o, bound


# queries, keys, heads, kv heads, dim, causal; kernel, tile rows and whether keys are split, as on 256 CUs
PLANS = [
    (1, 20000, 8, 8, 128, True, ("few", 1, True)), (3, 6000, 600, 300, 64, True, ("few", 6, False)),
    (40, 20000, 2, 2, 128, True, ("tiles", 64, True)), (100, 6000, 200, 200, 128, True, ("tiles", 128, False)),
    (64, 6000, 300, 300, 64, False, ("tiles", 128, False)), (64, 200, 128, 128, 128, True, ("tiles", 64, False)),
    (1100, 6000, 32, 32, 128, False, ("tiles", 256, False)), (1100, 6000, 32, 32, 64, False, ("tiles", 256, False)),
    (20, 900, 3, 1, 33, True, ("rows", 1, False))]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("softcap,slope", [(0.0, False), (60.0, False), (0.0, True), (60.0, True)])
@pytest.mark.parametrize("at", [0, 70])
@pytest.mark.parametrize("nq,nk,heads,kv,dim,causal,plan", PLANS)
def test_one_key_outweighs_the_others(nq, nk, heads, kv, dim, causal, plan, at, softcap, slope, dtype):
    """Key `at`, whose value is zero, scores 17 to 18 above the others, whose weights, 2^-25
    of its, are all that the output is made of."""
    g = torch.Generator(device="cuda").manual_seed(nk + dim + at)
    randn = lambda *s: torch.randn(s, generator=g, device="cuda")
    q, k, v = 0.01 * randn(nq, heads, dim), 0.05 * randn(nk, kv, dim), 1.0 + 0.25 * randn(nk, kv, dim)
    q[..., 0] = 16.0
    k[..., 0] = 0.0
    k[at, :, 0] = 17.3 * dim ** 0.5 / 16.0 if not softcap else 17.8 * dim ** 0.5 / 16.0
    v[at] = 0.0
    q, k, v = q.to(dtype), k.to(dtype), v.to(dtype)
    slopes = torch.full((heads,), 2.0 ** -16, device="cuda") if slope else None
    kw = dict(causal=causal, softcap=softcap, slopes=slopes)
    if torch.cuda.get_device_properties(0).multi_processor_count == 256:
        p = imq.attention_plan(q, k, v, **kw)
        assert (p["kernel"], p["tile_rows"], p["splits"] > 1) == plan, p
    got = imq.attention(q, k, v, **kw)
    some = list(range(0, heads, max(1, heads // 4)))  # heads are alike
    kv_of = [i * kv // heads for i in some]
    want, bound = exact(q[:, some], k[:, kv_of], v[:, kv_of], dim ** -0.5, causal, softcap, slopes)
    check(got[:, some], want, bound, f"{nq} x {nk}")


@pytest.mark.parametrize("softcap", [0.0, 60.0])
@pytest.mark.parametrize("nq,heads,kv,dim,causal,at,plan", [
    (3, 600, 300, 64, False, 200, ("few", 6, False)), (1, 300, 300, 128, True, 200, ("few", 1, False)),
    (40, 2, 2, 128, False, 100, ("tiles", 64, False)), (100, 200, 200, 128, False, 100, ("tiles", 128, False)),
    (1100, 32, 32, 64, False, 100, ("tiles", 256, False)), (20, 3, 1, 33, False, 100, ("rows", 1, False))])
def test_large_values(nq, heads, kv, dim, causal, at, plan, softcap):
    """bf16 values of 2^121, of 250 keys of which one, behind a first tile of 32 or 64, weighs 2^7 times
    the others: their sums with weights of 1 and less stay under 2^128, with weights of 2^7 they do not."""
    q, k = torch.zeros(nq, heads, dim, device="cuda"), torch.zeros(250, kv, dim, device="cuda")
    q[..., 0] = 16.0
    k[at, :, 0] = 4.9 * dim ** 0.5 / 16.0
    v = torch.full((250, kv, dim), 2.0 ** 121, device="cuda")
    q, k, v = q.to(BF16), k.to(BF16), v.to(BF16)
    kw = dict(causal=causal, softcap=softcap)
    if torch.cuda.get_device_properties(0).multi_processor_count == 256:
        p = imq.attention_plan(q, k, v, **kw)
        assert (p["kernel"], p["tile_rows"], p["splits"] > 1) == plan, p
    got = imq.attention(q, k, v, **kw)
    want, bound = exact(q[:, :1], k[:, :1], v[:, :1], dim ** -0.5, causal, softcap, None)
    for head in (0, heads - 1):
        check(got[:, head:head + 1], want, bound, f"head {head}")
