"""LoraAdapters and quantized_matmul_lora where other tests do not go."""

from __future__ import annotations

import gc
import weakref

import pytest
import torch

import aestrix_amd as imq
from core_reference import check
from test_gpu_lora import each, gen, ints, pairs, projection, randn, runs, wanted

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


BF16, F16 = torch.bfloat16, torch.float16


def run(m, k, n, ranks, which, t, **plan):
    """As the plan says, against the definition."""
    g = gen(m + 3 * k + 5 * n)
    proj, ab, x = projection(g, n, k, t), pairs(g, n, k, ranks, t), randn(g, m, k, dtype=t)
    ad = imq.LoraAdapters(ab, [1.0 + i % 3 for i in range(len(ab))])
    p = imq.quantized_matmul_lora_plan(ad, m)
    assert plan.items() <= p.items(), p
    ids = ints(which(m))
    got = imq.quantized_matmul_lora(x, *proj, ad, ids)
    check(got, *wanted(x, proj, ab, [1.0 + i % 3 for i in range(len(ab))], ids), f"[{m} x {n}] K {k}")


@pytest.mark.parametrize("t", [BF16, F16])
@pytest.mark.parametrize("m,k,n,ranks,plan", [
    (1, 2560, 500, [16] * 8, dict(kernel="few", u="rows", join="outputs")),
    (32, 2560, 600, [64] * 16, dict(kernel="few", u="rows", join="outputs")),
    (33, 256, 300, [40] * 3, dict(kernel="split", splits=1, u="rows", join="outputs")),
    (100, 9728, 600, [16] * 24, dict(kernel="split", u="rows", join="outputs")),
    (64, 2560, 6144, [256], dict(kernel="split", u="tiles", join="tiles")),
    (200, 9728, 2560, [256, 33], dict(kernel="split", u="tiles", join="tiles")),
    (300, 64, 100, [8, 17], dict(kernel="tiles_reg", u="rows", grouped=False, join=None)),
    (4100, 192, 60, [64, 64], dict(kernel="tiles_reg", u="tiles", grouped=False, join=None)),
    (300, 2560, 6144, [64], dict(kernel="tiles", u="tiles", grouped=False, join=None)),
    (512, 2560, 2560, [64] * 32, dict(kernel="tiles", u="tiles", grouped=True, join=None)),
    (4000, 256, 4000, [16] * 1000, dict(kernel="tiles", u="rows", grouped=True, join=None))])
def test_each_way(m, k, n, ranks, plan, t):
    run(m, k, n, ranks, each(len(ranks)), t, **plan)
    run(m, k, n, ranks, runs(len(ranks), 50), t, **plan)


@pytest.mark.parametrize("count", [1023, 1024, 1500])
def test_as_many_adapters_as_are_grouped_and_more(count):
    run(6000, 256, 5000, [1 + i % 16 for i in range(count)], lambda m: [(i * 37) % (count + 1) - 1 for i in range(m)], BF16,
        kernel="tiles", grouped=True)


@pytest.mark.parametrize("m", [16383, 16384, 16385, 20000])
@pytest.mark.parametrize("which", [each(5), runs(5, 3001)])
def test_more_rows_than_stay_in_lds(m, which):
    run(m, 256, 300, [16, 8, 1, 16, 3], which, BF16, kernel="tiles", grouped=True)


@pytest.mark.parametrize("m,join", [(65535, "outputs"), (65536, "tiles"), (70000, "tiles")])
@pytest.mark.parametrize("n", [1, 8])
def test_a_join_of_many_rows(m, n, join):
    run(m, 256, n, [16, 8, 1, 16, 3], runs(5, 3001), F16, kernel="split", join=join)


def test_refusals_of_the_plan():
    ad = imq.LoraAdapters(pairs(gen(1), 96, 128, [8], BF16))
    with pytest.raises(imq.ImqInvalid):
        imq.quantized_matmul_lora_plan(ad, 0)
    assert imq.quantized_matmul_lora_plan(ad, 1)["workspace_bytes"] >= 16
