"""attention_shared on each of its kernels, which the tests ask the plan for first, against its
definition in 64 bits."""

from __future__ import annotations

import pytest
import torch

import aestrix_amd as imq

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16
NAN, INF = float("nan"), float("inf")


@pytest.fixture(autouse=True)
def _need_gpu(request):
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")
    print(request.node.name, flush=True)


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, dtype):
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


@pytest.mark.parametrize("n,nq,nk,heads,kv,dim", [(3, 1, 3000, 8, 2, 128), (2, 5, 40, 4, 4, 64), (1, 300, 300, 8, 2, 128),
                                                  (8, 2048, 2048, 32, 8, 128), (2, 3, 50, 4, 2, 136), (0, 3, 5, 2, 2, 64)])
def test_the_plan_of_no_shared_keys_is_attentions(n, nq, nk, heads, kv, dim):
    q = torch.zeros((n, nq, heads, dim), dtype=BF16, device="cuda")
    k = q.new_zeros((n, nk, kv, dim))
    none = q.new_empty((0, kv, dim))
    plan, own = imq.attention_shared_plan(q, k, k, none, none, causal=True), imq.attention_plan(q, k, k, causal=True)
    few = own["kernel"] == "few"
    assert plan == {"kernel": "stream" if few else own["kernel"], "tile_rows": own["tile_rows"],
                    "splits": 0 if few else own["splits"], "own_splits": own["splits"] if few else 0,
                    "workspace_bytes": own["workspace_bytes"]}
