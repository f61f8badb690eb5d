"""Attention with NaN and infinities in what the queries see: the outputs say so, in the time that
finite ones take."""

from __future__ import annotations

import time

import pytest
import torch

import aestrix_amd as imq

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16
NAN, INF = float("nan"), float("inf")

# queries, keys, heads, kv heads, dim, causal; kernel, tile rows and whether keys are split, as on 256 CUs
PLANS = [
    (1, 4000, 8, 8, 128, True, ("few", 1, True)), (3, 700, 600, 300, 64, True, ("few", 6, False)),
    (40, 4000, 2, 2, 128, True, ("tiles", 64, True)), (100, 700, 200, 200, 128, True, ("tiles", 128, False)),
    (64, 200, 128, 128, 128, True, ("tiles", 64, False)), (1100, 300, 32, 32, 128, False, ("tiles", 256, False)),
    (6000, 6000, 32, 32, 64, True, ("tiles", 256, False)), (20, 900, 3, 1, 33, True, ("rows", 1, False))]


@pytest.fixture(autouse=True)
def _need_gpu(request):
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")
    print(request.node.name, flush=True)


def inputs(nq, nk, heads, kv, dim, dtype=BF16):
    g = torch.Generator(device="cuda").manual_seed(nq + nk)
    return (torch.randn(n, h, dim, generator=g, device="cuda").to(dtype) for n, h in ((nq, heads), (nk, kv), (nk, kv)))


def plan_is(q, k, v, plan, **kw):
    if torch.cuda.get_device_properties(0).multi_processor_count == 256:
        p = imq.attention_plan(q, k, v, **kw)
        assert (p["kernel"], p["tile_rows"], p["splits"] > 1) == plan, p


def expected(q, k, v, head, causal):
    """What IEEE arithmetic gives for one head, with what a query does not see left out: float64 [nq, dim]."""
    nq, nk = q.shape[0], k.shape[0]
    j = torch.arange(nk, device="cuda")
    seen = j <= (torch.arange(nq, device="cuda")[:, None] + nk - nq) if causal else torch.ones(nq, nk, dtype=torch.bool, device="cuda")
    kh = head * k.shape[1] // q.shape[1]
    e = (q[:, head].double() @ k[:, kh].double().T.contiguous()) * q.shape[2] ** -0.5
    p = torch.softmax(e.masked_fill(~seen, -INF), -1)
    # 0 of a hidden key times its value is nothing, whatever the value: a product a part.
    vd = v[:, kh].double()
    odd = ~torch.isfinite(vd)
    o = p @ torch.where(odd, 0.0, vd)
    for i in odd.any(1).nonzero().flatten().tolist():
        term = p[:, i:i + 1] * torch.where(odd[i], vd[i], 0.0)[None]
        o = o + torch.where(seen[:, i:i + 1], term, 0.0)
    return o


def same(got, want, what):
    """Where `want` is not finite the same, elsewhere near (the bounds of the numbers are tested elsewhere)."""
    odd = ~torch.isfinite(want)
    assert torch.equal(got.isnan(), want.isnan()), (what, "NaN")
    assert torch.equal(got.isinf(), want.isinf()) and torch.equal(got[got.isinf()].double(), want[want.isinf()]), (what, "infinities")
    if not odd.all():
        assert float((got.double() - want)[~odd].abs().max()) < 0.05, what


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("nq,nk,heads,kv,dim,causal,plan", PLANS)
def test_visible_ones_reach_the_output(nq, nk, heads, kv, dim, causal, plan, dtype):
    """A NaN and an infinity in the keys, in the values and in a query, seen by some of the queries."""
    for where in ("k", "v", "v late", "q", "v all"):
        q, k, v = inputs(nq, nk, heads, kv, dim, dtype)
        plan_is(q, k, v, plan, causal=causal)
        if where == "k":
            k[nk // 3, 0, 3] = NAN
            k[nk - 2, -1, 5] = INF
        elif where == "v":
            v[1, 0, 3], v[nk // 3, 0, 4], v[2, -1, 7] = INF, -INF, NAN
        elif where == "v late":
            v[nk - 1, 0, 3], v[nk - 2, 0, 4], v[max(nk - 40, 0), -1, 7] = INF, -INF, NAN
        elif where == "q":
            q[nq // 2, 0, 3], q[0, -1, 1] = NAN, INF
            k[0, -1, 1] = 1.0  # a score of +infinity
        else:
            v[..., 2], v[..., 4] = INF, NAN
        got = imq.attention(q, k, v, causal=causal)
        for head in (0, heads - 1):
            same(got[:, head], expected(q, k, v, head, causal), (where, head))


@pytest.mark.parametrize("nq,nk,heads,kv,dim,causal,plan", PLANS)
def test_hidden_ones_beside_visible_ones(nq, nk, heads, kv, dim, causal, plan):
    """Keys behind a sequence's own hold anything, in one tile with keys that hold a NaN."""
    q, k, v = inputs(nq, nk, heads, kv, dim)
    n = nk - 45
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    k[n:], v[n:] = NAN, INF
    v[n - 1, 0, 1] = NAN
    got = imq.attention(q[None], k[None], v[None], causal=causal, k_lens=lens)[0]
    for head in (0, heads - 1):
        same(got[:, head], expected(q, k[:n], v[:n], head, causal) if n >= nq or not causal else
             torch.cat([torch.zeros(nq - n, dim, dtype=torch.float64, device="cuda"),
                        expected(q[nq - n:], k[:n], v[:n], head, True)]), head)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("nq,nk,heads,kv,dim,causal,plan", PLANS)
def test_scores_of_minus_infinity(nq, nk, heads, kv, dim, causal, plan, dtype):
    """A query whose scores are all -infinity has no softmax, whichever kernel it takes; one that sees
    no key gives zeros, and keys of such a score beside others have no weight."""
    q, k, v = inputs(nq, nk, heads, kv, dim, dtype)
    plan_is(q, k, v, plan, causal=causal)
    k[..., 0] = 1.0
    q[nq // 2, 0, 0] = -INF
    q[nq // 3, -1, 0] = 1.0
    k[nk // 2, -1, 0] = -INF
    got = imq.attention(q, k, v, causal=causal)
    for head in (0, heads - 1):
        same(got[:, head], expected(q, k, v, head, causal), head)
    none = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = imq.attention(q[None], k[None], v[None], causal=causal, k_lens=none)
    assert not got.any()


def test_overlapping_rows_of_values():
    """Rows of values that begin inside the one before (a window over a sequence): what a tile
    reads behind the last is part of those in front."""
    g = torch.Generator(device="cuda").manual_seed(3)
    flat = torch.randn(8 * 200 + 128, generator=g, device="cuda").to(BF16)
    flat[8 * 199 + 100] = INF  # of the last row alone, whose element 100 it is; of the row before: 108
    v = flat.as_strided((200, 1, 128), (8, 128, 1))
    q, k = (torch.randn(n, 1, 128, generator=g, device="cuda").to(BF16) for n in (40, 200))
    got = imq.attention(q, k, v)
    same(got[:, 0], expected(q, k, v, 0, False), "overlapping")


@pytest.mark.parametrize("nq,nk,heads,kv,causal,what", [
    (*size, what) for size in [(4096, 4096, 32, 8, True), (1, 65536, 32, 8, True), (4096, 4096, 24, 24, False)]
    for what in ("q", "k", "v", "v all") if what != "v all" or size[0] == 1 or not size[4]])
def test_they_cost_no_more_than_finite_ones(nq, nk, heads, kv, causal, what):
    """The rows that hidden keys may have spoilt are made again, one after another, some thousand times
    slower than a tile's: not those that what they see has spoilt.  (Where every key holds one, those
    behind the diagonal do, and the causal rows are made again.)"""
    q, k, v = inputs(nq, nk, heads, kv, 128)

    def timed():
        torch.cuda.synchronize()
        t = time.perf_counter()
        imq.attention(q, k, v, causal=causal)
        torch.cuda.synchronize()
        return time.perf_counter() - t

    timed()
    plain = min(timed() for _ in range(5))
    if what == "q":
        q[:, :, 0] = NAN
    elif what == "k":
        k[0] = NAN
    elif what == "v":
        v[0, :, 5] = INF
    else:
        v[:, :, 5] = NAN
    odd = min(timed() for _ in range(3))
    print(f"  {plain * 1e6:.0f} us, {odd * 1e6:.0f} us", flush=True)
    assert odd < 4 * plain + 1e-3
