"""attention_shared on each of its kernels, which the tests ask the plan for first, against its
definition in 64 bits."""

from __future__ import annotations

import ctypes

import pytest
import torch

import aestrix_amd as imq
from aestrix_amd import _lib
from aestrix_amd.ops import context
from core_reference import check
from test_gpu_shared import falls, ints, packed, run_batch, wanted

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


def plan(shared, n, nq, nk, heads, kv, dim, dtype, *, causal=True, softcap=0.0, slope=False, qn=None, kn=None, prefix=None):
    q = torch.empty((n, nq, heads, dim), dtype=dtype, device="cuda")
    k, sk = q.new_empty((n, nk, kv, dim)), q.new_empty((shared, kv, dim))
    return imq.attention_shared_plan(q, k, k, sk, sk, causal=causal, softcap=softcap, slopes=falls(heads) if slope else None,
                                     q_lens=ints(qn), k_lens=ints(kn), prefix_lens=ints(prefix))


def packed_plan(shared, rows, n, longest, heads, kv, dim, dtype, longest_k=None, **kw):
    q = torch.empty((rows, heads, dim), dtype=dtype, device="cuda")
    k, sk = q.new_empty((rows, kv, dim)), q.new_empty((shared, kv, dim))
    at = ints([0] * (n + 1))
    return imq.attention_shared_plan(q, k, k, sk, sk, causal=True, q_offsets=at, k_offsets=at, max_q=longest,
                                     max_k=longest if longest_k is None else longest_k, **kw)


def whole(p, tile_rows):
    assert p["kernel"] == "tiles" and p["tile_rows"] == tile_rows and p["splits"] == 1, p


SCORES = [(0.0, False), (0.0, True), (30.0, False), (5.0, True)]


# Of few tiles a sequence (a CU's second place from the least keys up), and of eight and more, one sequence
# after the other; keys that end inside a tile, a pair of tiles, at one and before one.
@pytest.mark.parametrize("softcap,slope", SCORES)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("shared,n,nq,nk,heads,kv,dim,dtype", [
    (333, 9, 260, 260, 32, 8, 128, BF16), (257, 24, 140, 140, 32, 8, 128, F16), (65, 24, 140, 150, 16, 8, 64, BF16),
    (128, 33, 260, 260, 8, 2, 72, F16), (1, 33, 260, 270, 8, 2, 64, F16), (191, 40, 130, 60, 32, 8, 128, BF16)])
def test_tiles_of_128_rows(shared, n, nq, nk, heads, kv, dim, dtype, causal, softcap, slope):
    whole(plan(shared, n, nq, nk, heads, kv, dim, dtype, causal=causal, softcap=softcap, slope=slope), 128)
    run_batch(shared, nq, nk, heads, kv, dim, dtype, n=n, causal=causal, softcap=softcap, slope=slope)


@pytest.mark.parametrize("softcap,slope", SCORES)
@pytest.mark.parametrize("shared,n,nq,nk,heads,kv,dim,dtype", [
    (333, 33, 260, 300, 8, 2, 128, BF16), (190, 24, 140, 160, 32, 8, 128, F16), (63, 20, 300, 200, 16, 4, 64, F16)])
def test_tiles_of_128_rows_of_uneven_lengths(shared, n, nq, nk, heads, kv, dim, dtype, softcap, slope):
    """More queries than keys among them, none of either, prefixes."""
    qn = [nq if s % 4 == 0 else s * 37 % (nq + 1) for s in range(n)]
    kn = [s * 53 % (nk + 1) for s in range(n)]
    prefix = [kn[s] * (s % 3) // 2 for s in range(n)]
    whole(plan(shared, n, nq, nk, heads, kv, dim, dtype, softcap=softcap, slope=slope, qn=qn, kn=kn, prefix=prefix), 128)
    run_batch(shared, nq, nk, heads, kv, dim, dtype, softcap=softcap, slope=slope, qn=qn, kn=kn, prefix=prefix)


@pytest.mark.parametrize("slope", [False, True])
def test_tiles_that_attention_would_have_of_256_rows(slope):
    q, k = (torch.empty((5, 1030, 8, 128), dtype=BF16, device="cuda") for _ in range(2))
    assert imq.attention_plan(q, k, k)["tile_rows"] == 256
    whole(plan(300, 5, 1030, 1030, 8, 8, 128, BF16, causal=False, slope=slope), 128)
    run_batch(300, 1030, 1030, 8, 8, 128, BF16, n=5, causal=False, slope=slope)


@pytest.mark.parametrize("softcap,slope", SCORES)
@pytest.mark.parametrize("dim,dtype", [(128, BF16), (64, F16), (72, BF16)])
def test_whole_tiles_of_64_rows(dim, dtype, softcap, slope):
    kw = dict(softcap=softcap, slope=slope)
    whole(plan(1000, 9, 200, 270, 8, 2, dim, dtype, **kw), 64)
    run_batch(1000, 200, 270, 8, 2, dim, dtype, n=9, **kw)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("n,nq,nk,heads,shared,tile_rows", [(40, 200, 200, 4, 103, 128), (9, 200, 200, 8, 1000, 64)])
def test_hidden_keys_of_whole_tiles(n, nq, nk, heads, shared, tile_rows, dtype):
    """NaN and infinities behind the keys, behind the diagonal and behind the shared rows."""
    g = gen(8)
    q = randn(g, n, nq, heads, 128, dtype=dtype)
    k, v = (randn(g, n, nk + 40, 2, 128, dtype=dtype) for _ in range(2))
    rows = [randn(g, shared + 60, 2, 128, dtype=dtype) for _ in range(2)]
    rows[0][shared:], rows[1][shared:] = NAN, INF
    sk, sv = rows[0][:shared], rows[1][:shared]
    kn = [nk - s * 7 % 70 for s in range(n)]
    for s, b in enumerate(kn):
        k[s, b:], v[s, b:] = NAN, INF
        # The last key: only the last query sees it.
        k[s, b - 1, 0], v[s, b - 1, 0, 5], v[s, b - 1, 1] = NAN, -INF, NAN
    whole(imq.attention_shared_plan(q, k, v, sk, sv, causal=True, k_lens=ints(kn)), tile_rows)
    got = imq.attention_shared(q, k, v, sk, sv, causal=True, k_lens=ints(kn))
    for s, b in enumerate(kn):
        want, bound = wanted(q[s, :-1], k[s, :b - 1], v[s, :b - 1], sk, sv, scale=128 ** -0.5, causal=True)
        check(got[s, :-1], want, bound, f"sequence {s}")
        assert bool(got[s, -1].isnan().all())


@pytest.mark.parametrize("softcap", [0.0, 20.0])
def test_packed_documents_of_hidden_keys(softcap):
    """The same in one stretch of rows; rows of no document are NaN."""
    g = gen(31)
    lens = [(13 * i) % 78 for i in range(44)]
    at = [sum(lens[:i]) + 3 for i in range(45)]  # three rows before the first document
    n = at[-1] + 4
    q, k, v = randn(g, n, 8, 128, dtype=BF16), *(randn(g, n, 2, 128, dtype=BF16) for _ in range(2))
    sk, sv = (randn(g, 900, 2, 128, dtype=BF16) for _ in range(2))
    for x, spoilt in ((q, NAN), (k, NAN), (v, INF)):
        x[:3], x[at[-1]:] = spoilt, spoilt
    for i, m in zip(at, lens):
        if m:
            k[i + m - 1], v[i + m - 1] = NAN, INF
    out = torch.full_like(q, 9.0)
    kw = dict(causal=True, softcap=softcap, q_offsets=ints(at), k_offsets=ints(at), max_q=77, max_k=77)
    assert imq.attention_shared_plan(q, k, v, sk, sv, **kw)["kernel"] == "packed"
    imq.attention_shared(q, k, v, sk, sv, out=out, **kw)
    for i, m in zip(at, lens):
        if m > 1:
            a = slice(i, i + m - 1)
            want, bound = wanted(q[a], k[a], v[a], sk, sv, scale=128 ** -0.5, causal=True, softcap=softcap)
            check(out[a], want, bound, f"document from {i}")
            assert bool(out[i + m - 1].isnan().all())
    assert bool((out[:3] == 9.0).all() and (out[at[-1]:] == 9.0).all())


def test_packed_batch_of_hidden_rows():
    """A padded batch of few rows a sequence; its padding is NaN in q, k and v."""
    g = gen(32)
    n, nq, nk = 64, 9, 100
    qn, kn = [1 + s * 5 % nq for s in range(n)], [9 + s * 11 % (nk - 8) for s in range(n)]
    q, k, v = randn(g, n, nq, 32, 128, dtype=F16), *(randn(g, n, nk, 8, 128, dtype=F16) for _ in range(2))
    sk, sv = (randn(g, 1000, 8, 128, dtype=F16) for _ in range(2))
    for s in range(n):
        q[s, qn[s]:], k[s, kn[s]:], v[s, kn[s]:] = NAN, NAN, -INF
    kw = dict(causal=True, q_lens=ints(qn), k_lens=ints(kn))
    assert imq.attention_shared_plan(q, k, v, sk, sv, **kw)["kernel"] == "packed"
    out = torch.full_like(q, 9.0)
    imq.attention_shared(q, k, v, sk, sv, out=out, **kw)
    for s, (a, b) in enumerate(zip(qn, kn)):
        want, bound = wanted(q[s, :a], k[s, :b], v[s, :b], sk, sv, scale=128 ** -0.5, causal=True)
        check(out[s, :a], want, bound, f"sequence {s}")
        assert bool((out[s, a:] == 9.0).all())


@pytest.mark.parametrize("softcap", [0.0, 20.0])
@pytest.mark.parametrize("dim,dtype", [(128, BF16), (64, F16)])
def test_packed_documents_without_keys_of_their_own(dim, dtype, softcap):
    lens = [(11 * i) % 78 for i in range(44)]
    assert packed_plan(900, sum(lens) + 5, 44, 77, 8, 2, dim, dtype, longest_k=0, softcap=softcap)["kernel"] == "packed"
    packed(900, lens, [0] * 44, 8, 2, dim, dtype, True, softcap=softcap)


def test_short_documents_with_slopes():
    lens = [(11 * i) % 78 for i in range(44)]
    for dim, dtype in ((128, BF16), (64, F16)):
        q = torch.empty((sum(lens) + 5, 8, dim), dtype=dtype, device="cuda")
        k, sk, at = q[:, :2].contiguous(), q.new_empty((900, 2, dim)), ints([0] * 45)
        whole(imq.attention_shared_plan(q, k, k, sk, sk, causal=True, q_offsets=at, k_offsets=at, max_q=77, max_k=77,
                                        slopes=falls(8)), 128)
        packed(900, lens, lens, 8, 2, dim, dtype, True, slope=True)


def new_stream():
    """A stream that no call has been on (torch hands its own out again)."""
    stream = ctypes.c_void_p()
    _lib.check(_lib.load().imq_stream_create(context(0), ctypes.byref(stream)), context(0))
    return torch.cuda.ExternalStream(stream.value)


@pytest.mark.parametrize("kernel,n,nq,nk,heads,shared", [("tiles", 3, 200, 270, 8, 3000), ("packed", 64, 9, 100, 32, 1000),
                                                         ("stream", 9, 1, 300, 8, 3000)])
def test_captured_without_a_workspace(kernel, n, nq, nk, heads, shared):
    """A stream's first call, captured, of each plan that has one."""
    g = gen(14)
    q, k, v = randn(g, n, nq, heads, 128, dtype=BF16), *(randn(g, n, nk, heads // 4, 128, dtype=BF16) for _ in range(2))
    sk, sv = (randn(g, shared, heads // 4, 128, dtype=BF16) for _ in range(2))
    p = imq.attention_shared_plan(q, k, v, sk, sv, causal=True)
    assert p["kernel"] == kernel and p["workspace_bytes"] > 0, p
    out, graph = torch.zeros_like(q), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=new_stream()):
        imq.attention_shared(q, k, v, sk, sv, causal=True, out=out)
    for i in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for s in (0, n - 1):
            want, bound = wanted(q[s], k[s], v[s], sk, sv, scale=128 ** -0.5, causal=True)
            check(out[s], want, bound, f"replay {i}, sequence {s}")
        imq.attention_shared(q, k, v, sk, sv, causal=True)
