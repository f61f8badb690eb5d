"""attention_shared (include/imq_core.h) against attention over the shared and the own keys
as one sequence, from its definition in 64 bits."""

from __future__ import annotations

import pytest
import torch

import aestrix_amd as imq
from core_reference import attention_sequence, check

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


def ints(x):
    return None if x is None else torch.tensor(x, dtype=torch.int32, device="cuda")


def falls(heads):
    return torch.exp2(-8.0 * torch.arange(1, heads + 1, device="cuda") / heads).float()


def wanted(q, k, v, sk, sv, *, prefix=0, **kw):
    """(o, bound) of one sequence: every query sees all of sk, which stand before k."""
    if kw.get("causal"):
        kw["prefix"] = sk.shape[0] + prefix
    return attention_sequence(q, torch.cat([sk, k]), torch.cat([sv, v]), **kw)


def run_batch(shared, nq, nk, heads, kv, dim, dtype, *, n=1, causal=True, softcap=0.0, slope=False, qn=None, kn=None,
              prefix=None, seed=0):
    g = gen(seed + shared + 3 * nq + 5 * nk + dim)
    n = len(kn) if kn else len(qn) if qn else n
    q = randn(g, n, nq, heads, dim, dtype=dtype)
    k, v = (randn(g, n, nk, kv, dim, dtype=dtype) for _ in range(2))
    sk, sv = (randn(g, shared, kv, dim, dtype=dtype) for _ in range(2))
    kw = dict(scale=dim ** -0.5, causal=causal, softcap=softcap, slopes=falls(heads) if slope else None)
    out = torch.full_like(q, 9.0)
    got = imq.attention_shared(q, k, v, sk, sv, q_lens=ints(qn), k_lens=ints(kn), prefix_lens=ints(prefix), out=out, **kw)
    assert got is out
    for s in range(n):
        a, b = qn[s] if qn else nq, kn[s] if kn else nk
        want, bound = wanted(q[s, :a], k[s, :b], v[s, :b], sk, sv, prefix=prefix[s] if prefix else 0, **kw)
        check(got[s, :a], want, bound, f"sequence {s} of {a} x {shared} + {b}")
        assert bool((got[s, a:] == 9.0).all()), "rows behind the last query changed"


SIZES = [  # shared keys, sequences, queries, own keys, heads, kv heads, dim
    (1, 1, 1, 1, 1, 1, 128), (64, 2, 1, 64, 4, 4, 64), (65, 3, 1, 1, 32, 8, 128), (4097, 8, 1, 300, 8, 2, 128),
    (300, 2, 2, 300, 6, 2, 64), (33, 7, 5, 7, 5, 1, 96), (31, 3, 31, 31, 2, 2, 128), (257, 2, 33, 40, 3, 1, 80),
    (64, 4, 64, 64, 4, 1, 128), (63, 5, 65, 65, 4, 2, 128), (129, 3, 200, 201, 2, 2, 64), (1000, 9, 3, 50, 16, 2, 128),
    (300, 2, 300, 300, 8, 2, 128), (515, 2, 515, 515, 3, 3, 64), (50, 2, 9, 20, 2, 1, 8), (130, 3, 130, 140, 2, 1, 40),
    (70, 2, 5, 6, 2, 2, 33), (90, 2, 3, 4, 3, 1, 256), (40, 2, 17, 17, 3, 1, 1), (2000, 40, 1, 90, 8, 8, 128),
    (777, 20, 1, 130, 40, 1, 128)]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("shared,n,nq,nk,heads,kv,dim", SIZES)
def test_sizes(shared, n, nq, nk, heads, kv, dim, causal, dtype):
    run_batch(shared, nq, nk, heads, kv, dim, dtype, n=n, causal=causal)


@pytest.mark.parametrize("softcap,slope", [(0.0, False), (0.0, True), (30.0, False), (5.0, True)])
@pytest.mark.parametrize("shared,n,nq,nk,heads,kv,dim,dtype",
                         [(4500, 9, 1, 90, 32, 8, 128, BF16), (8300, 33, 2, 40, 16, 16, 64, F16),
                          (7400, 5, 4, 3, 32, 8, 72, F16), (9100, 70, 1, 130, 12, 4, 128, F16)])
def test_long_shared_keys(shared, n, nq, nk, heads, kv, dim, dtype, softcap, slope):
    """More than 32 rows of the batch behind keys that no cache keeps: 64 a workgroup."""
    run_batch(shared, nq, nk, heads, kv, dim, dtype, n=n, causal=True, softcap=softcap, slope=slope)


@pytest.mark.parametrize("softcap,causal", [(0.0, True), (0.0, False), (20.0, True)])
@pytest.mark.parametrize("shared,n,nq,nk,heads,kv,dim,dtype",
                         [(1030, 40, 9, 40, 32, 8, 128, BF16), (600, 70, 20, 20, 8, 4, 64, F16),
                          (777, 50, 12, 33, 18, 6, 72, BF16), (520, 33, 33, 260, 32, 8, 128, F16)])
def test_batches_of_few_tiles(shared, n, nq, nk, heads, kv, dim, dtype, softcap, causal):
    """All rows of a padded batch together against the shared keys; lengths down to none."""
    qn = [nq if s % 3 == 0 else s * 7 % (nq + 1) for s in range(n)]
    kn = [min(nk, qn[s] + s % 5) for s in range(n)]
    run_batch(shared, nq, nk, heads, kv, dim, dtype, causal=causal, softcap=softcap, qn=qn, kn=kn)


@pytest.mark.parametrize("dtype,dim", [(BF16, 128), (F16, 64), (F16, 72)])
@pytest.mark.parametrize("softcap,slope", [(0.0, True), (30.0, False), (5.0, True)])
@pytest.mark.parametrize("shared,n,nq,nk,causal", [(500, 6, 1, 60, True), (129, 3, 3, 9, False), (200, 2, 200, 200, True),
                                                   (333, 3, 70, 90, True), (90, 2, 150, 160, False)])
def test_scores(shared, n, nq, nk, causal, softcap, slope, dtype, dim):
    run_batch(shared, nq, nk, 6, 2, dim, dtype, n=n, causal=causal, softcap=softcap, slope=slope)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dim,heads,kv", [(128, 8, 2), (64, 4, 4), (24, 3, 1)])
def test_lengths(dim, heads, kv, causal):
    """Lengths from none to all, as keys alone and as whole prompts."""
    run_batch(100, 100, 200, heads, kv, dim, BF16, causal=causal, kn=[200, 100, 101, 163, 164, 165, 199])
    run_batch(70, 130, 130, heads, kv, dim, F16, causal=causal, qn=[0, 130, 1, 64, 129], kn=[0, 130, 1, 64, 129])
    run_batch(513, 1, 700, heads, kv, dim, F16, causal=causal, kn=[700, 0, 1, 31, 32, 33, 699, 128])
    run_batch(513, 2, 300, heads, kv, dim, BF16, causal=causal, qn=[2, 1, 0, 2], kn=[300, 1, 7, 0])


def test_more_queries_than_keys():
    """Queries before the first own key see the shared ones alone."""
    run_batch(90, 200, 50, 4, 2, 128, BF16, kn=[50, 0, 33])
    run_batch(90, 5, 3, 4, 2, 64, F16, kn=[3, 0, 1], slope=True)
    for softcap in (0.0, 20.0):
        run_batch(333, 200, 50, 4, 2, 128, BF16, kn=[50, 0, 33], slope=True, softcap=softcap)
        run_batch(333, 200, 50, 4, 2, 64, F16, kn=[50, 0, 33], slope=True, softcap=softcap, causal=False)


@pytest.mark.parametrize("nq,nk", [(90, 90), (1, 80), (8, 300), (257, 257)])
def test_prefix(nq, nk):
    run_batch(77, nq, nk, 4, 2, 128, BF16, kn=[nk] * 5, prefix=[0, 1, nk // 2, nk, nk - 1])
    run_batch(77, nq, nk, 4, 2, 64, F16, kn=[nk] * 5, prefix=[0, 1, nk // 2, nk, nk - 1], slope=True)


def packed(shared, lens_q, lens_k, heads, kv, dim, dtype, causal, prefix=None, softcap=0.0, slope=False):
    g = gen(3)
    at = [[0], [0]]
    for a, b in zip(lens_q, lens_k):
        at[0].append(at[0][-1] + a)
        at[1].append(at[1][-1] + b)
    q = randn(g, at[0][-1] + 5, heads, dim, dtype=dtype)
    k, v = (randn(g, at[1][-1] + 3, kv, dim, dtype=dtype) for _ in range(2))
    sk, sv = (randn(g, shared, kv, dim, dtype=dtype) for _ in range(2))
    out = torch.full_like(q, 9.0)
    kw = dict(scale=dim ** -0.5, causal=causal, softcap=softcap, slopes=falls(heads) if slope else None)
    got = imq.attention_shared(q, k, v, sk, sv, prefix_lens=ints(prefix), q_offsets=ints(at[0]), k_offsets=ints(at[1]),
                               max_q=max(lens_q), max_k=max(lens_k), out=out, **kw)
    for s, (a, b) in enumerate(zip(lens_q, lens_k)):
        i, j = at[0][s], at[1][s]
        want, bound = wanted(q[i:i + a], k[j:j + b], v[j:j + b], sk, sv, prefix=prefix[s] if prefix else 0, **kw)
        check(got[i:i + a], want, bound, f"document {s} of {a} x {shared} + {b}")
    assert bool((got[at[0][-1]:] == 9.0).all()), "rows behind the last document changed"


@pytest.mark.parametrize("dim,dtype", [(128, BF16), (64, F16), (96, BF16)])
@pytest.mark.parametrize("causal", [False, True])
def test_documents(dim, dtype, causal):
    lens = [1, 0, 70, 64, 200, 3, 0, 129]
    packed(150, lens, lens, 6, 2, dim, dtype, causal)
    packed(64, lens, [5, 2, 0, 64, 130, 300, 1, 128], 4, 4, dim, dtype, causal, slope=True)
    packed(777, [1] * 7, [5, 200, 1, 64, 63, 65, 129], 8, 2, dim, dtype, causal)
    packed(1500, [1, 2] * 20, [1, 30] * 20, 8, 2, dim, dtype, causal, slope=True)
    if causal:
        packed(65, lens, lens, 6, 3, dim, dtype, True, prefix=[1, 0, 30, 64, 100, 0, 0, 5], softcap=20.0)


def test_documents_shorter_than_the_offsets_say():
    """max_q and max_k cut what the offsets would give, as attention does."""
    g = gen(4)
    q, k, v = (randn(g, 90, h, 128, dtype=BF16) for h in (4, 2, 2))
    sk, sv = (randn(g, 130, 2, 128, dtype=BF16) for _ in range(2))
    at = ints([0, 40, 90])
    out = torch.full_like(q, 9.0)
    imq.attention_shared(q, k, v, sk, sv, causal=True, q_offsets=at, k_offsets=at, max_q=30, max_k=30, out=out)
    for i in (0, 40):
        want, bound = wanted(q[i:i + 30], k[i:i + 30], v[i:i + 30], sk, sv, scale=128 ** -0.5, causal=True)
        check(out[i:i + 30], want, bound, f"document from {i}")
    assert bool((out[30:40] == 9.0).all() and (out[70:] == 9.0).all())


@pytest.mark.parametrize("dim,dtype,softcap", [(128, BF16, 0.0), (64, F16, 30.0), (72, BF16, 5.0)])
def test_documents_of_few_tiles(dim, dtype, softcap):
    """Many short documents in one stretch of rows: whole tiles of several against the shared keys."""
    lens = [(7 * i) % 78 for i in range(40)]
    q, k = torch.zeros(sum(lens) + 5, 6, dim, dtype=dtype, device="cuda"), torch.zeros(sum(lens) + 3, 2, dim, dtype=dtype, device="cuda")
    sk = k.new_zeros((1000, 2, dim))
    at = ints([sum(lens[:i]) for i in range(41)])
    plan = imq.attention_shared_plan(q, k, k, sk, sk, q_offsets=at, k_offsets=at, max_q=77, max_k=77, softcap=softcap)
    assert plan["kernel"] == "packed", plan
    packed(1000, lens, lens, 6, 2, dim, dtype, True, softcap=softcap)
    packed(777, lens, [max(0, 90 - n) for n in lens], 6, 2, dim, dtype, True, softcap=softcap)
    packed(513, lens, lens, 12, 4, dim, dtype, False, softcap=softcap)
    packed(600, lens, lens, 6, 3, dim, dtype, True, prefix=[n // 2 for n in lens], softcap=softcap)
    packed(600, [1, 77, 0, 64], [0, 0, 0, 0], 6, 1, dim, dtype, True, softcap=softcap)


def test_documents_of_few_tiles_hidden_keys():
    """NaN and infinities behind the documents' keys and behind the diagonal; rows of no document."""
    g = gen(31)
    lens = [60, 5, 77, 0, 33, 64, 77, 40]
    at = [sum(lens[:i]) + 3 for i in range(9)]  # three rows before the first document
    n = at[-1] + 4
    q, k, v = randn(g, n, 8, 128, dtype=BF16), *(randn(g, n, 2, 128, dtype=BF16) for _ in range(2))
    sk, sv = (randn(g, 900, 2, 128, dtype=BF16) for _ in range(2))
    q[:3], q[at[-1]:], k[:3], v[:3], k[at[-1]:], v[at[-1]:] = NAN, NAN, NAN, INF, NAN, INF
    for i, m in zip(at, lens):
        if m:
            k[i + m - 1], v[i + m - 1] = NAN, INF
    out = torch.full_like(q, 9.0)
    imq.attention_shared(q, k, v, sk, sv, causal=True, q_offsets=ints(at), k_offsets=ints(at), max_q=77, max_k=77, out=out)
    for i, m in zip(at, lens):
        if m > 1:
            want, bound = wanted(q[i:i + m - 1], k[i:i + m - 1], v[i:i + m - 1], sk, sv, scale=128 ** -0.5, causal=True)
            check(out[i:i + m - 1], want, bound, f"document from {i}")
    assert bool((out[:3] == 9.0).all() and (out[at[-1]:] == 9.0).all())


def test_no_shared_keys_is_attention():
    g = gen(5)
    for nq, nk in ((1, 300), (100, 100)):
        q, k, v = randn(g, 3, nq, 8, 128, dtype=BF16), *(randn(g, 3, nk, 2, 128, dtype=BF16) for _ in range(2))
        none = q.new_empty((0, 2, 128))
        assert torch.equal(imq.attention_shared(q, k, v, none, none, causal=True), imq.attention(q, k, v, causal=True))


@pytest.mark.parametrize("nq", [1, 3, 150])
def test_no_own_keys(nq):
    run_batch(333, nq, 0, 8, 2, 128, BF16, n=3)
    run_batch(333, nq, 0, 8, 2, 64, F16, n=3, causal=False, slope=True)


def test_nothing_to_see_gives_zeros():
    q = torch.ones((2, 3, 4, 64), dtype=BF16, device="cuda")
    none, sk = q.new_empty((2, 0, 2, 64)), q.new_empty((0, 2, 64))
    assert bool((imq.attention_shared(q, none, none, sk, sk) == 0).all())
    empty = q.new_empty((0, 3, 4, 64))
    assert imq.attention_shared(empty, q.new_empty((0, 5, 2, 64)), q.new_empty((0, 5, 2, 64)), sk, sk).shape == empty.shape


def test_views():
    """q, k, v as columns of one product, the output a column block, shared keys as rows of a
    cache [kv, rows, dim] and keys that one row stands for (stride 0)."""
    g = gen(12)
    for nq in (1, 200):
        qkv = randn(g, 3, nq, 12 * 128, dtype=F16)
        q, k, v = (t.unflatten(2, (-1, 128)) for t in qkv.split([1024, 256, 256], 2))
        sk, sv = (randn(g, 2, 500, 128, dtype=F16).transpose(0, 1)[100:] for _ in range(2))
        wide = torch.full((3, nq, 1024 + 256), 9.0, dtype=F16, device="cuda")
        out = wide[..., 256:].unflatten(2, (8, 128))
        imq.attention_shared(q, k, v, sk, sv, causal=True, out=out)
        for s in range(3):
            want, bound = wanted(q[s], k[s], v[s], sk, sv, scale=128 ** -0.5, causal=True)
            check(out[s], want, bound, f"columns {s}")
        assert bool((wide[..., :256] == 9.0).all())
        one = sk[:1].expand(70, 2, 128)
        got = imq.attention_shared(q, k, v, one, sv[:70], causal=True)
        want, bound = wanted(q[0], k[0], v[0], one, sv[:70], scale=128 ** -0.5, causal=True)
        check(got[0], want, bound, "one row for all")


@pytest.mark.parametrize("dim", [128, 64])
def test_odd_alignment(dim):
    """Pointers and strides that no 16-byte load takes."""
    g = gen(13)
    for nq in (1, 70):
        q = randn(g, 2, nq, 4, dim + 1, dtype=BF16)[..., 1:]
        k, v = (randn(g, 2, 80, 2, dim + 2, dtype=BF16)[..., :dim] for _ in range(2))
        sk, sv = (randn(g, 99, 2, dim + 3, dtype=BF16)[..., 3:] for _ in range(2))
        got = imq.attention_shared(q, k, v, sk, sv, causal=True)
        for s in range(2):
            want, bound = wanted(q[s], k[s], v[s], sk, sv, scale=dim ** -0.5, causal=True)
            check(got[s], want, bound, f"sequence {s}")
        # The shared keys alone off their alignment.
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
        got = imq.attention_shared(q, k, v, sk, sv, causal=True)
        want, bound = wanted(q[1], k[1], v[1], sk, sv, scale=dim ** -0.5, causal=True)
        check(got[1], want, bound, "shared keys")


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("nq,nk", [(1, 300), (3, 200), (200, 200), (40, 170)])
def test_hidden_keys_may_hold_anything(nq, nk, dtype):
    """NaN and infinities behind a sequence's keys, behind the diagonal and behind the shared
    rows leave the queries that do not see them alone; a NaN that is seen shows."""
    g = gen(8)
    q = randn(g, 3, nq, 4, 128, dtype=dtype)
    k, v = (randn(g, 3, nk + 40, 2, 128, dtype=dtype) for _ in range(2))
    rows = [randn(g, 163, 2, 128, dtype=dtype) for _ in range(2)]
    rows[0][103:], rows[1][103:] = NAN, INF
    sk, sv = rows[0][:103], rows[1][:103]
    kn = (nk, nk - 7, nk - 64)
    for s, b in enumerate(kn):
        k[s, b:], v[s, b:] = NAN, INF
        if nq > 1:  # the last key: only the last query sees it
            k[s, b - 1, 0], v[s, b - 1, 0, 5], v[s, b - 1, 1] = NAN, -INF, NAN
    got = imq.attention_shared(q, k, v, sk, sv, causal=True, k_lens=ints(kn))
    for s, b in enumerate(kn):
        a = nq - 1 if nq > 1 else nq
        want, bound = wanted(q[s, :a], k[s, :b - (nq - a)], v[s, :b - (nq - a)], sk, sv, scale=128 ** -0.5, causal=True)
        check(got[s, :a], want, bound, f"sequence {s}")
        if nq > 1:
            assert bool(got[s, -1].isnan().all())
    # One sequence's spoilt keys stay its own.
    k[1], v[1] = NAN, NAN
    got = imq.attention_shared(q, k, v, sk, sv, causal=True, k_lens=ints(kn))
    assert bool(got[1, -1].isnan().all())
    for s in (0, 2):
        a = nq - 1 if nq > 1 else nq
        want, bound = wanted(q[s, :a], k[s, :kn[s] - (nq - a)], v[s, :kn[s] - (nq - a)], sk, sv, scale=128 ** -0.5, causal=True)
        check(got[s, :a], want, bound, f"beside it {s}")


@pytest.mark.parametrize("nq", [1, 150])
def test_spoilt_shared_keys_show(nq):
    g = gen(9)
    q = randn(g, 2, nq, 4, 128, dtype=BF16)
    k, v, sk, sv = (randn(g, *s, 2, 128, dtype=BF16) for s in ((2, nq), (2, nq), (300,), (300,)))
    sv[299, 1, 7] = INF
    got = imq.attention_shared(q, k, v, sk, sv, causal=True)
    assert bool((got[:, :, 2:, 7] == INF).all()) and bool(torch.isfinite(got[:, :, :2]).all())
    sk[0, 0, 3] = NAN
    got = imq.attention_shared(q, k, v, sk, sv, causal=True)
    assert bool(got[:, :, :2].isnan().all())


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("nq", [1, 130])
def test_large_values_and_scores(nq, dtype):
    """Values near the type's largest, scores far apart: sums stay finite.  All values are one:
    what weights lose cancels, and the output is off by its rounding and those of 32-bit sums."""
    g = gen(10)
    q = randn(g, 2, nq, 4, 128, dtype=dtype)
    k, sk = randn(g, 2, nq + 9, 2, 128, dtype=dtype), 8 * randn(g, 200, 2, 128, dtype=dtype)
    top = 60000.0 if dtype == F16 else 3e38
    v, sv = torch.full_like(k, top), torch.full_like(sk, top)
    got = imq.attention_shared(q, k, v, sk, sv, causal=True)
    assert bool(((got.double() - v[0, 0, 0, 0].double()).abs() <= (torch.finfo(dtype).eps / 2 + 1e-4) * top).all())


def test_streams_graph_and_threads_of_calls():
    """Another stream, and a captured call replayed between eager calls of other sizes."""
    g = gen(11)
    q, k, v = randn(g, 16, 1, 8, 128, dtype=BF16), *(randn(g, 16, 200, 2, 128, dtype=BF16) for _ in range(2))
    sk, sv = (randn(g, 3000, 2, 128, dtype=BF16) for _ in range(2))
    lens = ints(list(range(1, 17)))
    run = lambda **kw: imq.attention_shared(q, k, v, sk, sv, causal=True, k_lens=lens, **kw)
    eager = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(run(), eager)
        out = torch.zeros_like(q)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            run(out=out)
    torch.cuda.synchronize()
    for i in range(4):
        out.zero_()
        q.copy_(randn(g, 16, 1, 8, 128, dtype=BF16))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, run()), i
        imq.attention_shared(q[:3], k[:3], v[:3], sk[:100], sv[:100])


@pytest.mark.parametrize("nq", [1, 200])
def test_captured_without_a_workspace(nq):
    """A stream's first call may be captured: it runs without a workspace."""
    g = gen(14)
    q, k, v = randn(g, 9, nq, 8, 128, dtype=BF16), *(randn(g, 9, nq + 70, 2, 128, dtype=BF16) for _ in range(2))
    sk, sv = (randn(g, 3000, 2, 128, dtype=BF16) for _ in range(2))
    out = torch.zeros_like(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        imq.attention_shared(q, k, v, sk, sv, causal=True, out=out)
    for i in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for s in (0, 8):
            want, bound = wanted(q[s], k[s], v[s], sk, sv, scale=128 ** -0.5, causal=True)
            check(out[s], want, bound, f"replay {i}, sequence {s}")


def test_decoding_continues_a_prompt():
    """A prompt behind shared keys, then tokens one at a time on a cache: the same outputs."""
    g = gen(15)
    n, total, first = 3, 40, 33
    q, k, v = randn(g, n, total, 8, 128, dtype=F16), *(randn(g, n, total, 2, 128, dtype=F16) for _ in range(2))
    sk, sv = (randn(g, 700, 2, 128, dtype=F16) for _ in range(2))
    rows = [imq.attention_shared(q[:, :first], k[:, :first], v[:, :first], sk, sv, causal=True)]
    for t in range(first, total):
        lens = torch.full((n,), t + 1, dtype=torch.int32, device="cuda")
        rows.append(imq.attention_shared(q[:, t:t + 1], k, v, sk, sv, causal=True, k_lens=lens))
    got = torch.cat(rows, 1)
    for s in range(n):
        want, bound = wanted(q[s], k[s], v[s], sk, sv, scale=128 ** -0.5, causal=True)
        check(got[s], want, bound, f"sequence {s}")


def test_refusals():
    z = lambda *s, t=BF16: torch.zeros(s, dtype=t, device="cuda")
    q, k, sk = z(2, 3, 4, 64), z(2, 5, 2, 64), z(7, 2, 64)
    call = imq.attention_shared
    for bad in (z(7, 4, 64), z(7, 2, 32), z(2, 64), z(1, 7, 2, 64), z(7, 2, 64, t=F16), torch.zeros(7, 2, 64, dtype=BF16)):
        with pytest.raises(ValueError):
            call(q, k, k, bad, bad)
    with pytest.raises(ValueError):
        call(q, k, k, sk, z(6, 2, 64))
    with pytest.raises(ValueError):
        call(q, k, k, sk.transpose(0, 2).contiguous().transpose(0, 2), sk)
    with pytest.raises(ValueError):
        call(q, k, z(2, 4, 2, 64), sk, sk)
    with pytest.raises(imq.ImqInvalid):
        call(q, k, k, sk, sk, scale=NAN)
    with pytest.raises(imq.ImqInvalid):
        call(z(1, 7, 2, 64), z(1, 0, 2, 64), z(1, 0, 2, 64), sk, sk, out=sk[None])
    with pytest.raises(imq.ImqUnsupported):
        call(*(x.float() for x in (q, k, k, sk, sk)))
