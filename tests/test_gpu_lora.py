"""quantized_matmul_lora (include/imq_lora.h) against its definition in 64 bits."""

from __future__ import annotations

import pytest
import torch

import aestrix_amd as imq
from core_reference import U32, check, half_step, least

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


def randn(g, *shape, dtype=torch.float32):
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def projection(g, n, k, t):
    w = torch.randint(-2 ** 31, 2 ** 31 - 1, (n, k // 8), generator=g, device="cuda", dtype=torch.int32)
    s = (randn(g, n, k // 64).abs() / (4 * k ** 0.5)).to(t)
    return w, s, (-7.5 * s.float() + randn(g, n, k // 64) / (10 * k ** 0.5)).to(t)


def pairs(g, n, k, ranks, t):
    return [((randn(g, r, k) / k ** 0.5).to(t), (0.3 * randn(g, n, r) / r ** 0.5).to(t)) for r in ranks]


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def wanted(x, proj, ab, c, which):
    """(y, bound).  fp32 sums of K, then of K and rank terms, in any order; u as two values of
    T (half a step of half a step is left; in f16, of values under 1 with B under 2, not
    under 2^-25); one rounding."""
    t, m, k = x.dtype, x.shape[0], x.shape[1]
    wd = imq.dequantize(*proj).double()
    xd = x.double()
    y, mag = xd @ wd.T.contiguous(), xd.abs() @ wd.abs().T.contiguous()
    err = (k + 8) * U32 * mag
    for i, (a, b) in enumerate(ab):
        rows = torch.nonzero(which == i)[:, 0]
        if len(rows) == 0:
            continue
        ad, bd, r = a.double(), b.double(), a.shape[0]
        u, um = abs(c[i]) * (xd[rows] @ ad.T.contiguous()), abs(c[i]) * (xd[rows].abs() @ ad.abs().T.contiguous())
        y[rows] += (u if c[i] >= 0 else -u) @ bd.T.contiguous()
        ba = bd.abs().T.contiguous()
        err[rows] += (k + r + 16) * U32 * (um @ ba) + (half_step(t) ** 2 + (k + 8) * U32) * (u.abs() @ ba)
        err[rows] += (r + 8) * U32 * mag[rows]
        if t == F16:
            err[rows] += r * 2.0 ** -24
    return y, half_step(t) * y.abs() + 1.02 * err + least(t)


def run(m, k, n, ranks, which, t, seed=0, c=None):
    g = gen(seed + m + 3 * k + 5 * n)
    proj, ab, x = projection(g, n, k, t), pairs(g, n, k, ranks, t), randn(g, m, k, dtype=t)
    c = [2.0 / (1 + i % 3) for i in range(len(ranks))] if c is None else c
    ids = ints(which(m) if callable(which) else which)
    out = torch.full((m, n), 9.0, dtype=t, device="cuda")
    got = imq.quantized_matmul_lora(x, *proj, imq.LoraAdapters(ab, c), ids, out=out)
    assert got is out
    check(got, *wanted(x, proj, ab, c, ids), f"[{m} x {n}] K {k}")


def each(count):
    return lambda m: [-1 if r % 5 == 4 else (7 * r + r // count) % count for r in range(m)]


def runs(count, longest):
    """Runs of uneven lengths, each its own adapter, some without."""
    def of(m):
        rows = []
        while len(rows) < m:
            i = len(rows)
            rows += [(i * 5 + 1) % (count + 1) - 1] * (1 + i * 7 % longest)
        return rows[:m]
    return of


MIXED = [64, 32, 16, 8, 1, 33, 100, 256]


@pytest.mark.parametrize("t", [BF16, F16])
@pytest.mark.parametrize("m", [1, 2, 3, 5, 16, 17, 31, 32, 33, 64, 65, 100, 130])
@pytest.mark.parametrize("k,n", [(256, 300), (2560, 1024), (1024, 2555), (4864, 640)])
def test_each_row_its_own(m, k, n, t):
    run(m, k, n, MIXED, each(len(MIXED)), t)


@pytest.mark.parametrize("t", [BF16, F16])
@pytest.mark.parametrize("m,k,n", [(130, 1024, 700), (257, 2560, 6144), (300, 4096, 2555), (777, 1024, 1000),
                                   (1000, 512, 4100), (2100, 256, 9728), (4608, 256, 2600)])
def test_prompts(m, k, n, t):
    run(m, k, n, [16, 64, 24, 128], runs(4, 97), t)
    run(m, k, n, [64], [0] * m, t)


@pytest.mark.parametrize("t", [BF16, F16])
@pytest.mark.parametrize("m", [1, 7, 40, 200])
@pytest.mark.parametrize("k,n", [(64, 1), (128, 257), (192, 100), (320, 5), (576, 640), (704, 1111), (1088, 96),
                                 (2624, 130)])
def test_odd_sizes(m, k, n, t):
    """K of few or odd groups (the register-staged tiles among them), few and odd columns."""
    run(m, k, n, [8, 17, 40], each(3), t)


@pytest.mark.parametrize("rank", [1, 2, 15, 16, 17, 64, 255, 256])
@pytest.mark.parametrize("m", [1, 20, 150])
def test_ranks(rank, m):
    run(m, 512, 390, [rank, 1, rank], each(3), BF16)


@pytest.mark.parametrize("t", [BF16, F16])
@pytest.mark.parametrize("m,k,n,rank,count", [(48, 2560, 6144, 64, 8), (64, 2560, 6144, 256, 1), (96, 9728, 2560, 64, 4),
                                              (160, 2560, 6144, 16, 24), (160, 9728, 2560, 64, 1),
                                              (256, 2560, 6144, 64, 2), (256, 2560, 6144, 64, 8),
                                              (512, 2560, 6144, 16, 32), (512, 2560, 2560, 64, 32)])
def test_rows_between_tokens_and_prompts(m, k, n, rank, count, t):
    """u by rows or by tiles, grouped or not; B u by either join or in the projection's tiles."""
    run(m, k, n, [rank] * count, each(count), t)


@pytest.mark.parametrize("m", [1, 40, 300, 1200])
def test_many_adapters(m):
    count = 200
    run(m, 256, 520, [1 + 5 * i % 48 for i in range(count)], lambda m: [(i * 37) % count for i in range(m)], BF16)


@pytest.mark.parametrize("m", [1, 4, 50, 300])
def test_rows_without_an_adapter(m):
    """All of them, and values that name none: the projection alone."""
    for ids in ([-1] * m, [2, -5, 1 << 30, -(1 << 31)] * m):
        run(m, 1024, 500, [16, 32], ids[:m], F16)


@pytest.mark.parametrize("m", [1, 3, 16, 40, 300])
def test_a_row_does_not_depend_on_the_others(m):
    """The same rows in another order, and beside other rows' adapters."""
    g = gen(m)
    proj, x = projection(g, 500, 1024, BF16), randn(g, m, 1024, dtype=BF16)
    ad = imq.LoraAdapters(pairs(g, 500, 1024, [64, 16, 32], BF16), [1.0, 0.5, -2.0])
    ids = ints(each(3)(m))
    got = imq.quantized_matmul_lora(x, *proj, ad, ids)
    p = torch.randperm(m, generator=g, device="cuda")
    assert torch.equal(imq.quantized_matmul_lora(x[p], *proj, ad, ids[p]), got[p])
    other = ids.clone()
    other[1:] = 1
    assert torch.equal(imq.quantized_matmul_lora(x, *proj, ad, other)[0], got[0])


@pytest.mark.parametrize("t", [BF16, F16])
@pytest.mark.parametrize("m", [5, 40, 300])
def test_an_adapters_nan_stays_with_its_rows(m, t):
    g = gen(m)
    proj, x, c = projection(g, 333, 512, t), randn(g, m, 512, dtype=t), [1.0, 1.0, 1.0, 1.0]
    ab = pairs(g, 333, 512, [16, 32, 16, 48], t)
    ab[1][1][:, 3] = NAN
    ab[2][0][5] = INF
    ids = ints([r % 5 - 1 for r in range(m)])
    x[2, 7] = NAN
    got = imq.quantized_matmul_lora(x, *proj, imq.LoraAdapters(ab, c), ids)
    assert bool(got[ids == 1].isnan().all()) and not bool(torch.isfinite(got[ids == 2]).any())
    assert bool(got[2].isnan().all())
    sound = (ids != 1) & (ids != 2)
    sound[2] = False
    ab[1][1][:, 3], ab[2][0][5], x[2, 7] = 0.0, 0.0, 0.0
    want, bound = wanted(x, proj, ab, c, ids)
    check(got[sound], want[sound], bound[sound], "the others")


def test_large_products_between_the_two_in_f16():
    """A x past f16's largest value, times a small B; and small ones times a large B."""
    g = gen(3)
    proj, x = projection(g, 200, 512, F16), randn(g, 40, 512, dtype=F16)
    big = [((3000 * randn(g, 16, 512)).to(F16), (randn(g, 200, 16) * 2.0 ** -19).to(F16)),
           ((2.0 ** -18 * randn(g, 16, 512)).to(F16), (4000 * randn(g, 200, 16)).to(F16))]
    ids = ints([r % 2 for r in range(40)])
    got = imq.quantized_matmul_lora(x, *proj, imq.LoraAdapters(big, 1.0), ids)
    check(got, *wanted(x, proj, big, [1.0, 1.0], ids), "large")


def test_scales():
    for c in ([0.0, -1.5], [1e-3, 100.0]):
        run(33, 512, 200, [16, 16], each(2), BF16, c=c)
    g = gen(1)
    ab = pairs(g, 200, 512, [16, 8], BF16)
    proj, x, ids = projection(g, 200, 512, BF16), randn(g, 3, 512, dtype=BF16), ints([0, 1, -1])
    one = imq.quantized_matmul_lora(x, *proj, imq.LoraAdapters(ab), ids)
    assert torch.equal(one, imq.quantized_matmul_lora(x, *proj, imq.LoraAdapters(ab, 1), ids))
    assert torch.equal(one, imq.quantized_matmul_lora(x, *proj, imq.LoraAdapters(ab, [1.0, 1.0]), ids))


def test_shapes_views_and_empty_batches():
    g = gen(7)
    proj = projection(g, 100, 256, BF16)
    ad = imq.LoraAdapters([(a.T.contiguous().T, b.T.contiguous().T) for a, b in pairs(g, 100, 256, [8, 24], BF16)])
    x, ids = randn(g, 2, 3, 512, dtype=BF16)[..., ::2], ints([[0, 1, -1], [1, 1, 0]])
    got = imq.quantized_matmul_lora(x, *proj, ad, ids)
    assert got.shape == (2, 3, 100)
    assert torch.equal(got.view(6, 100), imq.quantized_matmul_lora(x.reshape(6, 256), *proj, ad, ids.view(6)))
    assert imq.quantized_matmul_lora(x[:0], *proj, ad, ids[:0]).shape == (0, 3, 100)
    alone = imq.quantized_matmul_lora(x[0, 0], *proj, ad, ids[0, 0])
    assert alone.shape == (100,)
    check(alone[None], *wanted(x[0, :1], proj, [(ad.a[:8], ad.b.view(-1)[:1600].view(100, 16)[:, :8])], [1.0], ids[0, :1]),
          "one row")


@pytest.mark.parametrize("m", [1, 24, 300])
def test_streams_and_graphs(m):
    """Another stream; two captured calls replayed beside each other and between eager ones."""
    g = gen(11)
    proj, ad = projection(g, 1024, 2560, BF16), imq.LoraAdapters(pairs(g, 1024, 2560, [16, 64, 8], BF16))
    xs = [randn(g, m, 2560, dtype=BF16) for _ in range(2)]
    ids = [ints(each(3)(m)), ints([r % 3 for r in range(m)])]
    call = lambda i, **kw: imq.quantized_matmul_lora(xs[i], *proj, ad, ids[i], **kw)
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs, graphs = [torch.zeros((m, 1024), dtype=BF16, device="cuda") for _ in range(2)], []
    for i, s in enumerate(streams):
        want = call(i)
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            assert torch.equal(call(i), want)
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[i], stream=s):
                call(i, out=outs[i])
    torch.cuda.synchronize()
    for n in range(4):
        for i in range(2):
            outs[i].zero_()
            xs[i].copy_(randn(g, m, 2560, dtype=BF16))
        torch.cuda.synchronize()
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                graphs[i].replay()
        eager = [call(i) for i in range(2)]
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(outs[i], eager[i]), (n, i)


def test_adapters_of_a_layer_together():
    """q, k, v and the way back of one layer, each with its set, for a mixed batch."""
    g = gen(21)
    m, dim = 21, 512
    ids, x = ints(each(4)(m)), randn(g, m, dim, dtype=BF16)
    for n in (1024, 256, 256):
        proj, ab = projection(g, n, dim, BF16), pairs(g, n, dim, [16, 32, 8, 64], BF16)
        got = imq.quantized_matmul_lora(x, *proj, imq.LoraAdapters(ab, 0.5), ids)
        check(got, *wanted(x, proj, ab, [0.5] * 4, ids), f"to {n}")


def test_batch_behind_a_shared_prompt():
    """What a server runs a layer: projections with adapters, then attention behind the shared
    keys, then the way out, tokens of several requests."""
    from core_reference import attention_sequence
    g = gen(22)
    n, dim, heads, kv, d = 6, 512, 8, 2, 64
    ids, x = ints([0, 1, -1, 2, 0, 1]), randn(g, n, dim, dtype=BF16)
    width = (heads + 2 * kv) * d
    qkv_p, out_p = projection(g, width, dim, BF16), projection(g, dim, heads * d, BF16)
    qkv_ab, out_ab = pairs(g, width, dim, [16, 8, 32], BF16), pairs(g, dim, heads * d, [16, 8, 32], BF16)
    sk, sv = (randn(g, 300, kv, d, dtype=BF16) for _ in range(2))
    cache = [randn(g, n, 50, kv, d, dtype=BF16) for _ in range(2)]
    lens = ints([1, 50, 7, 33, 20, 49])
    qkv = imq.quantized_matmul_lora(x, *qkv_p, imq.LoraAdapters(qkv_ab), ids)
    check(qkv, *wanted(x, qkv_p, qkv_ab, [1.0] * 3, ids), "qkv")
    q, k, v = (t.unflatten(1, (-1, d)) for t in qkv.split([heads * d, kv * d, kv * d], 1))
    at = (torch.arange(n, device="cuda"), (lens - 1).long())
    cache[0][at], cache[1][at] = k, v
    o = imq.attention_shared(q[:, None], cache[0], cache[1], sk, sv, causal=True, k_lens=lens)
    for s in range(n):
        b = int(lens[s])
        want, bound = attention_sequence(q[s:s + 1], torch.cat([sk, cache[0][s, :b]]), torch.cat([sv, cache[1][s, :b]]),
                                         scale=d ** -0.5)
        check(o[s], want, bound, f"attention {s}")
    flat = o.reshape(n, heads * d)
    y = imq.quantized_matmul_lora(flat, *out_p, imq.LoraAdapters(out_ab), ids)
    check(y, *wanted(flat, out_p, out_ab, [1.0] * 3, ids), "out")


def test_refusals():
    g = gen(1)
    proj, ab, x = projection(g, 96, 128, BF16), pairs(g, 96, 128, [8, 16], BF16), randn(g, 3, 128, dtype=BF16)
    ad, ids = imq.LoraAdapters(ab), ints([0, 1, 0])
    call = imq.quantized_matmul_lora
    for bad in (ids.long(), ids[:2], ids[None], ids.cpu(), ints([0, 0, 1, 0, 0, 0])[::2]):
        with pytest.raises(ValueError):
            call(x, *proj, ad, bad)
    for other in (imq.LoraAdapters(pairs(g, 97, 128, [8], BF16)), imq.LoraAdapters(pairs(g, 96, 64, [8], BF16)),
                  imq.LoraAdapters(pairs(g, 96, 128, [8], F16))):
        with pytest.raises(ValueError):
            call(x, *proj, other, ids)
    with pytest.raises(ValueError):
        call(x, *proj, ad, ids, out=torch.empty((3, 97), dtype=BF16, device="cuda"))
    with pytest.raises(imq.ImqUnsupported):
        call(x, *proj, ad, ids, group_size=32)
    square = projection(g, 128, 128, BF16)
    with pytest.raises(imq.ImqInvalid):
        call(x, *square, imq.LoraAdapters(pairs(g, 128, 128, [8], BF16)), ids, out=x)
    a, b = ab[0]
    for bad in ([], [(a,)], [(a, b[:, :7])], [(a[:0], b[:, :0])], [(a, b), (a[:, :64], b)], [(a, b), (a.half(), b.half())],
                [(a, b), (a, b[:90])], [(a[0], b)], [(a.cpu(), b.cpu())], [(a, b), (a.cpu(), b.cpu())],
                [(a.new_zeros(257, 128), b.new_zeros(96, 257))], [(a[:, :100], b)]):
        with pytest.raises(ValueError):
            imq.LoraAdapters(bad)
    for bad in ([1.0], [1.0, NAN], INF, [1.0, 1e39]):
        with pytest.raises(ValueError):
            imq.LoraAdapters(ab, bad)
    with pytest.raises(imq.ImqUnsupported):
        imq.LoraAdapters([(a.float(), b.float())])
