"""ln_mod, rope and attention (include/imq_core.h) against their definitions in 64 bits."""

from __future__ import annotations

import pytest
import torch

import aestrix_amd as imq
from core_reference import attention_sequence, check, ln_mod, rope

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True)
def _need_gpu(request):
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")
    print(request.node.name, flush=True)


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, dtype=F32):
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


# ------------------------------------------------------------------- ln_mod


@pytest.mark.parametrize("rows,cols,sets,xt,yt", [
    (1, 64, 0, F32, F16), (3, 1, 0, F32, BF16), (5, 333, 2, F32, F16), (17, 2560, 0, BF16, BF16),
    (9, 3072, 3, F32, BF16), (300, 1000, 4, F16, F16), (1, 8192, 1, F32, F16), (1025, 264, 5, F32, F16),
    (33, 5120, 2, F32, F16), (7, 20000, 2, F32, BF16), (2050, 2052, 2, BF16, BF16),
    (4101, 1000, 3, F32, F16), (4096, 516, 2, BF16, BF16)])
def test_ln_mod(rows, cols, sets, xt, yt):
    g = gen(rows + cols)
    n = max(sets, 1)
    x = (randn(g, rows, cols) * 2 + 0.5).to(xt)
    shift, scale = 0.3 * randn(g, n, cols), 0.3 * randn(g, n, cols)
    idx = torch.randint(0, n, (rows,), generator=g, device="cuda", dtype=torch.int32) if sets else None
    got = imq.ln_mod(x, shift, scale, sets=idx, eps=1e-6, post_scale=0.0625, out_dtype=yt)
    want, bound = ln_mod(x, shift, scale, idx, 1e-6, 0.0625, yt)
    check(got, want, bound, f"ln_mod {rows}x{cols}")


def test_ln_mod_means_and_constant_rows():
    """A mean far above the spread, a constant row (variance 0) and huge values."""
    g = gen(5)
    x = randn(g, 6, 512)
    x[0] += 1000.0
    x[1] = 3.25
    x[2] *= 1e15
    x[3] = 0.0
    shift, scale = randn(g, 512), randn(g, 512)
    got = imq.ln_mod(x, shift, scale, eps=1e-6, out_dtype=BF16)
    want, bound = ln_mod(x, shift, scale, None, 1e-6, 1.0, BF16)
    check(got, want, bound, "ln_mod odd rows")


@pytest.mark.parametrize("cols", [4, 3])
def test_ln_mod_of_more_rows_than_a_launch(cols):
    rows = (1 << 24) + 7
    g = gen(cols)
    x, sh, sc = randn(g, rows, cols, dtype=F16), randn(g, 2, cols), randn(g, 2, cols)
    sets = (torch.arange(rows, device="cuda") % 3 == 0).int()
    got = imq.ln_mod(x, sh, sc, sets=sets)
    for a in (0, (1 << 23) - 64, (1 << 24) - 64, rows - 64):
        b = min(a + 128, rows)
        want, bound = ln_mod(x[a:b], sh, sc, sets[a:b], 1e-6, 1.0, F16)
        check(got[a:b], want, bound, f"rows from {a}")


@pytest.mark.parametrize("dim", [16, 6])
def test_rope_of_more_rows_than_a_launch(dim):
    rows = (1 << 23) + 77
    g = gen(dim)
    x, k = randn(g, rows, 1, dim, dtype=BF16), randn(g, rows, 2, dim, dtype=BF16)
    pos = torch.arange(rows, dtype=torch.int32, device="cuda") % 100003
    f, _ = imq.rope_frequencies(dim, device="cuda")
    out = imq.rope(x, k, positions=pos, inv_freq=f)
    for t, got in zip((x, k), out):
        for a in (0, (1 << 23) - 64, rows - 64):
            b = min(a + 128, rows)
            want, bound = rope(t[a:b], pos[a:b], f, None, False, 1.0, None, 1e-6)
            check(got[a:b], want, bound, f"rows from {a}")


def test_ln_mod_in_place_and_clamped_sets():
    g = gen(6)
    x = randn(g, 40, 768, dtype=F16)
    shift, scale = 0.1 * randn(g, 2, 768), 0.1 * randn(g, 2, 768)
    idx = torch.randint(0, 2, (40,), generator=g, device="cuda", dtype=torch.int32)
    want = imq.ln_mod(x, shift, scale, sets=idx)
    wild = torch.where(idx == 0, -7, 1 << 30).to(torch.int32)
    y = imq.ln_mod(x, shift, scale, sets=wild, out=x)
    assert y.data_ptr() == x.data_ptr() and torch.equal(y, want)


# --------------------------------------------------------------------- rope


ROPE = [  # rows, heads, kv, dim, rot, axes, interleaved, norm
    (1, 32, 8, 128, 128, 1, False, True), (3, 1, 1, 2, 2, 1, True, False),
    (33, 24, 24, 128, 128, 4, True, True), (70, 5, 1, 96, 48, 3, False, True),
    (129, 3, 3, 80, 80, 2, True, False), (9, 2, 2, 6, 4, 2, False, True),
    (1030, 4, 2, 64, 32, 1, False, False), (5, 2, 1, 256, 256, 1, True, True),
    (11, 3, 1, 70, 0, 1, False, True), (4100, 2, 1, 64, 64, 1, False, True),
    (6, 2, 2, 512, 96, 1, False, True), (2, 40, 3, 112, 64, 1, True, True)]


def rope_case(rows, heads, kv, dim, rot, axes, norm, dtype, seed=0, far=1 << 20):
    g = gen(seed + rows + dim)
    qkv = randn(g, rows, (heads + 2 * kv) * dim, dtype=dtype)
    q = qkv[:, :heads * dim].unflatten(1, (heads, dim))
    k = qkv[:, heads * dim:(heads + kv) * dim].unflatten(1, (kv, dim))
    f, _ = imq.rope_frequencies(max(rot, 2), 1e4, device="cuda")
    f = f[:rot // 2].contiguous()
    pos = torch.randint(-far, far, (rows, axes), generator=g, device="cuda", dtype=torch.int32)
    half = rot // 2
    sections = [half // axes + (1 if a < half % axes else 0) for a in range(axes)] if axes > 1 else None
    w = [1 + 0.2 * randn(g, dim) if norm else None for _ in range(2)]
    return q, k, pos, f, sections, w


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("rows,heads,kv,dim,rot,axes,interleaved,norm", ROPE)
def test_rope(rows, heads, kv, dim, rot, axes, interleaved, norm, dtype):
    q, k, pos, f, sections, w = rope_case(rows, heads, kv, dim, rot, axes, norm, dtype)
    got = imq.rope(q, k, positions=pos, inv_freq=f, sections=sections, interleaved=interleaved,
                   amplitude=1.25, q_weight=w[0], k_weight=w[1], eps=1e-6)
    for x, y, wt, name in ((q, got[0], w[0], "q"), (k, got[1], w[1], "k")):
        want, bound = rope(x, pos, f, sections, interleaved, 1.25, wt, 1e-6)
        check(y, want, bound, name)
    # One group alone, and in place, give the same bits.
    alone = imq.rope(q, positions=pos, inv_freq=f, sections=sections, interleaved=interleaved,
                     amplitude=1.25, q_weight=w[0], eps=1e-6)
    assert torch.equal(alone, got[0])
    imq.rope(q, k, positions=pos, inv_freq=f, sections=sections, interleaved=interleaved,
             amplitude=1.25, q_weight=w[0], k_weight=w[1], eps=1e-6, q_out=q, k_out=k)
    assert torch.equal(q, got[0]) and torch.equal(k, got[1])


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rope_far_positions(dtype):
    """Positions to the ends of int32: the angle keeps its fraction of a turn."""
    q, k, pos, f, _, w = rope_case(64, 4, 2, 128, 128, 1, True, dtype)
    pos[:4, 0] = torch.tensor([2 ** 31 - 1, -2 ** 31, 2 ** 30 + 1, 0], device="cuda", dtype=torch.int32)
    got = imq.rope(q, k, positions=pos[:, 0].contiguous(), inv_freq=f, q_weight=w[0], k_weight=w[1])
    for x, y, wt in ((q, got[0], w[0]), (k, got[1], w[1])):
        want, bound = rope(x, pos, f, None, False, 1.0, wt, 1e-6)
        check(y, want, bound, "far")


def test_rope_into_a_cache_and_unaligned_views():
    """Keys go to rows of a cache; the slots around them stay.  Views off 16 bytes agree."""
    q, k, pos, f, _, w = rope_case(6, 8, 2, 64, 64, 1, True, BF16)
    pos = pos[:, 0].contiguous()
    kw = dict(positions=pos, inv_freq=f, q_weight=w[0], k_weight=w[1])
    want = imq.rope(q, k, **kw)
    cache = torch.full((6, 9, 2, 64), 7.0, dtype=BF16, device="cuda")
    imq.rope(q, k, k_out=cache[:, 4], **kw)
    assert torch.equal(cache[:, 4], want[1])
    cache[:, 4] = 7.0
    assert bool((cache == 7.0).all())
    wide = torch.zeros((6, 8 * 65 + 3), dtype=BF16, device="cuda")
    view = wide[:, 1:1 + 8 * 65].unflatten(1, (8, 65))[..., :64]
    view.copy_(q)
    got = imq.rope(view, positions=pos, inv_freq=f, q_weight=w[0])
    exact, bound = rope(q, pos, f, None, False, 1.0, w[0], 1e-6)
    check(got, exact, bound, "unaligned")


# ---------------------------------------------------------------- attention


def sequences(q, k, qn, kn):
    """Views of every sequence of a padded batch."""
    return [(q[s, :a], k[s, :b]) for s, (a, b) in enumerate(zip(qn, kn))]


def run_batch(nq, nk, heads, kv, dim, dtype, *, causal=False, softcap=0.0, slope=False, qn=None,
              kn=None, prefix=None, seed=0, scale=None, n=None):
    g = gen(seed + nq + 3 * nk + dim)
    n = len(kn) if kn else len(qn) if qn else n or 1
    q = randn(g, n, nq, heads, dim, dtype=dtype)
    k, v = randn(g, n, nk, kv, dim, dtype=dtype), randn(g, n, nk, kv, dim, dtype=dtype)
    slopes = torch.exp2(-8.0 * torch.arange(1, heads + 1, device="cuda") / heads).float() if slope else None
    ints = [None if x is None else torch.tensor(x, dtype=torch.int32, device="cuda") for x in (qn, kn, prefix)]
    scale = dim ** -0.5 if scale is None else scale
    out = torch.full_like(q, 9.0)
    got = imq.attention(q, k, v, scale=scale, causal=causal, softcap=softcap, slopes=slopes, q_lens=ints[0],
                        k_lens=ints[1], prefix_lens=ints[2], out=out)
    for s in range(n):
        a, b = qn[s] if qn else nq, kn[s] if kn else nk
        want, bound = attention_sequence(q[s, :a], k[s, :b], v[s, :b], scale=scale, causal=causal, softcap=softcap,
                                         slopes=slopes, prefix=prefix[s] if prefix else 0)
        check(got[s, :a], want, bound, f"sequence {s} of {a} x {b}")
        assert bool((got[s, a:] == 9.0).all()), "rows behind the last query changed"


SIZES = [  # queries, keys, heads, kv heads, dim
    (1, 1, 1, 1, 128), (1, 64, 4, 4, 64), (1, 65, 32, 8, 128), (1, 4097, 8, 2, 128), (2, 300, 6, 2, 64),
    (7, 33, 5, 1, 96), (31, 31, 2, 2, 128), (33, 257, 3, 1, 80), (64, 64, 4, 1, 128), (65, 63, 4, 2, 128),
    (129, 200, 2, 2, 64), (300, 300, 8, 2, 128), (515, 515, 3, 3, 64), (40, 1000, 16, 2, 128),
    (9, 50, 2, 1, 8), (130, 130, 2, 1, 40), (5, 70, 2, 2, 33), (3, 90, 2, 1, 256), (17, 40, 3, 1, 1)]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("nq,nk,heads,kv,dim", SIZES)
def test_attention_sizes(nq, nk, heads, kv, dim, causal, dtype):
    run_batch(nq, nk, heads, kv, dim, dtype, causal=causal)


@pytest.mark.parametrize("dtype,dim", [(BF16, 128), (F16, 64), (F16, 72)])
@pytest.mark.parametrize("softcap,slope", [(0.0, True), (30.0, False), (5.0, True)])
@pytest.mark.parametrize("nq,nk,causal", [(1, 500, True), (3, 129, False), (200, 200, True), (70, 333, True),
                                          (150, 90, False)])
def test_attention_scores(nq, nk, causal, softcap, slope, dtype, dim):
    run_batch(nq, nk, 6, 2, dim, dtype, causal=causal, softcap=softcap, slope=slope)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dim,heads,kv", [(128, 8, 2), (64, 4, 4), (24, 3, 1)])
def test_attention_padded_batch(dim, heads, kv, causal):
    """Lengths from none to all, as keys alone and as whole prompts."""
    run_batch(100, 200, heads, kv, dim, BF16, causal=causal, kn=[200, 0, 1, 63, 64, 65, 199])
    run_batch(130, 130, heads, kv, dim, F16, causal=causal, qn=[0, 130, 1, 64, 129], kn=[0, 130, 1, 64, 129])
    run_batch(1, 700, heads, kv, dim, F16, causal=causal, kn=[700, 0, 1, 31, 32, 33, 699, 128])


@pytest.mark.parametrize("nq,nk", [(90, 90), (1, 80), (8, 300), (257, 257)])
def test_attention_prefix(nq, nk):
    """A prefix seen whole, empty, inside a tile and past the end."""
    run_batch(nq, nk, 4, 2, 128, BF16, causal=True, kn=[nk] * 5, prefix=[0, 1, nk // 2, nk, nk - 1])


def test_attention_more_queries_than_keys():
    """Causal with fewer keys than queries: the first queries see nothing and give zeros."""
    run_batch(200, 50, 4, 2, 128, BF16, causal=True, kn=[50, 0, 33])
    run_batch(5, 3, 4, 2, 64, F16, causal=True, kn=[3, 0, 1])


@pytest.mark.parametrize("scale", [3.0, 1e-3])
@pytest.mark.parametrize("nq,nk", [(1, 900), (150, 150)])
def test_attention_sharp_and_flat(nq, nk, scale):
    run_batch(nq, nk, 4, 2, 128, BF16, causal=True, scale=scale)
    run_batch(nq, nk, 4, 2, 128, F16, causal=False, scale=scale)


def packed(lens_q, lens_k, heads, kv, dim, dtype, causal, prefix=None, softcap=0.0, seed=3):
    g = gen(seed)
    at = [[0], [0]]
    for a, b in zip(lens_q, lens_k):
        at[0].append(at[0][-1] + a)
        at[1].append(at[1][-1] + b)
    q = randn(g, at[0][-1] + 5, heads, dim, dtype=dtype)
    k, v = (randn(g, at[1][-1] + 3, kv, dim, dtype=dtype) for _ in range(2))
    offs = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in at]
    pre = torch.tensor(prefix, dtype=torch.int32, device="cuda") if prefix else None
    out = torch.full_like(q, 9.0)
    got = imq.attention(q, k, v, causal=causal, softcap=softcap, prefix_lens=pre, q_offsets=offs[0], k_offsets=offs[1],
                        max_q=max(lens_q), max_k=max(lens_k), out=out)
    for s, (a, b) in enumerate(zip(lens_q, lens_k)):
        i, j = at[0][s], at[1][s]
        want, bound = attention_sequence(q[i:i + a], k[j:j + b], v[j:j + b], scale=dim ** -0.5, causal=causal,
                                         softcap=softcap, prefix=prefix[s] if prefix else 0)
        check(got[i:i + a], want, bound, f"document {s} of {a} x {b}")
    assert bool((got[at[0][-1]:] == 9.0).all()), "rows behind the last document changed"


@pytest.mark.parametrize("dim,dtype", [(128, BF16), (64, F16), (96, BF16)])
@pytest.mark.parametrize("causal", [False, True])
def test_attention_documents(dim, dtype, causal):
    lens = [1, 0, 70, 64, 200, 3, 0, 129]
    packed(lens, lens, 6, 2, dim, dtype, causal)
    packed(lens, [5, 2, 0, 64, 130, 300, 1, 128], 4, 4, dim, dtype, causal)
    packed([1] * 7, [5, 200, 1, 64, 63, 65, 129], 8, 2, dim, dtype, causal)
    if causal:
        packed(lens, lens, 6, 3, dim, dtype, True, prefix=[1, 0, 30, 64, 100, 0, 0, 5], softcap=20.0)


@pytest.mark.parametrize("softcap,slope", [(0.0, False), (30.0, False), (0.0, True), (5.0, True)])
@pytest.mark.parametrize("dim,dtype", [(128, BF16), (64, F16), (72, F16)])
def test_attention_wide_tiles(dim, dtype, softcap, slope):
    """256 rows a workgroup: its last tile partly, one key and keys past a tile, prompts of all lengths."""
    rows = lambda n, nq, nk, heads, kv, causal: imq.attention_plan(
        *(torch.empty((n, a, b, dim), dtype=dtype, device="cuda") for a, b in ((nq, heads), (nk, kv), (nk, kv))),
        causal=causal)["tile_rows"]
    kw = dict(softcap=softcap, slope=slope)
    if rows(1, 1100, 65, 32, 32, False) == rows(10, 1031, 1100, 16, 4, True) == 256:  # as on 256 CUs
        run_batch(1100, 65, 32, 32, dim, dtype, **kw)
        run_batch(1026, 1, 32, 32, dim, dtype, **kw)
        run_batch(1031, 1100, 16, 4, dim, dtype, causal=True, qn=[1031, 1, 0, 1030, 65, 700, 1031, 257, 64, 1031],
                  kn=[1100, 9, 70, 3, 1030, 700, 1031, 257, 64, 0], **kw)
    else:
        pytest.skip("this card's plan takes other tiles")


def tile_rows(n, nq, nk, heads, kv, dim, dtype, causal):
    p = imq.attention_plan(*(torch.empty((n, a, b, dim), dtype=dtype, device="cuda")
                             for a, b in ((nq, heads), (nk, kv), (nk, kv))), causal=causal)
    return p["tile_rows"], p["splits"]


@pytest.mark.parametrize("softcap,slope", [(0.0, False), (30.0, False), (0.0, True), (5.0, True)])
@pytest.mark.parametrize("dim,dtype", [(128, BF16), (128, F16), (72, BF16), (64, F16)])
def test_attention_128_row_tiles(dim, dtype, softcap, slope):
    if tile_rows(7, 301, 333, 16, 4, dim, dtype, True) != (128, 1):  # as on 256 CUs
        pytest.skip("this card's plan takes other tiles")
    kw = dict(softcap=softcap, slope=slope)
    qn, kn = [301, 0, 1, 300, 64, 129, 301], [333, 70, 9, 3, 64, 130, 0]
    run_batch(301, 333, 16, 4, dim, dtype, causal=True, qn=qn, kn=kn, **kw)
    run_batch(301, 333, 16, 4, dim, dtype, n=7, **kw)
    run_batch(301, 333, 16, 4, dim, dtype, causal=True, kn=[333] * 7, prefix=[0, 1, 64, 100, 333, 31, 200], **kw)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim", [128, 64])
def test_attention_128_row_tiles_of_documents(dim, dtype):
    lens = [301, 0, 70, 64, 200, 3, 0, 129, 301, 256, 130]
    packed(lens, lens, 16, 4, dim, dtype, True, prefix=[0, 0, 30, 64, 100, 0, 0, 5, 301, 1, 2], softcap=20.0)
    packed(lens, lens, 12, 4, dim, dtype, False)


def test_attention_128_row_tiles_split():
    if tile_rows(1, 1100, 12400, 16, 16, 128, BF16, False) != (128, 3):
        pytest.skip("this card's plan takes other tiles")
    run_batch(1100, 12400, 16, 16, 128, BF16)


def test_attention_128_row_tiles_views_and_hidden_keys():
    """Columns of a projection, an output between other columns, NaN and infinities behind the keys."""
    g = gen(28)
    qkv = randn(g, 7, 301, 24 * 128, dtype=F16)
    q, k, v = (t.unflatten(2, (-1, 128)) for t in qkv.split([16 * 128, 4 * 128, 4 * 128], 2))
    kn = [301, 290, 64, 65, 1, 0, 200]
    for s, b in enumerate(kn):
        k[s, b:], v[s, b:, 0], v[s, b:, 1] = float("nan"), float("inf"), float("nan")
    wide = torch.full((7, 301, 18 * 128), 9.0, dtype=F16, device="cuda")
    out = wide[..., 128:17 * 128].unflatten(2, (16, 128))
    lens = torch.tensor(kn, dtype=torch.int32, device="cuda")
    imq.attention(q, k, v, causal=True, q_lens=lens, k_lens=lens, out=out)
    for s, b in enumerate(kn):
        want, bound = attention_sequence(q[s, :b], k[s, :b], v[s, :b], scale=128 ** -0.5, causal=True)
        check(out[s, :b], want, bound, f"sequence {s}")
        assert bool((out[s, b:] == 9.0).all()), "rows behind the last query changed"
    assert bool((wide[..., :128] == 9.0).all() and (wide[..., 17 * 128:] == 9.0).all())


@pytest.mark.parametrize("n,nq,nk,heads,kv,causal", [(150, 1000, 40, 7, 7, False), (45, 4000, 33, 6, 6, False),
                                                     (301, 150, 150, 24, 8, True)])
def test_attention_many_sequences(n, nq, nk, heads, kv, causal):
    """So many tiles that a few sequences' and key heads' run at a time, the last few fewer."""
    run_batch(nq, nk, heads, kv, 64, BF16, causal=causal, seed=n, n=n)


def test_attention_wide_tiles_hidden_keys():
    """NaN and infinities behind a sequence's keys and behind the diagonal, 256 rows a workgroup."""
    g = gen(18)
    q, k, v = (randn(g, 10, 1040, h, 128, dtype=BF16) for h in (16, 4, 4))
    kn = [1040 - 9 * s for s in range(10)]
    for s, b in enumerate(kn):
        k[s, b:], v[s, b - 3:, 1], v[s, b:, 2] = float("nan"), float("inf"), float("nan")
    got = imq.attention(q, k, v, causal=True, k_lens=torch.tensor(kn, dtype=torch.int32, device="cuda"))
    for s, b in enumerate(kn):  # the queries that see none of the last three keys
        want, bound = attention_sequence(q[s, :1037], k[s, :b - 3], v[s, :b - 3], scale=128 ** -0.5, causal=True)
        check(got[s, :1037], want, bound, f"sequence {s}")


def test_attention_views_of_a_projection_and_of_a_cache():
    """q, k, v as columns of one product, the output a column block, the cache [n, kv, rows, dim]."""
    g = gen(12)
    qkv = randn(g, 200, 12 * 128, dtype=F16)
    q, k, v = qkv[:, :1024].unflatten(1, (8, 128)), qkv[:, 1024:1280].unflatten(1, (2, 128)), qkv[:, 1280:].unflatten(1, (2, 128))
    wide = torch.full((200, 1024 + 256), 9.0, dtype=F16, device="cuda")
    imq.attention(q, k, v, causal=True, out=wide[:, 256:].unflatten(1, (8, 128)))
    want, bound = attention_sequence(q, k, v, scale=128 ** -0.5, causal=True)
    check(wide[:, 256:].unflatten(1, (8, 128)), want, bound, "columns")
    assert bool((wide[:, :256] == 9.0).all())
    cache = randn(g, 2, 3, 2, 333, 128, dtype=F16)  # k | v, sequence, head, row
    q1 = randn(g, 3, 1, 8, 128, dtype=F16)
    ck, cv = cache[0].transpose(1, 2), cache[1].transpose(1, 2)
    got = imq.attention(q1, ck, cv, causal=True)
    for s in range(3):
        want, bound = attention_sequence(q1[s], ck[s], cv[s], scale=128 ** -0.5, causal=True)
        check(got[s], want, bound, f"cache {s}")


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("nq,nk", [(1, 300), (100, 100), (200, 200), (40, 170)])
def test_attention_hidden_keys_may_hold_anything(nq, nk, dtype):
    """NaN and infinities in keys and values that a query does not see leave it alone:
    behind a sequence's keys, and behind the diagonal."""
    g = gen(8)
    q = randn(g, 2, nq, 4, 128, dtype=dtype)
    k, v = randn(g, 2, nk + 40, 2, 128, dtype=dtype), randn(g, 2, nk + 40, 2, 128, dtype=dtype)
    lens = torch.tensor([nk, nk - 7], dtype=torch.int32, device="cuda")
    for s, b in enumerate((nk, nk - 7)):
        k[s, b:], v[s, b:] = float("nan"), float("inf")
        if nq > 1:  # the last key: only the last query sees it
            k[s, b - 1, 0], v[s, b - 1, 0, 5], v[s, b - 1, 1] = float("nan"), float("-inf"), float("nan")
    got = imq.attention(q, k, v, causal=True, k_lens=lens)
    for s, b in enumerate((nk, nk - 7)):
        a = nq - 1 if nq > 1 else nq
        want, bound = attention_sequence(q[s, :a], k[s, :b - (nq - a)], v[s, :b - (nq - a)], scale=128 ** -0.5, causal=True)
        check(got[s, :a], want, bound, f"sequence {s}")
        if nq > 1:
            assert bool(got[s, -1].isnan().all())


def test_attention_plan_names_the_kernel():
    q, k = torch.zeros((1, 1, 8, 128), dtype=BF16, device="cuda"), torch.zeros((1, 4096, 2, 128), dtype=BF16, device="cuda")
    p = imq.attention_plan(q, k, k, causal=True)
    assert p["kernel"] in ("rows", "tiles", "few") and p["splits"] >= 1
    assert (p["workspace_bytes"] > 0) == (p["splits"] > 1)
