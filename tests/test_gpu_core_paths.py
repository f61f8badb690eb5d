"""The block core as it is used: a text-encoder layer, a denoise step, caches, streams and graphs."""

from __future__ import annotations

import pytest
import torch

import aestrix_amd as imq
from aestrix_amd import dit
from aestrix_amd.ops import Q
from aestrix_amd.step import DitDims, DitStep, random_head, random_projections
from aestrix_amd.te import EPS, TextEncoderLayers, random_te_layers
from core_reference import attention_sequence, check, rope

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


def wide(q: Q) -> torch.Tensor:
    """The packed weight as float64, a weight held in its scales' type."""
    return imq.dequantize(q.w, q.s, q.b).double()


def mm(x, q):
    return x @ wide(q).T.contiguous()


def rms(x, w, eps):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * w.double()


def near(got, want, what, normwise, cosine):
    g, w = got.double().flatten(), want.double().flatten()
    n = float((g - w).abs().max() / w.abs().max())
    c = float(torch.dot(g, w) / (g.norm() * w.norm()))
    print(f"  {what}: normwise {n:.2e} cosine {c:.8f}", flush=True)
    assert torch.isfinite(got).all() and n <= normwise and c >= cosine, (what, n, c)


# -------------------------------------------------------------- text encoder

SMALL = dict(hidden=512, nq=1024, nkv=256, inter=768)


def te(dtype, n_layers=2, seed=3, norms=True, **dims):
    layers = random_te_layers(n_layers, dtype=dtype, seed=seed, **(dims or SMALL))
    g = gen(seed)
    for l in layers:
        if norms:
            l.norm_q, l.norm_k = 1 + 0.1 * randn(g, 128), 1 + 0.1 * randn(g, 128)
    return TextEncoderLayers(layers, max_rows=512)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("prompts,window,lens", [(1, 1, None), (1, 30, None), (3, 40, [40, 1, 17]), (2, 200, [0, 133])])
def test_te_attn_core_is_rope_and_attention(prompts, window, lens, dtype):
    plan = te(dtype)
    x = randn(gen(9), prompts * window, plan.hidden, dtype=dtype)
    qkv = plan.attn_in(0, x)
    want_qkv = qkv.clone()
    ln = None if lens is None else torch.tensor(lens, dtype=torch.int32, device="cuda")
    got = plan.attn_core(0, qkv, prompts, ln)
    l = plan.layers[0]
    f, _ = imq.rope_frequencies(128, 1e6, device="cuda")
    pos = torch.arange(window, dtype=torch.int32, device="cuda").repeat(prompts)
    for a, n, w in ((0, plan.nq, l.norm_q), (plan.nq, plan.nkv, l.norm_k)):
        y, bound = rope(want_qkv[:, a:a + n].unflatten(1, (-1, 128)), pos, f, None, False, 1.0, w, EPS)
        check(qkv[:, a:a + n].unflatten(1, (-1, 128)), y, bound, "rope in place")
    assert torch.equal(qkv[:, plan.nq + plan.nkv:], want_qkv[:, plan.nq + plan.nkv:])
    q, k, v = (t.unflatten(-1, (-1, 128)) for t in qkv.split([plan.nq, plan.nkv, plan.nkv], -1))
    for s in range(prompts):
        n = window if lens is None else lens[s]
        r = slice(s * window, s * window + n)
        want, bound = attention_sequence(q[r], k[r], v[r], scale=128 ** -0.5, causal=True)
        check(got[r].unflatten(1, (-1, 128)), want, bound, f"prompt {s}")
        assert not got[s * window + n:(s + 1) * window].any(), "padding rows"


def te_layer_exact(l, x, prompts):
    """A layer in float64, no rounding between its steps."""
    rows = x.shape[0]
    w = rows // prompts
    qkv = mm(rms(x, l.norm_in, EPS), l.qkv)
    nq, nkv = l.o.k, (l.qkv.n - l.o.k) // 2
    q, k, v = (t.unflatten(-1, (-1, 128)) for t in qkv.split([nq, nkv, nkv], -1))
    f, _ = imq.rope_frequencies(128, 1e6, device="cuda")
    pos = torch.arange(w, dtype=torch.int32, device="cuda").repeat(prompts)
    q = rope(q, pos, f, None, False, 1.0, l.norm_q, EPS)[0]
    k = rope(k, pos, f, None, False, 1.0, l.norm_k, EPS)[0]
    o = torch.cat([_softmax(q[i:i + w], k[i:i + w], v[i:i + w], True) for i in range(0, rows, w)])
    r = x + mm(o.flatten(1), l.o)
    g, u = mm(rms(r, l.norm_post, EPS), l.gate_up).chunk(2, -1)
    return r + mm(g * torch.sigmoid(g) * u, l.down)


def _softmax(q, k, v, causal):
    n, h, d = q.shape
    rep = h // k.shape[1]
    k, v = k.repeat_interleave(rep, 1), v.repeat_interleave(rep, 1)
    s = torch.bmm(q.transpose(0, 1).contiguous(), k.permute(1, 2, 0).contiguous()) * d ** -0.5
    if causal:
        s = s.masked_fill(torch.ones(n, n, device="cuda").triu(1).bool(), -torch.inf)
    return torch.bmm(torch.softmax(s, -1), v.transpose(0, 1).contiguous()).transpose(0, 1)


@pytest.mark.parametrize("dtype,prompts,window", [(BF16, 1, 30), (BF16, 2, 100), (F16, 1, 1), (F16, 1, 257)])
def test_te_layers_against_64_bits(dtype, prompts, window):
    """Two whole layers; the bars are those of the layer halves (test_gpu_te.py): each of the
    dozen roundings to T of a layer is half a step, 2^-9 in bf16, and they add up in squares:
    sqrt(24) * 2^-9 = 9.6e-3 of the values' own size, against the largest value here."""
    plan = te(dtype)
    x = randn(gen(10), prompts * window, plan.hidden, dtype=dtype)
    keep = x.clone()
    got = plan.encode(x, prompts, taps=(1, 2))
    assert torch.equal(x, keep)
    want = x.double()
    for i in range(2):
        want = te_layer_exact(plan.layers[i], want, prompts)
        near(got[i], want, f"layer {i + 1}", 1e-2, 0.9999)


def test_te_padding_leaves_prompts_alone():
    """A prompt's rows are the same bits alone, beside others and with other padding."""
    plan = te(BF16)
    g = gen(4)
    a, b = randn(g, 40, plan.hidden, dtype=BF16), randn(g, 40, plan.hidden, dtype=BF16)
    lens = torch.tensor([40, 23], dtype=torch.int32, device="cuda")
    one = plan.encode(torch.cat([a, b]), 2, lens, taps=(2,))[0]
    b[23:] = randn(g, 17, plan.hidden, dtype=BF16)
    two = plan.encode(torch.cat([a, b]), 2, lens, taps=(2,))[0]
    assert torch.equal(one[:63], two[:63])


def test_te_first_core_in_a_graph():
    """A layer's core captured before any eager call of it."""
    plan = te(BF16)
    qkv = randn(gen(15), 48, plan.nq + 2 * plan.nkv, dtype=BF16)
    start, out = qkv.clone(), torch.zeros((48, plan.nq), dtype=BF16, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan.attn_core(0, qkv, 2, out=out)
    qkv.copy_(start)
    want = plan.attn_core(0, qkv, 2)
    for _ in range(3):
        qkv.copy_(start)
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_te_without_head_norms_and_refusals():
    plan = te(BF16, norms=False)
    x = randn(gen(5), 6, plan.hidden, dtype=BF16)
    assert torch.isfinite(plan.layer(0, x)).all()
    with pytest.raises(ValueError):
        plan.attn_core(0, plan.attn_in(0, x), prompts=4)
    with pytest.raises(ValueError):
        plan.encode(x, taps=(3,))
    with pytest.raises(ValueError):
        plan.set_rope(head_dim=96)


# ------------------------------------------------------------- denoise step

TINY = DitDims(l_img=96, l_txt=32, dim=512, ff_inner=512, n_double=2, n_single=2)


def dit_parts(dims, seed=21):
    g = gen(seed)
    projs, head = random_projections(dims, F16, seed), random_head(dims, 128, F16, seed)
    step = DitStep(dims, projs)
    step.set_head(*head)
    gates = 0.5 * randn(g, 4 * dims.n_double + dims.n_single, dims.dim)
    step.set_conditioning(gates=gates.contiguous())
    w = lambda: 1 + 0.1 * randn(g, 128)
    norms = [dit.DitNorms(w(), w(), w(), w()) for _ in range(dims.n_double)]
    norms += [dit.DitNorms(w(), w()) for _ in range(dims.n_single)]
    pos = torch.zeros((dims.joint, 4), dtype=torch.int32, device="cuda")
    pos[:dims.l_txt, 3] = torch.arange(dims.l_txt, device="cuda")
    i = torch.arange(dims.l_img, device="cuda")
    pos[dims.l_txt:, 1], pos[dims.l_txt:, 2] = i // 8, i % 8
    d = dims.dim
    m = [0.3 * randn(g, 2, d) for _ in range(4)] + [0.3 * randn(g, d) for _ in range(4)]
    return dit.DitModel(step, norms, pos), dit.DitModulation(*m), projs, head, gates, pos, g


def dit_exact(model, mod, projs, head, gates, lat, e, dt):
    d = model.step.dims
    t, i = slice(0, d.l_txt), slice(d.l_txt, d.joint)

    def ln(x, shift, scale):
        x = x - x.mean(-1, keepdim=True)
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)
        if shift.dim() == 2:
            n = torch.cat([torch.zeros(d.l_txt), torch.ones(d.l_img)]).long().cuda()
            return x * (1 + scale.double()[n]) + shift.double()[n]
        return x * (1 + scale.double()) + shift.double()

    def core(q, k, v, nq, nk):
        q, k, v = (z.unflatten(-1, (-1, 128)) for z in (q, k, v))
        turn = lambda z, n: torch.cat([rope(z[r], model.positions[r], model.freq, model.sections, True, 1.0, w, 1e-5)[0]
                                       for r, w in n])
        return _softmax(turn(q, nq), turn(k, nk), v, False).flatten(1)

    def swiglu(x):
        a, b = x.chunk(2, -1)
        return a * torch.sigmoid(a) * b

    g = gates.double()
    x = torch.cat([e.double(), mm(lat.double(), head[0])])
    for b in range(d.n_double):
        w, n = projs[12 * b:12 * b + 12], model.norms[b]
        nx = ln(x, mod.attn_shift, mod.attn_scale)
        q, k, v = (torch.cat([mm(nx[t], w[3 + j]), mm(nx[i], w[j])]) for j in range(3))
        a = core(q, k, v, ((t, n.added_q), (i, n.q)), ((t, n.added_k), (i, n.k)))
        x = torch.cat([x[t] + g[4 * b + 1] * mm(a[t], w[7]), x[i] + g[4 * b] * mm(a[i], w[6])])
        nx = ln(x, mod.mlp_shift, mod.mlp_scale)
        x = torch.cat([x[t] + g[4 * b + 3] * mm(swiglu(mm(nx[t], w[10])), w[11]),
                       x[i] + g[4 * b + 2] * mm(swiglu(mm(nx[i], w[8])), w[9])])
    for b in range(d.n_single):
        w, n = projs[12 * d.n_double + 2 * b:][:2], model.norms[d.n_double + b]
        y = mm(ln(x, mod.single_shift, mod.single_scale), w[0])
        q, k, v = y[:, :3 * d.dim].split(d.dim, -1)
        every = slice(None)
        a = core(q, k, v, ((every, n.q),), ((every, n.k),))
        x = x + g[4 * d.n_double + b] * mm(torch.cat([a, swiglu(y[:, 3 * d.dim:])], 1), w[1])
    return lat.double() + dt * mm(ln(x[i], mod.out_shift, mod.out_scale), head[1])


def test_dit_denoise_against_64_bits():
    """The whole step in float64 without a rounding between.  About 12 roundings to f16 a
    block, each half a step, 2^-11, added up in squares over 4 blocks: sqrt(48) * 2^-11 =
    3.4e-3 of the values' own size; the bar is three times that against the largest value."""
    model, mod, projs, head, gates, _, g = dit_parts(TINY)
    lat, e = randn(g, TINY.l_img, 128), randn(g, TINY.l_txt, TINY.dim)
    got = model.denoise(lat, e, -0.25, mod)
    want = dit_exact(model, mod, projs, head, gates, lat, e, -0.25)
    near(got - lat, want - lat.double(), "denoise", 1e-2, 0.9999)
    assert torch.equal(got, model.denoise(lat, e, -0.25, mod))


def test_dit_denoise_in_a_graph():
    model, mod, _, _, _, _, g = dit_parts(TINY, 22)
    lat, e = randn(g, TINY.l_img, 128), randn(g, TINY.l_txt, TINY.dim)
    out = torch.empty_like(lat)
    model.denoise(lat, e, -0.25, mod, out=out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        model.denoise(lat, e, -0.25, mod, out=out)
    for seed in range(3):
        lat.copy_(randn(gen(100 + seed), *lat.shape))
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(got, model.denoise(lat, e, -0.25, mod))


def test_dit_refusals():
    model, *_ = dit_parts(TINY, 23)
    with pytest.raises(ValueError):
        dit.DitModel(model.step, model.norms[:-1], model.positions)
    with pytest.raises(ValueError):
        dit.DitModel(model.step, model.norms, model.positions[:-1])
    with pytest.raises(ValueError):
        dit.DitModel(model.step, model.norms, model.positions, head_dim=100)
    with pytest.raises(ValueError):
        dit.DitModel(model.step, model.norms, model.positions, sections=(16, 16, 16, 8))


# ----------------------------------------------- attention among other work


def cache_case(seed=1, n=4, longest=3000, dtype=BF16):
    g = gen(seed)
    q = randn(g, n, 1, 16, 128, dtype=dtype)
    k, v = randn(g, n, longest, 4, 128, dtype=dtype), randn(g, n, longest, 4, 128, dtype=dtype)
    lens = torch.tensor([longest, 7, 1000, 2049][:n], dtype=torch.int32, device="cuda")
    return q, k, v, lens


def test_attention_split_in_a_graph():
    """Captured on a stream whose workspace has grown: the split plan, the eager bits, with
    lengths that change between the replays; captured where it would have to grow: unsplit."""
    q, k, v, lens = cache_case()
    assert imq.attention_plan(q, k, v, causal=True, k_lens=lens)["splits"] > 1
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        imq.attention(q, k, v, causal=True, k_lens=lens)
    torch.cuda.synchronize()
    out = torch.empty_like(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        imq.attention(q, k, v, causal=True, k_lens=lens, out=out)
    fresh = torch.cuda.CUDAGraph()
    out2 = torch.empty_like(q)
    with torch.cuda.graph(fresh, stream=torch.cuda.Stream()):
        imq.attention(q, k, v, causal=True, k_lens=lens, out=out2)
    for i in range(4):
        lens.copy_(torch.tensor([3000 - i, 7 * i, 1000 + i, 1], dtype=torch.int32))
        with torch.cuda.stream(s):
            graph.replay()
        s.synchronize()
        fresh.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, imq.attention(q, k, v, causal=True, k_lens=lens))
        for b, n in enumerate(lens.tolist()):
            want, bound = attention_sequence(q[b], k[b, :n], v[b, :n], scale=128 ** -0.5, causal=True)
            check(out[b], want, bound, f"replay {i} sequence {b}")
            check(out2[b], want, bound, f"unsplit replay {i} sequence {b}")


def test_attention_on_two_streams_at_once():
    """Each stream has a workspace of its own."""
    a, b = cache_case(1), cache_case(2)
    want = [imq.attention(*c[:3], causal=True, k_lens=c[3]) for c in (a, b)]
    torch.cuda.synchronize()
    s = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(8):
        for i, c in enumerate((a, b)):
            with torch.cuda.stream(s[i]):
                got[i].append(imq.attention(*c[:3], causal=True, k_lens=c[3]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])


@pytest.mark.parametrize("row", [1 << 22, 1 << 24])
@pytest.mark.parametrize("nq", [1, 40])
def test_attention_rows_past_32_bits(row, nq):
    """Rows 8 and 32 MiB apart: the last ones begin past 2^32 bytes (the second distance is
    past what a tile's 32-bit offsets hold, and takes the kernel by rows)."""
    n = 600 if row == 1 << 22 else 140
    flat = torch.empty(row * n + 4096, dtype=BF16, device="cuda")
    g = gen(row)
    k = flat.as_strided((1, n, 1, 128), (0, row, 128, 1))
    v = flat.as_strided((1, n, 1, 128), (0, row, 128, 1), 1024)
    k.copy_(randn(g, 1, n, 1, 128))
    v.copy_(randn(g, 1, n, 1, 128))
    q = randn(g, 1, nq, 2, 128, dtype=BF16)
    got = imq.attention(q, k, v, causal=True)
    assert (imq.attention_plan(q, k, v, causal=True)["kernel"] == "rows") == (row == 1 << 24)
    want, bound = attention_sequence(q[0], k[0], v[0], scale=128 ** -0.5, causal=True)
    check(got[0], want, bound, "far rows")
    o = flat.as_strided((1, nq, 2, 128), (0, row, 128, 1), 2048)
    imq.attention(q, k, v, causal=True, out=o)
    assert torch.equal(o, got)


def test_attention_sequences_past_32_bits():
    """A cache whose later sequences begin past 2^32 elements."""
    flat = torch.empty((1 << 32) + (1 << 24), dtype=F16, device="cuda")
    g = gen(77)
    k = flat.as_strided((3, 200, 2, 64), (1 << 31, 128, 64, 1))
    v = flat.as_strided((3, 200, 2, 64), (1 << 31, 128, 64, 1), 1 << 20)
    k.copy_(randn(g, 3, 200, 2, 64))
    v.copy_(randn(g, 3, 200, 2, 64))
    for nq in (1, 50):
        q = randn(g, 3, nq, 4, 64, dtype=F16)
        got = imq.attention(q, k, v, causal=True)
        for s in range(3):
            want, bound = attention_sequence(q[s], k[s], v[s], scale=0.125, causal=True)
            check(got[s], want, bound, f"sequence {s}")


def test_attention_broadcast_keys():
    """Keys shared by all sequences (stride 0), and one key head for all heads."""
    g = gen(5)
    k, v = randn(g, 1, 333, 1, 128, dtype=BF16), randn(g, 1, 333, 1, 128, dtype=BF16)
    q = randn(g, 3, 20, 8, 128, dtype=BF16)
    got = imq.attention(q, k.expand(3, -1, -1, -1), v.expand(3, -1, -1, -1))
    for s in range(3):
        want, bound = attention_sequence(q[s], k[0], v[0], scale=128 ** -0.5)
        check(got[s], want, bound, f"sequence {s}")


def test_attention_wild_lengths_are_clamped():
    """Device lengths and offsets outside what the arguments allow touch nothing outside."""
    g = gen(6)
    q, k, v = randn(g, 2, 33, 4, 128, dtype=BF16), randn(g, 2, 90, 2, 128, dtype=BF16), randn(g, 2, 90, 2, 128, dtype=BF16)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
    want = imq.attention(q, k, v, causal=True, prefix_lens=i32(90, 0))
    got = imq.attention(q, k, v, causal=True, q_lens=i32(1 << 30, 33), k_lens=i32(2 ** 31 - 1, 90), prefix_lens=i32(1 << 20, -5))
    assert torch.equal(got, want)
    out = torch.full_like(q, 3.0)
    imq.attention(q, k, v, q_lens=i32(-4, 0), k_lens=i32(90, 90), out=out)
    assert bool((out == 3.0).all())
    flat = lambda x: x.flatten(0, 1)
    out = torch.full_like(flat(q), 3.0)
    imq.attention(flat(q), flat(k), flat(v), q_offsets=i32(-9, 33, 1 << 30), k_offsets=i32(-1, 90, 1 << 29), max_q=33, max_k=90, out=out)
    want = imq.attention(q, k, v)
    assert torch.equal(out, flat(want))


def test_attention_nothing_to_do():
    z = lambda *s: torch.zeros(s, dtype=BF16, device="cuda")
    assert imq.attention(z(0, 5, 2, 64), z(0, 9, 2, 64), z(0, 9, 2, 64)).shape == (0, 5, 2, 64)
    assert imq.attention(z(0, 2, 64), z(9, 2, 64), z(9, 2, 64)).numel() == 0
    assert not imq.attention(z(3, 2, 64) + 1, z(0, 2, 64), z(0, 2, 64)).any()
    assert not imq.attention(z(100, 2, 64) + 1, z(0, 2, 64), z(0, 2, 64), causal=True).any()
    assert imq.rope(z(0, 2, 64), positions=torch.zeros(0, dtype=torch.int32, device="cuda"),
                    inv_freq=imq.rope_frequencies(64, device="cuda")[0]).numel() == 0
    assert imq.ln_mod(z(0, 64), torch.zeros(64, device="cuda"), torch.zeros(64, device="cuda")).numel() == 0


def test_rope_and_ln_mod_in_graphs():
    g = gen(12)
    q, k = randn(g, 5, 8, 128, dtype=F16), randn(g, 5, 2, 128, dtype=F16)
    pos = torch.arange(5, dtype=torch.int32, device="cuda")
    f, _ = imq.rope_frequencies(128, device="cuda")
    x, sh, sc = randn(g, 9, 512), randn(g, 512), randn(g, 512)
    qo, ko, y = torch.empty_like(q), torch.empty_like(k), torch.empty((9, 512), dtype=F16, device="cuda")
    run = lambda: (imq.rope(q, k, positions=pos, inv_freq=f, q_out=qo, k_out=ko), imq.ln_mod(x, sh, sc, out=y))
    run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for i in range(3):
        pos.add_(1000 * i)
        x.add_(0.5)
        graph.replay()
        torch.cuda.synchronize()
        got = qo.clone(), ko.clone(), y.clone()
        run()
        assert all(torch.equal(a, b) for a, b in zip(got, (qo, ko, y)))


# ------------------------------------------------------------------ refusals


def test_refusals():
    z = lambda *s, t=BF16: torch.zeros(s, dtype=t, device="cuda")
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
    q, k = z(2, 5, 4, 64), z(2, 9, 2, 64)
    bad = [dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=1e300), dict(softcap=-1.0),
           dict(softcap=float("inf")), dict(prefix_lens=i32(1, 1)), dict(q_lens=i32(1)), dict(k_lens=i32(1, 2).long()),
           dict(slopes=z(4)), dict(slopes=z(3, t=F32)), dict(out=z(2, 5, 4, 32)), dict(out=z(2, 5, 4, 64, t=F16)),
           dict(max_q=5), dict(q_offsets=i32(0, 5, 10), k_offsets=i32(0, 9, 18), max_q=5, max_k=9),
           dict(out=z(1, 5, 4, 64).expand(2, -1, -1, -1))]
    for kw in bad:
        with pytest.raises(ValueError):
            imq.attention(q, k, k, **kw)
    for a in ((q, z(2, 9, 3, 64), z(2, 9, 3, 64)), (q, z(2, 9, 2, 32), z(2, 9, 2, 32)), (q, k, z(2, 8, 2, 64)),
              (q, z(3, 9, 2, 64), z(3, 9, 2, 64)), (q, z(9, 2, 64), z(9, 2, 64)), (q[..., ::2], k[..., ::2], k[..., ::2]),
              (q, k.half(), k.half()), (q.cpu(), k, k), (q, k.cpu(), k.cpu())):
        with pytest.raises(ValueError):
            imq.attention(*a)
    with pytest.raises(ValueError, match="out is q"):
        imq.attention(q, k, k, out=q)
    with pytest.raises(NotImplementedError, match="softcap"):
        imq.attention(q, k, k, softcap=1e4)
    p = q.flatten(0, 1), k.flatten(0, 1), k.flatten(0, 1)
    for kw in (dict(q_offsets=i32(0, 5, 10)), dict(q_offsets=i32(0, 5, 10), k_offsets=i32(0, 9, 18)),
               dict(q_offsets=i32(0, 5, 10), k_offsets=i32(0, 18), max_q=5, max_k=9),
               dict(q_offsets=i32(0, 5, 10), k_offsets=i32(0, 9, 18), max_q=5, max_k=9, k_lens=i32(1, 1)),
               dict(q_offsets=i32(0, 5, 10), k_offsets=i32(0, 9, 18), max_q=-1, max_k=9)):
        with pytest.raises(ValueError):
            imq.attention(*p, **kw)
    for a in ((z(2, 5, 4, 64, t=F32),) + (z(2, 9, 2, 64, t=F32),) * 2, (z(2, 5, 4, 264),) + (z(2, 9, 2, 264),) * 2):
        with pytest.raises(NotImplementedError):
            imq.attention(*a)

    x, f = z(5, 4, 64), imq.rope_frequencies(64, device="cuda")[0]
    pos = i32(0, 1, 2, 3, 4)
    ok = dict(positions=pos, inv_freq=f)
    for kw in (dict(ok, positions=pos.long()), dict(ok, positions=pos[:4]), dict(ok, inv_freq=f.float()),
               dict(ok, inv_freq=f.cpu()), dict(ok, inv_freq=torch.cat([f, f])), dict(ok, sections=(16, 16)),
               dict(ok, positions=torch.stack([pos, pos], 1).contiguous()), dict(ok, sections=(31,)),
               dict(ok, positions=torch.stack([pos, pos], 1).contiguous(), sections=(40, -8)),
               dict(ok, q_weight=z(64)), dict(ok, q_weight=z(32, t=F32)), dict(ok, k_weight=z(64, t=F32)),
               dict(ok, eps=-1.0), dict(ok, amplitude=float("nan")), dict(ok, q_out=z(5, 4, 32)),
               dict(ok, q_out=z(1, 4, 64).expand(5, -1, -1)), dict(ok, q_out=z(4, 5, 64).transpose(0, 1)[..., :64].expand(5, 4, 64)[:, :1].expand(5, 4, 64))):
        with pytest.raises(ValueError):
            imq.rope(x, **kw)
    with pytest.raises(ValueError):
        imq.rope(x, x[:4], **ok)
    with pytest.raises(ValueError):
        imq.rope(z(5, 4, 63)[..., :63], **ok)
    with pytest.raises(NotImplementedError):
        imq.rope(z(5, 1, 1026), **ok)

    y, s = z(6, 64, t=F32), z(64, t=F32)
    for kw in (dict(eps=-1.0), dict(eps=float("nan")), dict(post_scale=float("inf")), dict(sets=i32(0, 0)),
               dict(sets=i32(*[0] * 6).long()), dict(out=z(6, 64, t=F32)[:, :32])):
        with pytest.raises(ValueError):
            imq.ln_mod(y, s, s, **kw)
    for a in ((y, s[0], s[0]), (y, s[:32], s[:32]), (y, s, s.half()), (y, torch.stack([s, s]), torch.stack([s, s])), (y.T, s[:6], s[:6]),
              (y.cpu(), s, s)):
        with pytest.raises(ValueError):
            imq.ln_mod(*a)
    with pytest.raises(NotImplementedError):
        imq.ln_mod(y, s, s, out_dtype=F32)
    with pytest.raises(NotImplementedError):
        imq.ln_mod(y.half(), s, s, out_dtype=BF16)
