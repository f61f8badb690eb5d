"""The core of a transformer block between its quantized projections, as cases that can be timed and checked.

The operators, by a case's ``kind``:

* ``lnmod``     -- LayerNorm with a modulation from the conditioning vector:
                   T(((x - mean) / sqrt(var + eps) * (1 + scale) + shift) * post);
* ``rope``      -- per-head RMSNorm (or none) and rotary positions of the query and key heads:
                   pairs in the half or the interleaved layout, all or a part of the head,
                   one to four position axes, frequencies scaled for long contexts;
* ``attention`` -- softmax attention with grouped heads: causal or not, a prefix that every query
                   sees, documents packed into one row sequence, scores capped by a tanh, a bias
                   that falls with the distance; whole prompts, images, and single tokens over a cache.

``own`` false computes them with elementary torch operations in 32 bits; true
calls the framework's entry points.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZES = {"bf16": 2, "f16": 2, "f32": 4}


def listed():
    return [
        # The joint residual of a 512 x 512 image: 1024 image and 512 text rows, each with its own modulation.
        {"name": "lnmod-512px", "kind": "lnmod", "rows": 1536, "cols": 3072, "sets": 2, "in": "f32", "dtype": "f16"},
        # The same of a 1024 x 1024 image, 4096 image rows.
        {"name": "lnmod-1024px", "kind": "lnmod", "rows": 4608, "cols": 3072, "sets": 2, "in": "f32", "dtype": "f16"},
        # The next token of four sequences: the keys go straight into the cache.
        {"name": "rope-token", "kind": "rope", "rows": 4, "heads": 32, "kv": 8, "dim": 128, "rot": 128, "axes": 1, "interleaved": False,
         "norm": True, "far": 4096, "scaling": "none", "cache": True, "dtype": "bf16"},
        # The query and key heads of a 1024 x 1024 image's joint rows: four axes, interleaved pairs.
        {"name": "rope-1024px", "kind": "rope", "rows": 4608, "heads": 24, "kv": 24, "dim": 128, "rot": 128, "axes": 4, "interleaved": True,
         "norm": True, "far": 64, "scaling": "none", "cache": False, "dtype": "f16"},
        # A long document, half of each head rotated, frequencies stretched to positions past a million.
        {"name": "rope-long", "kind": "rope", "rows": 16001, "heads": 32, "kv": 8, "dim": 128, "rot": 64, "axes": 1, "interleaved": False,
         "norm": False, "far": 1 << 20, "scaling": "yarn", "cache": False, "dtype": "bf16"},
        # The next token of eight sequences of many lengths: the latency of the smallest calls.
        {"name": "attention-token", "kind": "attention", "form": "cache", "seqs": 8, "q": 1, "k": 2048, "heads": 32, "kv": 8, "dim": 128,
         "causal": True, "prefix": False, "cap": 0.0, "slopes": False, "dtype": "bf16"},
        # One token over one very long cache.
        {"name": "attention-token-long", "kind": "attention", "form": "cache", "seqs": 1, "q": 1, "k": 131072, "heads": 32, "kv": 8, "dim": 128,
         "causal": True, "prefix": False, "cap": 0.0, "slopes": False, "dtype": "bf16"},
        # A padded window of four prompts through a text-encoder layer.
        {"name": "attention-prompts", "kind": "attention", "form": "batch", "seqs": 4, "q": 512, "k": 512, "heads": 32, "kv": 8, "dim": 128,
         "causal": True, "prefix": False, "cap": 0.0, "slopes": False, "dtype": "bf16"},
        # Many short documents packed into one sequence of rows, each with a prefix that it sees whole.
        {"name": "attention-documents", "kind": "attention", "form": "packed", "seqs": 61, "q": 777, "k": 777, "heads": 16, "kv": 8, "dim": 64,
         "causal": True, "prefix": True, "cap": 30.0, "slopes": False, "dtype": "f16"},
        # The joint rows of a 1024 x 1024 image: every row sees every row.
        {"name": "attention-1024px", "kind": "attention", "form": "batch", "seqs": 1, "q": 4608, "k": 4608, "heads": 24, "kv": 24, "dim": 128,
         "causal": False, "prefix": False, "cap": 0.0, "slopes": False, "dtype": "f16"},
        # One long prompt, scores that fall with the distance.
        {"name": "attention-long", "kind": "attention", "form": "batch", "seqs": 1, "q": 16384, "k": 16384, "heads": 32, "kv": 8, "dim": 128,
         "causal": True, "prefix": False, "cap": 0.0, "slopes": True, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_rope(rng):
    cache = rng.random() < 0.3
    dim = rng.choice([64, 80, 96, 128, 128, 128, 256])
    kv = rng.choice([1, 2, 4, 8, 24])
    heads = kv * rng.choice([1, 1, 2, 4, 5])
    c = {"kind": "rope", "rows": _log(rng, 1, 64) if cache else _log(rng, 1, 16384), "heads": heads, "kv": kv, "dim": dim,
         "rot": rng.choice([dim, dim, dim // 2]), "axes": rng.choice([1, 1, 2, 3, 4]), "interleaved": rng.random() < 0.5,
         "norm": rng.random() < 0.6, "far": _log(rng, 64, 1 << 20), "scaling": rng.choice(["none", "none", "linear", "yarn"]),
         "cache": cache, "dtype": rng.choice(["bf16", "bf16", "f16", "f32"])}
    while c["rows"] * (heads + kv) * dim * SIZES[c["dtype"]] > 16001 * 40 * 128 * 2:
        c["rows"] = c["rows"] * 2 // 3
    return c


def _draw_attention(rng):
    form = rng.choice(["cache", "cache", "batch", "packed"])
    kv = rng.choice([1, 2, 4, 8, 24])
    heads = kv * rng.choice([1, 1, 2, 3, 4, 8])
    c = {"kind": "attention", "form": form, "heads": heads, "kv": kv, "dim": rng.choice([64, 128, 128, 128, 80, 96])}
    if form == "cache":
        c["seqs"], c["q"] = _log(rng, 1, 64), rng.choice([1, 1, 1, 2, 7, 65])
        c["k"] = max(c["q"], _log(rng, 1, 131072))
    else:
        c["seqs"] = _log(rng, 1, 8 if form == "batch" else 100)
        c["q"] = c["k"] = _log(rng, 1, 8192 if form == "batch" else 2048)
        if form == "batch" and rng.random() < 0.3:  # a window that reads the rows of another
            c["k"] = _log(rng, 1, 4096)
    c["causal"] = rng.random() < 0.6
    c["prefix"] = c["causal"] and rng.random() < 0.3
    c["cap"] = rng.choice([0.0, 0.0, 30.0, 50.0])
    c["slopes"] = rng.random() < 0.3
    c["dtype"] = rng.choice(["bf16", "bf16", "f16"])
    while c["seqs"] > 1 and c["seqs"] * c["k"] * kv * c["dim"] > 1 << 28:
        c["seqs"] = c["seqs"] * 2 // 3
    while c["seqs"] * c["q"] * c["k"] * heads > 16384 * 16384 * 16:
        c["k"] = c["k"] * 2 // 3
        c["q"] = min(c["q"], c["k"])
    return c


def draw(rng):
    kind = rng.choice(["lnmod", "rope", "rope", "attention", "attention", "attention"])
    if kind == "rope":
        return _draw_rope(rng)
    if kind == "attention":
        return _draw_attention(rng)
    dtype = rng.choice(["f16", "bf16"])
    return {"kind": kind, "rows": _log(rng, 1, 8192), "cols": rng.choice([64 * rng.randint(4, 80), rng.randint(200, 5120)]),
            "sets": rng.choice([1, 2, 5]), "in": rng.choice(["f32", "f32", dtype]), "dtype": dtype}


# ---- inputs


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(1000003 * (seed + 1))


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _lengths(n, longest, least):
    """n lengths spread over [least, longest], the longest first."""
    return [max(least, int(longest * ((1.0 + 0.6180339887 * i) % 1.0 or 1.0))) for i in range(n)]


def _lens(case):
    """(query rows, key rows) of every sequence."""
    n, q, k = case["seqs"], case["q"], case["k"]
    if case["form"] == "cache":
        return [q] * n, _lengths(n, k, q)
    if case["form"] == "packed":
        ln = _lengths(n, q, 0)
        return ln, ln
    if q == k:
        ln = _lengths(n, q, 1)
        return ln, ln
    return [q] * n, _lengths(n, k, 1)


def _prefixes(case):
    return [n // 3 for n in _lens(case)[1]] if case["prefix"] else None


def _frequencies(case):
    """Radians a position of every pair (float64), the pairs of each axis, and the amplitude."""
    pairs = case["rot"] // 2
    axes = min(case["axes"], pairs)
    sections = [pairs // axes + (1 if a < pairs % axes else 0) for a in range(axes)]
    base = 2000.0 if axes > 1 else 1e6
    f = torch.cat([base ** -(torch.arange(s, dtype=torch.float64) / s) for s in sections])
    amplitude = 1.0
    if case["scaling"] == "linear":
        f = f / 8.0
    elif case["scaling"] == "yarn":  # slow pairs stretched by the factor, fast ones kept, a ramp between
        factor, old = 32.0, 32768.0
        turns = old * f / (2.0 * math.pi)
        keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0.0, 1.0)
        f = f * keep + f / factor * (1.0 - keep)
        amplitude = 0.1 * math.log(factor) + 1.0
    return f.cuda(), sections, amplitude


def _rope_inputs(case, seed):
    g, t = _gen(seed), DTYPES[case["dtype"]]
    rows, h, kv, d = case["rows"], case["heads"], case["kv"], case["dim"]
    f, sections, amplitude = _frequencies(case)
    i = {"qkv": _randn(g, rows, (h + 2 * kv) * d).to(t), "freq": f, "sections": sections, "amplitude": amplitude}
    if case["cache"] or len(sections) > 1:  # one position a sequence, or rows of patches and words
        i["pos"] = torch.randint(0, case["far"], (rows, len(sections)), generator=g, device="cuda", dtype=torch.int32)
    else:
        first = int(torch.randint(0, max(1, case["far"] - rows), (1,), generator=torch.Generator().manual_seed(seed)))
        i["pos"] = torch.arange(first, first + rows, device="cuda", dtype=torch.int32)[:, None]
    if case["norm"]:
        i["qw"], i["kw"] = 1.0 + 0.1 * _randn(g, d), 1.0 + 0.1 * _randn(g, d)
    else:
        i["qw"] = i["kw"] = None
    i["q"] = i["qkv"][:, :h * d].unflatten(1, (h, d))
    i["k"] = i["qkv"][:, h * d:(h + kv) * d].unflatten(1, (kv, d))
    i["interleaved"] = case["interleaved"]
    i["kcache"] = torch.zeros((rows, 8, kv, d), dtype=t, device="cuda")[:, 5] if case["cache"] else None
    return i


def _attention_inputs(case, seed):
    g, t = _gen(seed), DTYPES[case["dtype"]]
    n, q, k, h, kv, d = (case[x] for x in ("seqs", "q", "k", "heads", "kv", "dim"))
    qn, kn = _lens(case)
    i = {"form": case["form"], "qn": qn, "kn": kn, "pre": _prefixes(case), "causal": case["causal"], "cap": case["cap"],
         "scale": d ** -0.5, "max": (q, k)}
    if case["form"] == "cache":
        i["q"] = _randn(g, n, q, h, d).to(t)
        i["k"], i["v"] = (torch.empty((n, k, kv, d), dtype=t, device="cuda") for _ in range(2))
        for b in range(n):
            i["k"][b], i["v"][b] = _randn(g, k, kv, d).to(t), _randn(g, k, kv, d).to(t)
    else:
        rows = [sum(qn)] if case["form"] == "packed" else [n, q]
        if q == k:  # columns of one projection's output
            qkv = _randn(g, *rows, (h + 2 * kv) * d).to(t)
            i["q"] = qkv[..., :h * d].unflatten(-1, (h, d))
            i["k"] = qkv[..., h * d:(h + kv) * d].unflatten(-1, (kv, d))
            i["v"] = qkv[..., (h + kv) * d:].unflatten(-1, (kv, d))
        else:
            i["q"], i["k"], i["v"] = _randn(g, n, q, h, d).to(t), _randn(g, n, k, kv, d).to(t), _randn(g, n, k, kv, d).to(t)
    i["slopes"] = torch.exp2(-8.0 * torch.arange(1, h + 1, device="cuda", dtype=torch.float32) / h) if case["slopes"] else None
    return i


def prepare(case, seed):
    kind = case["kind"]
    if kind == "rope":
        st = _rope_inputs(case, seed)
    elif kind == "attention":
        st = _attention_inputs(case, seed)
        ints = {"qn": st["qn"], "kn": st["kn"], "pre": st["pre"]}
        st["lens"] = {x: None if v is None else torch.tensor(v, dtype=torch.int32, device="cuda") for x, v in ints.items()}
        if case["form"] == "packed":
            at = [0]
            for m in st["qn"]:
                at.append(at[-1] + m)
            st["offsets"] = torch.tensor(at, dtype=torch.int32, device="cuda")
        # Rows behind a sequence's last are nobody's: they stay zero.
        st["out"] = torch.zeros(st["q"].shape, dtype=st["q"].dtype, device="cuda")
    else:
        g = _gen(seed)
        rows, cols, n = case["rows"], case["cols"], case["sets"]
        st = {"x": (2.0 * _randn(g, rows, cols) + 0.5).to(DTYPES[case["in"]]), "shift": 0.3 * _randn(g, n, cols), "scale": 0.3 * _randn(g, n, cols),
              "t": DTYPES[case["dtype"]]}
        # Runs of rows that share a modulation: the text rows, then the image rows.
        st["sets"] = (torch.arange(rows, device="cuda") * n // rows).to(torch.int32) if n > 1 else None
    st["kind"] = kind
    return st


# ---- the plain forms


def _turn(x, cos, sin, interleaved):
    """The pairs of x [rows, heads, rot] turned by the angles [rows, 1, rot / 2]."""
    if interleaved:
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    a, b = x.chunk(2, -1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _plain_rope(st):
    axis = torch.cat([torch.full((n,), a, device="cuda") for a, n in enumerate(st["sections"])])
    angle = st["pos"].double()[:, axis] * st["freq"]  # far positions: 32 bits keep no angle
    cos, sin = ((f(angle) * st["amplitude"]).float()[:, None] for f in (torch.cos, torch.sin))
    out = []
    for x, w in ((st["q"], st["qw"]), (st["k"], st["kw"])):
        y = x.float()
        if w is not None:
            y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-6) * w
        rot = 2 * cos.shape[-1]
        out.append(torch.cat([_turn(y[..., :rot], cos, sin, st["interleaved"]), y[..., rot:]], -1).to(x.dtype))
    if st["kcache"] is not None:
        st["kcache"].copy_(out[1])
        out[1] = st["kcache"]
    return {"q": out[0], "k": out[1]}


def _sequences(st):
    """(queries, keys, values, where the output goes, prefix) of every sequence."""
    a = 0
    for s, (nq, nk) in enumerate(zip(st["qn"], st["kn"])):
        pre = st["pre"][s] if st["pre"] else 0
        if st["form"] == "packed":
            r = slice(a, a + nq)
            a += nq
            yield st["q"][r], st["k"][r], st["v"][r], r, pre
        else:
            yield st["q"][s, :nq], st["k"][s, :nk], st["v"][s, :nk], (s, slice(0, nq)), pre


def _plain_attention(st):
    out = torch.zeros_like(st["out"])
    for q, k, v, where, pre in _sequences(st):
        nq, nk, h = q.shape[0], k.shape[0], q.shape[1]
        if nq == 0 or nk == 0:
            continue
        # The last query stands at the last key.
        i, j = torch.arange(nk - nq, nk, device="cuda")[:, None], torch.arange(nk, device="cuda")
        seen = (j <= i) | (j < pre) if st["causal"] else None
        away = -(i - j).abs().float() if st["slopes"] is not None else None
        group = h // k.shape[1]
        step = max(1, min(k.shape[1], (1 << 30) // (nq * nk * group)))  # key heads at a time
        for a in range(0, k.shape[1], step):
            n = min(step, k.shape[1] - a)
            qs = q[:, a * group:(a + n) * group].float().unflatten(1, (n, group)).permute(1, 2, 0, 3).reshape(n, group * nq, -1)
            s = torch.bmm(qs * st["scale"], k[:, a:a + n].float().permute(1, 2, 0).contiguous()).view(n, group, nq, nk)
            if st["cap"]:
                s = torch.tanh(s / st["cap"]) * st["cap"]
            if away is not None:
                s = s + st["slopes"][a * group:(a + n) * group].view(n, group, 1, 1) * away
            if seen is not None:
                s = s.masked_fill(~seen, -math.inf)
            top = s.amax(-1, keepdim=True)
            s = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
            total = s.sum(-1, keepdim=True)
            o = torch.bmm(s.view(n, group * nq, nk), v[:, a:a + n].float().permute(1, 0, 2).contiguous()).view(n, group, nq, -1)
            o = o / torch.where(total == 0, 1.0, total)  # a row that sees nothing is zero
            out[where][:, a * group:(a + n) * group] = o.permute(2, 0, 1, 3).flatten(1, 2).to(out.dtype)
    return out


def _plain_lnmod(st):
    x = st["x"].float()
    x = x - x.mean(-1, keepdim=True)
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)
    if st["sets"] is None:
        y = x * (1.0 + st["scale"][0]) + st["shift"][0]
    else:
        y = x * (1.0 + st["scale"])[st["sets"]] + st["shift"][st["sets"]]
    return (y * 0.0625).to(st["t"])


# ---- a pass


def run(st):
    kind = st["kind"]
    if not own:
        return {"rope": _plain_rope, "attention": _plain_attention, "lnmod": _plain_lnmod}[kind](st)
    import aestrix_amd as imq

    if kind == "rope":
        q, k = imq.rope(st["q"], st["k"], positions=st["pos"], inv_freq=st["freq"], sections=st["sections"], interleaved=st["interleaved"],
                        amplitude=st["amplitude"], q_weight=st["qw"], k_weight=st["kw"], eps=1e-6, k_out=st["kcache"])
        return {"q": q, "k": k}
    if kind == "lnmod":
        return imq.ln_mod(st["x"], st["shift"], st["scale"], sets=st["sets"], eps=1e-6, post_scale=0.0625, out_dtype=st["t"])
    lens = st["lens"]
    if st["form"] == "packed":
        where = {"q_offsets": st["offsets"], "k_offsets": st["offsets"], "max_q": st["max"][0], "max_k": st["max"][1]}
    else:
        where = {"q_lens": None if st["form"] == "cache" else lens["qn"], "k_lens": lens["kn"]}
    return imq.attention(st["q"], st["k"], st["v"], scale=st["scale"], causal=st["causal"], softcap=st["cap"], slopes=st["slopes"],
                         prefix_lens=lens["pre"], out=st["out"], **where)


# ---- the same in 64 bits


def _exact_rope(case, seed):
    i = _rope_inputs(case, seed)
    pairs = case["rot"] // 2
    angle, a = torch.empty((case["rows"], pairs), dtype=torch.float64, device="cuda"), 0
    for axis, n in enumerate(i["sections"]):
        angle[:, a:a + n] = torch.outer(i["pos"][:, axis].double(), i["freq"][a:a + n])
        a += n
    z = torch.polar(torch.full_like(angle, i["amplitude"]), angle)[:, None]  # a turn is a complex product
    out = {}
    for name, w in (("q", i["qw"]), ("k", i["kw"])):
        y = i[name].double()
        if w is not None:
            y = y / torch.sqrt((y * y).sum(-1, keepdim=True) / case["dim"] + 1e-6) * w.double()
        r = y[..., :2 * pairs]
        order = torch.arange(2 * pairs, device="cuda").view(*((pairs, 2) if case["interleaved"] else (2, pairs)))
        order = order if case["interleaved"] else order.T
        c = torch.complex(r[..., order[:, 0]], r[..., order[:, 1]]) * z
        y[..., order[:, 0]], y[..., order[:, 1]] = c.real, c.imag
        out[name] = y
    return out


def _exact_attention(case, seed):
    i = _attention_inputs(case, seed)
    qn, kn = _lens(case)
    group = case["heads"] // case["kv"]
    out = torch.zeros(i["q"].shape, dtype=torch.float64, device="cuda")
    a = 0
    for s in range(case["seqs"]):
        nq, nk = qn[s], kn[s]
        r = slice(a, a + nq)
        a += nq
        packed = case["form"] == "packed"
        q, o = (x[r] if packed else x[s, :nq] for x in (i["q"], out))
        k, v = (x[r] if packed else x[s, :nk] for x in (i["k"], i["v"]))
        for b in range(0, nq, 4096):
            rows = torch.arange(b, min(nq, b + 4096), device="cuda")
            if len(rows) == 0 or nk == 0:
                continue
            at = rows + (nk - nq)
            hide = None
            if case["causal"]:
                hide = torch.arange(nk, device="cuda")[None] > at[:, None]
                if i["pre"]:
                    hide[:, :i["pre"][s]] = False
            for h in range(case["heads"]):
                e = q[rows, h].double() @ k[:, h // group].double().T.contiguous() * case["dim"] ** -0.5
                if case["cap"]:
                    e = case["cap"] * torch.tanh(e / case["cap"])
                if case["slopes"]:
                    e -= 2.0 ** (-8.0 * (h + 1) / case["heads"]) * (at[:, None] - torch.arange(nk, device="cuda")).abs()
                if hide is not None:
                    e[hide] = -math.inf
                p = torch.softmax(e, -1)
                if hide is not None:
                    p = torch.nan_to_num(p, nan=0.0)
                o[rows, h] = p @ v[:, h // group].double()
    return out


def exact(case, seed):
    if case["kind"] == "rope":
        return _exact_rope(case, seed)
    if case["kind"] == "attention":
        return _exact_attention(case, seed)
    st = prepare(case, seed)
    x = st["x"].double()
    x = (x - x.mean(-1, keepdim=True)) / torch.sqrt(x.var(-1, unbiased=False, keepdim=True) + 1e-6)
    rows = torch.zeros(case["rows"], dtype=torch.long, device="cuda") if st["sets"] is None else st["sets"].long()
    return (x * (1.0 + st["scale"].double()[rows]) + st["shift"].double()[rows]) / 16.0


# ---- what a pass cannot do without


def _pairs(nq, nk, causal, pre):
    """Visible (query, key) pairs of a sequence."""
    if not causal:
        return nq * nk
    total = 0
    first = nk - nq + 1  # keys the first query sees
    lo, hi = max(0, min(pre, nk)), nk
    # queries whose own count is above the prefix
    for a, b in ((first, nk),):
        n_low = max(0, min(nq, lo - a + 1))  # those with count <= lo
        total += n_low * lo
        a2 = a + n_low
        total += (a2 + b) * (b - a2 + 1) // 2 if a2 <= b else 0
    return total


def work(case):
    kind = case["kind"]
    size = SIZES[case["dtype"]]
    if kind == "lnmod":
        n = case["rows"] * case["cols"]
        return {"bytes": n * (SIZES[case["in"]] + size) + 8 * case["sets"] * case["cols"] + (4 * case["rows"] if case["sets"] > 1 else 0),
                "flops": 8 * n}
    if kind == "rope":
        n = case["rows"] * (case["heads"] + case["kv"]) * case["dim"]
        return {"bytes": 2 * n * size + 4 * case["rows"] * min(case["axes"], case["rot"] // 2) + 4 * case["rot"] + (8 * case["dim"] if case["norm"] else 0),
                "flops": n * (3 + (4 if case["norm"] else 0))}
    qn, kn = _lens(case)
    pre = _prefixes(case) or [0] * len(qn)
    d, h, kv = case["dim"], case["heads"], case["kv"]
    pairs = sum(_pairs(a, b, case["causal"], p) for a, b, p in zip(qn, kn, pre))
    keys = sum(b if a else 0 for a, b in zip(qn, kn))
    return {"bytes": size * d * (2 * h * sum(qn) + 2 * kv * keys) + 8 * len(qn), "flops": 4 * d * h * pairs}
