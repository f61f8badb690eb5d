"""What a text encoder needs to serve many requests in one batch, as cases that can be timed and checked.

The operators, by a case's ``kind``:

* ``lora``   -- low-rank adapters of many requests beside a shared 4-bit projection:
                T(x . deq(W)^T + scale_i * (x . A_i^T) . B_i^T), i the adapter of the row, or none;
* ``shared`` -- softmax attention of sequences that all begin with the same keys (a system prompt, a
                template): the shared keys, which every query sees, then each sequence's own.

``own`` false computes them with elementary torch operations in 32 bits; true
calls the framework's entry points.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
SLOPES = 2.0 ** -8  # of the last head


def listed():
    return [
        # One token of one request through gate and up: the latency of the smallest calls.
        {"name": "lora-token", "kind": "lora", "m": 1, "k": 2560, "n": 9728, "rank": 16, "count": 8, "mixed": False, "rows": "runs",
         "requests": 1, "dtype": "bf16"},
        # The next tokens of 16 requests, each with its own adapter, of ranks from 8 to 64.
        {"name": "lora-tokens", "kind": "lora", "m": 16, "k": 2560, "n": 6144, "rank": 64, "count": 16, "mixed": True, "rows": "each",
         "requests": 16, "dtype": "bf16"},
        # The next tokens of 64 requests in any order through the way down, every fifth without an adapter.
        {"name": "lora-tokens-many", "kind": "lora", "m": 64, "k": 9728, "n": 2560, "rank": 32, "count": 24, "mixed": False, "rows": "each",
         "requests": 64, "dtype": "bf16"},
        # Eight short prompts of uneven lengths, an odd width.
        {"name": "lora-prompts", "kind": "lora", "m": 777, "k": 4096, "n": 2555, "rank": 24, "count": 5, "mixed": True, "rows": "runs",
         "requests": 8, "dtype": "bf16"},
        # The joint rows of a 1024 x 1024 image under one style's adapter.
        {"name": "lora-image", "kind": "lora", "m": 4608, "k": 2560, "n": 19456, "rank": 64, "count": 2, "mixed": False, "rows": "runs",
         "requests": 1, "dtype": "f16"},
        # Many prompts in one window, each with its adapter.
        {"name": "lora-window", "kind": "lora", "m": 4000, "k": 2560, "n": 6144, "rank": 16, "count": 32, "mixed": False, "rows": "runs",
         "requests": 40, "dtype": "bf16"},
        # The next token of eight requests behind a short template.
        {"name": "shared-token", "kind": "shared", "form": "cache", "seqs": 8, "q": 1, "k": 256, "shared": 512, "heads": 32, "kv": 8, "dim": 128,
         "causal": True, "cap": 0.0, "slopes": False, "dtype": "bf16"},
        # The next token of 64 requests behind one long system prompt.
        {"name": "shared-token-batch", "kind": "shared", "form": "cache", "seqs": 64, "q": 1, "k": 1024, "shared": 8192, "heads": 32, "kv": 8,
         "dim": 128, "causal": True, "cap": 0.0, "slopes": False, "dtype": "bf16"},
        # 16 questions about one book.
        {"name": "shared-token-long", "kind": "shared", "form": "cache", "seqs": 16, "q": 1, "k": 500, "shared": 65536, "heads": 32, "kv": 8,
         "dim": 128, "causal": True, "cap": 0.0, "slopes": False, "dtype": "bf16"},
        # Short prompts of uneven lengths, packed, behind an odd prefix; capped scores.
        {"name": "shared-documents", "kind": "shared", "form": "packed", "seqs": 61, "q": 77, "k": 77, "shared": 3001, "heads": 16, "kv": 8,
         "dim": 64, "causal": True, "cap": 30.0, "slopes": False, "dtype": "f16"},
        # A padded window of prompts behind a system prompt.
        {"name": "shared-prompts", "kind": "shared", "form": "batch", "seqs": 16, "q": 128, "k": 128, "shared": 2048, "heads": 32, "kv": 8,
         "dim": 128, "causal": True, "cap": 0.0, "slopes": False, "dtype": "bf16"},
        # Long prompts behind a long context, scores that fall with the distance.
        {"name": "shared-prompts-long", "kind": "shared", "form": "batch", "seqs": 4, "q": 2048, "k": 2048, "shared": 8192, "heads": 32, "kv": 8,
         "dim": 128, "causal": True, "cap": 0.0, "slopes": True, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_lora(rng):
    rows = rng.choice(["runs", "runs", "each"])
    m = _log(rng, 1, 64) if rng.random() < 0.5 else _log(rng, 17, 4608)
    c = {"kind": "lora", "m": m, "k": 64 * rng.choice([4 * rng.randint(1, 38), rng.randint(2, 152)]),
         "n": rng.choice([64 * rng.randint(2, 304), rng.randint(100, 19456)]), "rank": _log(rng, 1, 128), "count": _log(rng, 1, 64),
         "mixed": rng.random() < 0.4, "rows": rows, "requests": m if rows == "each" else min(m, _log(rng, 1, 48)),
         "dtype": rng.choice(["bf16", "bf16", "f16"])}
    while c["m"] * c["n"] * c["k"] > 4608 * 2560 * 19456:
        c["m"] = c["m"] * 2 // 3
        c["requests"] = min(c["requests"], c["m"])
    return c


def _draw_shared(rng):
    form = rng.choice(["cache", "cache", "batch", "packed"])
    kv = rng.choice([1, 2, 4, 8, 24])
    c = {"kind": "shared", "form": form, "heads": kv * rng.choice([1, 1, 2, 4, 5, 8]), "kv": kv, "dim": rng.choice([64, 128, 128, 128, 80, 96])}
    c["seqs"] = _log(rng, 1, 100)
    if form == "cache":
        c["q"] = rng.choice([1, 1, 1, 2, 5])
        c["k"] = max(c["q"], _log(rng, 1, 4096))
    else:
        c["q"] = c["k"] = _log(rng, 1, 2048)
    c["shared"] = _log(rng, 1, 65536)
    c["causal"] = rng.random() < 0.8
    c["cap"] = rng.choice([0.0, 0.0, 30.0, 50.0])
    c["slopes"] = rng.random() < 0.3
    c["dtype"] = rng.choice(["bf16", "bf16", "f16"])
    while c["seqs"] > 1 and c["seqs"] * c["k"] * kv * c["dim"] > 1 << 28:
        c["seqs"] = c["seqs"] * 2 // 3
    while c["seqs"] * c["q"] * (c["shared"] + c["k"]) * c["heads"] > 1_500_000_000 or c["seqs"] * (c["shared"] + c["k"]) * kv > 1 << 24:
        c["shared"] = max(1, c["shared"] * 2 // 3)
        c["seqs"] = max(1, c["seqs"] * 4 // 5)
    return c


def draw(rng):
    return _draw_lora(rng) if rng.random() < 0.5 else _draw_shared(rng)


# ---- inputs


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(1000003 * (seed + 1))


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _lengths(n, longest, least):
    """n lengths spread over [least, longest], the longest first."""
    return [max(least, int(longest * ((1.0 + 0.6180339887 * i) % 1.0 or 1.0))) for i in range(n)]


def _ranks(case):
    return [max(1, case["rank"] >> (i % 4)) if case["mixed"] else case["rank"] for i in range(case["count"])]


def _which(case):
    """The adapter of every row, -1 for every fifth request (but the first)."""
    m, n, count = case["m"], case["requests"], case["count"]
    of = [-1 if r % 5 == 4 else (7 * r + r // count) % count for r in range(n)]
    if case["rows"] == "each":
        return of
    weight = _lengths(n, 1000, 100)
    end, rows = 0, []
    for r in range(n):
        end += weight[r]
        rows += [of[r]] * (m * end // sum(weight) - len(rows))
    return rows


def _lora_inputs(case, seed):
    g, t = _gen(seed), DTYPES[case["dtype"]]
    m, k, n = case["m"], case["k"], case["n"]
    i = {"x": _randn(g, m, k).to(t),
         "w": torch.randint(-2 ** 31, 2 ** 31 - 1, (n, k // 8), generator=g, device="cuda", dtype=torch.int32),
         # Weights of about 1 / sqrt(K).
         "s": (_randn(g, n, k // 64).abs() / (4.0 * k ** 0.5)).to(t)}
    i["b"] = (-7.5 * i["s"].float() + _randn(g, n, k // 64) / (10.0 * k ** 0.5)).to(t)
    i["ab"] = [((_randn(g, r, k) / k ** 0.5).to(t), (0.2 * _randn(g, n, r) / r ** 0.5).to(t)) for r in _ranks(case)]
    i["c"] = [2.0 / (1 + a % 3) for a in range(case["count"])]
    i["rows"] = _which(case)
    return i


def _seq_lens(case):
    """(query rows, own key rows) of every sequence."""
    n, q, k = case["seqs"], case["q"], case["k"]
    if case["form"] == "cache":
        return [q] * n, _lengths(n, k, q)
    ln = _lengths(n, q, 0 if case["form"] == "packed" else 1)
    return ln, ln


def _shared_inputs(case, seed):
    g, t = _gen(seed), DTYPES[case["dtype"]]
    n, q, k, p, h, kv, d = (case[x] for x in ("seqs", "q", "k", "shared", "heads", "kv", "dim"))
    qn, kn = _seq_lens(case)
    i = {"form": case["form"], "qn": qn, "kn": kn, "causal": case["causal"], "cap": case["cap"], "scale": d ** -0.5, "max": (q, k),
         "sk": _randn(g, p, kv, d).to(t), "sv": _randn(g, p, kv, d).to(t)}
    if case["form"] == "cache":
        i["q"] = _randn(g, n, q, h, d).to(t)
        i["k"], i["v"] = _randn(g, n, k, kv, d).to(t), _randn(g, n, k, kv, d).to(t)
    else:  # columns of one projection's output
        rows = [sum(qn)] if case["form"] == "packed" else [n, q]
        qkv = _randn(g, *rows, (h + 2 * kv) * d).to(t)
        i["q"] = qkv[..., :h * d].unflatten(-1, (h, d))
        i["k"] = qkv[..., h * d:(h + kv) * d].unflatten(-1, (kv, d))
        i["v"] = qkv[..., (h + kv) * d:].unflatten(-1, (kv, d))
    i["slopes"] = torch.exp2(math.log2(SLOPES) * torch.arange(1, h + 1, device="cuda", dtype=torch.float32) / h) if case["slopes"] else None
    return i


def prepare(case, seed):
    if case["kind"] == "lora":
        st = _lora_inputs(case, seed)
        st["which"] = torch.tensor(st["rows"], dtype=torch.int32, device="cuda")
        if own:  # a server lays its adapters out once
            import aestrix_amd as imq

            st["adapters"] = imq.LoraAdapters(st["ab"], st["c"])
    else:
        st = _shared_inputs(case, seed)
        st["lens"] = {x: torch.tensor(st[x], dtype=torch.int32, device="cuda") for x in ("qn", "kn")}
        if case["form"] == "packed":
            at = [0]
            for m in st["qn"]:
                at.append(at[-1] + m)
            st["offsets"] = torch.tensor(at, dtype=torch.int32, device="cuda")
        # Rows behind a sequence's last are nobody's: they stay zero.
        st["out"] = torch.zeros(st["q"].shape, dtype=st["q"].dtype, device="cuda")
    st["kind"] = case["kind"]
    return st


# ---- the plain forms


def _weights(st):
    """deq(W) in the scales' type: scale * code + bias, rounded once."""
    w, s, b = st["w"], st["s"].float(), st["b"].float()
    codes = (w[..., None] >> torch.arange(0, 32, 4, device="cuda", dtype=torch.int32)) & 15
    codes = codes.reshape(w.shape[0], -1, 64).float()
    return (codes * s[..., None] + b[..., None]).to(st["s"].dtype).flatten(1)


def _plain_lora(st):
    x = st["x"].float()
    y = x @ _weights(st).float().t()
    for i, (a, b) in enumerate(st["ab"]):
        rows = torch.nonzero(st["which"] == i)[:, 0]
        if len(rows):
            y[rows] += (x[rows] @ a.float().t()) * st["c"][i] @ b.float().t()
    return y.to(st["x"].dtype)


def _plain_shared(st):
    out = torch.zeros_like(st["out"])
    a, p = 0, st["sk"].shape[0]
    for s, (nq, nk) in enumerate(zip(st["qn"], st["kn"])):
        where = slice(a, a + nq) if st["form"] == "packed" else (s, slice(0, nq))
        keys = slice(a, a + nk) if st["form"] == "packed" else (s, slice(0, nk))
        a += nq
        if nq == 0:
            continue
        q, k, v = st["q"][where], st["k"][keys], st["v"][keys]
        h, kv = q.shape[1], k.shape[1]
        group = h // kv
        # The last query stands at the last key.
        i, j = torch.arange(p + nk - nq, p + nk, device="cuda")[:, None], torch.arange(p + nk, device="cuda")
        step = max(1, min(kv, (1 << 29) // (nq * (p + nk) * group)))  # key heads at a time
        for b in range(0, kv, step):
            n = min(step, kv - b)
            qs = q[:, b * group:(b + n) * group].float().unflatten(1, (n, group)).permute(1, 2, 0, 3).reshape(n, group * nq, -1)
            kk = torch.cat([st["sk"][:, b:b + n], k[:, b:b + n]]).float()
            vv = torch.cat([st["sv"][:, b:b + n], v[:, b:b + n]]).float()
            e = torch.bmm(qs * st["scale"], kk.permute(1, 2, 0).contiguous()).view(n, group, nq, p + nk)
            if st["cap"]:
                e = torch.tanh(e / st["cap"]) * st["cap"]
            if st["slopes"] is not None:
                e = e - st["slopes"][b * group:(b + n) * group].view(n, group, 1, 1) * (i - j).abs().float()
            if st["causal"]:
                e = e.masked_fill((j > i) & (j >= p), -math.inf)
            e = torch.exp(e - e.amax(-1, keepdim=True))
            o = torch.bmm(e.view(n, group * nq, -1), vv.permute(1, 0, 2).contiguous()).view(n, group, nq, -1)
            o = o / e.sum(-1, keepdim=True)
            out[where][:, b * group:(b + n) * group] = o.permute(2, 0, 1, 3).flatten(1, 2).to(out.dtype)
    return out


# ---- a pass


def run(st):
    if not own:
        return _plain_lora(st) if st["kind"] == "lora" else _plain_shared(st)
    import aestrix_amd as imq

    if st["kind"] == "lora":
        return imq.quantized_matmul_lora(st["x"], st["w"], st["s"], st["b"], st["adapters"], st["which"])
    lens = st["lens"]
    if st["form"] == "packed":
        where = {"q_offsets": st["offsets"], "k_offsets": st["offsets"], "max_q": st["max"][0], "max_k": st["max"][1]}
    else:
        where = {"q_lens": None if st["form"] == "cache" else lens["qn"], "k_lens": lens["kn"]}
    return imq.attention_shared(st["q"], st["k"], st["v"], st["sk"], st["sv"], scale=st["scale"], causal=st["causal"], softcap=st["cap"],
                                slopes=st["slopes"], out=st["out"], **where)


# ---- the same in 64 bits


def _exact_lora(case, seed):
    i = _lora_inputs(case, seed)
    n, k = case["n"], case["k"]
    x = i["x"].double()
    out = torch.empty((case["m"], n), dtype=torch.float64, device="cuda")
    words = i["w"].long()
    for a in range(0, n, 4096):
        r = slice(a, min(n, a + 4096))
        w = torch.empty((r.stop - a, k // 8, 8), dtype=torch.float64, device="cuda")
        for c in range(8):
            w[..., c] = torch.bitwise_and(torch.bitwise_right_shift(words[r], 4 * c), 15).double()
        w = w.view(-1, k // 64, 64)
        # The projection's weights are values of its type: that rounding is part of its definition.
        w = (w * i["s"][r].double()[..., None] + i["b"][r].double()[..., None]).to(torch.float32).to(i["s"].dtype).double()
        out[:, r] = torch.mm(x, w.view(-1, k).T)
    start = 0
    while start < case["m"]:  # runs of rows of one adapter
        end = start + 1
        while end < case["m"] and i["rows"][end] == i["rows"][start]:
            end += 1
        which = i["rows"][start]
        if which >= 0:
            a, b = i["ab"][which]
            out[start:end] += i["c"][which] * torch.mm(torch.mm(x[start:end], a.double().T), b.double().T)
        start = end
    return out


def _exact_shared(case, seed):
    i = _shared_inputs(case, seed)
    qn, kn = _seq_lens(case)
    group = case["heads"] // case["kv"]
    p = case["shared"]
    out = torch.zeros(i["q"].shape, dtype=torch.float64, device="cuda")
    a = 0
    for s in range(case["seqs"]):
        nq, nk = qn[s], kn[s]
        r = slice(a, a + nq)
        a += nq
        if nq == 0:
            continue
        packed = case["form"] == "packed"
        q, o = (x[r] if packed else x[s, :nq] for x in (i["q"], out))
        k, v = (x[r] if packed else x[s, :nk] for x in (i["k"], i["v"]))
        for h in range(case["heads"]):
            kh = h // group
            at = torch.arange(nq, device="cuda")[:, None] + (nk - nq)  # of the own keys
            scores = []
            for keys, first in ((i["sk"], -p), (k, 0)):
                e = q[:, h].double() @ keys[:, kh].double().T.contiguous() * case["dim"] ** -0.5
                if case["cap"]:
                    e = case["cap"] * torch.tanh(e / case["cap"])
                j = torch.arange(first, first + len(keys), device="cuda")[None]
                if case["slopes"]:
                    e -= SLOPES ** ((h + 1) / case["heads"]) * (at - j).abs()
                if case["causal"] and first == 0:
                    e[j > at] = -math.inf
                scores.append(e)
            w = torch.softmax(torch.cat(scores, 1), -1)
            o[:, h] = w[:, :p] @ i["sv"][:, kh].double() + w[:, p:] @ v[:, kh].double()
    return out


def exact(case, seed):
    return _exact_lora(case, seed) if case["kind"] == "lora" else _exact_shared(case, seed)


# ---- what a pass cannot do without


def _seen(nq, nk, causal):
    """Visible pairs of a sequence's queries and own keys."""
    return nq * nk - (nq * (nq - 1) // 2 if causal else 0) if nq <= nk else nk * nk - nk * (nk - 1) // 2 if causal else nq * nk


def work(case):
    if case["kind"] == "lora":
        m, n, k = case["m"], case["n"], case["k"]
        ranks, rows = _ranks(case), _which(case)
        used = sorted({r for r in rows if r >= 0})
        return {"bytes": n * k // 2 + 4 * n * (k // 64) + 2 * m * (k + n) + 4 * m + 2 * (k + n) * sum(ranks[i] for i in used),
                "flops": 2 * m * n * k + 2 * (k + n) * sum(ranks[r] for r in rows if r >= 0)}
    qn, kn = _seq_lens(case)
    d, h, kv = case["dim"], case["heads"], case["kv"]
    pairs = sum(a * case["shared"] + _seen(a, b, case["causal"]) for a, b in zip(qn, kn))
    keys = case["shared"] + sum(b if a else 0 for a, b in zip(qn, kn))
    return {"bytes": 2 * d * (2 * h * sum(qn) + 2 * kv * keys) + 8 * len(qn), "flops": 4 * d * h * pairs}
