"""The block core's operators from their definitions in 64 bits, with the error
that the kernels' number formats allow (used by test_gpu_core*.py).

Every bound counts the roundings that the definition names: half a step of T at
the end (eps(T) / 2 relative), the softmax's weights rounded to T, and 32-bit
sums and products (2^-24 each, worst case: as many as there are terms)."""

from __future__ import annotations

import torch

U32 = 2.0 ** -24  # half a step of float32


def half_step(t: torch.dtype) -> float:
    return torch.finfo(t).eps / 2


def least(t: torch.dtype) -> float:
    """Half the smallest subnormal step: what rounding can cost next to zero."""
    return torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2


def seen_keys(nq: int, nk: int, causal: bool, prefix: int, device) -> torch.Tensor:
    """[nq, nk] of what each query sees."""
    if not causal:
        return torch.ones((nq, nk), dtype=torch.bool, device=device)
    p = torch.arange(nq, device=device)[:, None] + (nk - nq)
    j = torch.arange(nk, device=device)[None]
    return (j <= p) | (j < prefix)


def attention_sequence(q, k, v, *, scale, causal=False, softcap=0.0, slopes=None, prefix=0):
    """(o, bound) of one sequence: q [nq, h, d], k and v [nk, hk, d]; float64 [nq, h, d].

    Keys that a query does not see are left out of its sums, so what they hold does not
    matter."""
    nq, h, d = q.shape
    nk, hk = k.shape[0], k.shape[1]
    t = q.dtype
    o = torch.zeros((nq, h, d), dtype=torch.float64, device=q.device)
    bound = torch.full_like(o, least(t))
    if nq == 0 or nk == 0:
        return o, bound
    seen = seen_keys(nq, nk, causal, prefix, q.device)
    away = (torch.arange(nq, device=q.device)[:, None] + (nk - nq) -
            torch.arange(nk, device=q.device)[None]).abs().double()
    n = seen.sum(-1, keepdim=True).double()
    for i in range(h):
        qi, ki, vi = q[:, i].double(), k[:, i // (h // hk)].double(), v[:, i // (h // hk)].double()
        # Hidden keys may hold anything: zero where no query sees them at all.
        used = seen.any(0)
        ki, vi = ki.clone(), vi.clone()
        ki[~used], vi[~used] = 0.0, 0.0
        e = scale * (qi @ ki.T.contiguous())
        mag = scale * (qi.abs() @ ki.abs().T.contiguous())
        err = (d + 8) * U32 * mag  # the dot product, then its scale
        if softcap:
            e = softcap * torch.tanh(e / softcap)
            err = err + 8 * U32 * softcap  # the capped score's own steps are of the cap's size
        if slopes is not None:
            e = e - slopes[i].double() * away
            err = err + 4 * U32 * slopes[i].double().abs() * away
        e = e.masked_fill(~seen, -torch.inf)
        top = e.amax(-1, keepdim=True)
        top = torch.where(top == -torch.inf, 0.0, top)
        # exp's argument is rounded (its size), and a weight near its limit moves by that.
        err = err + 4 * U32 * (e - top).abs().nan_to_num(posinf=0.0)
        w = torch.exp(e - top)
        total = w.sum(-1, keepdim=True)
        p = torch.where(total > 0, w / total, 0.0)
        oi = torch.zeros((nq, d), dtype=torch.float64, device=q.device)
        ai = torch.zeros_like(oi)
        ei = torch.zeros_like(oi)
        big = torch.zeros_like(oi)
        av = vi.abs()
        oi += p @ vi
        ai += p @ av
        # A weight's relative error moves its term, and the sum that divides it.
        ei += (p * (err * 1.01).nan_to_num(posinf=0.0)) @ av
        ei += (p * err.nan_to_num(posinf=0.0)).sum(-1, keepdim=True) * ai
        if t == torch.float16:  # weights under 2^-14 keep an absolute 2^-25
            big += torch.where(total > 0, 2.0 ** -25 / total, 0.0) * (seen.double() @ av)
        o[:, i] = oi
        bound[:, i] += half_step(t) * oi.abs() + 1.02 * (
            ei + (half_step(t) + (2 * n + 32) * U32) * ai + big)
    return o, bound


def rope(x, positions, inv_freq, sections, interleaved, amplitude, weight, eps):
    """(y, bound) of x [rows, heads, dim]; float64."""
    rows, _, dim = x.shape
    y = x.double()
    err = torch.zeros_like(y)
    if weight is not None:
        y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + eps) * weight.double()
        err = y.abs() * (dim / 2 + 8) * U32  # half of the sum of squares' worst case, and the rest
    half = inv_freq.shape[0]
    pos = positions.view(rows, -1).double()
    sections = [half] if sections is None else list(sections)
    axis = torch.cat([torch.full((n,), a, dtype=torch.long) for a, n in enumerate(sections)]).to(x.device)
    angle = pos[:, axis] * inv_freq
    c, s = (torch.cos(angle) * amplitude)[:, None], (torch.sin(angle) * amplitude)[:, None]
    r, re = y[..., :2 * half], err[..., :2 * half]
    if interleaved:
        a, b, ea, eb = r[..., 0::2], r[..., 1::2], re[..., 0::2], re[..., 1::2]
    else:
        a, b, ea, eb = r[..., :half], r[..., half:], re[..., :half], re[..., half:]
    # cos and sin: 2 steps each from sincospi, 2 more from the reduced angle and the amplitude.
    turn = abs(amplitude) * (a.abs() + b.abs()) * 8 * U32
    out = [a * c - b * s, b * c + a * s]
    e = [ea * c.abs() + eb * s.abs() + turn, eb * c.abs() + ea * s.abs() + turn]
    if interleaved:
        out, e = torch.stack(out, -1).flatten(-2), torch.stack(e, -1).flatten(-2)
    else:
        out, e = torch.cat(out, -1), torch.cat(e, -1)
    y = torch.cat([out, y[..., 2 * half:]], -1)
    err = torch.cat([e, err[..., 2 * half:]], -1)
    return y, half_step(x.dtype) * y.abs() + 1.02 * err + least(x.dtype)


def ln_mod(x, shift, scale, sets, eps, post, t):
    """(y, bound) of x [rows, cols]; float64."""
    cols = x.shape[-1]
    xd = x.double()
    mean = xd.mean(-1, keepdim=True)
    inv = torch.rsqrt((xd - mean).square().mean(-1, keepdim=True) + eps)
    n = (xd - mean) * inv
    if sets is None:
        sc, sh = scale.view(-1, cols)[:1].double(), shift.view(-1, cols)[:1].double()
    else:
        sc, sh = scale.double()[sets.long()], shift.double()[sets.long()]
    y = (n * (1 + sc) + sh) * post
    # The mean's error (a sum of cols terms) moves every difference; inv's is relative.
    at = (cols + 8) * U32 * xd.abs().mean(-1, keepdim=True) + 2 * U32 * xd.abs()
    err = ((1 + sc).abs() * (at * inv + n.abs() * (cols / 2 + 8) * U32) + 4 * U32 * sh.abs()) * abs(post)
    return y, half_step(t) * y.abs() + 1.02 * err + least(t)


def check(got: torch.Tensor, want: torch.Tensor, bound: torch.Tensor, what: str) -> None:
    assert torch.isfinite(got).all(), f"{what}: not finite"
    over = (got.double() - want).abs() / bound
    worst = float(over.max()) if over.numel() else 0.0
    print(f"  {what}: {worst:.3f} of the bound", flush=True)
    assert worst <= 1.0, (what, worst)
