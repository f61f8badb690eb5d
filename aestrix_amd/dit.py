"""A whole DiT denoise step: the block halves of ``aestrix_amd.step`` with their
core (``include/imq_core.h``) between them.

``DitModel`` is ``encodeDenoiseStep`` (``Sources/ImarelloDirect/DirectDiTStep.swift:908-971``)
without stand-ins: every ``lnMod`` is a modulated LayerNorm, and the attention of a
block is per-head RMSNorm, RoPE over the joint rows' position axes and attention of
every row to every row (``DirectDiTStep.swift:360-373,408-503``).
"""

from __future__ import annotations

from dataclasses import dataclass, fields
from typing import Sequence

import torch

from .core import attention, ln_mod, rope, rope_frequencies
from .ops import _require
from .step import DitStep

HEAD_DIM, AXES, ROPE_BASE = 128, (16, 16, 16, 16), 2000.0  # FLUX.2 klein: pairs of each axis
LN_EPS, HEAD_EPS = 1e-6, 1e-5


@dataclass
class DitNorms:
    """A block's per-head RMSNorm weights, float32 [head_dim]: q and k of the image rows
    (single blocks: of all rows), added_q and added_k of the text rows (double blocks)."""

    q: torch.Tensor
    k: torch.Tensor
    added_q: torch.Tensor | None = None
    added_k: torch.Tensor | None = None


@dataclass
class DitModulation:
    """One timestep's shift and scale, float32 [2, dim] (row 0 the text rows', 1 the image
    rows') before the double blocks' attention and MLPs, [dim] in the single blocks and
    before proj_out (the fields of the reference's Flux2StepConditioning)."""

    attn_shift: torch.Tensor
    attn_scale: torch.Tensor
    mlp_shift: torch.Tensor
    mlp_scale: torch.Tensor
    single_shift: torch.Tensor
    single_scale: torch.Tensor
    out_shift: torch.Tensor
    out_scale: torch.Tensor


_MODULATIONS = tuple(f.name for f in fields(DitModulation))


class DitModel:
    """A step plan with its head set, and what its blocks need between the projections.

    norms: one ``DitNorms`` a block, double blocks first; positions: int32 [J, axes], text
    rows first; sections: the pairs of each axis (sum head_dim / 2).  The buffers between
    the halves are allocated here, once; a model runs one step at a time, on one stream."""

    def __init__(self, step: DitStep, norms: list[DitNorms], positions: torch.Tensor,
                 head_dim: int = HEAD_DIM, sections: Sequence[int] = AXES, base: float = ROPE_BASE):
        d = step.dims
        _require(len(norms) == d.n_double + d.n_single, f"{len(norms)} norms for "
                 f"{d.n_double + d.n_single} blocks")
        _require(all(n.added_q is not None and n.added_k is not None for n in norms[:d.n_double]),
                 "double blocks need added_q and added_k")
        _require(head_dim > 0 and d.dim % head_dim == 0, f"dim {d.dim} is not heads of {head_dim}")
        _require(tuple(positions.shape) == (d.joint, len(sections)), f"positions must be "
                 f"[{d.joint}, {len(sections)}]")
        _require(2 * sum(sections) == head_dim, "the sections must hold all pairs of a head")
        self.step, self.norms, self.head_dim, self.sections = step, norms, head_dim, tuple(sections)
        self.positions = positions
        dev, t, j = step.device, step.dtype, d.joint
        self.freq = torch.cat([rope_frequencies(2 * s, base)[0] for s in sections if s]).to(dev)
        self.sets = (torch.arange(j, device=dev) >= d.l_txt).to(torch.int32)  # text rows 0, image 1

        def buf(rows, cols, dtype=t):
            return torch.empty((rows, cols), dtype=dtype, device=dev)

        self.x, self.nx = buf(j, d.dim, torch.float32), buf(j, d.dim)
        self.q, self.k, self.v, self.attn = (buf(j, d.dim) for _ in range(4))
        self.qkv, self.concat = buf(j, 3 * d.dim), buf(j, d.dim + d.ff_inner)
        self.nh = buf(d.l_img, d.dim)

    def _heads(self, x: torch.Tensor) -> torch.Tensor:
        return x.unflatten(-1, (-1, self.head_dim))

    def _rope(self, rows: slice, q, k, q_weight, k_weight) -> None:
        q, k = q[rows], k[rows]
        rope(q, k, positions=self.positions[rows], inv_freq=self.freq, sections=self.sections,
             interleaved=True, q_weight=q_weight, k_weight=k_weight, eps=HEAD_EPS, q_out=q, k_out=k)

    def double_core(self, block: int) -> None:
        """q, k, v to attn: the double block's attention between its halves."""
        n, l = self.norms[block], self.step.dims.l_txt
        q, k = self._heads(self.q), self._heads(self.k)
        self._rope(slice(0, l), q, k, n.added_q, n.added_k)
        self._rope(slice(l, None), q, k, n.q, n.k)
        attention(q, k, self._heads(self.v), out=self._heads(self.attn))

    def single_core(self, block: int) -> None:
        """qkv to concat[:, :dim]: the single block's attention between its halves."""
        d = self.step.dims
        n = self.norms[d.n_double + block]
        q, k, v = (self._heads(t) for t in self.qkv.split(d.dim, -1))
        self._rope(slice(None), q, k, n.q, n.k)
        attention(q, k, v, out=self._heads(self.concat[:, :d.dim]))

    def denoise(self, lat: torch.Tensor, e: torch.Tensor, dt: float, mod: DitModulation,
                out: torch.Tensor | None = None) -> torch.Tensor:
        """lat_out [l_img, C] float32 = lat + 16 dt times the head's prediction
        (gates: ``step.set_conditioning``)."""
        s, d, x = self.step, self.step.dims, self.x
        _require(e.dtype == torch.float32 and tuple(e.shape) == (d.l_txt, d.dim) and
                 e.device == x.device, f"e must be float32 [{d.l_txt}, {d.dim}] on {x.device}")
        for name in _MODULATIONS:  # another number of rows would go to the wrong ones
            t = getattr(mod, name)
            both = name.startswith(("attn", "mlp"))
            _require(t.dtype == torch.float32 and t.device == x.device and
                     (t.shape == (2, d.dim) if both else t.shape in ((d.dim,), (1, d.dim))),
                     f"{name} must be float32 {'[2, ' if both else '['}{d.dim}] on {x.device}")
        if out is None:
            out = torch.empty_like(lat)
        x[:d.l_txt].copy_(e)
        s.head_embed(lat, x)
        for b in range(d.n_double):
            ln_mod(x, mod.attn_shift, mod.attn_scale, sets=self.sets, eps=LN_EPS, out=self.nx)
            s.double_attn_in(b, None, self.q, self.k, self.v, nx=self.nx)
            self.double_core(b)
            s.double_attn_out(b, self.attn, x)
            ln_mod(x, mod.mlp_shift, mod.mlp_scale, sets=self.sets, eps=LN_EPS, out=self.nx)
            s.double_mlp(b, x, nx=self.nx)
        for b in range(d.n_single):
            ln_mod(x, mod.single_shift, mod.single_scale, eps=LN_EPS, out=self.nx)
            s.single_attn_in(b, None, self.qkv, self.concat, nx=self.nx)
            self.single_core(b)
            s.single_attn_out(b, self.concat, x)
        ln_mod(x[d.l_txt:], mod.out_shift, mod.out_scale, eps=LN_EPS, post_scale=0.0625, out=self.nh)
        s.head_out(None, lat, dt, out, nh=self.nh)
        return out
