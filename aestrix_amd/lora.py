"""Low-rank adapters of many requests beside a shared 4-bit projection (include/imq_lora.h).

The reference has no adapters.  A server runs the rows of all its requests through one
quantized projection; every row has its request's adapter, or none.
"""

from __future__ import annotations

import ctypes
import math
from typing import Sequence

import torch

from . import _lib
from .ops import _DTYPES, BITS, GROUP_SIZE, _epi_args, _require, context, new_out, raw_stream, run_on

_MAX_RANK = 256
_FILL = 16  # ranks are filled up to multiples of this


def _ups(b: torch.Tensor) -> torch.Tensor:
    """Exponents [sets, rank] for float16 B [sets, N, rank]: of the powers of two that bring the columns'
    largest finite elements to [1, 2), but no element's lowest bit under float16's, 2^-24."""
    units = (torch.where(torch.isfinite(b), b, 0).double() * 2.0 ** 24).long()  # whole numbers
    top, low = units.abs().amax(1), units & -units
    low = low.masked_fill(low == 0, 1 << 62).amin(1)
    at = lambda v: torch.frexp(v.double()).exponent - 1  # of the highest bit
    return torch.where(top > 0, torch.maximum(24 - at(top), -at(low)), 0)


class LoraAdapters:
    """A set of adapters for one projection, laid out once, a copy outside any autograd graph.

    ``pairs``: (A [rank, K], B [N, rank]) of every adapter, bfloat16 or float16 on one device,
    ranks from 1 to 256, not all alike if they are not; ``scales``: a factor each (alpha / rank),
    one for all, or none.  Adapter i adds ``scales[i] * (x . A^T) . B^T``.

    The tensors are copied: in bytes about what the adapters have, ranks filled up to multiples
    of 16.  In float16 each column of B is multiplied by a power of two, which its rank's scale takes
    back, so that the products between A and B, which have that type's range, leave it only where one
    of them times its element of B does."""

    @torch.no_grad()  # parameters would otherwise stay referenced by the copies
    def __init__(self, pairs: Sequence[tuple[torch.Tensor, torch.Tensor]],
                 scales: float | Sequence[float] | None = None):
        pairs = [tuple(p) for p in pairs]
        _require(len(pairs) > 0 and all(len(p) == 2 for p in pairs), "pairs must be (A, B), one at least")
        if scales is None or isinstance(scales, (int, float)):
            scales = [1.0 if scales is None else scales] * len(pairs)
        scales = [float(s) for s in scales]
        _require(len(scales) == len(pairs), f"{len(scales)} scales for {len(pairs)} adapters")
        _require(all(math.isfinite(s) and abs(s) < 3e38 for s in scales), "scales must be finite float32")
        a0, b0 = pairs[0]
        _require(a0.dim() == 2 and b0.dim() == 2, "A must be [rank, K] and B [N, rank]")
        self.k, self.n, self.dtype, self.device = a0.shape[1], b0.shape[0], a0.dtype, a0.device
        _require(a0.is_cuda, "tensors must be on a HIP device")
        if self.dtype not in (torch.bfloat16, torch.float16):
            raise _lib.ImqUnsupported(_lib.IMQ_EUNSUPPORTED, f"{self.dtype}: bfloat16 and float16 are provided")
        _require(self.k > 0 and self.k % GROUP_SIZE == 0 and self.n > 0, f"K = {self.k} must be a multiple of 64, N > 0")
        first = [0]
        for a, b in pairs:
            _require(a.dim() == 2 and b.dim() == 2 and a.shape[1] == self.k and b.shape[0] == self.n and
                     a.shape[0] == b.shape[1], f"A must be [rank, {self.k}] and B [{self.n}, rank], "
                     f"got {tuple(a.shape)} and {tuple(b.shape)}")
            _require(1 <= a.shape[0] <= _MAX_RANK, f"rank {a.shape[0]}: 1 to {_MAX_RANK} are taken")
            _require(a.dtype == b.dtype == self.dtype and a.device == b.device == self.device,
                     "all A and B must share a dtype and a device")
            first.append(first[-1] + -(-a.shape[0] // _FILL) * _FILL)
        self.count, self.rows = len(pairs), first[-1]
        self.max_rank = max(q - p for p, q in zip(first, first[1:]))
        self.a = torch.zeros((self.rows, self.k), dtype=self.dtype, device=self.device)
        self.b = torch.zeros(self.rows * self.n, dtype=self.dtype, device=self.device)
        by_rank = self.dtype == torch.float16
        self.scale = torch.tensor([s for s, p, q in zip(scales, first, first[1:]) for _ in range(q - p)]
                                  if by_rank else scales, dtype=torch.float32, device=self.device)
        self.first = torch.tensor(first, dtype=torch.int32, device=self.device)
        for i, (a, b) in enumerate(pairs):
            rank = a.shape[0]
            self.a[first[i]:first[i] + rank] = a
            at = self.b[first[i] * self.n:first[i + 1] * self.n].view(self.n, -1)[:, :rank]
            at.copy_(b)
        if by_rank:
            self._bring_up(first)
        self._c = _lib.Lora(self.a.data_ptr(), self.b.data_ptr(), self.first.data_ptr(), self.scale.data_ptr(),
                            self.count, self.rows, self.max_rank, int(by_rank))
        self._p = ctypes.addressof(self._c)
        self._bytes: dict[int, int] = {}  # of the workspace, by a call's rows

    def _bring_up(self, first: list[int]) -> None:
        """B's columns multiplied by 2^up each, the ranks' scales divided by it; adapters of one rank together."""
        i = 0
        while i < self.count:
            fill = first[i + 1] - first[i]
            end = i + 1
            while end < self.count and first[end + 1] - first[end] == fill and (end + 1 - i) * self.n * fill <= 1 << 24:
                end += 1
            b = self.b[first[i] * self.n:first[end] * self.n].view(end - i, self.n, fill)
            scale = self.scale[first[i]:first[end]].view(end - i, fill)
            up = _ups(b)
            b.copy_(torch.ldexp(b.float(), up[:, None]))
            # (A product that is zero stays zero where this would leave float32.)
            scale.copy_(torch.ldexp(scale, -up).clamp(-3.4e38, 3.4e38))
            i = end


def quantized_matmul_lora(x: torch.Tensor, w: torch.Tensor, scales: torch.Tensor, biases: torch.Tensor,
                          adapters: LoraAdapters, which: torch.Tensor, group_size: int = GROUP_SIZE,
                          bits: int = BITS, out: torch.Tensor | None = None) -> torch.Tensor:
    """y[..., N] = T(x . deq(W)^T + scale_i * (x . A_i^T) . B_i^T), i = which[...] the adapter of
    each row of x, rounded once.

    which: int32, x's leading shape; a row whose value is not one of 0 to count - 1 (-1) has no
    adapter.  x, scales and biases as in ``quantized_matmul``, bfloat16 or float16, of the
    adapters' type; ``out`` is not x.  The workspace is torch's, so that calls may be captured
    into graphs and graphs replayed beside each other; a call's result does not depend on any of that."""
    n, k, m, lead, x = _epi_args(x, w, scales, biases, group_size, bits)
    idx = w.get_device()
    device = x.device
    if not (adapters.k == k and adapters.n == n and adapters.dtype == x.dtype and adapters.device == device):
        raise ValueError(f"adapters of a {adapters.dtype} [{adapters.n}, {adapters.k}] projection on {adapters.device}, "
                         f"this is {x.dtype} [{n}, {k}] on {device}")
    if not (which.dtype == torch.int32 and which.shape == lead and which.is_contiguous() and which.device == device):
        raise ValueError(f"which must be a contiguous int32 tensor of shape {lead} on x's device")
    shape = lead + (n,)
    if out is None:
        out = new_out(x, shape)
    elif not (out.is_contiguous() and out.shape == shape and out.dtype == x.dtype and out.device == device):
        raise ValueError("out must be a contiguous [..., N] tensor of x's dtype and device")
    if m == 0:
        return out
    ctx = context(idx)
    lib, dtype = _lib.load(), _DTYPES.get(x.dtype, -1)
    need = adapters._bytes.get(m)
    if need is None:
        size = ctypes.c_size_t()
        _lib.check(lib.imq_qmm_lora_workspace(ctx, adapters._p, k, n, m, dtype, ctypes.byref(size)), ctx)
        need = adapters._bytes[m] = size.value
    ws = x.new_empty((need + 1) // 2) if type(x) is torch.Tensor else \
        torch.empty((need + 1) // 2, dtype=x.dtype, device=x.device)
    rc = run_on(idx, lib.imq_qmm_lora, ctx, w.data_ptr(), scales.data_ptr(), biases.data_ptr(), x.data_ptr(),
                adapters._p, which.data_ptr(), out.data_ptr(), k, n, m, group_size, bits, dtype, ws.data_ptr(),
                need, raw_stream(idx))
    if rc:
        _lib.check(rc, ctx)
    return out


LORA_KERNELS = {0: "few", 1: "split", 2: "tiles", 3: "tiles_reg"}


def quantized_matmul_lora_plan(adapters: LoraAdapters, m: int) -> dict:
    """The kernel, tile height, ranges of K, way to u ("rows", "tiles"), grouping, join ("outputs", "tiles" or
    None) and workspace that ``quantized_matmul_lora`` would use for m rows."""
    ctx = context(adapters.device.index)
    p = _lib.LoraPlanInfo()
    _lib.check(_lib.load().imq_qmm_lora_plan(ctx, adapters._p, adapters.k, adapters.n, m, _DTYPES[adapters.dtype],
                                             ctypes.byref(p)), ctx)
    kernel = LORA_KERNELS[p.kernel]
    join = ("tiles" if p.join_tiles else "outputs") if kernel in ("few", "split") else None
    return {"kernel": kernel, "tile_rows": p.tile_rows, "splits": p.splits, "u": "rows" if p.u_rows else "tiles",
            "grouped": bool(p.grouped), "join": join, "workspace_bytes": p.workspace_bytes}
