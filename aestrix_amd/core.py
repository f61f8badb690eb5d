"""What stands between the quantized projections of a block (include/imq_core.h).

* ``ln_mod``    -- LayerNorm with the block's modulation (``lnMod``,
  ``Sources/ImarelloDirect/DirectDiTKernels.swift:16-59``);
* ``rope``      -- per-head RMSNorm and rotary positions of queries and keys
  (``DirectDiTKernels.swift:61-122``, ``DirectGlueKernels.swift:14-75``), and
  ``rope_frequencies`` for the frequencies, scaled for long contexts or not;
* ``attention`` -- softmax attention over padded batches, packed documents and
  caches (``DirectDiTStep.swift:457-488``, ``DirectTEEncoder.swift:159-202``).

Calls run on torch's current HIP stream; tensors may be strided views (columns
of a projection's output, rows of a cache) whose last dimension is contiguous.
"""

from __future__ import annotations

import ctypes
import math
import struct
from typing import Sequence

import torch

from . import _lib
from .ops import _DTYPES, _require, context, new_out, raw_stream, run_on

_i32 = torch.int32

# Calls of one row cost mostly what happens here: shapes and strides are read
# once, a C struct is packed as bytes (a ctypes.Structure of as many fields
# takes three times as long), messages are only formatted when a check fails.


def _device_of(x: torch.Tensor, what: str) -> int:
    if not x.is_cuda:
        raise ValueError(f"{what} must be on a HIP device")
    return x.get_device()


def _side(t: torch.Tensor | None, idx: int, dtype: torch.dtype, shape: tuple, what: str) -> int:
    """Pointer of a contiguous side tensor (0 where it is not given)."""
    if t is None:
        return 0
    if not (t.dtype == dtype and t.is_cuda and t.get_device() == idx and t.shape == shape and
            t.is_contiguous()):
        raise ValueError(f"{what} must be a contiguous {dtype} tensor of shape {tuple(shape)} on "
                         f"the inputs' device")
    return t.data_ptr()


def _int32(n: int, what: str) -> int:
    if not 0 <= n < 1 << 31:
        raise ValueError(f"{n} {what}: fewer than 2^31 are taken")
    return n


def _packed(fields: struct.Struct, *values) -> bytes:
    """values as a C struct."""
    try:
        return fields.pack(*values)
    except (struct.error, OverflowError) as e:  # a size past 32 bits, a float past float32
        raise ValueError(f"an argument does not fit its C type: {e}") from None


def ln_mod(x: torch.Tensor, shift: torch.Tensor, scale: torch.Tensor, *,
           sets: torch.Tensor | None = None, eps: float = 1e-6, post_scale: float = 1.0,
           out_dtype: torch.dtype | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """T(((x - mean) * rsqrt(var + eps) * (1 + scale) + shift) * post_scale) over x's last dim.

    x: contiguous float32 or T [..., cols], up to 2^20 columns; shift, scale: float32 [cols], or
    [n, cols] with sets: int32, x's leading shape: the modulation each row takes (text and
    image rows of a joint residual in one launch).  T: ``out_dtype``, float16 or bfloat16
    (default: x's own type, or float16 for float32)."""
    idx = _device_of(x, "x")
    shape = x.shape
    if not (len(shape) >= 1 and x.is_contiguous()):
        raise ValueError("x must be contiguous [..., cols]")
    cols = shape[-1]
    if out_dtype is None:
        out_dtype = out.dtype if out is not None else \
            torch.float16 if x.dtype == torch.float32 else x.dtype
    n = shift.shape[0] if shift.dim() == 2 else 1
    side = (n, cols) if shift.dim() == 2 else (cols,)
    psh = _side(shift, idx, torch.float32, side, "shift")
    psc = _side(scale, idx, torch.float32, side, "scale")
    pse = _side(sets, idx, _i32, shape[:-1], "sets")
    if out is None:
        out = torch.empty(shape, dtype=out_dtype, device=x.device)
    elif not (out.dtype == out_dtype and out.shape == shape and out.is_contiguous() and
              out.is_cuda and out.get_device() == idx):
        raise ValueError("out must be a contiguous tensor of out_dtype shaped like x")
    ctx = context(idx)
    rc = run_on(idx, _lib.load().imq_ln_mod, ctx, x.data_ptr(), _DTYPES.get(x.dtype, -1), psh, psc,
                pse, n, out.data_ptr(), _DTYPES.get(out_dtype, -1),
                _int32(x.numel() // cols if cols else 0, "rows"), _int32(cols, "columns"), eps,
                post_scale, raw_stream(idx))
    if rc:
        _lib.check(rc, ctx)
    return out


def rope_frequencies(rot_dim: int, base: float = 1e6, *, scaling: str | None = None,
                     factor: float = 1.0, original_len: int = 32768, beta_fast: float = 32.0,
                     beta_slow: float = 1.0, device=None) -> tuple[torch.Tensor, float]:
    """(inv_freq, amplitude) of ``rope``: float64 [rot_dim / 2] radians a position,
    base^(-2 j / rot_dim), and the factor on cos and sin (1 without YaRN).

    ``scaling`` for contexts ``factor`` times ``original_len``:

    * ``"linear"``: every frequency divided by factor (position interpolation);
    * ``"ntk"``: base * factor^(rot_dim / (rot_dim - 2)), which divides the slowest
      frequency by factor and keeps the fastest;
    * ``"yarn"``: pairs that turn more than beta_fast times over original_len are kept,
      those under beta_slow divided by factor, between them a line over the pair's index,
      from the last pair that is kept (at least the first) to the first that is divided,
      which may lie past the last of rot_dim; amplitude 0.1 ln(factor) + 1 (after Peng et
      al., YaRN, 2023, whose formula has the line over the turns)."""
    _require(rot_dim >= 2 and rot_dim % 2 == 0, "rot_dim must be even and positive")
    _require(base > 1.0 and factor >= 1.0, "base must be above 1 and factor at least 1")
    amplitude = 1.0
    if scaling == "ntk":
        _require(rot_dim > 2, "ntk scaling needs rot_dim above 2")
        base = base * factor ** (rot_dim / (rot_dim - 2))
    j = torch.arange(rot_dim // 2, dtype=torch.float64)
    f = base ** (-2.0 * j / rot_dim)
    if scaling == "linear":
        f = f / factor
    elif scaling == "yarn":
        _require(beta_fast > beta_slow > 0.0 and original_len > 0,
                 "yarn needs beta_fast > beta_slow > 0 and a positive original_len")

        def pair_of(turns: float) -> float:
            return rot_dim * math.log(original_len / (turns * 2.0 * math.pi)) / (2.0 * math.log(base))

        lo, hi = max(math.floor(pair_of(beta_fast)), 0), math.ceil(pair_of(beta_slow))
        slow = ((j - lo) / (hi - lo)).clamp(0.0, 1.0) if hi > lo else (j >= hi).double()
        f = f * (1.0 - slow) + f / factor * slow
        amplitude = 0.1 * math.log(factor) + 1.0
    elif scaling not in (None, "ntk"):
        raise ValueError(f"scaling {scaling!r}: None, 'linear', 'ntk' or 'yarn'")
    return (f if device is None else f.to(device)), amplitude


# imq_rope_heads: x, y, heads, strides, weight.
_ROPE_HEADS = struct.Struct("@PPi4x4qP")


def _rope_group(x, out, weight, rows, dim, dtype, idx, what):
    """(out, the packed imq_rope_heads) of one group of heads."""
    shape = x.shape
    if not (len(shape) == 3 and shape[0] == rows and shape[2] == dim and x.dtype == dtype and
            x.is_cuda and x.get_device() == idx):
        raise ValueError(f"{what} must be a {dtype} [{rows}, heads, {dim}] tensor on one device "
                         "with the others")
    if out is None:
        out = new_out(x, shape)
    elif not (out.shape == shape and out.dtype == dtype and out.is_cuda and
              out.get_device() == idx):
        raise ValueError(f"{what}_out must be a {dtype} tensor shaped like {what}")
    xr, xh, xd = x.stride()
    yr, yh, yd = out.stride()
    if not (xd == 1 and yd == 1) and x.numel():
        raise ValueError(f"{what} and {what}_out must be contiguous in the head dim")
    w = _side(weight, idx, torch.float32, (dim,), f"{what}_weight")
    return out, _packed(_ROPE_HEADS, x.data_ptr(), out.data_ptr(), shape[1], xr, xh, yr, yh, w)


def rope(q: torch.Tensor, k: torch.Tensor | None = None, *, positions: torch.Tensor,
         inv_freq: torch.Tensor, sections: Sequence[int] | None = None, interleaved: bool = False,
         amplitude: float = 1.0, q_weight: torch.Tensor | None = None,
         k_weight: torch.Tensor | None = None, eps: float = 1e-6,
         q_out: torch.Tensor | None = None, k_out: torch.Tensor | None = None):
    """Per-head RMSNorm (where a weight is given) and rotary positions, one launch.

    q [rows, heads, dim] and k [rows, kv_heads, dim], strided views allowed; the first
    2 * len(inv_freq) elements of a head are turned (``rot_dim``), the rest only normed.
    positions: int32 [rows] or [rows, axes]; inv_freq: float64 [rot_dim / 2] on the
    device (``rope_frequencies``); sections: pairs an axis, where there are more than one.
    interleaved False pairs j with j + rot_dim / 2, True 2j with 2j + 1.  q_out / k_out:
    where the results go (``q_out=q`` in place, ``k_out`` the rows of a cache), else new
    contiguous tensors.  Returns q's result, or (q's, k's) where k is given."""
    idx = _device_of(q, "q")
    if q.dim() != 3:
        raise ValueError("q must be [rows, heads, dim]")
    rows, _, dim = q.shape
    _int32(rows, "rows")
    dtype = q.dtype
    if not (inv_freq.dtype == torch.float64 and inv_freq.dim() == 1):
        raise ValueError("inv_freq must be a float64 [rot_dim / 2] tensor")
    half = inv_freq.shape[0]
    pf = _side(inv_freq, idx, torch.float64, (half,), "inv_freq")
    axes = 1 if positions.dim() == 1 else positions.shape[1] if positions.dim() == 2 else 0
    pp = _side(positions, idx, _i32, (rows,) if positions.dim() == 1 else (rows, axes), "positions")
    sec = None
    if sections is not None:
        if len(sections) != axes:
            raise ValueError(f"{len(sections)} sections for {axes} axes of positions")
        sec = _packed(struct.Struct(f"@{axes}i"), *sections)
    q_out, groups = _rope_group(q, q_out, q_weight, rows, dim, dtype, idx, "q")
    n = 1
    if k is not None:
        k_out, group = _rope_group(k, k_out, k_weight, rows, dim, dtype, idx, "k")
        groups += group
        n = 2
    elif k_out is not None or k_weight is not None:
        raise ValueError("k_out and k_weight need k")
    ctx = context(idx)
    rc = run_on(idx, _lib.load().imq_rope, ctx, groups, n, rows, dim, 2 * half,
                1 if interleaved else 0, pp, axes, sec, pf, amplitude, eps, _DTYPES.get(dtype, -1),
                raw_stream(idx))
    if rc:
        _lib.check(rc, ctx)
    return q_out if k is None else (q_out, k_out)


# imq_attention_args: pointers, strides, sizes, side arrays, scale, softcap, causal, dtype.
_ATTENTION_ARGS = struct.Struct("@4P12q8i6P2f2i")


class AttentionPlanInfo(ctypes.Structure):
    """imq_attention_plan_info."""
    _fields_ = [("kernel", ctypes.c_int), ("tile_rows", ctypes.c_int), ("splits", ctypes.c_int),
                ("workspace_bytes", ctypes.c_size_t)]


ATTENTION_KERNELS = {0: "rows", 1: "tiles", 2: "few"}


def _attention_args(q, k, v, scale, causal, softcap, slopes, q_lens, k_lens, prefix_lens,
                    q_offsets, k_offsets, max_q, max_k, out):
    idx = _device_of(q, "q")
    dtype = q.dtype
    qs, ks = q.shape, k.shape
    nd = len(qs)
    if not (nd == len(ks) and (nd == 3 or nd == 4)):
        raise ValueError("q, k and v must be all [rows, heads, dim] or all [seqs, rows, heads, dim]")
    if not (k.dtype == dtype and v.dtype == dtype and k.is_cuda and v.is_cuda and
            k.get_device() == idx and v.get_device() == idx):
        raise ValueError("q, k and v must share a dtype and a device")
    q_rows, heads, dim = qs[-3:]
    k_rows, kv, kd = ks[-3:]
    if not (ks == v.shape and kd == dim):
        raise ValueError(f"k and v must be [..., kv_heads, {dim}] of one shape, "
                         f"got {tuple(ks)} and {tuple(v.shape)}")
    if q_offsets is not None or k_offsets is not None:
        if nd != 3 or q_offsets is None or k_offsets is None:
            raise ValueError("packed documents are [rows, heads, dim] with q_offsets and k_offsets")
        if max_q is None or max_k is None:
            raise ValueError("packed documents need max_q and max_k, the longest document's rows")
        if q_lens is not None or k_lens is not None:
            raise ValueError("offsets and lengths exclude each other")
        n = q_offsets.shape[0] - 1 if q_offsets.dim() == 1 else -1
        if n < 0:
            raise ValueError("q_offsets must be int32 [n + 1]")
    else:
        if max_q is not None or max_k is not None:
            raise ValueError("max_q and max_k are for packed documents")
        n = qs[0] if nd == 4 else 1
        if nd == 4 and ks[0] != n:
            raise ValueError(f"q has {n} sequences, k and v {ks[0]}")
        max_q, max_k = q_rows, k_rows
    if out is None:
        out = new_out(q, qs)
    elif not (out.shape == qs and out.dtype == dtype and out.is_cuda and out.get_device() == idx):
        raise ValueError("out must be shaped like q, of its dtype and device")
    if nd == 3:
        sq, sk, sv, so = (0, *q.stride()), (0, *k.stride()), (0, *v.stride()), (0, *out.stride())
    else:
        sq, sk, sv, so = q.stride(), k.stride(), v.stride(), out.stride()
    if not (sq[3] == 1 and sk[3] == 1 and sv[3] == 1 and so[3] == 1) and \
            (q.numel() and not sq[3] == so[3] == 1 or k.numel() and not sk[3] == sv[3] == 1):
        raise ValueError("q, k, v and out must be contiguous in the head dim")
    return idx, out, _packed(
        _ATTENTION_ARGS, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), *sq[:3], *sk[:3], *sv[:3],
        *so[:3], n, heads, kv, dim, max_q, max_k, q_rows, k_rows,
        _side(q_offsets, idx, _i32, (n + 1,), "q_offsets"),
        _side(k_offsets, idx, _i32, (n + 1,), "k_offsets"),
        _side(q_lens, idx, _i32, (n,), "q_lens"), _side(k_lens, idx, _i32, (n,), "k_lens"),
        _side(prefix_lens, idx, _i32, (n,), "prefix_lens"),
        _side(slopes, idx, torch.float32, (heads,), "slopes"),
        scale if scale is not None else dim ** -0.5 if dim else 1.0, softcap, 1 if causal else 0,
        _DTYPES.get(dtype, -1))


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, scale: float | None = None,
              causal: bool = False, softcap: float = 0.0, slopes: torch.Tensor | None = None,
              q_lens: torch.Tensor | None = None, k_lens: torch.Tensor | None = None,
              prefix_lens: torch.Tensor | None = None, q_offsets: torch.Tensor | None = None,
              k_offsets: torch.Tensor | None = None, max_q: int | None = None,
              max_k: int | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """softmax(scores) v with heads sharing key heads in whole groups, bf16 or f16.

    Scores are scale * q . k (scale: 1 / sqrt(dim) by default), then capped to
    softcap * tanh(score / softcap) where softcap > 0 (up to 4096), then lowered by slopes[head] times
    the distance (float32 [heads], up to 2^20 in size; scale then from 2^-64 on).  The last query stands at the last key; ``causal`` hides later keys but
    for the first prefix_lens[s] of a sequence.  A query that sees nothing gives zeros.

    * one sequence: q [rows, heads, dim], k and v [keys, kv_heads, dim];
    * a batch, or a cache: q [n, rows, heads, dim], k and v [n, keys, kv_heads, dim], of
      which sequence s uses the first q_lens[s] rows and k_lens[s] keys (int32 [n]);
    * packed documents: q, k, v [rows, ...], document s in rows q_offsets[s] to
      q_offsets[s + 1] (int32 [n + 1]), max_q and max_k the longest one's rows.

    Views with a contiguous last dim are taken as they are; ``out`` overlaps none of
    q, k and v.  Rows of ``out`` that are no
    query's are left as they were (in a new tensor: undefined).

    Few queries over many keys split the keys over a workspace of the stream, which grows on
    its first such call.  A call captured into a graph on a stream without one runs unsplit
    (much slower for a token over a long cache: run it once on the stream that the graph is
    then captured on); graphs captured on one stream share its workspace, so that replays of
    two of them do not run at once, nor one beside calls on that stream."""
    idx, out, args = _attention_args(q, k, v, scale, causal, softcap, slopes, q_lens, k_lens,
                                     prefix_lens, q_offsets, k_offsets, max_q, max_k, out)
    ctx = context(idx)
    rc = run_on(idx, _lib.load().imq_attention, ctx, args, raw_stream(idx))
    if rc:
        _lib.check(rc, ctx)
    return out


def attention_plan(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, scale=None, causal=False,
                   softcap=0.0, slopes=None, q_lens=None, k_lens=None, prefix_lens=None,
                   q_offsets=None, k_offsets=None, max_q=None, max_k=None, out=None) -> dict:
    """The kernel ("rows", "tiles" or "few"), tile height and key splits that
    ``attention`` with these arguments would run, without launching anything."""
    idx, _, args = _attention_args(q, k, v, scale, causal, softcap, slopes, q_lens, k_lens,
                                   prefix_lens, q_offsets, k_offsets, max_q, max_k, out)
    ctx = context(idx)
    info = AttentionPlanInfo()
    _lib.check(_lib.load().imq_attention_plan(ctx, args, ctypes.byref(info)), ctx)
    return {"kernel": ATTENTION_KERNELS[info.kernel], "tile_rows": info.tile_rows,
            "splits": info.splits, "workspace_bytes": info.workspace_bytes}
