"""The text encoder's quantized-linear layer halves (include/imq_te.h) from Python.

Mirrors ``DirectTEEncoder.encodeLayer`` (``Sources/ImarelloDirect/DirectTEEncoder.swift:364-412``)
over the layers ``DirectTEForward.loadLayers`` uploads (``DirectTEForward.swift:97-138``):
``attn_in`` is RMSNorm + the q/k/v projections (one launch), ``attn_out_mlp`` is
o_proj + dq_add, RMSNorm, gate/up with dq_silu_mul (one launch) and down_proj +
dq_add.  ``attn_core`` is the attention core between them (per-head norms, RoPE,
causal attention over padded prompts, ``include/imq_core.h``), or a caller
brings its own; ``layer`` and ``encode`` run whole layers.
"""

from __future__ import annotations

import ctypes
from dataclasses import dataclass

import torch

from . import _lib
from .core import attention, rope, rope_frequencies
from .ops import Q, _require, context, device_index, new_out, raw_stream, run_on
from .step import _qweight

# Qwen3 4B text encoder (DirectTEForward.swift:12-22).
HIDDEN, N_HEADS, N_KV, HEAD_DIM, INTER, N_LAYERS, EPS = 2560, 32, 8, 128, 9728, 27, 1e-6
ROPE_BASE = 1e6  # Qwen3's rope_theta
TAPS = (9, 18, 27)  # layers whose output encode returns (DirectTEForward.swift:20)


@dataclass
class TeLayer:
    """One layer's resident projections and norm weights: q/k/v and gate/up
    concatenated along N (rows q | k | v, gate | up)."""

    qkv: Q
    o: Q
    gate_up: Q
    down: Q
    norm_in: torch.Tensor    # input_layernorm.weight, float32 [hidden]
    norm_post: torch.Tensor  # post_attention_layernorm.weight, float32 [hidden]
    norm_q: torch.Tensor | None = None  # self_attn.q_norm.weight, float32 [head_dim] (attn_core)
    norm_k: torch.Tensor | None = None  # self_attn.k_norm.weight


def _rand_q(n, k, dtype, g, dev) -> Q:
    w = torch.randint(-2 ** 31, 2 ** 31 - 1, (n, k // 8), dtype=torch.int32, device=dev, generator=g)
    unit = 1.0 / (4.0 * k ** 0.5)
    s = torch.randn((n, k // 64), device=dev, generator=g).abs() * unit
    b = -8.0 * s + torch.randn((n, k // 64), device=dev, generator=g) * (0.1 * unit)
    return Q(w=w, s=s.to(dtype), b=b.to(dtype), n=n, k=k)


def random_te_layers(n_layers: int = 1, hidden: int = HIDDEN, nq: int = N_HEADS * HEAD_DIM,
                     nkv: int = N_KV * HEAD_DIM, inter: int = INTER,
                     dtype: torch.dtype = torch.bfloat16, seed: int = 0,
                     device=None) -> list[TeLayer]:
    """Synthetic layers of the given shapes (scale law of ``step.random_projections``:
    outputs at the scale of the normalized input) and norm weights 1 + N(0, 0.1)."""
    dev = torch.device("cuda", device_index(device))
    g = torch.Generator(device=dev).manual_seed(seed)
    out = []
    for _ in range(n_layers):
        out.append(TeLayer(
            qkv=_rand_q(nq + 2 * nkv, hidden, dtype, g, dev), o=_rand_q(hidden, nq, dtype, g, dev),
            gate_up=_rand_q(2 * inter, hidden, dtype, g, dev), down=_rand_q(hidden, inter, dtype, g, dev),
            norm_in=1.0 + 0.1 * torch.randn(hidden, device=dev, generator=g),
            norm_post=1.0 + 0.1 * torch.randn(hidden, device=dev, generator=g)))
    return out


def load_te_layers(st, n_layers: int = N_LAYERS, prefix: str = "layers",
                   scales: torch.dtype = torch.bfloat16, device=None) -> list[TeLayer]:
    """``DirectTEForward.loadLayers`` (``:97-138``) from an opened ``SafetensorsSet``:
    ``<prefix>.<i>.self_attn.{q,k,v,o}_proj``, ``mlp.{gate,up,down}_proj`` with their
    scales and biases kept in ``scales`` (the TE's raw bf16 by default), the norm
    weights (``self_attn.{q,k}_norm`` too, where the set has them) as float32."""
    from .weights import load_qlinear, load_qlinear_cat
    out = []
    names = set(st.names())
    for i in range(n_layers):
        p = f"{prefix}.{i}"
        head = [st.upload(n, torch.float32, device) if n in names else None
                for n in (f"{p}.self_attn.q_norm.weight", f"{p}.self_attn.k_norm.weight")]
        qkv = load_qlinear_cat(st, [f"{p}.self_attn.{n}_proj" for n in "qkv"], scales, device)
        gate_up = load_qlinear_cat(st, [f"{p}.mlp.gate_proj", f"{p}.mlp.up_proj"], scales, device)
        out.append(TeLayer(
            qkv=qkv, o=load_qlinear(st, f"{p}.self_attn.o_proj", scales, device), gate_up=gate_up,
            down=load_qlinear(st, f"{p}.mlp.down_proj", scales, device),
            norm_in=st.upload(f"{p}.input_layernorm.weight", torch.float32, device),
            norm_post=st.upload(f"{p}.post_attention_layernorm.weight", torch.float32, device),
            norm_q=head[0], norm_k=head[1]))
    return out


class TeLayerWeights(ctypes.Structure):
    """imq_te_layer_weights."""
    _fields_ = [("qkv", _lib.QWeight), ("o", _lib.QWeight), ("gate_up", _lib.QWeight),
                ("down", _lib.QWeight), ("norm_in", ctypes.c_void_p), ("norm_post", ctypes.c_void_p)]


class TextEncoderLayers:
    """A created plan over resident layers (kept alive here)."""

    def __init__(self, layers: list[TeLayer], max_rows: int = 512, eps: float = EPS, device=None):
        self.layers = layers
        self.device = torch.device("cuda", device_index(device))
        self.dtype = layers[0].qkv.s.dtype
        self.max_rows = max_rows
        self.eps = float(eps)
        self._L = _lib.load()
        self._ctx = context(self.device)
        arr = (TeLayerWeights * len(layers))()
        for i, l in enumerate(layers):
            for name in ("qkv", "o", "gate_up", "down"):
                setattr(arr[i], name, _qweight(getattr(l, name)))
            _require(l.norm_in.dtype == torch.float32 and l.norm_post.dtype == torch.float32,
                     "norm weights must be float32")
            arr[i].norm_in = l.norm_in.data_ptr()
            arr[i].norm_post = l.norm_post.data_ptr()
        out = ctypes.c_void_p()
        with torch.cuda.device(self.device):
            _lib.check(self._L.imq_te_create(self._ctx, arr, len(layers), max_rows, self.eps,
                                             ctypes.byref(out)), self._ctx)
        self._h = out
        dims = [ctypes.c_int() for _ in range(4)]
        _lib.check(self._L.imq_te_dims(self._h, *[ctypes.byref(d) for d in dims]), self._ctx)
        self.hidden, self.nq, self.nkv, self.inter = (d.value for d in dims)
        if self.nq % HEAD_DIM == 0 and self.nkv % HEAD_DIM == 0:
            self.set_rope()  # here, so that a first attn_core may be captured

    def close(self) -> None:
        if self._h:
            self._L.imq_te_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def _rows(self, x: torch.Tensor, width: int, name: str) -> int:
        if not (x.dim() == 2 and x.shape[1] == width and x.dtype == self.dtype and
                x.is_contiguous() and x.device == self.device):
            raise ValueError(f"{name} must be a contiguous {self.dtype} [rows, {width}] tensor "
                             f"on {self.device}")
        return x.shape[0]

    def attn_in(self, layer: int, x: torch.Tensor, qkv: torch.Tensor | None = None) -> torch.Tensor:
        """qkv [rows, nq + 2 nkv] (q | k | v columns) = RMSNorm(x) . [Wq; Wk; Wv]^T."""
        rows = self._rows(x, self.hidden, "x")
        width = self.nq + 2 * self.nkv
        if qkv is None:
            qkv = new_out(x, (rows, width))
        _require(self._rows(qkv, width, "qkv") == rows, "qkv rows must match x")
        idx = self.device.index
        _lib.check(run_on(idx, self._L.imq_te_attn_in, self._h, layer, x.data_ptr(), qkv.data_ptr(),
                          rows, raw_stream(idx)), self._ctx)
        return qkv

    def attn_out_mlp(self, layer: int, x: torch.Tensor, attn_o: torch.Tensor,
                     out: torch.Tensor | None = None) -> torch.Tensor:
        """The layer output [rows, hidden] from its input x and the attention output
        attn_o [rows, nq]; ``out=x`` updates x in place."""
        rows = self._rows(x, self.hidden, "x")
        _require(self._rows(attn_o, self.nq, "attn_o") == rows, "attn_o rows must match x")
        if out is None:
            out = torch.empty_like(x)
        _require(self._rows(out, self.hidden, "out") == rows, "out rows must match x")
        idx = self.device.index
        _lib.check(run_on(idx, self._L.imq_te_attn_out_mlp, self._h, layer, x.data_ptr(),
                          attn_o.data_ptr(), out.data_ptr(), rows, raw_stream(idx)), self._ctx)
        return out

    # ---- the attention core, and whole layers ------------------------------

    def set_rope(self, head_dim: int = HEAD_DIM, base: float = ROPE_BASE, **scaling) -> None:
        """Head size and rotary frequencies of ``attn_core`` (``rope_frequencies``' scaling
        for windows past the trained length); without a call, the Qwen3 encoder's, where the
        columns are heads of its size."""
        _require(head_dim > 0 and self.nq % head_dim == 0 and self.nkv % head_dim == 0,
                 f"q and k / v of {self.nq} and {self.nkv} columns are not heads of {head_dim}")
        self.head_dim = head_dim
        self.freq, self.amplitude = rope_frequencies(head_dim, base, device=self.device, **scaling)

    def attn_core(self, layer: int, qkv: torch.Tensor, prompts: int = 1,
                  lens: torch.Tensor | None = None, positions: torch.Tensor | None = None,
                  out: torch.Tensor | None = None) -> torch.Tensor:
        """``encodeLayer`` between the q/k/v and the o projection (DirectTEEncoder.swift:382-389):
        per-head RMSNorm (where the layer has ``norm_q`` / ``norm_k``; the encoder's eps) and RoPE of q and k,
        in place in ``qkv``, then causal attention; attn_o [rows, nq].

        rows = prompts * window, prompt after prompt; lens (int32 [prompts]): the prompts'
        own lengths, the rows behind them padding, whose attention output is zero (with
        ``out`` given: left as it was).  positions: int32 [rows], by default 0, 1, ... of
        each window."""
        rows = self._rows(qkv, self.nq + 2 * self.nkv, "qkv")
        _require(prompts >= 1 and rows % prompts == 0, f"{rows} rows are not {prompts} windows")
        _require(hasattr(self, "freq"), f"q and k / v of {self.nq} and {self.nkv} columns are not "
                 f"heads of {HEAD_DIM}: set_rope first")
        if positions is None:
            positions = torch.arange(rows // prompts, dtype=torch.int32, device=self.device)
            if prompts > 1:
                positions = positions.repeat(prompts)
        if out is None:
            out = new_out(qkv, (rows, self.nq)) if lens is None else \
                torch.zeros((rows, self.nq), dtype=self.dtype, device=self.device)
        _require(self._rows(out, self.nq, "out") == rows, "out rows must match qkv")
        # What attention would refuse, before q and k are turned in place.
        _require(lens is None or (lens.dtype == torch.int32 and lens.shape == (prompts,) and
                                  lens.is_contiguous() and lens.device == qkv.device),
                 f"lens must be a contiguous int32 [{prompts}] tensor on {qkv.device}")
        a, b = qkv.data_ptr(), out.data_ptr()
        _require(b >= a + qkv.nbytes or a >= b + out.nbytes, "out lies in qkv")
        d, l = self.head_dim, self.layers[layer]
        q, k, v = (t.unflatten(-1, (-1, d)) for t in qkv.split([self.nq, self.nkv, self.nkv], -1))
        rope(q, k, positions=positions, inv_freq=self.freq, amplitude=self.amplitude,
             q_weight=l.norm_q, k_weight=l.norm_k, eps=self.eps, q_out=q, k_out=k)
        window = (prompts, rows // prompts)
        attention(q.unflatten(0, window), k.unflatten(0, window), v.unflatten(0, window),
                  causal=True, q_lens=lens, k_lens=lens,
                  out=out.view(*window, self.nq // d, d))
        return out

    def layer(self, layer: int, x: torch.Tensor, prompts: int = 1,
              lens: torch.Tensor | None = None, positions: torch.Tensor | None = None,
              out: torch.Tensor | None = None) -> torch.Tensor:
        """One whole layer (``encodeLayer``, DirectTEEncoder.swift:364-412): x [rows, hidden]
        to the layer's output, ``out=x`` in place."""
        qkv = self.attn_in(layer, x)
        return self.attn_out_mlp(layer, x, self.attn_core(layer, qkv, prompts, lens, positions), out)

    def encode(self, x: torch.Tensor, prompts: int = 1, lens: torch.Tensor | None = None,
               taps=TAPS) -> list[torch.Tensor]:
        """The hidden states after the layers ``taps`` counts (from 1), of the embedding rows
        x [rows, hidden] (``DirectTEForward``'s layer loop; x is left as it is)."""
        rows = self._rows(x, self.hidden, "x")
        _require(prompts >= 1 and rows % prompts == 0, f"{rows} rows are not {prompts} windows")
        _require(all(1 <= t <= len(self.layers) for t in taps), f"taps {taps} of {len(self.layers)}")
        pos = torch.arange(rows // prompts, dtype=torch.int32, device=self.device).repeat(prompts)
        out = {}
        for i in range(max(taps, default=0)):
            x = self.layer(i, x, prompts, lens, pos)
            if i + 1 in taps:
                out[i + 1] = x
        return [out[t] for t in taps]
