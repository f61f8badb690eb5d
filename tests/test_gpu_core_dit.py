"""``DitModel``: the modulations that a step takes."""

from __future__ import annotations

import dataclasses

import pytest
import torch

from aestrix_amd import dit
from aestrix_amd.step import DitDims, DitStep, random_head, random_projections

pytestmark = pytest.mark.gpu

F16, F32 = torch.float16, torch.float32
TINY = DitDims(l_img=64, l_txt=32, dim=256, ff_inner=512, n_double=1, n_single=1)


@pytest.fixture(autouse=True)
def _need_gpu(request):
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")
    print(request.node.name, flush=True)


def test_modulations_of_other_shapes_are_refused():
    """A modulation without a row of its own for the text, or with one too many, would go to the wrong rows."""
    d = TINY.dim
    step = DitStep(TINY, random_projections(TINY, F16, 3))
    step.set_head(*random_head(TINY, 128, F16, 3))
    g = torch.Generator(device="cuda").manual_seed(3)
    randn = lambda *s: torch.randn(s, generator=g, device="cuda")
    step.set_conditioning(gates=randn(5, d))
    norms = [dit.DitNorms(*(1 + 0.1 * randn(128) for _ in range(4))) for _ in range(2)]
    model = dit.DitModel(step, norms, torch.zeros((TINY.joint, 4), dtype=torch.int32, device="cuda"))
    names = [f.name for f in dataclasses.fields(dit.DitModulation)]
    good = {n: 0.1 * (randn(d) if n[:3] in ("sin", "out") else randn(2, d)) for n in names}
    lat, e = randn(TINY.l_img, 128), randn(TINY.l_txt, d)
    out = torch.full_like(lat, 7.0)
    for n in names:
        shapes = [(2, d), (d - 64,), (1, 1, d)] if n[:3] in ("sin", "out") else [(d,), (1, d), (3, d), (d, 2), (2, d - 64)]
        for bad in [torch.zeros(s, device="cuda") for s in shapes] + [good[n].half(), good[n].cpu()]:
            with pytest.raises(ValueError):
                model.denoise(lat, e, -0.25, dit.DitModulation(**{**good, n: bad}), out=out)
            # Both of a pair alike.
            pair = n.replace("shift", "scale") if n.endswith("shift") else n.replace("scale", "shift")
            with pytest.raises(ValueError):
                model.denoise(lat, e, -0.25, dit.DitModulation(**{**good, n: bad, pair: bad}), out=out)
    torch.cuda.synchronize()
    assert bool((out == 7.0).all())
    mod = dit.DitModulation(**good)
    mod.timestep = 3  # a caller's own
    assert torch.isfinite(model.denoise(lat, e, -0.25, mod, out=out)).all()
