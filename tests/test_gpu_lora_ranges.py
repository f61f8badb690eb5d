"""quantized_matmul_lora in f16 where an adapter's ranks, or the rows of its B, differ much in
size, against its definition in 64 bits."""

from __future__ import annotations

import pytest
import torch

import aestrix_amd as imq
from core_reference import U32, check, half_step, least

pytestmark = pytest.mark.gpu

F16 = torch.float16
NAN, INF = float("nan"), float("inf")
# (rows, K, N): the few-row kernel, partial sums and either join, the register-staged and the other
# tiles, u by rows and by tiles (test_the_ways_there).
SHAPES = [(1, 2560, 300), (5, 2560, 500), (40, 256, 300), (300, 256, 300), (70, 64, 300), (64, 2560, 6144), (1000, 512, 4100)]


@pytest.fixture(autouse=True)
def _need_gpu(request):
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")
    print(request.node.name, flush=True)


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def projection(g, n, k):
    w = torch.randint(-2 ** 31, 2 ** 31 - 1, (n, k // 8), generator=g, device="cuda", dtype=torch.int32)
    s = (randn(g, n, k // 64).abs() / (4 * k ** 0.5)).half()
    return w, s, (-7.5 * s.float() + randn(g, n, k // 64) / (10 * k ** 0.5)).half()


def held(b):
    """|B| as it is held: a power of two for each column brings its largest element to [1, 2), but
    takes no bit of any element (f16's smallest step is 2^-24)."""
    out = b.double().abs().cpu().nan_to_num(0.0, 0.0, 0.0)
    for r in range(out.shape[1]):
        column = [int(v * 2 ** 24) for v in out[:, r].tolist()]
        if any(column):
            up = 25 - max(column).bit_length()
            least_bit = min((v & -v).bit_length() - 1 for v in column if v)
            out[:, r] *= 2.0 ** max(up, -least_bit)
    return out.to(b.device)


def wanted(x, proj, ab, c, ids):
    """(y, bound).  fp32 sums of K, then of K and rank terms; u as two values of f16, of which half
    a step of half a step is left, or half of f16's smallest step, times B as it is held; one
    rounding."""
    k = x.shape[1]
    wd, xd = imq.dequantize(*proj).double(), x.double()
    y, mag = xd @ wd.T.contiguous(), xd.abs() @ wd.abs().T.contiguous()
    err = (k + 8) * U32 * mag
    for i, (a, b) in enumerate(ab):
        rows = torch.nonzero(ids == i)[:, 0]
        ad, bt, r = a.double(), b.double().T.contiguous(), a.shape[0]
        u, um = c[i] * (xd[rows] @ ad.T.contiguous()), abs(c[i]) * (xd[rows].abs() @ ad.abs().T.contiguous())
        y[rows] += u @ bt
        err[rows] += (k + r + 16) * U32 * (um @ bt.abs())
        err[rows] += (half_step(F16) ** 2 + (k + 8) * U32) * (u.abs() @ bt.abs())
        err[rows] += (r + 8) * U32 * mag[rows] + 2.0 ** -25 * held(b).sum(1)
    return y, half_step(F16) * y.abs() + 1.02 * err + least(F16)


def run(ab, shape, c=None):
    m, k, n = shape
    g = gen(m)
    proj, x = projection(g, n, k), randn(g, m, k).half()
    c = [1.0] * len(ab) if c is None else c
    ids = torch.tensor([-1 if r % 7 == 6 else r % len(ab) for r in range(m)], dtype=torch.int32, device="cuda")
    got = imq.quantized_matmul_lora(x, *proj, imq.LoraAdapters(ab, c), ids)
    want, bound = wanted(x, proj, ab, c, ids)
    assert float(want.abs().max()) < 60000.0
    check(got, want, bound, f"{m} rows")


def test_what_is_held():
    """B comes back from what is held, bit for bit, with its columns' largest elements at 1 or more."""
    g = gen(1)
    b = (randn(g, 90, 24) * torch.exp2(torch.randint(-20, 12, (90, 24), generator=g, device="cuda"))).half()
    b[:, 3], b[:, 4] = 0.0, torch.where(torch.arange(90, device="cuda") == 7, 2.0 ** -24, 0.0).half()
    b[:, 5] = 2.0 ** 10 * (1 + torch.arange(90, device="cuda")).half()
    b[5, 6], b[6, 6], b[7, 7] = NAN, INF, -INF
    ad = imq.LoraAdapters([(randn(g, 24, 64).half(), b)], 3.0)
    at = ad.b.view(90, 32)
    assert bool((at[:, 24:] == 0).all())
    up = ad.scale[:24].double() / 3.0
    assert torch.equal((at[:, :24].double() * up).half().nan_to_num(7.0), b.nan_to_num(7.0))
    assert torch.equal(at[:, :24].double().abs().nan_to_num(0.0, 0.0, 0.0), held(b))


def test_the_ways_there():
    g = gen(2)
    seen = []
    for m, k, n in SHAPES:
        for rank in (16, 64, 256):
            plan = imq.quantized_matmul_lora_plan(imq.LoraAdapters([(randn(g, rank, k).half(), randn(g, n, rank).half())] * 2), m)
            seen.append((plan["kernel"], plan["u"], plan["join"]))
    assert {("few", "rows", "outputs"), ("split", "rows", "outputs"), ("split", "tiles", "tiles"), ("tiles", "tiles", None),
            ("tiles_reg", "rows", None)} <= set(seen), seen


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("rank", [2, 24, 64, 256])
def test_ranks_of_mixed_size(shape, rank):
    """Large rows of A before small columns of B, up to A x of some 2^26, and the other way round."""
    g = gen(rank)
    s = torch.arange(rank, device="cuda") % 27 - 13.0
    _, k, n = shape
    ab = [((randn(g, rank, k) / k ** 0.5 * torch.exp2(s if i else -s)[:, None]).half(),
           (randn(g, n, rank) * torch.exp2(-s if i else s)).half()) for i in range(2)]
    run(ab, shape, c=[-2.0, 16.0])


@pytest.mark.parametrize("shape", SHAPES)
def test_one_ordinary_rank_and_one_of_large_a(shape):
    """A x of 2e5 and more in one rank times elements of 2^-14, beside a rank of B of about 1."""
    g = gen(3)
    _, k, n = shape
    a = torch.stack([randn(g, k) / 16, 12000.0 * randn(g, k)]).half()
    b = torch.stack([randn(g, n), 2.0 ** -14 * randn(g, n)], 1).half()
    b[::9, 1] = 0.0
    run([(a, b)], shape)


@pytest.mark.parametrize("shape", SHAPES)
def test_rows_of_b_of_mixed_size(shape):
    """Elements of 2^-12 to 2^10 in every column; one of 1000 among others of 0.01."""
    g = gen(4)
    _, k, n = shape
    rows = torch.exp2(10.0 - torch.arange(n, device="cuda") % 23)
    mixed = ((randn(g, 16, k) / 4 / k ** 0.5).half(), (randn(g, n, 16) * rows[:, None]).half())
    one = ((randn(g, 16, k) / 4 / k ** 0.5).half(), (0.01 * randn(g, n, 16)).half())
    one[1][17] = 1000.0
    run([mixed, one], shape)


@pytest.mark.parametrize("shape", SHAPES)
def test_an_element_that_is_not_finite_leaves_its_column_in_range(shape):
    """NaN or infinite in one output; the others of that adapter have a large A before a small B."""
    g = gen(5)
    m, k, n = shape
    proj, x = projection(g, n, k), randn(g, m, k).half()
    a, b = (3000 * randn(g, 16, k)).half(), (2.0 ** -18 * randn(g, n, 16)).half()
    ids = torch.tensor([r % 2 - 1 for r in range(m)], dtype=torch.int32, device="cuda")
    ids[0] = 0
    want, bound = wanted(x, proj, [(a, b)], [1.0], ids)
    b[7, 2], b[8, 3] = NAN, INF
    got = imq.quantized_matmul_lora(x, *proj, imq.LoraAdapters([(a, b)]), ids)
    assert not bool(torch.isfinite(got[ids == 0][:, 7:9]).any())
    got[:, 7:9], want[:, 7:9] = 0.0, 0.0
    check(got, want, bound, f"{m} rows")


def test_a_factor_that_ends_the_range_of_fp32():
    """A factor near fp32's largest takes nothing from zeros."""
    g = gen(6)
    proj, x = projection(g, 100, 128), randn(g, 5, 128).half()
    ab = [(torch.zeros(8, 128, dtype=F16, device="cuda"), (4000 * randn(g, 100, 8)).half())]
    ids = torch.zeros(5, dtype=torch.int32, device="cuda")
    got = imq.quantized_matmul_lora(x, *proj, imq.LoraAdapters(ab, 2.9e38), ids)
    assert torch.equal(got, imq.quantized_matmul_lora(x, *proj, imq.LoraAdapters(ab, 2.9e38), ids - 1))


@pytest.mark.parametrize("shape", SHAPES)
def test_small_a_and_x(shape):
    """A and x under f16's smallest normal value, whose bits count behind a large factor."""
    g = gen(7)
    m, k, n = shape
    ab = [((2.0 ** -17 * randn(g, 24, k)).half(), randn(g, n, 24).half())]
    run(ab, shape, c=[2.0 ** 13])
    proj, x = projection(g, n, k), (2.0 ** -17 * randn(g, m, k)).half()
    ab = [((64 * randn(g, 24, k)).half(), randn(g, n, 24).half())]
    ids = torch.zeros(m, dtype=torch.int32, device="cuda")
    got = imq.quantized_matmul_lora(x, *proj, imq.LoraAdapters(ab, 8.0), ids)
    check(got, *wanted(x, proj, ab, [8.0], ids), f"small x, {m} rows")


def test_scales_by_adapter_or_by_rank():
    """The same set with its factors given either way, and a value that is neither."""
    g = gen(8)
    proj, x = projection(g, 100, 128), randn(g, 33, 128).half()
    ab = [((randn(g, r, 128) / 16).half(), randn(g, 100, r).clamp(-1.5, 1.5).half()) for r in (16, 32)]
    for _, b in ab:
        b[0] = 1.0  # every column is held as it is
    ad = imq.LoraAdapters(ab, [0.5, -3.0])
    ids = torch.arange(33, device="cuda", dtype=torch.int32) % 3 - 1
    want = imq.quantized_matmul_lora(x, *proj, ad, ids)
    two = torch.tensor([0.5, -3.0], device="cuda")
    assert torch.equal(ad.scale, two.repeat_interleave(torch.tensor([16, 32], device="cuda")))
    ad._c.scale, ad._c.rank_scales = two.data_ptr(), 0
    assert torch.equal(imq.quantized_matmul_lora(x, *proj, ad, ids), want)
    ad._c.rank_scales = 2
    with pytest.raises(imq.ImqInvalid):
        imq.quantized_matmul_lora(x, *proj, ad, ids)
