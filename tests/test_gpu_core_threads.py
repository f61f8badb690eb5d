"""Host threads that call on one stream: split calls' two kernels meet in one workspace."""

from __future__ import annotations

import threading

import pytest
import torch

import aestrix_amd as imq
from aestrix_amd import synth

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _need_gpu(request):
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")
    print(request.node.name, flush=True)


def test_threads_on_one_stream_get_their_own_results():
    g = torch.Generator(device="cuda").manual_seed(2)
    randn = lambda *s: torch.randn(s, generator=g, device="cuda").to(torch.bfloat16)
    work = []
    for keys in (3000, 5000, 9000):
        q, k, v = randn(1, 1, 16, 128), randn(1, keys, 4, 128), randn(1, keys, 4, 128)
        assert imq.attention_plan(q, k, v, causal=True)["splits"] > 1
        work.append(lambda q=q, k=k, v=v: imq.attention(q, k, v, causal=True))
    for m in (8, 100):
        x, w, s, b = synth.to_device(synth.make_problem(m, 2560, 9728, seed=m), "cuda:0")
        work.append(lambda x=x, w=w, s=s, b=b: imq.quantized_matmul(x, w, s, b))
    want = [f() for f in work]
    torch.cuda.synchronize()
    got = [[] for _ in work]
    start = threading.Barrier(len(work))

    def run(i):
        start.wait()
        for _ in range(40):
            got[i].append(work[i]())

    threads = [threading.Thread(target=run, args=(i,)) for i in range(len(work))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for i, outs in enumerate(got):
        assert len(outs) == 40 and all(torch.equal(o, want[i]) for o in outs), i
