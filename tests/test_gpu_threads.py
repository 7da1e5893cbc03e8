"""Calls from a thread that has made no CUDA call before."""
import threading

import pytest
import torch

import fastgate_b200 as fg

pytestmark = pytest.mark.gpu


def _cases(dev):
    g = torch.Generator().manual_seed(1)
    x8, w8 = (torch.randint(-9, 10, (n, 1024), generator=g, dtype=torch.int8).to(dev) for n in (16, 512))
    x, w = (torch.randn(n, 1024, generator=g).half().to(dev) for n in (16, 512))
    s, sw = torch.full((16,), 2.0 ** -10, device=dev), torch.ones(512, dtype=torch.half, device=dev)
    norm = torch.ones(1024, dtype=torch.half, device=dev)
    out = lambda m, n=512: torch.empty(m, n, dtype=torch.half, device=dev)
    return {
        "linear_int8": lambda c=out(16): (fg.linear_int8(x8, w8, c, s), c)[1],
        "linear_int8_pairs": lambda c=out(16): (fg.linear_int8(x8[:2], w8, c[:2], s[:2]), c[:2])[1],
        "edgemm": lambda c=out(16): (fg.edgemm_m8n128k64x4_bt(x, w, c), c)[1],
        "fastgemv": lambda c=out(1): (fg.fastgemv(w, x[:1], c), c)[1],
        "fastgemv_int8": lambda c=out(16): (fg.fastgemv_int8(w8, x, c, sw), c)[1],
        "add_rmsnorm": lambda c=out(16, 1024): (fg.add_rmsnorm(x, norm, c), c)[1],
    }


@pytest.mark.parametrize("name", ["linear_int8", "linear_int8_pairs", "edgemm", "fastgemv", "fastgemv_int8", "add_rmsnorm"])
def test_first_cuda_call_of_a_thread(name):
    """What the process knows of its device it knows already; the context is not yet current in the new thread."""
    dev = torch.device("cuda:0")
    run = _cases(dev)[name]
    want = run().clone()
    torch.cuda.synchronize()
    run().zero_()
    torch.cuda.synchronize()
    got, errors = [], []

    def other():
        try:
            got.append(run())
        except Exception as e:  # reported in the test's own thread
            errors.append(e)

    thread = threading.Thread(target=other)
    thread.start()
    thread.join()
    torch.cuda.synchronize()
    assert not errors and torch.equal(got[0], want), errors
