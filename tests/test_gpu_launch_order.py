"""A buffer that one call writes is the weight of the second call after it, whatever stands in between."""
import pytest
import torch

import fastgate_b200 as fg
from fastgate_b200.kvcache import KVCacheInt4, rotation_table

pytestmark = pytest.mark.gpu

N, K = 4096, 2048  # the weight that is written: rows enough that its writer runs for several microseconds


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda:0")


def _rand(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


def _writers(dev):
    """Calls that write a weight [N, K]: fp16 into w16, int8 into w8."""
    x, ones = _rand(1, N, K).half().to(dev), torch.ones(K, dtype=torch.half, device=dev)
    w16, w8, scales = torch.empty(N, K, dtype=torch.half, device=dev), torch.empty(N, K, dtype=torch.int8, device=dev), torch.empty(N, device=dev)
    a8, b8 = (torch.randint(-9, 10, (n, 512), generator=torch.Generator().manual_seed(n), dtype=torch.int8).to(dev) for n in (N, K))
    sa = torch.full((N,), 2.0 ** -12, device=dev)
    a16, b16 = (_rand(n, n, 512).half().to(dev) / 16 for n in (N, K))
    cache, slots = KVCacheInt4(N // 64, 1, 128), torch.arange(N, device=dev)
    q, table = _rand(3, N, K // 128, 128).half().to(dev), rotation_table(N, 128)
    k = _rand(4, N, 1, 128).half().to(dev)
    cache.append(k, k, slots)
    pages, lens = torch.zeros(N, 1, dtype=torch.int32, device=dev), torch.full((N,), 40, dtype=torch.int32, device=dev)
    return w16, w8, {
        "norm": (w16, lambda: fg.add_rmsnorm(x, ones, w16)),
        "norm_int8": (w8, lambda: fg.add_rmsnorm(x, ones, w8, scales=scales)),
        "linear_int8": (w16, lambda: fg.linear_int8(a8, b8, w16, sa)),
        "linear_fp16": (w16, lambda: fg.edgemm_m8n128k64x4_bt(a16[:64], b16, w16[:64])),
        "append": (w16, lambda: cache.append(k, k, slots, table, slots, q, w16.view(N, K // 128, 128))),
        "attention": (w16, lambda: cache.attend(q, pages, lens, w16.view(N, K // 128, 128))),
    }


def _between(dev):
    """Short calls that write nothing of the weight."""
    x, w = _rand(5, 4, 512).half().to(dev), torch.ones(512, dtype=torch.half, device=dev)
    y, x8, sx = torch.empty_like(x), torch.ones(4, 512, dtype=torch.int8, device=dev), torch.ones(4, device=dev)
    c, wl, wl8 = torch.empty(4, 256, dtype=torch.half, device=dev), _rand(6, 256, 512).half().to(dev), torch.ones(256, 512, dtype=torch.int8, device=dev)
    cache, k = KVCacheInt4(2, 1, 64, 16), _rand(7, 4, 1, 64).half().to(dev)
    slots, o = torch.arange(4, device=dev), torch.empty(4, 1, 64, dtype=torch.half, device=dev)
    table, lens = torch.zeros(4, 1, dtype=torch.int32, device=dev), torch.ones(4, dtype=torch.int32, device=dev)
    w4, s4 = fg.quantize_int4(wl)
    q8, s8 = fg.quantize_int8(wl)
    return {
        "norm": lambda: fg.add_rmsnorm(x, w, y),
        "linear_int8_rows": lambda: fg.linear_int8(x8[:1], wl8, c[:1], sx[:1]),
        "linear_int8_tiles": lambda: fg.linear_int8(x8, wl8, c, sx),
        "linear_fp16": lambda: fg.edgemm_m8n128k64x4_bt(x, wl, c),
        "linear_fp16_rows": lambda: fg.fastgemv(wl, x[:1], c[:1]),
        "linear_w8": lambda: fg.fastgemv_int8(q8, x, c, s8),
        "linear_w4": lambda: fg.fastgemv_int4(w4, x, c, s4),
        "append": lambda: cache.append(k, k, slots),
        "attention": lambda: cache.attend(k, table, lens, o),
        "two": lambda: (fg.add_rmsnorm(x, w, y), cache.append(k, k, slots)),
    }


@pytest.mark.parametrize("writer", ["norm", "norm_int8", "linear_int8", "linear_fp16", "append", "attention"])
def test_weight_written_two_calls_earlier(writer, dev):
    w16, w8, writers = _writers(dev)
    weight, write = writers[writer]
    if weight is w8:
        rows = [torch.randint(-9, 10, (m, K), generator=torch.Generator().manual_seed(m), dtype=torch.int8).to(dev) for m in (1, 16)]
        read = lambda x, c: fg.linear_int8(x, w8, c, torch.full((x.shape[0],), 2.0 ** -12, device=dev))
    else:
        rows = [_rand(m, m, K).half().to(dev) / 64 for m in (1, 16)]
        read = lambda x, c: fg.fastgemv(w16, x, c) if x.shape[0] == 1 else fg.edgemm_m8n128k64x4_bt(x, w16, c)
    scales = [torch.full((x.shape[0],), 2.0 ** -12, device=dev) for x in rows]
    weight.zero_()
    torch.cuda.synchronize()
    write()
    torch.cuda.synchronize()
    want = []
    for x in rows:
        want.append(torch.empty(x.shape[0], N, dtype=torch.half, device=dev))
        read(x, want[-1])
    torch.cuda.synchronize()
    assert bool((want[1] != 0).any())
    if weight is w8:  # nothing but the three calls on the stream
        read = lambda x, c: fg.linear_int8(x, w8, c, scales[0] if x.shape[0] == 1 else scales[1])
    for name, between in _between(dev).items():
        for x, w in zip(rows, want):
            got = [torch.empty_like(w) for _ in range(10)]
            for c in got:
                weight.zero_()
                write()
                between()
                read(x, c)
            torch.cuda.synchronize()
            assert all(torch.equal(c, w) for c in got), (name, x.shape[0])


@pytest.mark.parametrize("writer", ["norm", "norm_int8", "linear_int8", "append", "attention"])
def test_captured_weight_written_two_calls_earlier(writer, dev):
    """The same three calls in a graph, where the early starts are edges between its nodes."""
    w16, w8, writers = _writers(dev)
    weight, write = writers[writer]
    if weight is w8:
        x = torch.randint(-9, 10, (16, K), generator=torch.Generator().manual_seed(16), dtype=torch.int8).to(dev)
        scales = torch.full((16,), 2.0 ** -12, device=dev)
        read = lambda c: fg.linear_int8(x, w8, c, scales)
    else:
        x = _rand(16, 16, K).half().to(dev) / 64
        read = lambda c: fg.edgemm_m8n128k64x4_bt(x, w16, c)
    between = _between(dev)
    want, got = (torch.empty(16, N, dtype=torch.half, device=dev) for _ in range(2))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # the stream's workspaces, too
        write()
        torch.cuda.synchronize()
        read(want)
        for call in between.values():
            call()
        torch.cuda.synchronize()
    for name, call in between.items():
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            weight.zero_()
            write()
            call()
            read(got)
        for _ in range(5):
            got.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got, want), name
