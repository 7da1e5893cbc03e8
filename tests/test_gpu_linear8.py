"""linear_int8 against 64 bits: the GEMV and every tiling of the tensor-core kernel, every epilogue, the largest sums, graphs."""
import ctypes
import os
import subprocess
import sys

import pytest
import torch

import fastgate_b200 as fg
from fastgate_b200 import capi
from tests import serving_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda:0")


def _data(M, N, K, seed, lim=127):
    g = torch.Generator().manual_seed(seed)
    x = torch.randint(-lim, lim + 1, (M, K), generator=g, dtype=torch.int8)
    w = torch.randint(-lim, lim + 1, (N, K), generator=g, dtype=torch.int8)
    sx = (torch.rand(M, generator=g) + 0.5) / 64
    sw = ((torch.rand(N, generator=g) + 0.5) / (64 * K ** 0.5)).half()
    return x, w, sx, sw, g


def _check(got, want, size):
    # the sum is exact; scales, bias, activation and residual take a few 32-bit roundings of terms of `size`
    tol = want.abs() * ref.HALF_STEP + size * 2.0 ** -20 + ref.TINY
    err = (got.cpu().to(torch.float64) - want).abs()
    assert bool((err <= tol).all()), float((err / tol).max())


@pytest.mark.parametrize("M", [1, 2, 16, 17, 33, 64, 65, 128, 129, 300])
@pytest.mark.parametrize("N,K", [(128, 128), (1152, 640), (256, 4096), (4224, 1408)])
def test_plain(M, N, K, dev):
    x, w, sx, sw, _ = _data(M, N, K, M + N)
    out = torch.full((M + 2, N), 123.0, dtype=torch.half, device=dev)
    fg.linear_int8(x.to(dev), w.to(dev), out[1:-1], sx.to(dev), sw.to(dev))
    _check(out[1:-1], *ref.linear_int8(x, w, sx, sw))
    assert bool((out[0] == 123).all()) and bool((out[-1] == 123).all())


@pytest.mark.parametrize("act", ["none", "gelu", "gelu_tanh", "silu", "silu_gate"])
@pytest.mark.parametrize("M", [1, 2, 40, 100, 700])
def test_epilogues(M, act, dev):
    N, K = 896, 512
    x, w, sx, sw, g = _data(M, N, K, M)
    width = N // 2 if act == "silu_gate" else N
    bias, res = torch.randn(N, generator=g).half(), torch.randn(M, width, generator=g).half()
    for b, r in ((bias, res), (None, res), (bias, None)):
        out = torch.empty(M, width, dtype=torch.half, device=dev)
        fg.linear_int8(x.to(dev), w.to(dev), out, sx.to(dev), sw.to(dev), None if b is None else b.to(dev), None if r is None else r.to(dev), act)
        _check(out, *ref.linear_int8(x, w, sx, sw, b, r, act))


@pytest.mark.parametrize("M", [3, 700])
def test_scales_of_both_types_and_none(M, dev):
    x, w, sx, sw, _ = _data(M, 384, 256, 5, lim=3)
    h = sx.half()
    out = torch.empty(M, 384, dtype=torch.half, device=dev)
    fg.linear_int8(x.to(dev), w.to(dev), out, h.to(dev))
    _check(out, *ref.linear_int8(x, w, h))
    fg.linear_int8(x.to(dev), w.to(dev), out, h.to(dev), sw.to(dev))
    _check(out, *ref.linear_int8(x, w, h, sw))


@pytest.mark.parametrize("M", [1, 2, 5, 200, 600])
def test_largest_sums(M, dev):
    """All -128 at the longest K allowed: the sum is 128 * 128 * 130944, just inside 32 bits."""
    K, N = 130944, 256
    x = torch.full((M, K), -128, dtype=torch.int8, device=dev)
    w = torch.full((N, K), -128, dtype=torch.int8, device=dev)
    w[1] = 127
    sx = torch.full((M,), 2.0 ** -20, device=dev)
    out = torch.empty(M, N, dtype=torch.half, device=dev)
    fg.linear_int8(x, w, out, sx)
    want = torch.full((M, N), 128.0 * 128 * K / 2 ** 20, dtype=torch.float64)
    want[:, 1] = -128.0 * 127 * K / 2 ** 20
    assert torch.equal(out.cpu(), want.half())
    with pytest.raises(ValueError):
        fg.linear_int8(torch.zeros(1, 131072, dtype=torch.int8, device=dev), torch.zeros(128, 131072, dtype=torch.int8, device=dev),
                       torch.zeros(1, 128, dtype=torch.half, device=dev), torch.ones(1, device=dev))


def test_rows_do_not_depend_on_their_company(dev):
    """Exact sums and the same roundings after them: row i of every path (GEMV, tiles of each width, clusters that share k, pairs)
    has the same bits, whatever the epilogue."""
    x, w, sx, sw, g = _data(2600, 8192, 384, 11)
    xd, wd, sxd, swd = x.to(dev), w.to(dev), sx.to(dev), sw.to(dev)
    bias, res = torch.randn(8192, generator=g).half().to(dev), torch.randn(2600, 8192, generator=g).half().to(dev)
    for act in ("none", "gelu_tanh", "silu_gate"):
        width = 4096 if act == "silu_gate" else 8192
        r = res[:, :width].contiguous()
        full = torch.empty(2600, width, dtype=torch.half, device=dev)
        fg.linear_int8(xd, wd, full, sxd, swd, bias, r, act)
        for n in (1, 2, 16, 31, 64, 128, 130, 513):
            out = torch.empty(n, width, dtype=torch.half, device=dev)
            fg.linear_int8(xd[:n], wd, out, sxd[:n], swd, bias, r[:n], act)
            assert torch.equal(out, full[:n]), (n, act)


@pytest.mark.parametrize("M", [5, 300])
def test_in_place_residual_and_quantize_int8(M, dev):
    """Activations from quantize_int8 (fp16 scales); the residual stream updated in place."""
    g = torch.Generator().manual_seed(2)
    xf = torch.randn(M, 1024, generator=g).half().to(dev)
    wf = (torch.randn(512, 1024, generator=g) / 32).half().to(dev)
    x8, sx = fg.quantize_int8(xf)
    w8, sw = fg.quantize_int8(wf)
    res = torch.randn(M, 512, generator=g).half().to(dev)
    want = ref.linear_int8(x8.cpu(), w8.cpu(), sx.cpu(), sw.cpu(), None, res.cpu())
    fg.linear_int8(x8, w8, res, sx, sw, residual=res)
    _check(res, *want)


@pytest.mark.parametrize("M", [4, 200])
def test_gate_from_two_weights(M, dev):
    g = torch.Generator().manual_seed(8)
    wg, wu = (torch.randint(-127, 128, (320, 384), generator=g, dtype=torch.int8) for _ in range(2))
    sg, su, bg, bu = ((torch.rand(320, generator=g) / 100).half() for _ in range(4))
    x = torch.randint(-127, 128, (M, 384), generator=g, dtype=torch.int8)
    sx = torch.rand(M, generator=g) / 100
    w, s, b = (fg.prepack_gate_up(p.to(dev), q.to(dev)) for p, q in ((wg, wu), (sg, su), (bg, bu)))
    out = torch.empty(M, 320, dtype=torch.half, device=dev)
    fg.linear_int8(x.to(dev), w, out, sx.to(dev), s, b, act="silu_gate")
    gate, s1 = ref.linear_int8(x, wg, sx, sg, bg)
    up, s2 = ref.linear_int8(x, wu, sx, su, bu)
    _check(out, ref.activation(gate, "silu") * up, (s1 + 1) * (s2 + 1))


@pytest.mark.parametrize("M", [8, 100, 160, 2048])
def test_two_graphs_of_one_stream_side_by_side(M, dev):
    """Graphs captured on one stream, replayed on two streams at once, do not meet (the operator keeps nothing between its CTAs
    but a cluster's shared memory)."""
    x, w, sx, sw, _ = _data(M, 4096, 2048, 21)
    xd, wd, sxd, swd = x.to(dev), w.to(dev), sx.to(dev), sw.to(dev)
    want = torch.empty(M, 4096, dtype=torch.half, device=dev)
    fg.linear_int8(xd, wd, want, sxd, swd)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    graphs, outs = [], []
    for _ in range(2):
        out = torch.zeros(M, 4096, dtype=torch.half, device=dev)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            for _ in range(4):
                fg.linear_int8(xd, wd, out, sxd, swd)
        graphs.append(graph)
        outs.append(out)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):
        for out in outs:
            out.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(s1):
            graphs[0].replay()
        with torch.cuda.stream(s2):
            graphs[1].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want)


def test_two_streams_and_mixed_with_fp16_linears(dev):
    """Eager calls on two streams, each between fp16 linears of the same streams (they share the stream's workspace)."""
    x, w, sx, sw, g = _data(48, 1024, 1024, 31)
    xd, wd, sxd, swd = x.to(dev), w.to(dev), sx.to(dev), sw.to(dev)
    xf, wf = torch.randn(48, 1024, generator=g).half().to(dev), (torch.randn(1024, 1024, generator=g) / 32).half().to(dev)
    want8, want16 = (torch.empty(48, 1024, dtype=torch.half, device=dev) for _ in range(2))
    fg.linear_int8(xd, wd, want8, sxd, swd)
    fg.edgemm_m8n128k64x4_bt(xf, wf, want16)
    torch.cuda.synchronize()
    got = []
    for stream in (torch.cuda.Stream(), torch.cuda.Stream()):
        with torch.cuda.stream(stream):
            for _ in range(10):
                a, b = torch.empty_like(want8), torch.empty_like(want16)
                fg.linear_int8(xd, wd, a, sxd, swd)
                fg.edgemm_m8n128k64x4_bt(xf, wf, b)
                got.append((a, b))
    torch.cuda.synchronize()
    for a, b in got:
        assert torch.equal(a, want8) and torch.equal(b, want16)


def test_refusals(dev):
    x, w = torch.zeros(2, 256, dtype=torch.int8, device=dev), torch.zeros(128, 256, dtype=torch.int8, device=dev)
    c, s = torch.empty(2, 128, dtype=torch.half, device=dev), torch.ones(2, device=dev)
    fg.linear_int8(x, w, c, s)
    fg.linear_int8(x[:0], w, c[:0], s[:0])
    for bad in (lambda: fg.linear_int8(x[:, :200].contiguous(), w[:, :200].contiguous(), c, s),
                lambda: fg.linear_int8(x, w[:100], torch.empty(2, 100, dtype=torch.half, device=dev), s),
                lambda: fg.linear_int8(x, w, c, s, act="relu")):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: fg.linear_int8(x, w, c, s[:1]),
                lambda: fg.linear_int8(x, w, c, s.double()),
                lambda: fg.linear_int8(x, w, c.float(), s),
                lambda: fg.linear_int8(x.half(), w, c, s),
                lambda: fg.linear_int8(x, w[:, :128].contiguous(), c, s),
                lambda: fg.linear_int8(x, w, c, s, bias=torch.zeros(64, dtype=torch.half, device=dev)),
                lambda: fg.linear_int8(x, w, c, s, act="silu_gate")):
        with pytest.raises(RuntimeError):
            bad()
    both = torch.empty(2 * 128 + 128, dtype=torch.half, device=dev)
    with pytest.raises(ValueError):  # the residual one row further in the same buffer
        fg.linear_int8(x, w, both[:256].view(2, 128), s, residual=both[128:].view(2, 128))
    args = lambda act=0, xs=s.data_ptr(): capi.lib.fg_linear_w8a8(x.data_ptr(), w.data_ptr(), xs, 1, None, c.data_ptr(), 2, 128, 256, None, None, act,
                                                                  None, ctypes.c_void_p(0))
    assert args(act=9) == capi.FG_ERR_PLAN and args(xs=None) == capi.FG_ERR_NULL


@pytest.mark.parametrize("M,N,K,act", [(3001, 4096, 1024, "none"), (2048, 5120, 1152, "gelu_tanh"), (3001, 3456, 1024, "none"), (4096, 4096, 1024, "silu_gate"),
                                       (1500, 8192, 1024, "silu")])
def test_last_columns_of_tiles_may_be_narrower(M, N, K, act, dev):
    """Sizes whose last wave of wide tiles would be far from full: narrower ones of 64, 128 or 192 weight rows take its place."""
    x8, w8, xs, ws, g = _data(M, N, K, M + N)
    bias = torch.randn(N, generator=g).half()
    width = N // 2 if act == "silu_gate" else N
    res = torch.randn(M, width, generator=g).half()
    d = [t.to(dev) for t in (x8, w8, xs, ws, bias, res)]
    c = torch.full((M, width), float("nan"), dtype=torch.half, device=dev)
    fg.linear_int8(d[0], d[1], c, d[2], d[3], d[4], d[5], act)
    rows = torch.cat([torch.arange(0, M, 97), torch.arange(M - 3, M)])
    _check(c[rows.to(dev)], *ref.linear_int8(x8[rows], w8, xs[rows], ws, bias, res[rows], act))
    again = torch.empty_like(c)  # every row, bit for bit, against calls of other tilings
    for m in range(0, M, 100):
        fg.linear_int8(d[0][m:m + 100], d[1], again[m:m + 100], d[2][m:m + 100], d[3], d[4], d[5][m:m + 100], act)
    assert torch.equal(c, again)


def test_captured_before_any_eager_call(dev):
    """A stream's first call may be a captured one; the status word that it holds is the one that workspace_status() reads."""
    x8, w8, xs, ws, *_ = _data(9, 256, 512, 77)
    a = [t.to(dev) for t in (x8, w8, xs, ws)]
    c = torch.empty(9, 256, dtype=torch.half, device=dev)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        fg.linear_int8(a[0], a[1], c, a[2], a[3])
    for _ in range(3):
        graph.replay()
    want = torch.empty_like(c)
    fg.linear_int8(a[0], a[1], want, a[2], a[3])
    assert torch.equal(c, want) and fg.workspace_status(0) == 0


def test_first_calls_from_several_threads():
    """What a process finds out once about its device is found out by whichever thread comes first."""
    code = """
import threading, torch
import fastgate_b200 as fg
dev = torch.device("cuda:0")
g = torch.Generator().manual_seed(1)
x, w = (torch.randint(-9, 10, (n, 1024), generator=g, dtype=torch.int8).to(dev) for n in (16, 512))
s = torch.full((16,), 2.0 ** -10, device=dev)
outs = [torch.empty(16, 512, dtype=torch.half, device=dev) for _ in range(8)]
torch.cuda.synchronize()
gate = threading.Barrier(8)
def run(i):
    with torch.cuda.stream(torch.cuda.Stream()):
        gate.wait()
        fg.linear_int8(x, w, outs[i], s)
threads = [threading.Thread(target=run, args=(i,)) for i in range(8)]
for t in threads: t.start()
for t in threads: t.join()
torch.cuda.synchronize()
want = (x.cpu().double() @ w.cpu().double().T * 2.0 ** -10).half()
assert all(torch.equal(o.cpu(), want) for o in outs)
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    subprocess.run([sys.executable, "-c", code], check=True, cwd=root, timeout=300)
