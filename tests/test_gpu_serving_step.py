"""The serving operators together: decoding steps of one block with 8-bit activations and a 4-bit cache, each stage held
against 64 bits on the inputs that it was given, the step then captured and replayed."""
import pytest
import torch

import fastgate_b200 as fg
from fastgate_b200.kvcache import KVCacheInt4, rotation_table
from tests import serving_ref as ref

pytestmark = pytest.mark.gpu

HIDDEN, HQ, HKV, D, FF, PAGE = 512, 8, 2, 64, 768, 16


class Block:
    def __init__(self, dev, batch):
        g = torch.Generator().manual_seed(77)
        weight = lambda n, k: fg.quantize_int8((torch.randn(n, k, generator=g) / k ** 0.5).half().to(dev))
        self.qkv, self.out = weight((HQ + 2 * HKV) * D, HIDDEN), weight(HIDDEN, HQ * D)
        gate, up = weight(FF, HIDDEN), weight(FF, HIDDEN)
        self.gate_up = (fg.prepack_gate_up(gate[0], up[0]), fg.prepack_gate_up(gate[1], up[1]))
        self.down = weight(HIDDEN, FF)
        self.norm1, self.norm2 = ((1 + 0.1 * torch.randn(HIDDEN, generator=g)).half().to(dev) for _ in range(2))
        self.bias = torch.randn((HQ + 2 * HKV) * D, generator=g).half().to(dev)
        self.cache = KVCacheInt4(64, HKV, D, PAGE)
        self.table = torch.randperm(64, generator=g)[: batch * 8].view(batch, 8).int().to(dev)
        self.angles = rotation_table(PAGE * 8, D)
        half = lambda *s: torch.empty(*s, dtype=torch.half, device=dev)
        self.x8, self.sx = torch.empty(batch, HIDDEN, dtype=torch.int8, device=dev), torch.empty(batch, device=dev)
        self.y, self.o, self.ff = half(batch, (HQ + 2 * HKV) * D), half(batch, HQ, D), half(batch, FF)
        self.attn, self.mlp, self.stream = half(batch, HIDDEN), half(batch, HIDDEN), torch.zeros(batch, HIDDEN, device=dev)
        self.lens = torch.zeros(batch, dtype=torch.int32, device=dev)
        self.pos = torch.zeros(batch, dtype=torch.int64, device=dev)
        self.rows = torch.arange(batch, device=dev)

    def step(self, x):
        """x [batch, HIDDEN] fp16: one token of each sequence, at position self.pos; the result lands in self.mlp."""
        fg.add_rmsnorm(x, self.norm1, self.x8, self.stream, scales=self.sx)
        fg.linear_int8(self.x8, self.qkv[0], self.y, self.sx, self.qkv[1], bias=self.bias)
        q, k, v = (t.unflatten(-1, (-1, D)) for t in self.y.split([HQ * D, HKV * D, HKV * D], -1))
        self.cache.append(k, v, self.cache.slots(self.table, self.rows, self.pos), self.angles, self.pos, q)
        self.cache.attend(q, self.table, self.lens, self.o)
        o8, so = fg.quantize_int8(self.o.flatten(1))
        fg.linear_int8(o8, self.out[0], self.attn, so, self.out[1])
        fg.add_rmsnorm(self.attn, self.norm2, self.x8, self.stream, scales=self.sx)
        fg.linear_int8(self.x8, self.gate_up[0], self.ff, self.sx, self.gate_up[1], act="silu_gate")
        f8, sf = fg.quantize_int8(self.ff)
        fg.linear_int8(f8, self.down[0], self.mlp, sf, self.down[1])
        return o8, so, f8, sf


def _close(got, want, size):
    err = (got.cpu().double() - want).abs()
    assert bool((err <= want.abs() * ref.HALF_STEP + size * 2.0 ** -18 + ref.TINY).all())


def test_decoding_steps():
    dev, batch = torch.device("cuda:0"), 5
    blk = Block(dev, batch)
    g = torch.Generator().manual_seed(5)
    begin = torch.tensor([0, 3, 15, 16, 40])  # how far each sequence is before the first step
    for b, n in enumerate(begin.tolist()):
        if n:
            k, v = (torch.randn(n, HKV, D, generator=g).half().to(dev) for _ in range(2))
            at = torch.arange(n, device=dev)
            blk.cache.append(k, v, blk.cache.slots(blk.table, torch.full((n,), b, device=dev), at), blk.angles, at)
    stream = torch.zeros(batch, HIDDEN, dtype=torch.float64)
    for step in range(4):
        blk.pos.copy_(begin + step)
        blk.lens.copy_((begin + step + 1).int())
        x = torch.randn(batch, HIDDEN, generator=g).half()
        o8, so, f8, sf = blk.step(x.to(dev))
        blk.cache.check()
        stream = stream + x.double() + blk.attn.cpu().double()
        assert bool(((blk.stream.cpu().double() - stream).abs() <= stream.abs() * 2.0 ** -20 + 2.0 ** -20).all())
        # the rows in the cache are those of this step's projection, turned; the attention is over what the cache holds
        v = blk.y[:, (HQ + HKV) * D:].unflatten(-1, (-1, D)).cpu().double()
        slots = blk.cache.slots(blk.table, blk.rows, blk.pos)
        vb = blk.cache.read(slots)[1].cpu().double()
        scale, _, _ = ref.quantise(v)
        assert bool(((vb - v).abs() <= scale * 0.51 + v.abs() * ref.HALF_STEP).all())
        q = blk.y[:, : HQ * D].unflatten(-1, (-1, D)).cpu()  # turned in place
        want, span, top = ref.attention(q, blk.cache.pages.cpu(), blk.table.cpu().tolist(), blk.lens.cpu().tolist(), PAGE)
        assert bool(((blk.o.cpu().double() - want).abs() <= ref.attention_tolerance(want, span, top)).all())
        _close(blk.attn, *ref.linear_int8(o8.cpu(), blk.out[0].cpu(), so.cpu(), blk.out[1].cpu()))
        _close(blk.ff, *ref.linear_int8(blk.x8.cpu(), blk.gate_up[0].cpu(), blk.sx.cpu(), blk.gate_up[1].cpu(), act="silu_gate"))
        _close(blk.mlp, *ref.linear_int8(f8.cpu(), blk.down[0].cpu(), sf.cpu(), blk.down[1].cpu()))
        # the second norm saw the stream after the attention
        tt = ref.rmsnorm(blk.stream.cpu(), blk.norm2.cpu())[2]
        assert float((blk.x8.cpu().double() - tt * 127 / tt.abs().amax(-1, keepdim=True)).abs().max()) <= 0.5 + 127 * 2.0 ** -20


def test_captured_step_equals_eager():
    """A step captured once and replayed at every position gives the bits of the eager steps."""
    dev, batch = torch.device("cuda:0"), 3
    eager, graphed = Block(dev, batch), Block(dev, batch)
    g = torch.Generator().manual_seed(6)
    xs = [torch.randn(batch, HIDDEN, generator=g).half().to(dev) for _ in range(5)]
    buf = torch.zeros_like(xs[0])
    graphed.lens.fill_(1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        graphed.step(buf)
    graphed.stream.zero_()
    graphed.cache.pages.zero_()
    for i, x in enumerate(xs):
        for blk in (eager, graphed):
            blk.pos.fill_(i)
            blk.lens.fill_(i + 1)
        eager.step(x)
        buf.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(eager.mlp, graphed.mlp) and torch.equal(eager.stream, graphed.stream), i
        assert torch.equal(eager.cache.pages, graphed.cache.pages), i
