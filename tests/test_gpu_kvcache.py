"""The 4-bit key/value cache (append, read, attention) against 64 bits: layouts, lengths, masks, bad indices, streams."""
import ctypes

import pytest
import torch

import fastgate_b200 as fg
from fastgate_b200 import capi
from fastgate_b200.kvcache import KVCacheInt4, rotation_table
from tests import serving_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda:0")


# ---- append and read -------------------------------------------------------------------------
def _check_rows(got, want):
    """Rows read back: within half a step of the exact row, plus what fp16 parameters and 32-bit angles add.  The top code
    moves by fifteen times the scale's rounding, half a step of an fp16: 2^-11 of it, or 2^-25 where the scale is below the
    normal range (127 * 2^-24 / 15 = 8.47 * 2^-24 is stored as 8 * 2^-24 and takes the top of the row from 127 to 120)."""
    scale, low, _ = ref.quantise(want)
    size = want.abs().amax(-1, keepdim=True)
    tol = scale * 0.5 + size * (2.0 ** -20 + ref.HALF_STEP) + 15 * (scale * ref.HALF_STEP + ref.TINY / 2) + ref.TINY
    err = (got.cpu().to(torch.float64) - want).abs()
    assert bool((err <= tol).all()), float((err / tol).max())


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
@pytest.mark.parametrize("tokens,hq,hkv,d,page", [(1, 1, 1, 64, 16), (3, 8, 2, 128, 32), (64, 7, 1, 128, 64), (257, 6, 3, 64, 16), (900, 32, 8, 128, 128)])
def test_append_and_read(tokens, hq, hkv, d, page, index, interleaved, dev):
    g = torch.Generator().manual_seed(tokens + d)
    pages = -(-tokens // page) + 3
    cache = KVCacheInt4(pages, hkv, d, page)
    qkv = torch.randn(tokens, (hq + 2 * hkv) * d + 8, generator=g).half()
    q, k, v = (t.unflatten(-1, (-1, d)) for t in qkv[:, 8:].split([hq * d, hkv * d, hkv * d], -1))
    slots = torch.randperm(pages * page, generator=g)[:tokens].to(index)
    positions = torch.randint(0, 5000, (tokens,), generator=g, dtype=index)
    table = rotation_table(5000, d, device="cpu")
    buf = qkv.to(dev)
    qd, kd, vd = (t.unflatten(-1, (-1, d)) for t in buf[:, 8:].split([hq * d, hkv * d, hkv * d], -1))
    q_out = torch.empty(tokens, hq, d, dtype=torch.half, device=dev)
    cache.append(kd, vd, slots.to(dev), table.to(dev), positions.to(dev), qd, q_out, interleaved)
    k_back, v_back = cache.read(slots.to(dev))
    cache.check()
    want_q = ref.rotate(q, table, positions, interleaved)
    assert bool(((q_out.cpu().to(torch.float64) - want_q).abs() <= want_q.abs() * ref.HALF_STEP + 2.0 ** -20 * q.abs().amax() + ref.TINY).all())
    _check_rows(k_back, ref.rotate(k, table, positions, interleaved))
    _check_rows(v_back, v.to(torch.float64))
    # the values are not rotated: their codes and parameters are known to the bit (codes away from a tie)
    codes, params = ref.unpack(cache.pages.cpu(), d)
    at = (1, slots.long() // page, slice(None), slots.long() % page)
    scale, low, exact = ref.quantise(v.to(torch.float64))
    assert torch.equal(params[at].to(torch.float64), torch.cat([scale, low], -1))
    clear = (exact - exact.floor() - 0.5).abs() > 1e-5
    assert bool((codes[at].to(torch.float64) == exact.round())[clear].all())
    # what is read is what is stored
    stored = ref.stored_rows(cache.pages.cpu(), d, slots.long(), page)
    assert torch.equal(k_back.cpu(), stored[0].float().half()) and torch.equal(v_back.cpu(), stored[1].float().half())
    # nothing else was written
    touched = torch.zeros(pages * page, dtype=torch.bool)
    touched[slots.long()] = True
    left = params.permute(1, 3, 0, 2, 4).reshape(pages * page, -1)[~touched]
    assert bool((left == 0).all()) and bool((codes.permute(1, 3, 0, 2, 4).reshape(pages * page, -1)[~touched] == 0).all())
    assert torch.equal(buf.cpu(), qkv)
    # the queries in place give the same
    cache.append(kd, vd, slots.to(dev), table.to(dev), positions.to(dev), qd, None, interleaved)
    assert torch.equal(qd, q_out)


def test_append_without_rotation_and_extremes(dev):
    """Keys as they are; constant rows, zero rows, the largest values, rows that are not finite."""
    d, page = 128, 16
    cache = KVCacheInt4(2, 1, d, page)
    k = torch.zeros(8, 1, d, dtype=torch.half)
    k[1] = 3.25
    k[2] = -0.0
    k[3] = 65504.0
    k[4, 0, ::2], k[4, 0, 1::2] = -65504.0, 65504.0
    k[5, 0, 3] = float("inf")
    k[6, 0, 3] = float("nan")
    k[7] = torch.arange(d) * 2.0 ** -24
    slots = torch.arange(8)
    cache.append(k.to(dev), k.flip(0).contiguous().to(dev), slots.to(dev))
    kb, vb = (t.cpu() for t in cache.read(slots.to(dev)))
    cache.check()
    assert torch.equal(kb, vb.flip(0)) or bool(torch.isnan(kb[5:7]).all())
    for i in range(4):
        assert torch.equal(kb[i].float(), k[i].float())
    assert float((kb[4].double() - k[4].double()).abs().max()) <= 65504 * 2.0 ** -10
    assert bool(torch.isnan(kb[5]).all()) and bool(torch.isnan(kb[6]).all())
    _check_rows(kb[7:], k[7:].double())


def test_append_leaves_out_padding_and_bad_indices(dev):
    d, page, T = 64, 16, 6
    cache = KVCacheInt4(2, 2, d, page)
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(T, 2, d, generator=g).half().to(dev) for _ in range(2))
    q = torch.randn(T, 4, d, generator=g).half().to(dev)
    q_out = torch.full_like(q, 7.0)
    table = rotation_table(100, d)
    cache.append(k, v, torch.tensor([0, -1, 5, -7, 31, 8], device=dev), table, torch.tensor([0, 1, 2, 999, 99, 3], device=dev), q, q_out)
    cache.check()  # padding is no error, whatever its position
    assert bool((q_out[[1, 3]] == 7).all()) and not bool((q_out[[0, 2, 4, 5]] == 7).all(-1).any())
    before = cache.pages.clone()
    for slots, positions in (([32, -1, -1, -1, -1, -1], [0] * 6), ([1, -1, -1, -1, -1, -1], [100] + [0] * 5), ([1, -1, -1, -1, -1, -1], [-1] + [0] * 5),
                             ([2 ** 40, -1, -1, -1, -1, -1], [0] * 6)):
        q_out.fill_(7.0)
        cache.append(k, v, torch.tensor(slots, device=dev), table, torch.tensor(positions, device=dev), q, q_out)
        assert torch.equal(cache.pages, before) and bool((q_out == 7).all())
        with pytest.raises(RuntimeError, match="out of range"):
            cache.check()
        cache.check()
    kb, vb = torch.full((3, 2, d), 9.0, dtype=torch.half, device=dev), torch.full((3, 2, d), 9.0, dtype=torch.half, device=dev)
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    fg.kv_read_int4(cache.pages, torch.tensor([-1, 5, 32], device=dev), kb, vb, page, status)
    assert bool((kb[[0, 2]] == 9).all()) and not bool((kb[1] == 9).any()) and int(status) == capi.FG_ERR_INDEX


# ---- attention -------------------------------------------------------------------------------
def _table(g, lens, page, pages, extra=2):
    width = max(1, max(-(-n // page) for n in lens)) + extra
    order = torch.randperm(pages, generator=g)
    table = torch.full((len(lens), width), -5, dtype=torch.int32)  # entries past a sequence's end are never looked at
    at = 0
    for b, n in enumerate(lens):
        need = -(-n // page)
        table[b, :need] = order[at:at + need].int()
        at += need
    return table


def _case(lens, news, hq, hkv, d, page, seed, spread=1.0, offset=0.0):
    g = torch.Generator().manual_seed(seed)
    pages = sum(-(-n // page) for n in lens) + 1
    pool = ref.random_pages(g, pages, hkv, d, page, spread, offset)
    table = _table(g, lens, page, pages)
    starts = None if news is None else [0]
    for n in news or []:
        starts.append(starts[-1] + n)
    tokens = len(lens) if news is None else starts[-1]
    q = torch.randn(tokens, hq, d, generator=g).half()
    return pool, table, q, starts


def _attend(pool, table, q, lens, page, starts, dev, scale=None, out=None, status=None):
    out = torch.full(q.shape, float("nan"), dtype=torch.half, device=dev) if out is None else out
    fg.kv_attention_int4(q.to(dev), pool.to(dev), table.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev), out, page,
                         None if starts is None else torch.tensor(starts, dtype=torch.int32, device=dev), scale, status)
    return out


def _check_attention(out, pool, table, q, lens, page, starts, scale=None):
    want, span, top = ref.attention(q, pool, table, lens, page, starts, scale)
    err = (out.cpu().to(torch.float64) - want).abs()
    tol = ref.attention_tolerance(want, span, top)
    assert bool((err <= tol).all()), float((err / tol).max())


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hq,hkv", [(1, 1), (6, 2), (8, 1), (14, 2), (16, 1), (17, 1), (40, 1)])
def test_heads(hq, hkv, d, dev):
    """Groups below, at and above the eight and sixteen columns of a tile."""
    lens = [1, 37, 300]
    pool, table, q, starts = _case(lens, None, hq, hkv, d, 32, hq + d)
    _check_attention(_attend(pool, table, q, lens, 32, starts, dev), pool, table, q, lens, 32, starts)


@pytest.mark.parametrize("page", [16, 32, 48, 128])
@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 31, 63, 64, 65, 255, 257, 1000, 2500])
def test_lengths(n, page, dev):
    """One sequence: lengths around a block, a unit, a page, a share of several CTAs, a set of 32 pages."""
    pool, table, q, starts = _case([n], None, 4, 2, 128, page, n)
    _check_attention(_attend(pool, table, q, [n], page, starts, dev), pool, table, q, [n], page, starts)


def test_ragged_batch_with_empty_sequences(dev):
    lens = [0, 700, 1, 0, 64, 129, 2000, 3, 16, 0]
    pool, table, q, starts = _case(lens, None, 8, 2, 64, 16, 5)
    out = _attend(pool, table, q, lens, 16, starts, dev)
    _check_attention(out, pool, table, q, lens, 16, starts)
    assert bool((out[[0, 3, 9]] == 0).all())


@pytest.mark.parametrize("d,hq,hkv", [(128, 4, 1), (64, 16, 2), (128, 9, 3)])
def test_several_new_tokens(d, hq, hkv, dev):
    """Each of a sequence's new tokens sees one row more; more new tokens than rows, no new token, and rows behind the last
    sequence, which stay as they were."""
    lens, news = [50, 3, 400, 0, 17, 1000], [5, 3, 17, 2, 0, 33]
    pool, table, q, starts = _case(lens, news, hq, hkv, d, 16, 7)
    lens[1] = 2  # three new tokens, two rows: the first sees nothing
    q = torch.cat([q, q[:4]])
    out = _attend(pool, table, q, lens, 16, starts, dev)
    assert bool(torch.isnan(out[-4:]).all())
    assert bool((out[starts[1]] == 0).all()) and bool((out[starts[3]:starts[4]] == 0).all())
    _check_attention(out[:-4], pool, table, q[:-4], lens, 16, starts)


@pytest.mark.parametrize("spread,offset", [(1e-3, 0.0), (1.0, 8.0), (30.0, 0.0), (1.0, -200.0)])
def test_ranges_of_keys_and_values(spread, offset, dev):
    """Small, shifted and large values; scores up to several hundred, so that one row takes nearly all the weight."""
    lens = [500, 90]
    pool, table, q, starts = _case(lens, None, 4, 1, 128, 16, 13, spread, offset)
    scale = 0.02 if offset else None
    _check_attention(_attend(pool, table, q, lens, 16, starts, dev, scale), pool, table, q, lens, 16, starts, scale)


@pytest.mark.parametrize("d", [64, 128])
def test_long_sums_keep_their_precision(d, dev):
    """Averages of thousands of values are small beside them: what sums of one sign lose on the way shows here.  Rounded once,
    exact outputs are at most half a step off each, in the mean 0.4 of that; so half a step bounds the error of all of them
    (weights of eleven bits alone make it 2^-11 * 2.7 / 2.4, sums that are cut off at every product 2^-11 * 3.3 / 2.4)."""
    n, page = 8000, 16
    pool, table, q, _ = _case([n], None, 8, 8, d, page, 71)
    lens = [n] * 40
    table, q = table.repeat(40, 1), torch.randn(40, 8, d, generator=torch.Generator().manual_seed(72)).half()
    out = _attend(pool, table, q, lens, page, None, dev).cpu().to(torch.float64)
    want, _, _ = ref.attention(q, pool, table, lens, page)
    assert float((out - want).norm()) <= 2.0 ** -11 * float(want.norm())


def test_constant_values_and_rising_scores(dev):
    """Rows whose values are all alike (the smallest scale) beside ordinary ones, and scores that rise along the sequence, so
    that the running maximum moves again and again."""
    d, page, n = 128, 16, 640
    cache = KVCacheInt4(n // page, 1, d, page)
    g = torch.Generator().manual_seed(3)
    q = torch.randn(1, 1, d, generator=g).half()
    k = (q[0, 0].double() * torch.linspace(-4, 4, n)[:, None]).half()[:, None]
    v = torch.randn(n, 1, d, generator=g).half()
    v[::3] = 5.0
    v[600:] = -7.0
    cache.append(k.to(dev), v.to(dev), torch.arange(n, device=dev))
    table = torch.arange(n // page, dtype=torch.int32)[None]
    out = torch.empty(1, 1, d, dtype=torch.half, device=dev)
    for length in (n, 601, 599, 4):
        cache.attend(q.to(dev), table.to(dev), torch.tensor([length], dtype=torch.int32, device=dev), out)
        _check_attention(out, cache.pages.cpu(), table, q, [length], page, None)


def test_masked_rows_may_hold_anything(dev):
    """Infinities and NaNs in rows behind the end of a sequence, and in rows that a new token does not see yet."""
    lens, news = [21, 40], [4, 1]
    pool, table, q, starts = _case(lens, news, 4, 1, 64, 16, 17)
    bad = pool.clone()
    for b, n in enumerate(lens):
        for r in range(n, -(-n // 16) * 16):
            page, row = int(table[b, r // 16]), r % 16
            for which in (0, 1):
                at = 16 * 64 + (which * 16 + row) * 4
                bad[page, 0, at:at + 4] = torch.tensor([0x00, 0x7E, 0x00, 0xFC], dtype=torch.uint8)  # (NaN, -inf)
    clean, dirty = (_attend(p, table, q, lens, 16, starts, dev) for p in (pool, bad))
    assert torch.equal(clean, dirty)
    last = (int(table[0, 20 // 16]), 20 % 16)  # row 20 is seen by the last new token of sequence 0 alone
    bad[last[0], 0, 16 * 64 + (16 + last[1]) * 4:][:4] = torch.tensor([0x00, 0x7E, 0x00, 0x7C], dtype=torch.uint8)
    dirty = _attend(bad, table, q, lens, 16, starts, dev)
    assert torch.equal(dirty[:3], clean[:3]) and torch.equal(dirty[4:], clean[4:]) and bool(torch.isnan(dirty[3]).any())


def test_bad_indices_are_reported(dev):
    lens, page = [100, 40], 16
    pool, table, q, starts = _case(lens, None, 2, 1, 64, page, 19)
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    good = _attend(pool, table, q, lens, page, None, dev, status=status)
    assert int(status) == 0
    for bad_page in (pool.shape[0], -1, 2 ** 31 - 1):
        t = table.clone()
        t[0, 2] = bad_page  # rows 32..47 of sequence 0 count as absent
        status.zero_()
        out = _attend(pool, t, q, lens, page, None, dev, status=status)
        assert int(status) == capi.FG_ERR_INDEX and torch.equal(out[1], good[1])
        keep = [i for i in range(7) if i != 2]
        _check_attention(out[:1], pool, [[int(table[0, i]) for i in keep]], q[:1], [100 - 16], page, None)
    status.zero_()
    out = _attend(pool, table, q, [100, table.shape[1] * page + 1], page, None, dev, status=status)
    assert int(status) == capi.FG_ERR_INDEX and bool((out[1] == 0).all()) and torch.equal(out[0], good[0])
    status.zero_()
    out = _attend(pool, table, q, [100, -3], page, None, dev, status=status)
    assert int(status) == capi.FG_ERR_INDEX and bool((out[1] == 0).all()) and torch.equal(out[0], good[0])
    for bad_starts in ([0, 1, 3], [0, 1, 0], [-1, 1, 2]):
        status.zero_()
        out = _attend(pool, table, q, lens, page, bad_starts, dev, status=status)
        assert int(status) == capi.FG_ERR_INDEX
    pool_out = _attend(pool, table, q, lens, page, None, dev)
    assert torch.equal(pool_out, good)


def test_overlapping_query_ranges_are_refused_before_they_overflow(dev):
    """q_starts that go back and forth give every other sequence all of q: more work units than 32 bits count."""
    tokens, batch, page = 16384, 64, 128
    q = torch.zeros(tokens, 64, 64, dtype=torch.half, device=dev)
    out = torch.full_like(q, 3.0)
    pool = torch.zeros(2, 8, page * 72, dtype=torch.uint8, device=dev)
    table = torch.zeros(1, 2048, dtype=torch.int32, device=dev).expand(batch, -1).contiguous()
    lens = torch.full((batch,), 2048 * page, dtype=torch.int32, device=dev)
    starts = torch.tensor([0, tokens] * (batch // 2) + [0], dtype=torch.int32, device=dev)
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    fg.kv_attention_int4(q, pool, table, lens, out, page, starts, None, status)
    assert int(status) == capi.FG_ERR_INDEX and bool((out == 3.0).all())


def test_rows_read_back_may_be_the_weight_of_the_next_call(dev):
    """A linear asks for its weight while the kernel before it still runs; rows that kv_read_int4 has just written are whole."""
    n, d, page = 4096, 128, 64
    pool = ref.random_pages(torch.Generator().manual_seed(3), n // page, 1, d, page).to(dev)
    slots = torch.arange(n, device=dev)
    x = torch.randn(16, d, generator=torch.Generator().manual_seed(4)).half().to(dev)
    k, v = (torch.empty(n, 1, d, dtype=torch.half, device=dev) for _ in range(2))
    c = torch.empty(16, n, dtype=torch.half, device=dev)
    fg.kv_read_int4(pool, slots, k, v, page)
    torch.cuda.synchronize()
    fg.edgemm_m8n128k64x4_bt(x, k.view(n, d), c)
    want = c.clone()
    torch.cuda.synchronize()
    for _ in range(50):
        k.zero_()
        fg.kv_read_int4(pool, slots, k, v, page)
        fg.edgemm_m8n128k64x4_bt(x, k.view(n, d), c)
        assert torch.equal(c, want)


def test_strides_and_scale(dev):
    """Queries out of a fused projection, output into a wider buffer, a table with a row stride."""
    lens, page = [70, 33, 90], 16
    pool, table, q, _ = _case(lens, None, 4, 2, 64, page, 23)
    wide = torch.full((3, 500 * 2 + 24), float("nan"), dtype=torch.half, device=dev)
    wide[:, 8:8 + 256] = q.flatten(1).to(dev)
    out = torch.full((3, 520), 3.0, dtype=torch.half, device=dev)
    big = torch.full((3, 40), -1, dtype=torch.int32, device=dev)
    big[:, :table.shape[1]] = table.to(dev)
    fg.kv_attention_int4(wide[:, 8:264].unflatten(1, (4, 64)), pool.to(dev), big[:, :table.shape[1]], torch.tensor(lens, dtype=torch.int32, device=dev),
                         out[:, 8:264].unflatten(1, (4, 64)), page, scale=0.3)
    _check_attention(out[:, 8:264].unflatten(1, (4, 64)), pool, table, q, lens, page, None, 0.3)
    assert bool((out[:, :8] == 3).all()) and bool((out[:, 264:] == 3).all())


def test_far_into_a_large_pool(dev):
    """Offsets past 2^32 bytes: the last pages of a 5 GB pool."""
    d, page, hkv = 128, 64, 8
    pages = 5 * 2 ** 30 // (hkv * page * (d + 8)) + 1
    cache = KVCacheInt4(pages, hkv, d, page)
    g = torch.Generator().manual_seed(29)
    n = 100
    table = torch.tensor([[pages - 1, pages - 2]], dtype=torch.int32)
    slots = cache.slots(table.to(dev), torch.zeros(n, dtype=torch.int64, device=dev), torch.arange(n, device=dev))
    k, v = (torch.randn(n, hkv, d, generator=g).half() for _ in range(2))
    cache.append(k.to(dev), v.to(dev), slots)
    kb, vb = cache.read(slots)
    _check_rows(kb, k.double())
    _check_rows(vb, v.double())
    q = torch.randn(1, 8, d, generator=g).half()
    out = torch.empty(1, 8, d, dtype=torch.half, device=dev)
    cache.attend(q.to(dev), table.to(dev), torch.tensor([n], dtype=torch.int32, device=dev), out)
    cache.check()
    near = cache.pages[pages - 2:].cpu().flip(0)
    _check_attention(out, near, [[0, 1]], q, [n], page, None)
    assert int(cache.pages[: pages - 2].max()) == 0


def test_reproducible_streams_and_graphs(dev):
    """The same bits twice, on another stream, and from two graphs of one stream that are replayed side by side; a graph
    follows the lengths in its tensors."""
    lens, page = [3000, 17, 900, 0], 32
    pool, table, q, _ = _case(lens, None, 16, 2, 128, page, 31)
    pd, td, qd = pool.to(dev), table.to(dev), q.to(dev)
    ld = torch.tensor(lens, dtype=torch.int32, device=dev)
    run = lambda out: fg.kv_attention_int4(qd, pd, td, ld, out, page)
    first = torch.empty_like(qd)
    run(first)
    side = torch.cuda.Stream()
    outs = [torch.empty_like(qd) for _ in range(3)]
    side.wait_stream(torch.cuda.current_stream())
    run(outs[0])
    with torch.cuda.stream(side):
        run(outs[1])
    torch.cuda.synchronize()
    assert torch.equal(outs[0], first) and torch.equal(outs[1], first)
    graphs = []
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            for _ in range(3):
                run(outs[i])
        graphs.append(graph)
    s = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        for out in outs:
            out.zero_()
        torch.cuda.synchronize()
        for i in range(2):
            with torch.cuda.stream(s[i]):
                graphs[i].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], first) and torch.equal(outs[1], first)
    ld.copy_(torch.tensor([100, 18, 901, 5], dtype=torch.int32))
    graphs[0].replay()
    torch.cuda.synchronize()
    t = table.clone()
    t[3, 0] = pool.shape[0] - 1
    td.copy_(t)
    graphs[0].replay()
    torch.cuda.synchronize()
    _check_attention(outs[0], pool, t, q, [100, 18, 901, 5], page, None)


def test_refusals(dev):
    cache = KVCacheInt4(4, 2, 64, 16)
    q = torch.zeros(2, 4, 64, dtype=torch.half, device=dev)
    out, table = torch.empty_like(q), torch.zeros(2, 2, dtype=torch.int32, device=dev)
    lens = torch.ones(2, dtype=torch.int32, device=dev)
    k = torch.zeros(2, 2, 64, dtype=torch.half, device=dev)
    slots = torch.arange(2, device=dev)
    cs, pos = rotation_table(8, 64), torch.zeros(2, dtype=torch.int64, device=dev)
    cache.attend(q, table, lens, out)
    cache.append(k, k, slots, cs, pos, q)
    for bad in (lambda: cache.attend(q, table, lens, q),
                lambda: cache.attend(q, table, lens[:1], out),
                lambda: cache.attend(q[:1], table, lens, out[:1]),
                lambda: cache.attend(q[:, :3].contiguous(), table, lens, out[:, :3].contiguous()),
                lambda: cache.attend(q, table, lens, out, scale=0.0),
                lambda: cache.attend(q, table, lens, out, scale=float("nan")),
                lambda: cache.attend(q, table, lens, out, q_starts=torch.zeros(2, dtype=torch.int32, device=dev)),
                lambda: fg.kv_attention_int4(q, cache.pages, table, lens, out, 32),
                lambda: cache.append(k, k[:1], slots),
                lambda: cache.append(k, k, slots[:1]),
                lambda: cache.append(k, k, slots, cs),
                lambda: cache.append(k, k, slots, q=q),
                lambda: cache.append(k, k, slots, cs, pos, q_out=q),
                lambda: cache.append(k, k, slots, cs[:, :32].contiguous(), pos),
                lambda: cache.append(k[:, :, :32].contiguous(), k[:, :, :32].contiguous(), slots),
                lambda: cache.append(k[:, :1], k[:, :1], slots),
                lambda: cache.append(torch.zeros(2, 64, 2, dtype=torch.half, device=dev).transpose(1, 2), k, slots),
                lambda: fg.kv_read_int4(cache.pages, slots, k, k, 16),
                lambda: KVCacheInt4(4, 2, 96),
                lambda: KVCacheInt4(4, 2, 64, 24)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: cache.attend(q.float(), table, lens, out),
                lambda: cache.attend(q, table.long(), lens, out),
                lambda: cache.attend(q, table, lens.long(), out),
                lambda: cache.append(k, k, slots.float()),
                lambda: cache.append(k.cpu(), k, slots)):
        with pytest.raises(RuntimeError):
            bad()
    empty = torch.zeros(0, 2, 64, dtype=torch.half, device=dev)
    cache.append(empty, empty, slots[:0])
    L, vp = capi.lib, ctypes.c_void_p
    ws = torch.empty(capi.lib.fg_kv_attention_workspace_bytes(), dtype=torch.uint8, device=dev)
    call = lambda **kw: L.fg_kv_attention_int4(q.data_ptr(), kw.get("ldq", 256), out.data_ptr(), 256, 2, 4, 2, kw.get("d", 64), cache.pages.data_ptr(), 4,
                                               kw.get("page", 16), table.data_ptr(), 2, 2, lens.data_ptr(), None, kw.get("batch", 2), kw.get("scale", 1.0),
                                               None, kw.get("ws", ws.data_ptr()), ws.numel(), vp(0))
    assert call(ldq=100) == call(d=96) == call(page=8) == call(batch=3) == call(scale=-1.0) == capi.FG_ERR_SHAPE
    assert call(ws=None) == call(ws=ws.data_ptr() + 16) == capi.FG_ERR_WORKSPACE


def test_joins_read_the_partials_of_their_own_call(dev):
    """Items of several CTAs, call after call on one stream and over other rows each time: whoever joins an item adds up the partial sums
    that its partners have just left in the workspace, not those of the call before."""
    page, d = 64, 128
    lens = [5000, 1800, 300]
    cases = []
    for seed in range(4):
        pool, table, q, _ = _case(lens, None, 8, 2, d, page, 100 + seed)
        cases.append((pool, table, q, [t.to(dev) for t in (pool, table, q)]))
    ld = torch.tensor(lens, dtype=torch.int32, device=dev)
    want = []
    for pool, table, q, (pd, td, qd) in cases:
        out = torch.empty_like(qd)
        fg.kv_attention_int4(qd, pd, td, ld, out, page)
        torch.cuda.synchronize()
        _check_attention(out, pool, table, q, lens, page, None)
        want.append(out)
    got = [torch.empty_like(want[0]) for _ in range(400)]
    for i, out in enumerate(got):
        _, _, _, (pd, td, qd) = cases[i % 4]
        fg.kv_attention_int4(qd, pd, td, ld, out, page)
    torch.cuda.synchronize()
    assert all(torch.equal(out, want[i % 4]) for i, out in enumerate(got))


def test_outputs_over_other_operands_are_refused(dev):
    """What a call writes may not lie over what it reads (nothing is launched); q_out may be q itself."""
    T, hq, hkv, d, page = 6, 4, 2, 64, 16
    n = T * hq * d
    g = torch.Generator().manual_seed(41)
    half = lambda *s: torch.randn(*s, generator=g).half().to(dev)
    big = half(4 * n)  # k at 0, v behind it, q at 2 n, room behind
    k, v, q = big[: T * hkv * d].view(T, hkv, d), big[T * hkv * d: n].view(T, hkv, d), big[2 * n: 3 * n].view(T, hq, d)
    over = lambda at: big[at: at + n].view(T, hq, d)
    bytes_ = torch.zeros(1 << 16, dtype=torch.uint8, device=dev)  # pages, and what is put over them
    pages = bytes_[: 2 * hkv * page * (d + 8)].view(2, hkv, page * (d + 8))
    in_pages = bytes_[512: 512 + 2 * n].view(torch.half).view(T, hq, d)
    slots, pos = torch.arange(T, device=dev), torch.arange(T, device=dev)
    table = rotation_table(8, d)
    ints = torch.arange(4 * n, device=dev)  # indices, and outputs over them
    in_ints = ints[:n // 4].view(torch.half).view(T, hq, d)
    in_table = rotation_table(1024, d)
    append = lambda q_out, k=k, q=q, slots=slots, cs=table, pos=pos, p=pages: fg.kv_append_int4(k, v, p, slots, page, cs, pos, q, q_out)
    before = big.clone()
    for bad in (lambda: append(over(0)), lambda: append(over(T * hkv * d)), lambda: append(over(2 * n - 8)), lambda: append(over(2 * n + 64)),
                lambda: append(in_pages), lambda: append(in_ints, slots=ints[:T]), lambda: append(in_ints, pos=ints[2:2 + T]),
                lambda: append(in_table.view(torch.half).flatten()[:n].view(T, hq, d), cs=in_table),
                lambda: append(None, q=in_pages), lambda: append(None, k=in_pages[:, :hkv].contiguous().copy_(0), q=in_pages),
                lambda: fg.kv_append_int4(bytes_[:2 * T * hkv * d].view(torch.half).view(T, hkv, d), v, pages, slots, page),
                lambda: fg.kv_append_int4(k, bytes_[:2 * T * hkv * d].view(torch.half).view(T, hkv, d), pages, slots, page),
                lambda: fg.kv_append_int4(k, v, pages, bytes_[:8 * T].view(torch.int64), page)):
        with pytest.raises(ValueError, match="overlap"):
            bad()
    assert torch.equal(big, before) and int(pages.max()) == 0
    block_table, lens, starts = torch.zeros(T, 1, dtype=torch.int32, device=dev), torch.ones(T, dtype=torch.int32, device=dev), torch.arange(T + 1, dtype=torch.int32, device=dev)
    i32 = torch.zeros(n, dtype=torch.int32, device=dev)
    in_i32 = i32[: n // 2].view(torch.half).view(T, hq, d)
    attend = lambda out, q=q, t=block_table, l=lens, s=starts: fg.kv_attention_int4(q, pages, t, l, out, page, s)
    for bad in (lambda: attend(q), lambda: attend(over(2 * n + 64)), lambda: attend(in_pages), lambda: attend(in_i32, t=i32[:T].view(T, 1)),
                lambda: attend(in_i32, l=i32[16:16 + T]), lambda: attend(in_i32, s=i32[8:9 + T])):
        with pytest.raises(ValueError, match="overlap"):
            bad()
    room = torch.empty(2 * T * hkv * d, dtype=torch.half, device=dev)
    with pytest.raises(ValueError, match="overlap"):
        fg.kv_read_int4(pages, room[: 4 * T].view(torch.int64), room[: T * hkv * d].view(T, hkv, d), room[T * hkv * d:].view(T, hkv, d), page)


def test_column_ranges_of_one_buffer_do_not_overlap(dev):
    """q, k, v, the turned queries and the attention's output side by side in one buffer of rows."""
    T, hq, hkv, d, page = 5, 4, 1, 64, 16
    g = torch.Generator().manual_seed(43)
    wide = torch.randn(T, (3 * hq + 2 * hkv) * d, generator=g).half()
    ranges = [hq * d, hkv * d, hkv * d, hq * d, hq * d]
    buf = wide.to(dev)
    q, k, v, q_out, out = (t.unflatten(1, (-1, d)) for t in buf.split(ranges, 1))
    cache, table, pos = KVCacheInt4(1, hkv, d, page), rotation_table(16, d), torch.arange(T, device=dev)
    cache.append(k, v, pos, table, pos, q, q_out)
    starts = torch.tensor([0, T], dtype=torch.int32, device=dev)
    block_table, lens = torch.zeros(1, 1, dtype=torch.int32, device=dev), torch.tensor([T], dtype=torch.int32, device=dev)
    cache.attend(q_out, block_table, lens, out, q_starts=starts)
    want_q = ref.rotate(wide[:, : hq * d].unflatten(1, (-1, d)), table.cpu(), pos.cpu(), False)
    assert bool(((q_out.cpu().double() - want_q).abs() <= want_q.abs() * ref.HALF_STEP + 2.0 ** -18).all())
    _check_attention(out, cache.pages.cpu(), [[0]], q_out.cpu(), [T], page, [0, T])
    assert torch.equal(buf.cpu()[:, : sum(ranges[:3])], wide[:, : sum(ranges[:3])])
    one = buf[:1]  # a single row
    q, k, v, q_out, out = (t.unflatten(1, (-1, d)) for t in one.split(ranges, 1))
    cache.append(k, v, pos[:1], table, pos[:1], q, q_out)
    cache.attend(q_out, block_table, lens[:1], out)
    # ranges that share a column do
    with pytest.raises(ValueError, match="overlap"):
        cache.append(k, v, pos[:1], table, pos[:1], q, one[:, 8: 8 + hq * d].unflatten(1, (-1, d)))
    with pytest.raises(ValueError, match="overlap"):
        cache.attend(buf[:, :hq * d].unflatten(1, (-1, d)), block_table, lens, buf[:, hq * d - 8: 2 * hq * d - 8].unflatten(1, (-1, d)), q_starts=starts)


def test_check_waits_for_every_stream(dev):
    """A bad index that a call on another stream meets later than the check is asked for."""
    cache = KVCacheInt4(2, 1, 64, 16)
    k, slots = torch.zeros(3, 1, 64, dtype=torch.half, device=dev), torch.tensor([0, 32, 1], device=dev)
    cache.append(k, k, slots.clamp(max=2))
    cache.check()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)  # about a tenth of a second
        cache.append(k, k, slots)
    with pytest.raises(RuntimeError, match="out of range"):
        cache.check()
    cache.check()


def test_extreme_rows_as_keys_and_as_values(dev):
    """Constant rows, zero rows, the largest values, the smallest, rows that are not finite: each row reads back alike whether it was
    stored as a key or as a value, whatever lies beside it."""
    d, page = 128, 16
    k = torch.zeros(8, 1, d, dtype=torch.half)
    k[1], k[2], k[3] = 3.25, -0.0, 65504.0
    k[4, 0, ::2], k[4, 0, 1::2] = -65504.0, 65504.0
    k[5, 0, 3], k[6, 0, 3] = float("inf"), float("nan")
    k[7] = torch.arange(d) * 2.0 ** -24
    cache, slots = KVCacheInt4(2, 1, d, page), torch.arange(8, device=dev)
    cache.append(k.to(dev), k.flip(0).contiguous().to(dev), slots)
    kb, vb = (t.cpu() for t in cache.read(slots))
    cache.check()
    vb = vb.flip(0)
    finite = [0, 1, 2, 3, 4, 7]
    assert torch.equal(kb[finite], vb[finite]) and bool(torch.isfinite(vb[finite]).all())
    assert bool(torch.isnan(kb[5:7]).all()) and bool(torch.isnan(vb[5:7]).all())
    assert torch.equal(vb[:4].float(), k[:4].float())
    assert float((vb[4].double() - k[4].double()).abs().max()) <= 65504 * 2.0 ** -10
    _check_rows(vb[7:], k[7:].double())


def _check_attention_error(out, pool, table, q, lens, page, starts):
    want, span, top = ref.attention(q, pool, table, lens, page, starts)
    err, tol = (out.cpu().to(torch.float64) - want).abs(), ref.attention_error(want, span, top)
    assert bool((err <= tol).all()), float((err / tol).max())


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hq,hkv", [(2, 2), (8, 1), (16, 1), (24, 2), (40, 1)])
def test_output_error_is_its_own_rounding(hq, hkv, d, dev):
    """Every column of the tiles of eight and of sixteen, one token and several, in items of one CTA and of many."""
    lens = [1, 40, 700, 2500]
    pool, table, q, starts = _case(lens, None, hq, hkv, d, 32, hq + d)
    _check_attention_error(_attend(pool, table, q, lens, 32, starts, dev), pool, table, q, lens, 32, starts)
    lens, news = [300, 5, 1200], [3, 5, 2]
    pool, table, q, starts = _case(lens, news, hq, hkv, d, 16, hq + d + 1)
    _check_attention_error(_attend(pool, table, q, lens, 16, starts, dev), pool, table, q, lens, 16, starts)


@pytest.mark.parametrize("d,hq", [(64, 8), (64, 16), (128, 8), (64, 13)])
def test_long_sums_of_shared_heads_keep_their_precision(d, hq, dev):
    """As for one query head per key/value head, with all columns of a tile in use: averages of thousands of values, whose errors
    together stay below half a step (what is exact but for the last rounding has 0.4 of it)."""
    n, page, batch = 8000, 16, 20
    pool, table, _, _ = _case([n], None, hq, 1, d, page, 73)
    lens = [n] * batch
    table, q = table.repeat(batch, 1), torch.randn(batch, hq, d, generator=torch.Generator().manual_seed(74)).half()
    out = _attend(pool, table, q, lens, page, None, dev).cpu().to(torch.float64)
    want, _, _ = ref.attention(q, pool, table, lens, page)
    assert float((out - want).norm()) <= 2.0 ** -11 * float(want.norm())


def test_graph_destroyed_while_it_runs(dev):
    """The workspace of a graph goes to the next capture only when nothing uses it any more."""
    page, lens = 64, [5000]
    pool, table, q, _ = _case(lens, None, 8, 2, 128, page, 51)
    pd, td, qd, ld = pool.to(dev), table.to(dev), q.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev)
    want = torch.empty_like(qd)
    fg.kv_attention_int4(qd, pd, td, ld, want, page)

    def capture(outs):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.stream(torch.cuda.Stream()):
            graph.capture_begin(capture_error_mode="relaxed")
            for out in outs:
                fg.kv_attention_int4(qd, pd, td, ld, out, page)
            graph.capture_end()
        return graph

    first, later = (torch.zeros(n, *q.shape, dtype=torch.half, device=dev) for n in (1000, 20))
    graph = capture(first)
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        graph.replay()
    del graph  # a thousand calls are still to run
    graphs = [capture(later) for _ in range(4)]
    for g in graphs:
        with torch.cuda.stream(torch.cuda.Stream()):
            g.replay()
    torch.cuda.synchronize()
    assert bool((first == want).all()) and bool((later == want).all())


@pytest.mark.parametrize("d,hq,hkv", [(128, 8, 2), (64, 12, 1)])
def test_prompt(d, hq, hkv, dev):
    """A sequence's first chunk, and a later one behind rows that are there already."""
    for rows, new in ((600, 600), (900, 333)):
        pool, table, q, starts = _case([rows], [new], hq, hkv, d, 32, rows + d)
        _check_attention_error(_attend(pool, table, q, [rows], 32, starts, dev), pool, table, q, [rows], 32, starts)


def test_keys_turned_out_of_range(dev):
    """A pair of the largest values turned by an eighth: above fp16's range the row saturates, below it the row has an infinity and
    reads back as NaN, as its fp16 low end says; its neighbours do not notice."""
    d, page = 64, 16
    cache = KVCacheInt4(1, 1, d, page)
    table = torch.zeros(2, d, device=dev)
    table[0, : d // 2] = 1.0
    table[1] = 0.5 ** 0.5
    k = torch.randn(4, 1, d, generator=torch.Generator().manual_seed(1)).half()
    k[1, 0, 0], k[1, 0, d // 2] = 65504.0, 65504.0    # (0, 92636)
    k[2, 0, 0], k[2, 0, d // 2] = -65504.0, -65504.0  # (0, -92636)
    slots, pos = torch.arange(4, device=dev), torch.tensor([0, 1, 1, 0], device=dev)
    cache.append(k.to(dev), k.to(dev), slots, table, pos)
    kb, vb = cache.read(slots)
    cache.check()
    _check_rows(kb[[0, 3]], k[[0, 3]].double())
    assert float(kb[1, 0, d // 2]) == 65504.0 and bool(torch.isfinite(kb[1]).all())
    assert bool(torch.isnan(kb[2]).any()) and not bool(torch.isfinite(kb[2]).any())
    _check_rows(vb, k.double())
