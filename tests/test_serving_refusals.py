"""What the serving operators refuse before they touch a device, and the host side of the cache (no GPU needed)."""
import ctypes
import os
import re

import pytest
import torch

import fastgate_b200 as fg
from fastgate_b200 import capi
from fastgate_b200.kvcache import KVCacheInt4, rotation_table

L = capi.lib
_buf = (ctypes.c_char * 8192)()
P = (ctypes.addressof(_buf) + 255) // 256 * 256  # aligned host address, never dereferenced


def test_norm_arguments():
    call = lambda x=P, ldx=64, w=P, r=None, ro=None, out=P, i8=0, s=None, M=2, K=64, eps=1e-6: L.fg_add_rmsnorm(x, ldx, w, r, ro, 0, out, i8, s, M, K, eps, None)
    assert call(x=None) == call(w=None) == call(out=None) == call(i8=1) == call(r=P) == call(ro=P) == capi.FG_ERR_NULL
    assert call(M=0) == call(K=0) == call(K=60) == call(ldx=32) == call(ldx=68) == call(eps=-1.0) == call(eps=float("nan")) == capi.FG_ERR_SHAPE
    assert call(x=P + 2) == call(w=P + 8) == call(out=P + 8) == call(r=P + 4, ro=P) == call(i8=1, s=P + 2) == capi.FG_ERR_ALIGN


def test_linear_arguments():
    call = lambda x=P, w=P, s=P, c=P, M=1, N=128, K=128, res=None, act=0, st=None: L.fg_linear_w8a8(x, w, s, 1, None, c, M, N, K, None, res, act, st, None)
    assert call(x=None) == call(w=None) == call(s=None) == call(c=None) == capi.FG_ERR_NULL
    assert call(M=0) == call(N=100) == call(K=64) == call(K=131072) == capi.FG_ERR_SHAPE
    assert call(act=5) == call(act=-1) == capi.FG_ERR_PLAN
    assert call(x=P + 8) == call(c=P + 8) == call(res=P + 2) == call(s=P + 2) == call(st=P + 1) == capi.FG_ERR_ALIGN


def test_cache_arguments():
    app = lambda k=P, ldk=128, T=1, heads=2, d=64, pages=P, n=4, page=16, slots=P, cs=None, plen=0, pos=None, q=None, ldq=0, qo=None, ldqo=0, qh=0: \
        L.fg_kv_append_int4(k, ldk, P, 128, T, heads, d, pages, n, page, slots, 1, cs, plen, pos, 1, q, ldq, qo, ldqo, qh, 0, None, None)
    assert app(k=None) == app(pages=None) == app(slots=None) == app(cs=P) == app(pos=P) == app(q=P, qo=P, qh=1, ldq=64, ldqo=64) == capi.FG_ERR_NULL
    assert app(T=0) == app(heads=0) == app(d=96) == app(n=0) == app(page=8) == app(page=24) == app(ldk=64) == app(ldk=132) == capi.FG_ERR_SHAPE
    assert app(qh=3) == app(cs=P, pos=P) == app(cs=P, plen=4, pos=P, q=P, qo=P, qh=2, ldq=64, ldqo=128) == capi.FG_ERR_SHAPE
    assert app(k=P + 8) == app(pages=P + 8) == app(slots=P + 4) == app(cs=P + 4, plen=4, pos=P) == capi.FG_ERR_ALIGN
    read = lambda pages=P, T=1, k=P, d=64: L.fg_kv_read_int4(pages, 4, 16, 2, d, P, 1, T, k, P, None, None)
    assert read(pages=None) == read(k=None) == capi.FG_ERR_NULL
    assert read(T=0) == read(d=32) == capi.FG_ERR_SHAPE
    assert read(k=P + 8) == capi.FG_ERR_ALIGN
    wsb = L.fg_kv_attention_workspace_bytes()
    att = lambda q=P, ldq=256, T=2, hq=4, hkv=2, d=64, n=4, page=16, ldt=2, width=2, starts=None, batch=2, scale=1.0, ws=P, wsb=wsb: \
        L.fg_kv_attention_int4(q, ldq, P, 256, T, hq, hkv, d, P, n, page, P, ldt, width, P, starts, batch, scale, None, ws, wsb, None)
    assert att(q=None) == capi.FG_ERR_NULL
    assert att(ldq=200) == att(T=3) == att(hq=3) == att(d=80) == att(page=20) == att(ldt=1) == att(width=0) == att(batch=0) == capi.FG_ERR_SHAPE
    assert att(scale=0.0) == att(scale=float("inf")) == att(width=2 ** 28, ldt=2 ** 28) == capi.FG_ERR_SHAPE
    assert att(q=P + 8) == att(starts=P + 2) == capi.FG_ERR_ALIGN
    assert att(ws=None) == att(ws=P + 64) == att(wsb=wsb - 1) == L.fg_kv_attention_workspace_init(None, wsb, None) == capi.FG_ERR_WORKSPACE


def test_valid_arguments_stop_at_the_device():
    """Without a GPU a call that is in order ends with an error, not with a crash."""
    if torch.cuda.is_available():
        pytest.skip("a device is there: host addresses would be used")
    assert L.fg_add_rmsnorm(P, 64, P, None, None, 0, P, 0, None, 2, 64, 1e-6, None) == capi.FG_ERR_NO_DEVICE
    assert L.fg_linear_w8a8(P, P, P, 1, None, P, 1, 128, 128, None, None, 0, None, None) == capi.FG_ERR_NO_DEVICE
    assert L.fg_kv_read_int4(P, 4, 16, 2, 64, P, 1, 1, P, P, None, None) == capi.FG_ERR_NO_DEVICE


def test_prepack_of_int8_weights_checks_its_sizes():
    assert L.fg_prepack_gate_up_w8(None, P, P, 64, 128, None) == capi.FG_ERR_NULL
    assert L.fg_prepack_gate_up_w8(P, P, P, 65, 128, None) == L.fg_prepack_gate_up_w8(P, P, P, 64, 64, None) == capi.FG_ERR_SHAPE


def test_operators_refuse_cpu_tensors():
    h = torch.zeros(2, 64, dtype=torch.half)
    with pytest.raises(RuntimeError, match="no CPU path"):
        fg.add_rmsnorm(h, h[0], h.clone())
    i8 = torch.zeros(2, 128, dtype=torch.int8)
    with pytest.raises(RuntimeError, match="no CPU path"):
        fg.linear_int8(i8, i8, h, h[:, 0])
    cache = KVCacheInt4(2, 1, 64, 16, device="cpu")
    with pytest.raises(RuntimeError, match="no CPU path"):
        cache.append(h[:, None], h[:, None], torch.arange(2))
    with pytest.raises(RuntimeError, match="no CPU path"):
        cache.read(torch.arange(2))
    with pytest.raises(RuntimeError, match="no CPU path"):
        cache.attend(h[:, None], torch.zeros(2, 1, dtype=torch.int32), torch.ones(2, dtype=torch.int32), h[:, None].clone())


def test_cache_bookkeeping():
    cache = KVCacheInt4(6, 2, 128, 32, device="cpu")
    assert cache.pages.shape == (6, 2, 32 * 136) and cache.pages.dtype == torch.uint8
    table = torch.tensor([[4, 1], [0, 3]], dtype=torch.int32)
    got = cache.slots(table, torch.tensor([0, 0, 1, 1, 0]), torch.tensor([0, 33, 31, 32, -1]))
    assert got.tolist() == [4 * 32, 32 + 1, 31, 3 * 32, -1]
    for bad in (lambda: KVCacheInt4(2, 1, 100), lambda: KVCacheInt4(2, 1, 64, 8), lambda: KVCacheInt4(0, 1, 64), lambda: KVCacheInt4(2, 0, 64)):
        with pytest.raises(ValueError):
            bad()


def test_rotation_table_keeps_far_angles():
    t = rotation_table(200001, 64, device="cpu")
    assert t.shape == (200001, 64) and t.dtype == torch.float32
    a = 200000.0 * 10000.0 ** (-torch.arange(0, 64, 2, dtype=torch.float64) / 64)
    assert float((t[200000].double() - torch.cat([a.cos(), a.sin()])).abs().max()) <= 2.0 ** -24


def test_slots_of_rows_without_a_page():
    """No page in the table, no such column, no such sequence: the slot behind the pool, which the kernels report."""
    cache = KVCacheInt4(8, 2, 64, page_size=32, device="cpu")
    table = torch.tensor([[3, -1], [5, 1]], dtype=torch.int32)
    got = cache.slots(table, torch.tensor([0, 0, 1, 1, 2, -1, 1]), torch.tensor([0, 40, 63, 64, 0, 0, -5]))
    assert got.tolist() == [96, 256, 63, 256, 256, 256, -1]


def test_pages_that_no_operator_takes_are_refused_at_once():
    with pytest.raises(ValueError, match="at most"):
        KVCacheInt4(1, 1, 64, page_size=(1 << 20) + 16, device="cpu")


@pytest.mark.parametrize("shape", [(0, 3), (3, 0), (0, 0)])
def test_slots_of_an_empty_table(shape):
    cache, table = KVCacheInt4(8, 2, 64, page_size=32, device="cpu"), torch.zeros(*shape, dtype=torch.int32)
    for index in (torch.int32, torch.int64):
        got = cache.slots(table, torch.tensor([0, 1, 0], dtype=index), torch.tensor([0, -1, 70], dtype=index))
        assert got.dtype == torch.int64 and got.tolist() == [256, -1, 256]
        assert cache.slots(table, torch.zeros(0, dtype=index), torch.zeros(0, dtype=index)).tolist() == []


def test_tilings_of_the_linear_are_launchable():
    """Every choice: a known tile, a cluster only where its tiles fit the card at once, no CTA without a stage of k, the
    followers' sums within the leader's ring."""
    blocks = {32: 2, 64: 2, 96: 2, 128: 2, 192: 1, 256: 1}
    for M in (3, 16, 17, 64, 100, 128, 129, 300, 1000, 3001, 8192):
        for N in (128, 512, 640, 1024, 4096, 11008, 28672, 65536):
            for K in (128, 256, 384, 2048, 4096, 11008, 130944):
                for gated in (0, 1):
                    t = L.fg_linear_w8a8_tiling(M, N, K, gated, 148, 232448)
                    bn, cg, splits = t & 0xFFFF, t >> 16 & 0xFF, t >> 24
                    assert bn in blocks and (cg, splits) in ((1, 1), (1, 2), (1, 4), (1, 8), (2, 1)) and (cg == 1 or bn == 256)
                    assert not gated or bn not in (96, 192)
                    if splits > 1:
                        tiles = -(-M // 128) * -(-N // bn)
                        per = blocks[bn]
                        stage = per * (128 + bn) * 128
                        ring = (232448 - 1024 - 64 - 8 * bn) // (stage + 16) * stage
                        assert tiles * splits <= 148 - 148 // 8 and -(-K // 128 // per) >= splits and (splits - 1) * bn * 512 <= ring


def test_entry_points_keep_no_containers():
    """A container's failing allocation would throw through the C interface: the library's own units use none."""
    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "fastgate_b200", "csrc")
    for name in ("fg_norm.cu", "fg_linear8.cu", "fg_kv4.cu", "fg_attn4.cu", "fg_host.h"):
        with open(os.path.join(csrc, name)) as f:
            assert not re.search(r"std::(map|unordered_map|vector|string|deque|list|set)\b|\bnew\b [a-z]|\bthrow\b [a-z]+::", re.sub(r"//.*", "", f.read())), name
