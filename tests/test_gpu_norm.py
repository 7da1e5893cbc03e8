"""add_rmsnorm against 64 bits: fp16 and int8 rows, residual streams of both types, strides, rows of the extremes."""
import pytest
import torch

import fastgate_b200 as fg
from fastgate_b200 import capi
from tests import serving_ref as ref

pytestmark = pytest.mark.gpu

# sums of K squares in 32 bits (at most 64 + 10 additions deep), a division, a square root, three products
REL = 2.0 ** -17


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda:0")


def _data(M, K, res, seed, dev, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(M, K, generator=g).half()
    w = (1 + 0.1 * torch.randn(K, generator=g)).half()
    r = None if res is None else (spread * torch.randn(M, K, generator=g)).to(res)
    return x, w, r


def _check_int8(q, scales, t, rstd):
    a = t.abs().amax(-1, keepdim=True)
    want = t * 127 / a
    # the code is the nearest integer of a product of two 32-bit roundings of at most 127
    assert float((q.to(torch.float64) - want).abs().max()) <= 0.5 + 127 * 4 * 2.0 ** -24
    want_s = (a * rstd / 127)[:, 0]
    assert float(((scales.to(torch.float64) - want_s).abs() / want_s).max()) <= REL
    assert int(q.abs().max()) == 127  # the largest element of a row uses the whole range


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("res", [None, torch.float16, torch.float32])
@pytest.mark.parametrize("M,K", [(1, 8), (3, 40), (2, 256), (5, 1000), (16, 4096), (1, 8192), (301, 4096), (400, 520), (2, 16384),
                                 (3, 32768), (2, 40000)])
def test_matches_64_bits(M, K, res, int8, dev):
    x, w, r = _data(M, K, res, M * 7 + K, dev)
    y, h, t, rstd = ref.rmsnorm(x, w, r, 1e-6)
    out = torch.empty(M, K, dtype=torch.int8 if int8 else torch.half, device=dev)
    scales = torch.empty(M, device=dev) if int8 else None
    rd = None if r is None else r.to(dev)
    fg.add_rmsnorm(x.to(dev), w.to(dev), out, rd, 1e-6, scales)
    if int8:
        _check_int8(out.cpu(), scales.cpu(), t, rstd)
    else:
        assert bool(((out.cpu().to(torch.float64) - y).abs() <= y.abs() * (ref.HALF_STEP + REL) + ref.TINY).all())
    if r is not None:
        step = ref.HALF_STEP if res == torch.float16 else 0
        assert bool(((rd.cpu().to(torch.float64) - h).abs() <= h.abs() * (step + 2.0 ** -23) + (ref.TINY if step else 0)).all())


def test_residual_out_and_strided_input(dev):
    """Rows of a wider buffer in, the residual stream to a buffer of its own; in place gives the same bits."""
    x, w, r = _data(33, 512, torch.float16, 3, dev)
    wide = torch.full((33, 1024), float("nan"), dtype=torch.half, device=dev)
    wide[:, 512:] = x.to(dev)
    rd, ro = r.to(dev), torch.empty(33, 512, dtype=torch.half, device=dev)
    a, b = torch.empty(33, 512, dtype=torch.half, device=dev), torch.empty(33, 512, dtype=torch.half, device=dev)
    fg.add_rmsnorm(wide[:, 512:], w.to(dev), a, rd, residual_out=ro)
    assert torch.equal(rd.cpu(), r)  # untouched
    fg.add_rmsnorm(x.to(dev), w.to(dev), b, rd)
    assert torch.equal(a, b) and torch.equal(ro, rd)
    c = x.to(dev)
    fg.add_rmsnorm(c, w.to(dev), c, r.to(dev))  # the output over x
    assert torch.equal(c, a)


def test_codes_do_not_depend_on_the_shape_of_the_call(dev):
    """A row gives the same codes alone (one vector a thread) and among many rows (four)."""
    x, w, r = _data(600, 2048, torch.float32, 9, dev)
    q = torch.empty(600, 2048, dtype=torch.int8, device=dev)
    s = torch.empty(600, device=dev)
    fg.add_rmsnorm(x.to(dev), w.to(dev), q, r.to(dev), scales=s)
    q1, s1 = torch.empty(1, 2048, dtype=torch.int8, device=dev), torch.empty(1, device=dev)
    for i in (0, 17, 599):
        fg.add_rmsnorm(x[i:i + 1].to(dev), w.to(dev), q1, r[i:i + 1].to(dev), scales=s1)
        assert torch.equal(q1[0], q[i])


def test_rows_of_the_extremes(dev):
    """Zero rows, rows with infinities and NaNs, the largest and smallest values: each row is its own."""
    K = 1024
    x = torch.ones(6, K, dtype=torch.half)
    x[1] = 0
    x[2, 5] = float("inf")
    x[3, 900] = float("nan")
    x[4] = 65504.0
    x[5] = 2.0 ** -24
    w = torch.ones(K, dtype=torch.half)
    q, s = torch.full((6, K), 77, dtype=torch.int8, device=dev), torch.empty(6, device=dev)
    fg.add_rmsnorm(x.to(dev), w.to(dev), q, scales=s, eps=0.0 + 1e-12)
    q, s = q.cpu(), s.cpu()
    assert bool((q[0] == 127).all()) and abs(float(s[0]) * 127 - 1) < 1e-5
    assert bool((q[1] == 0).all()) and float(s[1]) == 1.0
    assert bool(torch.isnan(s[2])) and bool(torch.isnan(s[3]))
    assert bool((q[4] == 127).all()) and abs(float(s[4]) * 127 - 1) < 1e-5
    assert bool((q[5] == 127).all())
    y = torch.empty(6, K, dtype=torch.half, device=dev)
    fg.add_rmsnorm(x.to(dev), w.to(dev), y)
    y = y.cpu().float()
    assert bool((y[0] == 1).all()) and bool((y[1] == 0).all()) and bool((y[4] == 1).all())
    assert not bool(torch.isfinite(y[2]).any() and (y[2] != 0).any() and torch.isfinite(y[2, 5]))
    assert bool(torch.isnan(y[3]).all())


@pytest.mark.parametrize("K", [64, 1024, 40000])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_weights_that_are_not_finite_show_in_the_scale(bad, K, dev):
    """Not finite is h * weight, whichever of the two is to blame, a zero times an infinity included; fp16 rows show it in its place."""
    x, w, r = _data(5, K, torch.float32, K, dev)
    at = K // 2 + 3
    x[2], r[2] = 0, 0
    w[at] = bad
    q, s = torch.empty(5, K, dtype=torch.int8, device=dev), torch.zeros(5, device=dev)
    fg.add_rmsnorm(x.to(dev), w.to(dev), q, r.to(dev), scales=s)
    assert bool(torch.isnan(s).all())
    y = torch.empty(5, K, dtype=torch.half, device=dev)
    fg.add_rmsnorm(x.to(dev), w.to(dev), y, r.to(dev))
    want = ref.rmsnorm(x, w, r)[0]
    other = torch.arange(K) != at
    assert not bool(torch.isfinite(y[:, at]).any()) and bool(torch.isfinite(y.cpu()[:, other]).all())
    assert bool(((y.cpu().double() - want).abs() <= want.abs() * (ref.HALF_STEP + REL) + ref.TINY)[:, other].all())


@pytest.mark.parametrize("K", [64, 4096, 40000])
@pytest.mark.parametrize("size", [1e17, 1e19, 1e25, 4e37])
def test_residuals_whose_squares_do_not_fit(size, K, dev):
    """A residual stream in 32 bits far beyond the root of the largest number: finite rows give what the formula says."""
    x, w, r = _data(6, K, torch.float32, 3, dev)
    r = r.clamp(-7, 7) * size / 3
    r[3] /= size  # an ordinary row between them
    y, h, t, rstd = ref.rmsnorm(x, w, r, 1e-6)
    out, rd = torch.empty(6, K, dtype=torch.half, device=dev), r.to(dev)
    fg.add_rmsnorm(x.to(dev), w.to(dev), out, rd)
    assert bool(((out.cpu().double() - y).abs() <= y.abs() * (ref.HALF_STEP + REL) + ref.TINY).all())
    q, s = torch.empty(6, K, dtype=torch.int8, device=dev), torch.empty(6, device=dev)
    fg.add_rmsnorm(x.to(dev), w.to(dev), q, r.to(dev), 1e-6, s)
    _check_int8(q.cpu(), s.cpu(), t, rstd)
    r[1, 5] = float("inf")
    r[2, 7] = float("nan")
    fg.add_rmsnorm(x.to(dev), w.to(dev), q, r.to(dev), 1e-6, s)
    assert torch.isnan(s).tolist() == [False, True, True, False, False, False]
    fg.add_rmsnorm(x.to(dev), w.to(dev), out, r.to(dev))
    assert bool(torch.isnan(out[1, 5])) and bool((out[1] == 0).sum() == K - 1) and bool(torch.isnan(out[2]).all())


def test_refusals(dev):
    x = torch.zeros(2, 64, dtype=torch.half, device=dev)
    w = torch.ones(64, dtype=torch.half, device=dev)
    y, q, s = torch.empty_like(x), torch.empty(2, 64, dtype=torch.int8, device=dev), torch.empty(2, device=dev)
    r = torch.zeros(2, 64, dtype=torch.half, device=dev)
    fg.add_rmsnorm(x, w, y, r)
    fg.add_rmsnorm(torch.zeros(0, 64, dtype=torch.half, device=dev), w, torch.zeros(0, 64, dtype=torch.half, device=dev))
    for bad in (lambda: fg.add_rmsnorm(x, w, q),                                # int8 without scales
                lambda: fg.add_rmsnorm(x, w, y, scales=s),                      # scales without int8
                lambda: fg.add_rmsnorm(x, w[:32], y),
                lambda: fg.add_rmsnorm(x, w, y, r[:1]),
                lambda: fg.add_rmsnorm(x, w, y, residual_out=r),
                lambda: fg.add_rmsnorm(x, w, y, eps=-1.0),
                lambda: fg.add_rmsnorm(x, w, y, eps=float("nan")),
                lambda: fg.add_rmsnorm(x, w, y, r, residual_out=y),             # two outputs in one buffer
                lambda: fg.add_rmsnorm(x, w, r, r),                             # out over the residual stream
                lambda: fg.add_rmsnorm(x[:, :60], w[:60].contiguous(), torch.empty(2, 60, dtype=torch.half, device=dev))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError):
        fg.add_rmsnorm(x.float(), w, y)
    with pytest.raises(RuntimeError):
        fg.add_rmsnorm(x, w, y, r.bfloat16())
    assert capi.lib.fg_add_rmsnorm(x.data_ptr() + 2, 64, w.data_ptr(), None, None, 0, y.data_ptr(), 0, None, 1, 64, 1e-6, None) == capi.FG_ERR_ALIGN
