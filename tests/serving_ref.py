"""64-bit plain implementations of the serving operators, for the tests (torch on the CPU, no code of the package)."""
from __future__ import annotations

import math

import torch

F64 = torch.float64
BLOCK = 16
HALF_STEP = torch.finfo(torch.float16).eps / 2  # a rounding to fp16 is off by at most this, relative (2^-11)
TINY = 2.0 ** -24                               # smallest positive fp16: roundings below the normal range


def rmsnorm(x, weight, residual=None, eps=1e-6):
    """(normalised rows, residual stream, t = h * weight, 1 / rms) in 64 bits."""
    h = x.to(F64) + (0 if residual is None else residual.to(F64))
    rstd = 1 / (h.pow(2).mean(-1, keepdim=True) + eps).sqrt()
    t = h * weight.to(F64)
    return t * rstd, h, t, rstd


def activation(v, act):
    if act == "gelu":
        return 0.5 * v * (1 + torch.erf(v / math.sqrt(2)))
    if act == "gelu_tanh":
        return 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)))
    if act == "silu":
        return v * torch.sigmoid(v)
    return v


def linear_int8(x8, w8, x_scales, w_scales=None, bias=None, residual=None, act="none"):
    """(result, size of the terms that were rounded on the way) in 64 bits."""
    v = x8.to(F64) @ w8.to(F64).T * x_scales.to(F64)[:, None]
    if w_scales is not None:
        v = v * w_scales.to(F64)
    size = v.abs()
    if bias is not None:
        v, size = v + bias.to(F64), size + bias.to(F64).abs()
    if act == "silu_gate":
        gs = [t.unflatten(-1, (-1, 2, 64)) for t in (v, size)]
        g, u = gs[0][:, :, 0], gs[0][:, :, 1]
        size = ((gs[1][:, :, 0] + 1) * (u.abs() + gs[1][:, :, 1])).flatten(-2)
        v = (g * torch.sigmoid(g) * u).flatten(-2)
    else:
        v = activation(v, act)
    if residual is not None:
        v, size = v + residual.to(F64), size + residual.to(F64).abs()
    return v, size


def rotate(x, cos_sin, positions, interleaved):
    """x [tokens, heads, d] turned, in 64 bits."""
    cos, sin = cos_sin.to(F64)[positions.long()][:, None].chunk(2, -1)
    x = x.to(F64)
    if interleaved:
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    a, b = x.chunk(2, -1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def quantise(rows):
    """(scale, low, exact codes before rounding) of 64-bit rows: the parameters as fp16 values."""
    low = rows.amin(-1, keepdim=True).half().to(F64)
    scale = ((rows.amax(-1, keepdim=True) - low) / 15).half().to(F64).clamp(min=TINY)
    return scale, low, ((rows - low) / scale).clamp(0, 15)


def unpack(pages, d):
    """pages [n, heads, page bytes] uint8 -> codes [2, n, heads, rows, d] and parameters [2, n, heads, rows, 2] (scale, low)."""
    n, heads = pages.shape[:2]
    blocks = pages.reshape(n, heads, -1, BLOCK * (d + 8))
    packed = blocks[..., :BLOCK * d].reshape(n, heads, -1, 2, BLOCK, d // 2)
    codes = torch.stack([packed & 15, packed >> 4], -1).flatten(-2)
    params = blocks[..., BLOCK * d:].contiguous().view(torch.float16).reshape(n, heads, -1, 2, BLOCK, 2)
    order = (3, 0, 1, 2, 4, 5)
    return codes.permute(order).flatten(3, 4), params.permute(order).flatten(3, 4)


def by_slot(t):
    """[2, pages, heads, rows, ...] -> [2, slots, heads, ...]."""
    return t.transpose(2, 3).flatten(1, 2)


def stored_rows(pages, d, slots, page_size):
    """The 64-bit rows [2, len(slots), heads, d] that the cache holds at `slots`."""
    codes, params = (by_slot(t)[:, torch.as_tensor(slots)].to(F64) for t in unpack(pages, d))
    return codes * params[..., :1] + params[..., 1:]


def attention(q, pages, table, lens, page_size, starts=None, scale=None):
    """Attention over the cache, sequence by sequence, in 64 bits.  Returns (out, largest 15 * scale, largest |value|)."""
    tokens, hq, d = q.shape
    heads = pages.shape[1]
    scale = d ** -0.5 if scale is None else scale
    out = torch.zeros(tokens, hq, d, dtype=F64)
    span, top = 0.0, 0.0
    codes, params = (by_slot(t) for t in unpack(pages, d))
    for b, n in enumerate(lens):
        q0, q1 = (b, b + 1) if starts is None else (starts[b], starts[b + 1])
        if n == 0 or q1 == q0:
            continue
        slots = torch.tensor([int(table[b][i // page_size]) * page_size + i % page_size for i in range(n)])
        par = params[:, slots].to(F64)
        k, v = codes[:, slots].to(F64) * par[..., :1] + par[..., 1:]  # [n, heads, d]
        span = max(span, 15 * float(par[1, :, :, 0].max()))
        top = max(top, float(v.abs().max()))
        for i in range(q0, q1):
            seen = n - (q1 - q0) + (i - q0) + 1
            if seen <= 0:
                continue
            for h in range(hq):
                g = h // (hq // heads)
                s = (k[:seen, g] @ q[i, h].to(F64)) * scale
                p = torch.softmax(s, 0)
                out[i, h] = p @ v[:seen, g]
    return out, span, top


def attention_tolerance(out, span, top):
    """What rounding explains: each weight times a value's scale is rounded to fp16 (half a step of a sum of terms of at most
    `span`), the result once more; scores of tens formed in 32 bits move a weight by a few 2^-17, the sums by less."""
    return HALF_STEP * (span + out.abs()) + 2.0 ** -15 * (top + span) + TINY


def attention_error(out, span, top):
    """A bound without the weights' rounding to fp16 (the kernel multiplies what it leaves over as well, so that 2^-22 of a weight is
    lost): half a step of the output, and what 32-bit scores move.  A score is at most eight truncated sums of sixteen
    products away from its own, each 2^-23 of at most 15 sk |scale| log2(e) sum|q|, which is below 100 for normal rows of 128 channels and
    less for 64: 8 * 100 * 2^-23 in log2, a weight moves by ln 2 of that, below 2^-13.8; the exponential and the sums add some
    2^-21.  Weights that are off by e move the output by at most e times its distance from the values, below top + span."""
    return HALF_STEP * out.abs() + 2.0 ** -13.8 * (top + span) + TINY


def random_pages(g, count, heads, d, page_size, spread=1.0, offset=0.0):
    """A pool whose rows are quantised normal rows (packed here, in 64 bits)."""
    rows = torch.randn(count, heads, page_size // BLOCK, 2, BLOCK, d, generator=g, dtype=F64) * spread + offset
    scale, low, codes = quantise(rows)
    codes = codes.round().to(torch.uint8)
    packed = (codes[..., 0::2] | (codes[..., 1::2] << 4)).reshape(count, heads, -1, BLOCK * d)
    params = torch.cat([scale, low], -1).half().reshape(count, heads, -1, 2 * BLOCK * 2).view(torch.uint8)
    return torch.cat([packed, params], -1).reshape(count, heads, -1)
