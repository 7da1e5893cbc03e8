"""The serving operators that surround the weight-streaming linears, as measurable cases.

Five operators of one decoding step with 8-bit activations and a 4-bit key/value cache:

  norm    add_rmsnorm        residual addition, RMS norm, fp16 output or int8 output with one scale per row
  linear  linear_int8        int8 activations x int8 weights with scales, bias, activation, residual
  append  kv_append_int4     rotation of queries and keys, 4-bit rows written into the pages of a cache
  read    kv_read_int4       rows of that cache back as fp16
  attend  kv_attention_int4  attention over the cached rows, grouped heads, ragged lengths

``run`` computes them with elementary torch operations in 32 bits, or, with ``own`` set, through the
package's entry points.  A page of the cache holds, for each key/value head, blocks of 16 rows:
16 rows of key codes (D/2 bytes, low nibble = even channel), 16 of value codes, then a (scale, low end) fp16
pair for each of the 16 key rows and each of the 16 value rows; a stored row is low end + scale * code.
"""
import math
import random

import torch

own = False

EPS = 1e-6
BLOCK = 16  # rows of a cache block


# ---- cases ----------------------------------------------------------------------------------------
def _norm(name, m, k, out, res):
    return {"name": name, "op": "norm", "m": m, "k": k, "out": out, "res": res}


def _linear(name, m, n, k, act, bias, residual):
    return {"name": name, "op": "linear", "m": m, "n": n, "k": k, "act": act, "bias": bias, "residual": residual}


def _append(name, tokens, hq, hkv, d, page, interleaved):
    return {"name": name, "op": "append", "tokens": tokens, "hq": hq, "hkv": hkv, "d": d, "page": page, "interleaved": interleaved}


def _read(name, tokens, hkv, d, page):
    return {"name": name, "op": "read", "tokens": tokens, "hkv": hkv, "d": d, "page": page}


def _attend(name, batch, longest, ragged, new, hq, hkv, d, page):
    return {"name": name, "op": "attend", "batch": batch, "longest": longest, "ragged": ragged, "new": new, "hq": hq, "hkv": hkv,
            "d": d, "page": page}


def listed():
    return [
        # one decoding step of sixteen sequences: the smallest call, all latency
        _norm("norm_decode_16x8192_int8", 16, 8192, "int8", "fp16"),
        # a prompt of 8192 tokens, the residual stream kept in 32 bits
        _norm("norm_prompt_8192x4096_int8", 8192, 4096, "int8", "fp32"),
        # the output projection of a 4096-wide model for one sequence
        _linear("linear_1x4096x4096", 1, 4096, 4096, "none", False, True),
        # gate and up projection together, sixteen sequences: the weight is all the traffic
        _linear("linear_gate_16x28672x8192", 16, 28672, 8192, "silu_gate", False, False),
        # the down projection of a prompt of odd length, bound by the tensor cores
        _linear("linear_prompt_3001x4096x11008", 3001, 4096, 11008, "none", True, True),
        # one new token for each of 64 sequences
        _append("append_decode_64", 64, 32, 8, 128, 64, False),
        # a chunk of a long prompt, heads of 64 channels rotated in interleaved pairs
        _append("append_prompt_6001_d64", 6001, 32, 8, 64, 16, True),
        # a short shared prefix
        _read("read_prefix_500", 500, 8, 128, 16),
        # a long context brought back
        _read("read_context_40000", 40000, 8, 128, 64),
        # one sequence with a middling context: latency, split over the length
        _attend("attend_1x5000", 1, 5000, False, 1, 32, 8, 128, 64),
        # drafted tokens checked for 24 sequences of uneven length, one of them padding
        _attend("attend_verify_24x3000", 24, 3000, True, 5, 32, 4, 64, 16),
        # 64 sequences with long contexts: the cache is all the traffic
        _attend("attend_64x8000", 64, 8000, True, 1, 64, 8, 128, 64),
    ]


def _between(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "linear", "append", "read", "attend", "attend", "linear"])
    if op == "norm":
        k = 8 * _between(rng, 32, 2048)
        m = _between(rng, 1, max(1, min(8192, 8192 * 4096 // k)))
        return {"op": op, "m": m, "k": k, "out": rng.choice(["int8", "fp16"]), "res": rng.choice(["none", "fp16", "fp32"])}
    if op == "linear":
        n, k = 128 * _between(rng, 4, 224), 128 * _between(rng, 4, 112)
        m = _between(rng, 1, 4096)
        while m > 1 and m * n * k > 3001 * 4096 * 11008:
            m = (m + 1) // 2
        act = rng.choice(["none", "none", "gelu_tanh", "silu", "silu_gate"])
        return {"op": op, "m": m, "n": n, "k": k, "act": act, "bias": rng.random() < 0.5, "residual": rng.random() < 0.5}
    d, page = rng.choice([64, 128]), rng.choice([16, 32, 64, 128])
    hkv = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 3, 4, 7, 8, 16])
    if op == "append":
        tokens = _between(rng, 1, 6001 * 32 // (hkv * max(group, 4)))
        return {"op": op, "tokens": min(tokens, 6001), "hq": hkv * group, "hkv": hkv, "d": d, "page": page, "interleaved": rng.random() < 0.5}
    if op == "read":
        return {"op": op, "tokens": _between(rng, 1, 40000), "hkv": hkv, "d": d, "page": page}
    batch = _between(rng, 1, 64)
    longest = _between(rng, 1, min(32000, 64 * 8000 // batch))
    new = rng.choice([1, 1, 1, 2, 3, 6])
    return {"op": op, "batch": batch, "longest": max(longest, new), "ragged": rng.random() < 0.7, "new": new, "hq": hkv * group, "hkv": hkv,
            "d": d, "page": page}


def _lengths(case):
    """Cached rows and new tokens of each sequence.  They belong to the case, not to the seed: the work depends on them."""
    b, longest, new = case["batch"], case["longest"], case["new"]
    if not case["ragged"]:
        return [longest] * b, [new] * b
    r = random.Random(b * 1000003 + longest * 101 + new)
    lens, news = [], []
    for i in range(b):
        if i == 1:  # an entry of the batch that is padding
            lens.append(0)
            news.append(0 if new > 1 else 1)
            continue
        n = r.randint(1, new)
        lens.append(longest if i == 0 else r.randint(max(n, longest // 3), longest))
        news.append(n)
    return lens, news


# ---- inputs ---------------------------------------------------------------------------------------
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def _pack_rows(rows):
    """[..., D] fp32 rows -> codes [..., D/2] uint8 and (scale, low end) [..., 2] fp16."""
    low = rows.amin(-1, keepdim=True).half()
    scale = ((rows.amax(-1, keepdim=True) - low.float()) / 15).half().clamp(min=2.0 ** -24)
    codes = torch.round((rows - low.float()) / scale.float()).clamp(0, 15).to(torch.uint8)
    return codes[..., 0::2] | (codes[..., 1::2] << 4), torch.cat([scale, low], -1)


def _unpack_rows(codes, params):
    """The fp32 rows that codes [..., D/2] and (scale, low end) [..., 2] stand for."""
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).float()
    return c * params[..., :1].float() + params[..., 1:].float()


def _views(pages, d):
    """Codes [pages, heads, blocks, 2 (key, value), 16, d/2] and parameters [pages, heads, blocks, 2, 16, 2] of a pool."""
    blocks = pages.view(pages.shape[0], pages.shape[1], -1, BLOCK * (d + 8))
    codes = blocks[..., : BLOCK * d].unflatten(-1, (2, BLOCK, d // 2))
    params = blocks[..., BLOCK * d:].view(torch.float16).unflatten(-1, (2, BLOCK, 2))
    return codes, params


def _pool(g, count, hkv, d, page):
    """A pool of `count` pages whose rows are normal keys and values."""
    pages = torch.empty(count, hkv, page * (d + 8), dtype=torch.uint8, device="cuda")
    codes, params = _views(pages, d)
    step = max(1, (1 << 25) // (hkv * page * d * 2))
    for at in range(0, count, step):
        n = min(step, count - at)
        c, p = _pack_rows(_randn(g, n, hkv, page // BLOCK, 2, BLOCK, d))
        codes[at:at + n] = c
        params[at:at + n] = p
    return pages


def _angles(positions, d):
    """cos and sin of a rotation table, [positions, d] fp32: the cosines of all pairs, then the sines."""
    inv = 10000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64, device="cuda") / d)
    a = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * inv
    return torch.cat([a.cos(), a.sin()], -1).float()


def prepare(case, seed):
    g, op = _generator(seed), case["op"]
    s = dict(case)
    if op == "norm":
        m, k = case["m"], case["k"]
        s["x"] = _randn(g, m, k).half()
        s["weight"] = (1 + 0.1 * _randn(g, k)).half()
        s["residual"] = None
        if case["res"] != "none":
            # a residual stream: larger than what is added to it, with some channels that stand out
            loud = torch.where(torch.rand(k, device="cuda", generator=g) < 0.01, 8.0, 1.0)
            s["residual"] = (3 * _randn(g, m, k) * loud).to(torch.float16 if case["res"] == "fp16" else torch.float32)
            s["residual_out"] = torch.empty_like(s["residual"])
        s["y"] = torch.empty(m, k, dtype=torch.float16 if case["out"] == "fp16" else torch.int8, device="cuda")
        if case["out"] == "int8":
            s["scales"] = torch.empty(m, dtype=torch.float32, device="cuda")
            s["values"] = torch.empty(m, k, dtype=torch.float16, device="cuda")
    elif op == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        width = n // 2 if case["act"] == "silu_gate" else n
        # normal activations and weights, quantised row by row to the range of their largest value
        s["x8"] = (_randn(g, m, k) * 32).round().clamp(-127, 127).to(torch.int8)
        s["w8"] = (_randn(g, n, k) * 32).round().clamp(-127, 127).to(torch.int8)
        s["x_scales"] = (0.5 + torch.rand(m, device="cuda", generator=g)) / 32
        s["w_scales"] = ((0.5 + torch.rand(n, device="cuda", generator=g)) / (32 * k ** 0.5)).half()
        s["bias_"] = _randn(g, n).half() if case["bias"] else None
        s["residual_"] = _randn(g, m, width).half() if case["residual"] else None
        s["c"] = torch.empty(m, width, dtype=torch.float16, device="cuda")
    elif op == "append":
        t, hq, hkv, d, page = (case[v] for v in ("tokens", "hq", "hkv", "d", "page"))
        # the three column ranges of one projection's output, as the fused projection leaves them
        qkv = _randn(g, t, (hq + 2 * hkv) * d).half()
        s["q"], s["k"], s["v"] = (x.unflatten(-1, (-1, d)) for x in qkv.split([hq * d, hkv * d, hkv * d], -1))
        s["q_out"] = torch.empty(t, hq, d, dtype=torch.float16, device="cuda")
        reach = 4 * t + 4096
        s["cos_sin"] = _angles(reach, d)
        s["positions"] = torch.randint(0, reach, (t,), device="cuda", generator=g, dtype=torch.int32)
        count = -(-t // page) + 16
        s["pages"] = torch.zeros(count, hkv, page * (d + 8), dtype=torch.uint8, device="cuda")
        s["slots"] = _slots(g, t, count, page)
        s["k_back"] = torch.empty(t, hkv, d, dtype=torch.float16, device="cuda")
        s["v_back"] = torch.empty_like(s["k_back"])
    elif op == "read":
        t, hkv, d, page = (case[v] for v in ("tokens", "hkv", "d", "page"))
        count = -(-t // page) + 16
        s["pages"] = _pool(g, count, hkv, d, page)
        s["slots"] = _slots(g, t, count, page)
        s["k_back"] = torch.empty(t, hkv, d, dtype=torch.float16, device="cuda")
        s["v_back"] = torch.empty_like(s["k_back"])
    else:
        hq, hkv, d, page = (case[v] for v in ("hq", "hkv", "d", "page"))
        lens, news = _lengths(case)
        per = [-(-n // page) for n in lens]
        table = torch.zeros(len(lens), max(1, max(per)), dtype=torch.int32)
        order = torch.randperm(sum(per) + 1, generator=torch.Generator().manual_seed(int(seed)))
        at = 0
        for b, n in enumerate(per):
            table[b, :n] = order[at:at + n]
            at += n
        s["pages"] = _pool(g, sum(per) + 1, hkv, d, page)
        s["table"] = table.cuda()
        s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        starts = [0]
        for n in news:
            starts.append(starts[-1] + n)
        s["starts"] = torch.tensor(starts, dtype=torch.int32, device="cuda") if case["new"] > 1 else None
        s["starts_"] = torch.tensor(starts, device="cuda")
        s["q"] = _randn(g, starts[-1], hq, d).half()
        s["o"] = torch.empty(starts[-1], hq, d, dtype=torch.float16, device="cuda")
    return s


def _slots(g, t, count, page):
    """Where t rows go: runs of consecutive slots in shuffled pages, as an allocator hands them out."""
    order = torch.randperm(count, device="cuda", generator=g)
    at = torch.arange(t, device="cuda")
    return order[at // page] * page + at % page


# ---- plain forms ----------------------------------------------------------------------------------
def _plain_norm(s):
    h = s["x"].float()
    if s["residual"] is not None:
        h = h + s["residual"].float()
    w = s["weight"].float()
    rstd = torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS)
    t = h * w
    if s["out"] == "fp16":
        got = {"y": (t * rstd).half()}
    else:
        top = t.abs().amax(-1, keepdim=True)
        q = torch.round(t * (127 / top))
        scales = top * rstd / 127
        got = {"y": (q * scales).half(), "scales": scales[:, 0]}
    if s["residual"] is not None:
        got["residual"] = h.to(s["residual"].dtype)
    return got


def _gelu_tanh(v):
    return 0.5 * v * (1 + torch.tanh(0.7978845608028654 * (v + 0.044715 * v * v * v)))


def _silu(v):
    return v / (1 + torch.exp(-v))


def _finish_linear(s, v):
    """Scales, bias, activation and residual of the raw products v [m, n], in v's type."""
    v = v * s["x_scales"].to(v.dtype)[:, None] * s["w_scales"].to(v.dtype)
    if s["bias_"] is not None:
        v = v + s["bias_"].to(v.dtype)
    if s["act"] == "gelu_tanh":
        v = _gelu_tanh(v)
    elif s["act"] == "silu":
        v = _silu(v)
    elif s["act"] == "silu_gate":
        pair = v.unflatten(-1, (-1, 2, 64))
        v = (_silu(pair[:, :, 0]) * pair[:, :, 1]).flatten(-2)
    if s["residual_"] is not None:
        v = v + s["residual_"].to(v.dtype)
    return v


def _plain_linear(s):
    return _finish_linear(s, s["x8"].float() @ s["w8"].float().t()).half()


def _rotated(x, cos_sin, positions, interleaved):
    """x [t, heads, d] turned by the table's angles, in the type of the table."""
    cos, sin = cos_sin[positions.long()].unsqueeze(1).chunk(2, -1)
    x = x.to(cos.dtype)
    if interleaved:
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    a, b = x.chunk(2, -1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _places(s):
    page, slot = s["page"], s["slots"]
    return slot // page, (slot % page) // BLOCK, slot % BLOCK


def _plain_read(s):
    codes, params = _views(s["pages"], s["d"])
    at, block, row = _places(s)
    return {"k": _unpack_rows(codes[at, :, block, 0, row], params[at, :, block, 0, row]).half(),
            "v": _unpack_rows(codes[at, :, block, 1, row], params[at, :, block, 1, row]).half()}


def _plain_append(s):
    k = _rotated(s["k"], s["cos_sin"], s["positions"], s["interleaved"])
    codes, params = _views(s["pages"], s["d"])
    at, block, row = _places(s)
    for which, rows in ((0, k), (1, s["v"].float())):
        c, p = _pack_rows(rows)
        codes[at, :, block, which, row] = c
        params[at, :, block, which, row] = p
    return {"q": _rotated(s["q"], s["cos_sin"], s["positions"], s["interleaved"]).half(), **_plain_read(s)}


def _attention(s, dtype):
    """Attention over the padded contexts of all sequences at once, in `dtype`."""
    hq, hkv, d, page = s["hq"], s["hkv"], s["d"], s["page"]
    codes, params = _views(s["pages"], d)
    lens, starts = s["lens"].long(), s["starts_"]
    b, width = s["table"].shape
    table = s["table"].long()
    kv = [_unpack_rows(codes[table, :, :, i], params[table, :, :, i]).to(dtype).transpose(1, 2).reshape(b, hkv, width * page, d) for i in (0, 1)]
    news = starts[1:] - starts[:-1]
    most = s["new"]
    inside = torch.arange(most, device=lens.device) < news[:, None]  # [b, most]
    rows = (starts[:-1, None] + torch.arange(most, device=lens.device)).clamp(max=s["q"].shape[0] - 1)
    q = s["q"].to(dtype)[rows].view(b, most, hkv, hq // hkv, d).permute(0, 2, 1, 3, 4).reshape(b, hkv, -1, d)
    scores = (q @ kv[0].transpose(-1, -2) * d ** -0.5).view(b, hkv, most, hq // hkv, -1)
    last = lens[:, None] - news[:, None] + torch.arange(most, device=lens.device)  # position of each new token
    seen = torch.arange(width * page, device=lens.device) <= last[..., None]  # [b, most, rows]
    seen &= torch.arange(width * page, device=lens.device) < lens[:, None, None]
    scores = scores.masked_fill(~seen[:, None, :, None], -math.inf)
    top = scores.amax(-1, keepdim=True).clamp(min=-1e30)
    p = torch.exp(scores - top)
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-30)  # a row that sees nothing gives zeros
    o = (p.view(b, hkv, -1, width * page) @ kv[1]).view(b, hkv, most, hq // hkv, d).permute(0, 2, 1, 3, 4).reshape(b, most, hq, d)
    return o[inside]


def run(s):
    op = s["op"]
    if own:
        return _own(s)
    if op == "norm":
        return _plain_norm(s)
    if op == "linear":
        return _plain_linear(s)
    if op == "append":
        return _plain_append(s)
    if op == "read":
        return _plain_read(s)
    return _attention(s, torch.float32).half()


# ---- the package's entry points -------------------------------------------------------------------
def _own(s):
    import fastgate_b200 as fg

    op = s["op"]
    if op == "norm":
        got = {"y": s["y"]}
        fg.add_rmsnorm(s["x"], s["weight"], s["y"], residual=s["residual"], residual_out=s.get("residual_out"), scales=s.get("scales"), eps=EPS)
        if s["out"] == "int8":
            got["scales"] = s["scales"]
            got["y"] = torch.mul(s["y"], s["scales"][:, None], out=s["values"])  # the values that the 8-bit rows stand for
        if s["residual"] is not None:
            got["residual"] = s["residual_out"]
        return got
    if op == "linear":
        fg.linear_int8(s["x8"], s["w8"], s["c"], s["x_scales"], s["w_scales"], bias=s["bias_"], residual=s["residual_"], act=s["act"])
        return s["c"]
    if op == "append":
        fg.kv_append_int4(s["k"], s["v"], s["pages"], s["slots"], s["page"], cos_sin=s["cos_sin"], positions=s["positions"], q=s["q"],
                          q_out=s["q_out"], interleaved=s["interleaved"])
        fg.kv_read_int4(s["pages"], s["slots"], s["k_back"], s["v_back"], s["page"])  # the values that the 4-bit rows stand for
        return {"q": s["q_out"], "k": s["k_back"], "v": s["v_back"]}
    if op == "read":
        fg.kv_read_int4(s["pages"], s["slots"], s["k_back"], s["v_back"], s["page"])
        return {"k": s["k_back"], "v": s["v_back"]}
    fg.kv_attention_int4(s["q"], s["pages"], s["table"], s["lens"], s["o"], s["page"], q_starts=s["starts"])
    return s["o"]


# ---- what a pass cannot do without ----------------------------------------------------------------
def work(case):
    op = case["op"]
    if op == "norm":
        m, k = case["m"], case["k"]
        stream = {"none": 0, "fp16": 4, "fp32": 8}[case["res"]]
        return {"bytes": m * k * (2 + stream + (2 if case["out"] == "fp16" else 1)) + 2 * k + (4 * m if case["out"] == "int8" else 0),
                "flops": 8 * m * k}
    if op == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        width = n // 2 if case["act"] == "silu_gate" else n
        return {"bytes": n * k + m * k + 2 * m * width * (2 if case["residual"] else 1) + 4 * m + 2 * n * (2 if case["bias"] else 1),
                "flops": 2 * m * n * k}
    if op == "append":
        t, hq, hkv, d = (case[v] for v in ("tokens", "hq", "hkv", "d"))
        return {"bytes": t * (4 * hq * d + 4 * hkv * d + hkv * (d + 8) + 4 * d + 12), "flops": t * d * (3 * hq + 12 * hkv)}
    if op == "read":
        t, hkv, d = case["tokens"], case["hkv"], case["d"]
        return {"bytes": t * (hkv * (d + 8) + 4 * hkv * d + 8), "flops": 4 * t * hkv * d}
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    lens, news = _lengths(case)
    rows = sum(max(0, n - new + i + 1) for n, new in zip(lens, news) for i in range(new))
    return {"bytes": sum(lens) * hkv * (d + 8) + 4 * sum(news) * hq * d + 4 * sum(-(-n // case["page"]) for n in lens) + 4 * len(lens),
            "flops": 4 * rows * hq * d}


# ---- the same in 64 bits --------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    op, f64 = case["op"], torch.float64
    if op == "norm":
        x = s["x"].to(f64) + (0 if s["residual"] is None else s["residual"].to(f64))
        norm = (x.pow(2).sum(1) / case["k"] + EPS).sqrt()
        y = x * s["weight"].to(f64) / norm[:, None]
        got = {"y": y}
        if case["out"] == "int8":
            got["scales"] = y.abs().max(1).values / 127
            got["y"] = (y / got["scales"][:, None]).round() * got["scales"][:, None]
        if s["residual"] is not None:
            got["residual"] = x
        return got
    if op == "linear":
        c = torch.empty(case["m"], case["n"], dtype=f64, device="cuda")
        w = s["w8"].to(f64)
        for at in range(0, case["m"], 512):
            c[at:at + 512] = torch.mm(s["x8"][at:at + 512].to(f64), w.T)
        c = c * torch.outer(s["x_scales"].to(f64), s["w_scales"].to(f64))
        if case["bias"]:
            c = c + s["bias_"].to(f64)
        if case["act"] == "silu":
            c = c * torch.sigmoid(c)
        elif case["act"] == "gelu_tanh":
            c = c * (1 + torch.tanh((2 / math.pi) ** 0.5 * (c + 0.044715 * c ** 3))) / 2
        elif case["act"] == "silu_gate":
            tiles = c.reshape(case["m"], -1, 128)
            c = (tiles[..., :64] * torch.sigmoid(tiles[..., :64]) * tiles[..., 64:]).reshape(case["m"], -1)
        return c + s["residual_"].to(f64) if case["residual"] else c
    if op in ("append", "read"):
        got = {}
        if op == "append":
            t, d = case["tokens"], case["d"]
            half = d // 2
            table = s["cos_sin"].to(f64)[s["positions"].long()]
            turn = torch.complex(table[:, :half], table[:, half:])[:, None]
            flat = []
            for x in (s["q"], s["k"]):
                x = x.to(f64)
                pair = (x[..., 0::2], x[..., 1::2]) if case["interleaved"] else (x[..., :half], x[..., half:])
                z = torch.complex(*pair) * turn
                flat.append(torch.stack([z.real, z.imag], -1).reshape(t, -1, d) if case["interleaved"] else torch.cat([z.real, z.imag], -1))
            got["q"] = flat[0]
            for name, x in (("k", flat[1]), ("v", s["v"].to(f64))):
                low = x.min(-1, keepdim=True).values.half().to(f64)
                step = torch.clamp(((x.max(-1, keepdim=True).values - low) / 15).half().to(f64), min=2.0 ** -24)
                got[name] = low + step * torch.clamp(torch.round((x - low) / step), 0, 15)
            return got
        raw, page, d = s["pages"], case["page"], case["d"]
        where = s["slots"]
        base = (where % page) // BLOCK * (BLOCK * (d + 8))
        own_page = raw[where // page]  # [t, heads, bytes]
        line = where % BLOCK
        for i, name in enumerate(("k", "v")):
            byte = base + i * (BLOCK * d // 2) + line * (d // 2)
            codes = torch.gather(own_page, 2, (byte[:, None] + torch.arange(d // 2, device="cuda"))[:, None].expand(-1, case["hkv"], -1)).long()
            byte = base + BLOCK * d + i * 4 * BLOCK + line * 4
            par = torch.gather(own_page, 2, (byte[:, None] + torch.arange(4, device="cuda"))[:, None].expand(-1, case["hkv"], -1))
            par = par.contiguous().view(torch.float16).to(f64)
            nibbles = torch.stack([codes % 16, codes // 16], -1).flatten(-2).to(f64)
            got[name] = nibbles * par[..., 0:1] + par[..., 1:2]
        return got
    # attention, one sequence after the other
    lens, news = _lengths(case)
    hq, hkv, d, page = (case[v] for v in ("hq", "hkv", "d", "page"))
    codes, params = _views(s["pages"], d)
    out, at = torch.zeros(sum(news), hq, d, dtype=f64, device="cuda"), 0
    for i, (n, new) in enumerate(zip(lens, news)):
        if n and new:
            mine = s["table"][i, : -(-n // page)].long()
            kv = []
            for which in (0, 1):
                c = codes[mine, :, :, which].transpose(0, 1).reshape(hkv, -1, d // 2)[:, :n]
                p = params[mine, :, :, which].transpose(0, 1).reshape(hkv, -1, 2)[:, :n].to(f64)
                c = torch.stack([c & 15, c >> 4], -1).flatten(-2).to(f64)
                kv.append((c * p[..., 0:1] + p[..., 1:2]).repeat_interleave(hq // hkv, 0))
            scores = torch.einsum("thd,hld->htl", s["q"][at:at + new].to(f64), kv[0]) / d ** 0.5
            hidden = torch.arange(n, device="cuda")[None] > torch.arange(n - new, n, device="cuda")[:, None]
            weights = torch.softmax(scores.masked_fill(hidden, -math.inf), -1)
            out[at:at + new] = torch.einsum("htl,hld->thd", weights, kv[1])
        at += new
    return out
