"""The operators of a decode step in eight bits, measured through the package's public entry points.  Eight bits are e4m3 codes with
power-of-two scales: a code times its scale is the value.

* ``attend``  attention over a cache held in eight bits with a scale for each block of tokens and head (``ops.Fp8Attention``).
* ``store``   key and value rows quantised as they are written into such a cache (``ops.Fp8KVCache.store``).
* ``read``    rows of such a cache in bf16 or fp32 again (``ops.Fp8KVCache.read``).
* ``norm``    root-mean-square norm with the residual's addition, rows in eight bits with a scale each (``ops.add_rmsnorm_fp8``).
* ``linear``  products of eight-bit rows with an eight-bit matrix, scales for each token and channel (``ops.fp8_linear``).

``own`` is set from outside: false computes the plain forms with elementary torch operations, true calls the package.
Keys are ~N(0, 1) with four outlier channels around a mean that the queries share, as in this repository's benchmark.
"""
import math

import torch

own = False

DEV = "cuda:0"
D = 128
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
F8 = torch.float8_e4m3fn
TOP = 448.0        # the largest e4m3 number
LEAST = -100       # exponent of the smallest scale


def listed():
    return [
        # a decode step of a serving batch over long documents, every cached row once: the bytes of the cache count
        dict(name="attend_64k_b4", kind="attend", bs=4, heads=8, group=4, tokens=1, rows=65536, form="dense", block=64, ragged=False,
             dtype="bf16"),
        # the retrieval's attended set (sink, selected rows, local window) of a full batch
        dict(name="attend_selected_b8", kind="attend", bs=8, heads=8, group=4, tokens=1, rows=32768, form="selected", block=64,
             ragged=False, dtype="bf16"),
        # fp32 queries, odd lengths, seven query heads to a KV head, five tokens a sequence, key counts of their own, rows with none
        dict(name="attend_9001_b3_f32", kind="attend", bs=3, heads=4, group=7, tokens=5, rows=9001, form="dense", block=16, ragged=True,
             dtype="f32"),
        # a prompt into the cache of one layer, straight from the fused projection
        dict(name="store_8k_b1", kind="store", bs=1, heads=8, group=4, tokens=8192, capacity=16384, block=64, ragged=False, dtype="bf16"),
        # one decoded token of each of eight sequences of different lengths: the launch is everything
        dict(name="store_token_b8", kind="store", bs=8, heads=8, group=4, tokens=1, capacity=4096, block=64, ragged=True, dtype="bf16"),
        # a whole cache in bf16 again
        dict(name="read_32k_b1", kind="read", bs=1, heads=8, rows=32768, select=0, block=64, dtype="bf16"),
        # selected rows of several sequences, fp32
        dict(name="read_selected_b3_f32", kind="read", bs=3, heads=4, rows=20011, select=515, block=32, dtype="f32"),
        # the norm before a projection of one token in the 8B shape
        dict(name="norm_1x4096", kind="norm", rows=1, width=4096, residual=True),
        # ... and of a batch of prompts
        dict(name="norm_4096x4096", kind="norm", rows=4096, width=4096, residual=True),
        # the logits of a batch: the largest matrix of the model, fp32 out
        dict(name="linear_head_m8", kind="linear", m=8, n=151936, k=4096, x="rows", bias=False, out="f32"),
        # a prompt through the QKV projection of the 8B shape, from bf16 rows: the matrix rate counts
        dict(name="linear_qkv_m4096", kind="linear", m=4096, n=6144, k=4096, x="bf16", bias=False, out="bf16"),
        # odd rows and columns, a bias
        dict(name="linear_odd_m13", kind="linear", m=13, n=1003, k=1185, x="rows", bias=True, out="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choices(["attend", "store", "read", "norm", "linear"], [32, 16, 12, 12, 28])[0]
    heads, group = rng.choice([(8, 4), (8, 4), (8, 4), (4, 7), (4, 8), (2, 8), (8, 8), (8, 5), (2, 4), (8, 1)])
    bs, block, dtype = rng.choice([1, 1, 2, 3, 4, 8]), rng.choice([16, 32, 64, 64, 128]), rng.choice(["bf16", "bf16", "bf16", "f32"])
    if kind == "attend":
        tokens = 1 if rng.random() < 0.6 else _log(rng, 2, 64)
        most = min((1 << 21) // (bs * heads), (1 << 25) // (bs * heads * group * tokens * (4 if dtype == "f32" else 1)))
        return dict(kind=kind, bs=bs, heads=heads, group=group, tokens=tokens, rows=_log(rng, 1, max(2, min(262144, most))),
                    form=rng.choice(["dense", "dense", "selected"]), block=block, ragged=rng.random() < 0.35, dtype=dtype)
    if kind == "store":
        tokens = 1 if rng.random() < 0.4 else _log(rng, 2, (1 << 15) // bs)
        return dict(kind=kind, bs=bs, heads=heads, group=group, tokens=tokens, capacity=tokens + _log(rng, 1, 8192), block=block,
                    ragged=rng.random() < 0.5, dtype=dtype)
    if kind == "read":
        rows = _log(rng, 1, (1 << 16) // bs)
        return dict(kind=kind, bs=bs, heads=heads, rows=rows, select=rng.choice([0, rng.randint(1, min(rows, 4096))]), block=block, dtype=dtype)
    if kind == "norm":
        width = rng.choice([1024, 2048, 4096, 5120, 12288, _log(rng, 100, 16384)])
        return dict(kind=kind, rows=_log(rng, 1, (1 << 24) // width), width=width, residual=rng.random() < 0.7)
    k, m = rng.choice([1024, 4096, 4096, 12288, _log(rng, 100, 16384)]), _log(rng, 1, 4096)
    most = min(151936, (1 << 29) // k, (1 << 36) // (m * k))
    return dict(kind=kind, m=m, n=_log(rng, 64, most), k=k, x=rng.choice(["rows", "rows", "bf16"]), bias=rng.random() < 0.3,
                out=rng.choice(["bf16", "bf16", "f32"]))


# ------------------------------------------------------------------ eight bits


def _pow2(e):
    """2^e in fp32, -126 <= e <= 127."""
    return ((e + 127) << 23).to(torch.int32).view(torch.float32)


def _exponent(top):
    """The least e >= LEAST with top <= 448 * 2^e, of the largest magnitudes `top` (fp32)."""
    _, e = torch.frexp(top / 1.75)  # 448 = 1.75 * 2^8: one too many where the quotient is a power of two
    e = e.clamp(min=LEAST + 8)
    e = torch.where((_pow2(e - 1) * 1.75 >= top) & (e > LEAST + 8), e - 1, e) - 8
    return torch.where(top > 0, e, LEAST)


def _codes(x, e):
    """Nearest e4m3 of x / 2^e; what is past 448 (infinities) is 448."""
    return (x * _pow2(-e)).clamp(-TOP, TOP).to(F8)


def _row_codes(x):
    """Codes and scales of rows, each with a scale of its own."""
    mag = x.abs()
    e = _exponent(torch.where(mag < math.inf, mag, 0.0).amax(-1, keepdim=True))
    return _codes(x, e), _pow2(e).squeeze(-1)


# ------------------------------------------------------------------ inputs


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _kv(c, g, rows):
    """K and V rows of a cache as floats, and the mean of the keys."""
    bs, h = c["bs"], c["heads"]
    mean = torch.randn(bs, h, 1, D, generator=g, device=DEV) * 0.5
    big = torch.randint(0, D, (4,), generator=g, device=DEV)
    k = torch.randn(bs, h, rows, D, generator=g, device=DEV)
    k[..., big] *= 3
    k += mean
    return k, torch.randn(bs, h, rows, D, generator=g, device=DEV), mean


def _filled(c, g, rows):
    """A cache of so many rows, some of its blocks short and some loud: codes and scales of K and of V, and the mean of the keys."""
    k, v, mean = _kv(c, g, rows)
    block, bs, h = c["block"], c["bs"], c["heads"]
    n = -(-rows // block)
    out = []
    for x in (k, v):
        x *= torch.exp(0.3 * torch.randn(bs, h, rows, 1, generator=g, device=DEV))
        padded = torch.zeros(bs, h, n * block, D, device=DEV)
        padded[:, :, :rows] = x
        codes, scales = _row_codes(padded.view(bs, h, n, block * D))
        out += [codes.view(bs, h, n * block, D), scales]
    return out, mean


def _attend_inputs(c, g):
    dt, bs, h, hq, t, n = DTYPES[c["dtype"]], c["bs"], c["heads"], c["heads"] * c["group"], c["tokens"], c["rows"]
    cache, mean = _filled(c, g, n)
    q = torch.randn(bs, t, hq, D, generator=g, device=DEV) * 0.5 + mean.view(bs, 1, h, 1, D).expand(bs, t, h, c["group"], D).reshape(bs, t, hq, D)
    s = dict(q=q.to(dt), cache=cache)
    if c["form"] == "dense":
        s["segments"] = [(0, n)]
    else:  # sink | selected rows of the zone | local window
        sink, tail = min(64, n // 4), min(529, n // 3)
        zone = n - sink - tail
        top = max(1, min(1024, zone // 2))
        idx = torch.rand(bs, h, zone, generator=g, device=DEV).argsort(dim=-1)[..., :top].contiguous()
        s["segments"] = [seg for seg in ((0, sink), (sink, top, idx), (n - tail, tail)) if seg[1] > 0]
    s["total"] = sum(seg[1] for seg in s["segments"])
    s["row_keys"] = None
    if c["ragged"]:
        rk = (torch.rand(bs, h, generator=g, device=DEV) * (s["total"] + 1)).to(torch.int32).clamp_(max=s["total"])
        rk.view(-1)[-1] = 0  # a row that has nothing in the cache yet
        s["row_keys"] = rk
    return s


def _store_inputs(c, g):
    bs, h, t, cap = c["bs"], c["heads"], c["tokens"], c["capacity"]
    cache, mean = _filled(c, g, cap)
    # what the fused projection holds: query, key and value heads side by side
    heads = (c["group"] + 2) * h
    x = torch.randn(bs, t, heads, D, generator=g, device=DEV)
    x[:, :, c["group"] * h:(c["group"] + 1) * h] += mean.view(bs, 1, h, D)
    x *= torch.exp(0.5 * torch.randn(bs, t, heads, 1, generator=g, device=DEV))
    x = x.to(DTYPES[c["dtype"]])
    s = dict(k=x[:, :, c["group"] * h:(c["group"] + 1) * h], v=x[:, :, (c["group"] + 1) * h:], cache=cache, start=0, lengths=None)
    if c["ragged"]:  # sequences of different lengths, shorter ones padded
        s["start"] = (torch.rand(bs, generator=g, device=DEV) * (cap - t + 1)).to(torch.int32).clamp_(max=cap - t)
        if t > 1:
            s["lengths"] = (torch.rand(bs, generator=g, device=DEV) * (t + 1)).to(torch.int32).clamp_(max=t)
    return s


def _matrix(n, k, g):
    """A matrix [n,k] in eight bits, ~N(0, 1/k), a scale for each of its rows."""
    w = torch.randn(n, k, generator=g, device=DEV) / math.sqrt(k)
    return _row_codes(w)


def _inputs(c, seed):
    g = _gen(seed)
    if c["kind"] == "attend":
        return _attend_inputs(c, g)
    if c["kind"] == "store":
        return _store_inputs(c, g)
    if c["kind"] == "read":
        cache, _ = _filled(c, g, c["rows"])
        idx = None
        if c["select"]:
            idx = torch.rand(c["bs"], c["heads"], c["rows"], generator=g, device=DEV).argsort(dim=-1)[..., :c["select"]].contiguous()
        return dict(cache=cache, idx=idx)
    if c["kind"] == "norm":
        x = torch.randn(c["rows"], c["width"], generator=g, device=DEV)
        x[:, torch.randint(0, c["width"], (4,), generator=g, device=DEV)] *= 12  # the outlier channels of a residual stream
        r = torch.randn(c["rows"], c["width"], generator=g, device=DEV) if c["residual"] else None
        return dict(x=x.to(torch.bfloat16), residual=None if r is None else r.to(torch.bfloat16),
                    weight=(1 + 0.1 * torch.randn(c["width"], generator=g, device=DEV)).to(torch.bfloat16))
    x = torch.randn(c["m"], c["k"], generator=g, device=DEV).to(torch.bfloat16)
    return dict(x=_row_codes(x.float()) if c["x"] == "rows" else x, w=_matrix(c["n"], c["k"], g),
                bias=torch.randn(c["n"], generator=g, device=DEV).to(torch.bfloat16) if c["bias"] else None)


EPS = 1e-6


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if not own:
        return s
    from pariskv_amd import ops

    if case["kind"] in ("attend", "store", "read"):
        s["cache"] = ops.Fp8KVCache.from_codes(*s["cache"], block=case["block"])
        if case["kind"] == "attend":
            s["plan"] = ops.Fp8Attention(case["bs"], case["heads"], case["group"], case["tokens"], s["total"], DEV)
    elif case["kind"] == "linear":
        s["w"] = ops.Fp8Weight.from_codes(*s["w"])
        if case["x"] == "rows":
            s["x"] = ops.Fp8Rows.from_codes(*s["x"])
    return s


# ------------------------------------------------------------- a pass


def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(s):
    from pariskv_amd import ops

    c = s["case"]
    if c["kind"] == "attend":
        return s["plan"].run(s["q"], s["cache"], s["segments"], row_keys=s["row_keys"])
    if c["kind"] == "store":
        cache = s["cache"]
        cache.store(s["k"], s["v"], s["start"], lengths=s["lengths"])
        return [cache.k, cache.k_scale, cache.v, cache.v_scale]
    if c["kind"] == "read":
        return s["cache"].read(0, None if s["idx"] is not None else c["rows"], idx=s["idx"], dtype=DTYPES[c["dtype"]])
    if c["kind"] == "norm":
        total, rows = ops.add_rmsnorm_fp8(s["x"], s["residual"], s["weight"], EPS)
        return [total, rows.codes, rows.scales]
    return ops.fp8_linear(s["x"], s["w"], bias=s["bias"], out_dtype=DTYPES[c["out"]])


def _values(codes, scales, block, row0, n, idx=None):
    """Rows of a cache in fp32: n from row0 on, or those that idx [bs,heads,n] names from there on."""
    bs, h = codes.shape[:2]
    at = torch.arange(row0, row0 + n, device=DEV).expand(bs, h, n) if idx is None else row0 + idx
    codes = codes[:, :, row0:row0 + n] if idx is None else codes.view(torch.uint8).gather(2, at.unsqueeze(-1).expand(-1, -1, -1, D)).view(F8)
    return codes.float() * scales.gather(2, at // block).unsqueeze(-1)


def _allowed(s, c):
    """[bs, heads, tokens, total]: which keys a token attends to: the last of its row's keys is the last token's own."""
    n, t = s["total"], c["tokens"]
    length = torch.full((c["bs"], c["heads"]), n, device=DEV) if s["row_keys"] is None else s["row_keys"]
    last = length.view(c["bs"], c["heads"], 1, 1) - (t - 1) + torch.arange(t, device=DEV).view(t, 1)
    return torch.arange(n, device=DEV) < last


def _attend_plain(s, c):
    bs, h, g, t = c["bs"], c["heads"], c["group"], c["tokens"]
    k, v = (torch.cat([_values(codes, scales, c["block"], *seg) for seg in s["segments"]], 2)
            for codes, scales in (s["cache"][:2], s["cache"][2:]))
    q = s["q"].float().view(bs, t, h, g, D).permute(0, 2, 1, 3, 4).reshape(bs, h, t * g, D)
    ok = _allowed(s, c).unsqueeze(3).expand(bs, h, t, g, -1).reshape(bs, h, t * g, -1)
    z = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(1 / math.sqrt(D)).masked_fill_(~ok, float("-inf"))
    p = z.sub_(z.amax(-1, keepdim=True).clamp_(min=-1e30)).exp_()
    o = torch.matmul(p, v) / p.sum(-1, keepdim=True).clamp_(min=1e-30)
    return o.view(bs, h, t, g, D).permute(0, 2, 1, 3, 4).reshape(bs, t, h * g, D).to(DTYPES[c["dtype"]])


def _store_plain(s, c):
    bs, h, t, block = c["bs"], c["heads"], c["tokens"], c["block"]
    start = torch.full((bs, 1), s["start"], device=DEV) if isinstance(s["start"], int) else s["start"].long().view(bs, 1)
    length = torch.full((bs, 1), t, device=DEV) if s["lengths"] is None else s["lengths"].long().view(bs, 1)
    # the blocks that the rows may reach into, [bs, n] of them, and what each of their places holds
    there = s["cache"][1].shape[2]
    n = min(there, (t + block - 2) // block + 1)
    blocks = (start // block).clamp(max=there - n) + torch.arange(n, device=DEV)
    at = (blocks.unsqueeze(-1) * block + torch.arange(block, device=DEV)).view(bs, n * block)
    token = at - start
    new = (token >= 0) & (token < length)
    old = (token < 0) & (length > 0) & (at // block == start // block)
    kept, touched = (m.view(bs, 1, n, block).any(-1) for m in (old, new))
    where, which = at.view(bs, 1, -1, 1).expand(bs, h, n * block, D), blocks.view(bs, 1, n).expand(bs, h, n)
    out = []
    for x, codes, scales in ((s["k"], *s["cache"][:2]), (s["v"], *s["cache"][2:])):
        x = x.gather(1, token.clamp(0, t - 1).view(bs, -1, 1, 1).expand(bs, n * block, h, D)).transpose(1, 2).float()
        x = torch.where(new.view(bs, 1, -1, 1), x, 0.0)
        before, s0 = codes.view(torch.uint8).gather(2, where), scales.gather(2, which)
        mag = x.abs().reshape(bs, h, n, -1)
        need = _pow2(_exponent(torch.where(mag < math.inf, mag, 0.0).amax(-1)))
        scale = torch.where(kept, torch.maximum(need, s0), need)
        wide, grown = (f.repeat_interleave(block, -1, output_size=n * block).unsqueeze(-1) for f in (scale, s0 / scale))
        now = torch.where(new.view(bs, 1, -1, 1), (x / wide).clamp(-TOP, TOP), before.view(F8).float() * grown).to(F8).view(torch.uint8)
        codes.view(torch.uint8).scatter_(2, where, torch.where((new | old).view(bs, 1, -1, 1), now, before))
        scales.scatter_(2, which, torch.where(touched, scale, s0))
        out += [codes, scales]
    return out


def _run_plain(s):
    c = s["case"]
    if c["kind"] == "attend":
        return _attend_plain(s, c)
    if c["kind"] == "store":
        return _store_plain(s, c)
    if c["kind"] == "read":
        n = c["select"] or c["rows"]
        return tuple(_values(codes, scales, c["block"], 0, n, s["idx"]).to(DTYPES[c["dtype"]])
                     for codes, scales in (s["cache"][:2], s["cache"][2:]))
    if c["kind"] == "norm":
        x = s["x"]
        if s["residual"] is not None:
            x = (x.float() + s["residual"].float()).to(torch.bfloat16)
        # 64 bits for the sum: a value next to the border of two codes goes by the last bit
        inv = (1 / torch.sqrt(x.double().square().mean(-1, keepdim=True) + EPS)).float()
        codes, scales = _row_codes(x.float() * inv * s["weight"].float())
        return [x, codes, scales]
    x, sx = s["x"] if c["x"] == "rows" else _row_codes(s["x"].float())
    w, sw = s["w"]
    y = torch.matmul(x.float(), w.float().t()) * sx.view(-1, 1) * sw
    if s["bias"] is not None:
        y += s["bias"].float()
    return y.to(DTYPES[c["out"]])


# ------------------------------------------------------- what it must cost, what it must give


def work(case):
    c = case
    if c["kind"] in ("norm", "linear"):
        if c["kind"] == "norm":
            n = c["rows"] * c["width"]
            return {"bytes": n * (2 + 1 + (4 if c["residual"] else 0)) + 4 * c["rows"] + 2 * c["width"], "flops": 0}
        m, n, k = c["m"], c["n"], c["k"]
        return {"bytes": n * k + 4 * n + m * ((k + 4) if c["x"] == "rows" else 2 * k) + m * n * (4 if c["out"] == "f32" else 2), "flops": 2 * m * n * k}
    es, bh = 2 if c["dtype"] == "bf16" else 4, c["bs"] * c["heads"]
    scale = 4 / c["block"]
    if c["kind"] == "store":
        n = bh * c["tokens"] * (0.5 if c["ragged"] and c["tokens"] > 1 else 1)
        return {"bytes": int(2 * n * (D * (es + 1) + scale)), "flops": 0}
    if c["kind"] == "read":
        n = bh * (c["select"] or c["rows"])
        return {"bytes": int(2 * n * (D * (es + 1) + scale)), "flops": 0}
    n = c["rows"]
    if c["form"] == "selected":
        sink, tail = min(64, n // 4), min(529, n // 3)
        n = sink + tail + max(1, min(1024, (n - sink - tail) // 2))
    if c["ragged"]:
        n = n / 2  # on average
    q = bh * c["group"] * c["tokens"]
    return {"bytes": int(2 * bh * n * (D + scale) + 2 * es * D * q), "flops": int(4 * D * q * n)}


def _exact_codes(x, top):
    """(codes, scale) of float64 x, of which `top` is the largest finite magnitude along a group, broadcast."""
    power = lambda e: ((e.long() + 1023) << 52).view(torch.float64)  # 2^e to the bit
    m, e = torch.frexp(top)  # top = m 2^e, 1/2 <= m < 1, and 448 = 7/8 2^9
    e = torch.where(top > 0, e - 9 + (m > 0.875), LEAST).clamp(min=LEAST)
    scale = power(e)
    x = (x / scale).clamp(-TOP, TOP)
    step = power(torch.frexp(x.abs().clamp(min=2.0 ** -6))[1] - 4)  # three bits behind the first
    return torch.round(x / step) * step, scale


def exact(case, seed):
    c, s = case, _inputs(case, seed)
    if c["kind"] == "attend":
        bs, h, g, t, block = c["bs"], c["heads"], c["group"], c["tokens"], c["block"]
        out = torch.zeros(bs, t, h * g, D, dtype=torch.float64, device=DEV)
        for b in range(bs):
            for j in range(h):
                at = torch.cat([seg[0] + (torch.arange(seg[1], device=DEV) if len(seg) < 3 else seg[2][b, j]) for seg in s["segments"]])
                n = s["total"] if s["row_keys"] is None else int(s["row_keys"][b, j])
                at = at[:n]
                k, v = (codes[b, j].view(torch.uint8)[at].view(F8).double() * scales[b, j][at // block].double().unsqueeze(-1)
                        for codes, scales in (s["cache"][:2], s["cache"][2:]))
                see = torch.arange(n, device=DEV) < n - (t - 1) + torch.arange(t, device=DEV).view(t, 1)
                for i in range(g):
                    z = torch.where(see, s["q"][b, :, j * g + i].double() @ k.t() / math.sqrt(D), -math.inf)
                    out[b, :, j * g + i] = torch.nan_to_num(torch.softmax(z, dim=1), nan=0.0) @ v  # nothing to attend to: zero
        return out
    if c["kind"] == "store":
        bs, t, block, out = c["bs"], c["tokens"], c["block"], []
        for x, codes, scales in ((s["k"], *s["cache"][:2]), (s["v"], *s["cache"][2:])):
            codes, scales = codes.double(), scales.double()
            for b in range(bs):
                start = s["start"] if isinstance(s["start"], int) else int(s["start"][b])
                end = start + (t if s["lengths"] is None else int(s["lengths"][b]))
                row = x[b].transpose(0, 1).double()
                if end <= start:
                    continue
                if start % block:  # behind rows that are there already
                    r0, r1 = start // block * block, min(end, (start // block + 1) * block)
                    was, before = codes[b, :, r0:start], scales[b, :, start // block].view(-1, 1, 1)
                    part = row[:, :r1 - start]
                    _, need = _exact_codes(part, part.abs().amax((1, 2), keepdim=True))
                    scale = torch.maximum(need, before)
                    codes[b, :, r0:start] = _exact_codes(was * before / scale, torch.full_like(scale, TOP))[0]
                    codes[b, :, start:r1] = _exact_codes(part / scale, torch.full_like(scale, TOP))[0]
                    scales[b, :, start // block] = scale.view(-1)
                    row, start = row[:, r1 - start:], r1
                if end > start:  # whole blocks, the last one filled up with nothing
                    n = -(-(end - start) // block)
                    full = torch.zeros(c["heads"], n * block, D, dtype=torch.float64, device=DEV)
                    full[:, :end - start] = row[:, :end - start]
                    full = full.view(c["heads"], n, block * D)
                    code, scale = _exact_codes(full, full.abs().amax(-1, keepdim=True))
                    codes[b, :, start:end] = code.view(c["heads"], n * block, D)[:, :end - start]
                    scales[b, :, start // block:start // block + n] = scale.squeeze(-1)
            out += [codes, scales]
        return out
    if c["kind"] == "read":
        out = []
        for codes, scales in (s["cache"][:2], s["cache"][2:]):
            x = codes.double() * scales.double().repeat_interleave(c["block"], -1).unsqueeze(-1)
            at = torch.arange(c["rows"], device=DEV).expand(c["bs"], c["heads"], -1) if s["idx"] is None else s["idx"]
            out.append(torch.take_along_dim(x, at.unsqueeze(-1), 2))
        return tuple(out)
    if c["kind"] == "norm":
        x = s["x"].double()
        if s["residual"] is not None:
            x = (x + s["residual"].double()).to(torch.bfloat16).double()
        y = x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + EPS) * s["weight"].double()
        codes, scales = _exact_codes(y, y.abs().amax(-1, keepdim=True))
        return [x, codes, scales.squeeze(-1)]
    if c["x"] == "rows":
        x = s["x"][0].double() * s["x"][1].double().unsqueeze(-1)
    else:
        x = s["x"].double()
        code, scale = _exact_codes(x, x.abs().amax(-1, keepdim=True))
        x = code * scale
    y = torch.empty(c["m"], c["n"], dtype=torch.float64, device=DEV)
    for r in range(0, c["n"], 8192):
        y[:, r:r + 8192] = x @ (s["w"][0][r:r + 8192].double() * s["w"][1][r:r + 8192].double().unsqueeze(-1)).t()
    return y if s["bias"] is None else y + s["bias"].double()
