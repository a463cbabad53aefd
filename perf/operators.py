"""The operators of a decode step over several drafted tokens, measured through the package's public entry points.

* ``tree``    attention of a tree of T drafted tokens over the cached rows and over each other (``ops.TreeAttention``).
* ``linear``  few rows times a matrix of 4-bit weights with group scales (``ops.w4_linear``).
* ``gated``   both projections of a gated feed-forward block with 4-bit weights, activation and product (``ops.w4_silu_mul``).
* ``append``  the accepted path of a drafted tree appended to the K/V rows of all layers (``ops.PathAppend``).

``own`` is set from outside: false computes the plain forms with elementary torch operations, true calls the package.
Keys are ~N(0, 1) with four outlier channels around a mean that the queries share, as in this repository's benchmark.
"""
import math

import torch

own = False

DEV = "cuda:0"
D = 128
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # one user, a short context, a handful of guesses: launches and latency are everything
        dict(name="tree_4k_b1", kind="tree", bs=1, heads=8, group=4, draft=5, rows=4096, form="dense", mask="tree", ragged=False,
             dtype="bf16"),
        # a serving batch over long documents: every cached row is read once for all drafted tokens
        dict(name="tree_64k_b4", kind="tree", bs=4, heads=8, group=4, draft=16, rows=65536, form="dense", mask="tree", ragged=False,
             dtype="bf16"),
        # the retrieval's attended set (sink, selected rows, local window) of a full batch, a wide tree: the matrix rate counts
        dict(name="tree_selected_b8", kind="tree", bs=8, heads=8, group=4, draft=64, rows=32768, form="selected", mask="tree",
             ragged=False, dtype="bf16"),
        # fp32 cache, odd lengths, seven query heads to a KV head, a key count for each row, masks that leave rows empty
        dict(name="tree_9001_b3_f32", kind="tree", bs=3, heads=4, group=7, draft=7, rows=9001, form="dense", mask="holes",
             ragged=True, dtype="f32"),
        # a single token's QKV projection in the 8B shape
        dict(name="linear_qkv_m1", kind="linear", m=1, n=6144, k=4096, g=128, bias=False, out="bf16"),
        # the logits of a batch: the largest matrix of the model, fp32 out
        dict(name="linear_head_m8", kind="linear", m=8, n=151936, k=4096, g=128, bias=False, out="f32"),
        # the down projection over a batch of drafted tokens, finer scales
        dict(name="linear_down_m64", kind="linear", m=64, n=4096, k=12288, g=64, bias=False, out="bf16"),
        # odd rows and columns, the finest scales, a bias
        dict(name="linear_odd_m13", kind="linear", m=13, n=1003, k=1184, g=32, bias=True, out="bf16"),
        # the feed-forward block of one token in the 8B shape
        dict(name="gated_m1", kind="gated", m=1, n=12288, k=4096, g=128),
        # a batch of drafted tokens through a block of odd width
        dict(name="gated_m40_odd", kind="gated", m=40, n=5001, k=2048, g=32),
        # four accepted tokens of each of eight sequences into all layers of the 8B shape
        dict(name="append_36l_b8", kind="append", layers=36, bs=8, heads=8, draft=16, path=4, rows=64, norms=False, dtype="bf16"),
        # fp32 caches that keep value norms, paths of different lengths
        dict(name="append_3l_b3_f32", kind="append", layers=3, bs=3, heads=4, draft=7, path=5, rows=300, norms=True, dtype="f32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choices(["tree", "linear", "gated", "append"], [40, 30, 18, 12])[0]
    if kind == "tree":
        f32 = rng.random() < 0.25
        heads, group = rng.choice([(8, 4), (8, 4), (8, 4), (4, 7), (4, 8), (2, 8), (8, 8), (8, 5), (2, 4), (8, 1)])
        bs, draft = rng.choice([1, 1, 2, 3, 4, 8]), _log(rng, 1, 64)
        most = (1 << 21) // (bs * heads * (2 if f32 else 1))
        most = min(most, (1 << 26) // (bs * heads * group * draft * (8 if f32 else 1)))
        return dict(kind=kind, bs=bs, heads=heads, group=group, draft=draft, rows=_log(rng, 1, max(2, min(262144, most))),
                    form=rng.choice(["dense", "dense", "two", "selected"]), mask=rng.choice(["chain", "tree", "tree", "holes"]),
                    ragged=rng.random() < 0.35, dtype="f32" if f32 else "bf16")
    g = rng.choice([32, 64, 128, 128])
    if kind == "linear":
        k = g * max(1, _log(rng, 256, 16384) // g)
        return dict(kind=kind, m=_log(rng, 1, 128), n=_log(rng, 100, min(151936, (1 << 28) // k)), k=k, g=g, bias=rng.random() < 0.3,
                    out=rng.choice(["bf16", "bf16", "f32"]))
    if kind == "gated":
        k = g * max(1, _log(rng, 256, 8192) // g)
        return dict(kind=kind, m=_log(rng, 1, 128), n=_log(rng, 100, min(28672, (1 << 26) // k)), k=k, g=g)
    f32 = rng.random() < 0.4
    draft = _log(rng, 1, 64)
    return dict(kind=kind, layers=_log(rng, 1, 48), bs=rng.choice([1, 1, 2, 3, 4, 8]), heads=rng.choice([2, 4, 8]), draft=draft,
                path=rng.randint(1, min(draft, 16)), rows=_log(rng, 17, 300), norms=f32 and rng.random() < 0.7, dtype="f32" if f32 else "bf16")


# ------------------------------------------------------------------ inputs


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _tree_inputs(c, g):
    dt, bs, h, hq, t, n = DTYPES[c["dtype"]], c["bs"], c["heads"], c["heads"] * c["group"], c["draft"], c["rows"]
    mean = torch.randn(bs, h, 1, D, generator=g, device=DEV) * 0.5
    big = torch.randint(0, D, (4,), generator=g, device=DEV)
    k = torch.randn(bs, h, n, D, generator=g, device=DEV)
    k[..., big] *= 3
    k = (k + mean).to(dt)
    v = torch.randn(bs, h, n, D, generator=g, device=DEV).to(dt)
    # what the fused projection of the drafted tokens holds: query, key and value heads side by side
    x = torch.randn(bs, t, hq + 2 * h, D, generator=g, device=DEV)
    x[:, :, :hq] = x[:, :, :hq] * 0.5 + mean.view(bs, 1, h, 1, D).expand(bs, 1, h, c["group"], D).reshape(bs, 1, hq, D)
    x[:, :, hq:hq + h] += mean.view(bs, 1, h, D)
    x = x.to(dt)
    s = dict(q=x[:, :, :hq].contiguous(), dk=x[:, :, hq:hq + h], dv=x[:, :, hq + h:])
    if c["form"] == "dense":
        s["segments"] = [(k, v, 0, n)]
    elif c["form"] == "two":  # the dense rows of an offloading cache beside the zone rows of a short sequence, in two tensors
        a = (n + 1) // 2
        s["segments"] = [(k[:, :, :a].contiguous(), v[:, :, :a].contiguous(), 0, a)] + ([(k, v, a, n - a)] if n > a else [])
    else:  # sink | selected rows of the zone | local window, in one tensor
        sink, tail = min(64, n // 4), min(529, n // 3)
        zone = n - sink - tail
        top = max(1, min(1024, zone // 2))
        idx = torch.rand(bs, h, zone, generator=g, device=DEV).argsort(dim=-1)[..., :top].contiguous()
        s["segments"] = [(k, v, a, m, i) for a, m, i in ((0, sink, None), (sink, top, idx), (n - tail, tail, None)) if m > 0]
    s["total"] = sum(seg[3] for seg in s["segments"])
    s["row_keys"] = None
    if c["ragged"]:
        rk = (torch.rand(bs, h, generator=g, device=DEV) * (s["total"] + 1)).to(torch.int32).clamp_(max=s["total"])
        rk.view(-1)[-1] = 0  # a row that has nothing in the cache yet
        s["row_keys"] = rk
    s["mask"] = None
    if c["mask"] != "chain":
        parent = (torch.rand(bs, t, generator=g, device=DEV) * (torch.arange(t, device=DEV) + 1)).long() - 1  # -1: after the cached rows
        m = torch.zeros(bs, t, t, dtype=torch.bool, device=DEV)
        at = torch.arange(t, device=DEV).expand(bs, t).clone()
        for _ in range(t):  # every token sees itself and what it descends from
            m |= (torch.arange(t, device=DEV) == at[..., None])
            at = torch.where(at >= 0, parent.gather(1, at.clamp(min=0)), at)
        if c["mask"] == "holes":  # tokens that are padding see nothing of the draft
            m[torch.rand(bs, t, generator=g, device=DEV) < 0.3] = False
        s["mask"] = m
    return s


def _w4_matrix(n, k, g, gen):
    codes = torch.randint(0, 16, (n, k), generator=gen, device=DEV, dtype=torch.uint8)
    scales = ((torch.rand(n, k // g, generator=gen, device=DEV) + 0.5) / (5 * math.sqrt(k))).to(torch.bfloat16)
    zeros = torch.randint(6, 10, (n, k // g), generator=gen, device=DEV, dtype=torch.uint8)
    return codes, scales, zeros


def _inputs(c, seed):
    g = _gen(seed)
    if c["kind"] == "tree":
        return _tree_inputs(c, g)
    if c["kind"] in ("linear", "gated"):
        s = dict(x=torch.randn(c["m"], c["k"], generator=g, device=DEV).to(torch.bfloat16), w=_w4_matrix(c["n"], c["k"], c["g"], g))
        if c["kind"] == "gated":
            s["up"] = _w4_matrix(c["n"], c["k"], c["g"], g)
        else:
            s["bias"] = torch.randn(c["n"], generator=g, device=DEV).to(torch.bfloat16) if c["bias"] else None
        return s
    dt, n, t = DTYPES[c["dtype"]], c["layers"], c["draft"]
    draft = torch.randn(n, c["bs"], t, 2 * c["heads"], D, generator=g, device=DEV).to(dt)
    cache = torch.randn(2, n, c["bs"], c["heads"], c["rows"], D, generator=g, device=DEV).to(dt)
    path = torch.rand(c["bs"], t, generator=g, device=DEV).argsort(dim=-1)[:, :c["path"]].sort(dim=-1).values
    if c["norms"]:  # caches of several sequences that accepted different numbers of tokens
        path = torch.where(torch.rand(path.shape, generator=g, device=DEV) < 0.2, -1, path)
    slots = [(7 * i) % (c["rows"] - c["path"] + 1) for i in range(n)]
    norms = torch.rand(n, c["bs"], c["heads"], c["rows"], generator=g, device=DEV) if c["norms"] else None
    return dict(dk=draft[:, :, :, :c["heads"]], dv=draft[:, :, :, c["heads"]:], k=cache[0], v=cache[1], path=path.contiguous(), slots=slots,
                norms=norms)


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if not own:
        return s
    from pariskv_amd import ops

    if case["kind"] == "tree":
        s["plan"] = ops.TreeAttention(case["bs"], case["heads"], case["group"], case["draft"], s["total"], DEV)
    elif case["kind"] in ("linear", "gated"):
        s["w"] = ops.W4Weight.from_codes(*s["w"])
        if case["kind"] == "gated":
            s["up"] = ops.W4Weight.from_codes(*s["up"])
    else:
        s["plan"] = ops.PathAppend(list(s["k"]), list(s["v"]), None if s["norms"] is None else list(s["norms"]))
    return s


# ------------------------------------------------------------- a pass


def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(s):
    from pariskv_amd import ops

    c = s["case"]
    if c["kind"] == "tree":
        return s["plan"].run(s["q"], s["segments"], s["dk"], s["dv"], mask=s["mask"], row_keys=s["row_keys"])
    if c["kind"] == "linear":
        return ops.w4_linear(s["x"], s["w"], bias=s["bias"], out_dtype=DTYPES[c["out"]])
    if c["kind"] == "gated":
        return ops.w4_silu_mul(s["x"], s["w"], s["up"])
    s["plan"].launch(s["dk"], s["dv"], s["path"], s["slots"])
    return _caches(s)


def _caches(s):
    return [s["k"], s["v"]] if s["norms"] is None else [s["k"], s["v"], s["norms"]]


def _rows(s, dtype):
    """The cached K and V rows that the segments name, side by side."""
    ks, vs = [], []
    for seg in s["segments"]:
        k, v, r0, n = seg[:4]
        i = seg[4] if len(seg) > 4 else None
        if i is None:
            ks.append(k[:, :, r0:r0 + n].to(dtype)), vs.append(v[:, :, r0:r0 + n].to(dtype))
        else:
            at = (r0 + i[:, :, :n]).unsqueeze(-1).expand(-1, -1, -1, D)
            ks.append(k.gather(2, at).to(dtype)), vs.append(v.gather(2, at).to(dtype))
    return torch.cat(ks, 2), torch.cat(vs, 2)


def _allowed(s, c):
    """[bs, heads, draft, total + draft]: which keys a drafted token attends to."""
    bs, h, t, n = c["bs"], c["heads"], c["draft"], s["total"]
    cached = torch.ones(bs, h, 1, n, dtype=torch.bool, device=DEV)
    if s["row_keys"] is not None:
        cached = torch.arange(n, device=DEV) < s["row_keys"].view(bs, h, 1, 1)
    m = s["mask"] if s["mask"] is not None else torch.ones(t, t, dtype=torch.bool, device=DEV).tril().expand(bs, t, t)
    return torch.cat([cached.expand(bs, h, t, n), m.view(bs, 1, t, t).expand(bs, h, t, t)], dim=-1)


def _silu(x):
    return x / (1 + torch.exp(-x))


def _dequant(w, dtype):
    codes, scales, zeros = w
    n, k = codes.shape
    x = codes.to(dtype).view(n, scales.shape[1], -1) - zeros.to(dtype).unsqueeze(-1)
    return (x * scales.to(dtype).unsqueeze(-1)).view(n, k)


def _run_plain(s):
    c = s["case"]
    if c["kind"] == "tree":
        bs, h, g, t = c["bs"], c["heads"], c["group"], c["draft"]
        k, v = _rows(s, torch.float32)
        k = torch.cat([k, s["dk"].float().transpose(1, 2)], 2)
        v = torch.cat([v, s["dv"].float().transpose(1, 2)], 2)
        q = s["q"].float().view(bs, t, h, g, D).permute(0, 2, 1, 3, 4).reshape(bs, h, t * g, D)
        ok = _allowed(s, c).unsqueeze(3).expand(bs, h, t, g, -1).reshape(bs, h, t * g, -1)
        z = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(1 / math.sqrt(D)).masked_fill_(~ok, float("-inf"))
        top = z.amax(-1, keepdim=True).clamp_(min=-1e30)
        p = z.sub_(top).exp_()
        o = torch.matmul(p, v) / p.sum(-1, keepdim=True).clamp_(min=1e-30)
        return o.view(bs, h, t, g, D).permute(0, 2, 1, 3, 4).reshape(bs, t, h * g, D).to(DTYPES[c["dtype"]])
    if c["kind"] == "linear":
        y = torch.matmul(s["x"].float(), _dequant(s["w"], torch.float32).t())
        if s["bias"] is not None:
            y += s["bias"].float()
        return y.to(DTYPES[c["out"]])
    if c["kind"] == "gated":
        x = s["x"].float()
        a = torch.matmul(x, _dequant(s["w"], torch.float32).t())
        b = torch.matmul(x, _dequant(s["up"], torch.float32).t())
        return (_silu(a) * b).to(torch.bfloat16)
    path = s["path"].clamp(min=0)
    keep = (s["path"] >= 0)[:, None, :, None]
    for i, slot in enumerate(s["slots"]):
        for src, dst in ((s["dk"][i], s["k"][i]), (s["dv"][i], s["v"][i])):
            rows = src.gather(1, path[:, :, None, None].expand(-1, -1, src.shape[2], D)).transpose(1, 2)
            at = dst[:, :, slot:slot + c["path"]]
            at.copy_(torch.where(keep, rows, at))
        if s["norms"] is not None:  # of the value rows, which came last
            at = s["norms"][i][:, :, slot:slot + c["path"]]
            at.copy_(torch.where(keep[..., 0], rows.float().square().sum(-1).sqrt(), at))
    return _caches(s)


# ------------------------------------------------------- what it must cost, what it must give


def work(case):
    c = case
    if c["kind"] == "tree":
        es = 2 if c["dtype"] == "bf16" else 4
        n = c["rows"]
        if c["form"] == "selected":
            sink, tail = min(64, n // 4), min(529, n // 3)
            n = sink + tail + max(1, min(1024, (n - sink - tail) // 2))
        if c["ragged"]:
            n = n / 2  # on average
        hq, t = c["heads"] * c["group"], c["draft"]
        return {"bytes": int(es * D * c["bs"] * (2 * c["heads"] * (n + t) + 2 * t * hq)), "flops": int(4 * D * c["bs"] * hq * t * (n + t))}
    if c["kind"] in ("linear", "gated"):
        m, n, k = c["m"], c["n"] * (2 if c["kind"] == "gated" else 1), c["k"]
        out = m * c["n"] * (4 if c.get("out") == "f32" else 2)
        return {"bytes": int(n * k / 2 + n * (k // c["g"]) * 2.5 + 2 * m * k + out), "flops": 2 * m * n * k}
    es = 2 if c["dtype"] == "bf16" else 4
    rows = c["layers"] * c["bs"] * c["heads"] * c["path"] * 2
    return {"bytes": rows * D * es * 2, "flops": 0}


def exact(case, seed):
    c, s = case, _inputs(case, seed)
    if c["kind"] == "tree":
        bs, h, g, t = c["bs"], c["heads"], c["group"], c["draft"]
        out = torch.zeros(bs, t, h * g, D, dtype=torch.float64, device=DEV)
        for b in range(bs):
            for j in range(h):
                ks, vs = [], []
                for seg in s["segments"]:
                    at = torch.arange(seg[3], device=DEV) if len(seg) < 5 or seg[4] is None else seg[4][b, j, :seg[3]]
                    ks.append(seg[0][b, j].index_select(0, seg[2] + at).double())
                    vs.append(seg[1][b, j].index_select(0, seg[2] + at).double())
                n = s["total"] if s["row_keys"] is None else int(s["row_keys"][b, j])
                k = torch.cat([torch.cat(ks)[:n], s["dk"][b, :, j].double()])
                v = torch.cat([torch.cat(vs)[:n], s["dv"][b, :, j].double()])
                see = torch.ones(t, n + t, dtype=torch.bool, device=DEV)
                see[:, n:] = torch.ones(t, t, device=DEV).tril().bool() if s["mask"] is None else s["mask"][b]
                for i in range(g):
                    z = s["q"][b, :, j * g + i].double() @ k.t() / math.sqrt(D)
                    z = torch.where(see, z, torch.full_like(z, -math.inf))
                    p = torch.nan_to_num(torch.softmax(z, dim=1), nan=0.0)  # nothing to attend to: zero
                    out[b, :, j * g + i] = p @ v
        return out
    if c["kind"] in ("linear", "gated"):
        def product(w):
            y = torch.empty(c["m"], c["n"], dtype=torch.float64, device=DEV)
            for r in range(0, c["n"], 8192):
                q, sc, z = (t[r:r + 8192] for t in w)
                real = (q.double() - z.double().repeat_interleave(c["g"], 1)) * sc.double().repeat_interleave(c["g"], 1)
                y[:, r:r + 8192] = s["x"].double() @ real.t()
            return y

        if c["kind"] == "gated":
            a = product(s["w"])
            return a * torch.sigmoid(a) * product(s["up"])
        y = product(s["w"])
        return y if s["bias"] is None else y + s["bias"].double()
    k, v = s["k"].double(), s["v"].double()
    norms = None if s["norms"] is None else s["norms"].double()
    for b, row in enumerate(s["path"].tolist()):
        for i, p in enumerate(row):
            if p < 0:
                continue
            for layer, slot in enumerate(s["slots"]):
                k[layer, b, :, slot + i] = s["dk"][layer, b, p].double()
                v[layer, b, :, slot + i] = s["dv"][layer, b, p].double()
                if norms is not None:
                    norms[layer, b, :, slot + i] = s["dv"][layer, b, p].double().norm(dim=-1)
    return [k, v] if norms is None else [k, v, norms]
