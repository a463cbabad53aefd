"""Operators of a step over several drafted tokens on the GPU, each against its definition in 64 bits: attention for a tree of
drafted tokens (ops.TreeAttention), products with 4-bit weights (ops.w4_linear, ops.w4_silu_mul), and the accepted path into the
caches of all layers (ops.PathAppend).

Tolerances, per element.  u = 2^-24 is half a step of fp32, h half a step of the output's type (2^-8 bf16, 2^-24 fp32).
Attention: with A = sum p |v| over the keys a row sees (p the exact weights), a score is off by at most 130 u S, S the largest sum of
|q| |k| times the scale (128 exact or rounded products and their sum, the scale), which moves a weight by that much and the normaliser
by as much again; the sum over n keys is off by (n + 200) u A (every key's addition, exponentials of 4 u, the merges), twice with the
normaliser.  bf16 weights are rounded to w (1 + d), |d| <= h, and summed up as they are: sum p (1 + d) v / sum p (1 + d) - sum p v
= sum p (d - mean d) v (1 + O(h)), with mean d = sum p d, at most h A + h |out|.  Together: A (4 * 130 u S + 2 (n + 200) u + h [bf16]) + h |out|,
and h |out| again for bf16.
4-bit products: with B = sum |x| s (16 + q + 16 + z), every partial sum is at most B and a path through the sums of a column has
at most 128 + K/128 + 20 additions: (148 + K/128) u B + h |y|.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV, D = "cuda:0", 128
U = 2.0 ** -24
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
BF, F32 = torch.bfloat16, torch.float32


def _randn(g, *shape, dtype=BF):
    return torch.randn(*shape, generator=g).to(dtype)


def _parents(g, bs, t):
    return (torch.rand(bs, t, generator=g) * (torch.arange(t) + 1)).long() - 1


def tree_case(seed, bs, h, group, t, rows, dtype, form="dense", mask="tree", ragged=False):
    """CPU tensors of one call: q, segments, draft_k, draft_v, mask, row_keys."""
    g = torch.Generator().manual_seed(seed)
    x = _randn(g, bs, t, (group + 2) * h, D, dtype=dtype)
    q, dk, dv = x[:, :, :group * h], x[:, :, group * h:(group + 1) * h], x[:, :, (group + 1) * h:]
    k, v = _randn(g, bs, h, max(rows, 1) + 3, D, dtype=dtype), _randn(g, bs, h, max(rows, 1) + 3, D, dtype=dtype)
    if rows == 0:
        segs = []
    elif form == "dense":
        segs = [(k, v, 2, rows)]
    elif form == "two":
        a = rows // 2
        k2, v2 = _randn(g, bs, h, rows, D, dtype=dtype), _randn(g, bs, h, rows, D, dtype=dtype)
        segs = [(k, v, 0, a), (k2, v2, 0, rows - a)]
    else:
        a = rows // 4
        idx = torch.rand(bs, h, rows, generator=g).argsort(-1)[..., :rows - 2 * a].contiguous()
        segs = [(k, v, 0, a), (k, v, 1, rows - 2 * a, idx), (k, v, rows - a, a)]
        if form == "index_two":
            segs[2] = (_randn(g, bs, h, a + 1, D, dtype=dtype), _randn(g, bs, h, a + 1, D, dtype=dtype), 1, a)
    m = None
    if mask != "chain":
        from pariskv_amd import ops

        m = ops.tree_mask(_parents(g, bs, t) if mask != "shared" else _parents(g, 1, t)[0])
        if mask == "holes":
            m = m & (torch.rand(bs, t, t, generator=g) < 0.7)
            m[:, t // 2] = False
    rk = None
    if ragged:
        rk = torch.randint(-1, rows + 3, (bs, h), generator=g, dtype=torch.int32)
        rk.view(-1)[-1] = 0
    return dict(q=q, segs=segs, dk=dk, dv=dv, mask=m, rk=rk)


def exact_tree(c, scale=None):
    """(output, tolerance), both fp64, by the definition."""
    q, dk, dv = c["q"].double(), c["dk"].double(), c["dv"].double()
    bs, t, hq, _ = q.shape
    h = dk.shape[2]
    group, scale = hq // h, scale or 1 / math.sqrt(D)
    out, tol = torch.zeros_like(q), torch.zeros_like(q)
    half = HALF[c["q"].dtype]
    for b in range(bs):
        for j in range(h):
            ks, vs = [dk[b, :, j]], [dv[b, :, j]]
            n = 0
            for seg in c["segs"]:
                at = seg[2] + (torch.arange(seg[3]) if len(seg) < 5 else seg[4][b, j, :seg[3]].clamp(0, seg[0].shape[2] - seg[2] - 1))
                ks.append(seg[0][b, j][at].double()), vs.append(seg[1][b, j][at].double())
                n += seg[3]
            if c["rk"] is not None:
                n = min(n, max(0, int(c["rk"][b, j])))
            k, v = torch.cat(ks[1:] + [torch.zeros(0, D, dtype=torch.float64)])[:n], torch.cat(vs[1:] + [torch.zeros(0, D, dtype=torch.float64)])[:n]
            for u in range(t):
                see = torch.arange(t) <= u if c["mask"] is None else (c["mask"][u] if c["mask"].dim() == 2 else c["mask"][b, u])
                kk, vv = torch.cat([k, ks[0][see]]), torch.cat([v, vs[0][see]])
                if len(kk) == 0:
                    continue
                qq = q[b, u, j * group:(j + 1) * group]
                p = torch.softmax(qq @ kk.T * scale, -1)
                o, a = p @ vv, p @ vv.abs()
                s = (qq.abs() @ kk.abs().T).amax(-1, keepdim=True) * abs(scale)
                out[b, u, j * group:(j + 1) * group] = o
                tol[b, u, j * group:(j + 1) * group] = (a * (520 * U * s + 2 * (len(kk) + 200) * U + (half if half > U else 0)) + half * (2 if half > U else 1) * o.abs())
    return out, tol


def to_gpu(c):
    """The same call on the GPU: K and V drafted rows and queries stay views of one tensor."""
    g = dict(c)
    hq, h = c["q"].shape[2], c["dk"].shape[2]
    x = torch.cat([c["q"], c["dk"], c["dv"]], 2).to(DEV)
    g["q"], g["dk"], g["dv"] = x[:, :, :hq], x[:, :, hq:hq + h], x[:, :, hq + h:]
    moved = {}
    put = lambda t: moved.setdefault(id(t), t.to(DEV))
    g["segs"] = [(put(s[0]), put(s[1]), *s[2:4], *[put(i) for i in s[4:]]) for s in c["segs"]]
    g["mask"], g["rk"] = (None if c[n] is None else c[n].to(DEV) for n in ("mask", "rk"))
    return g


def run_tree(c, **more):
    from pariskv_amd import ops

    bs, t, hq, _ = c["q"].shape
    h = c["dk"].shape[2]
    att = ops.TreeAttention(bs, h, hq // h, t, sum(s[3] for s in c["segs"]), DEV)
    return att.run(c["q"], c["segs"], c["dk"], c["dv"], mask=c["mask"], row_keys=c["rk"], **more)


def check(got, want, tol, what=""):
    assert got.shape == want.shape
    bad = ~((got.double().cpu() - want).abs() <= tol)
    assert not bad.any(), (what, int(bad.sum()), (got.double().cpu() - want).abs().max().item(), tol.max().item())


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("bs,h,group,t", [(1, 1, 1, 1), (1, 8, 4, 5), (2, 2, 7, 3), (1, 2, 8, 9), (2, 1, 4, 16), (1, 2, 5, 33), (1, 1, 4, 64), (1, 2, 1, 100)])
@pytest.mark.parametrize("rows", [0, 1, 33, 700])
def test_tree_attention_shapes(dtype, bs, h, group, t, rows):
    c = tree_case(rows * 7 + t, bs, h, group, t, rows, dtype)
    check(run_tree(to_gpu(c)), *exact_tree(c))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rows", [15, 16, 17, 31, 32, 63, 64, 65, 127, 128, 129, 511, 1025, 5000, 20000])
def test_tree_attention_lengths(dtype, rows):
    c = tree_case(rows, 1, 2, 4, 6, rows, dtype, mask="shared")
    check(run_tree(to_gpu(c)), *exact_tree(c))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("form", ["dense", "two", "index", "index_two"])
@pytest.mark.parametrize("mask", ["chain", "tree", "shared", "holes"])
@pytest.mark.parametrize("ragged", [False, True])
def test_tree_attention_segments_masks_and_counts(dtype, form, mask, ragged):
    c = tree_case(11, 3, 2, 4, 7, 601, dtype, form, mask, ragged)
    got = run_tree(to_gpu(c))
    want, tol = exact_tree(c)
    check(got, want, tol)
    if mask == "holes" and ragged:  # the row without cached keys has tokens that see nothing at all
        assert (want[-1, 3, -4:] == 0).all() and (got[-1, 3, -4:] == 0).all()


def test_tree_attention_of_one_token_is_decode_attention():
    """One drafted token sees the cached keys and itself: the keys that a decode step has after its append."""
    from pariskv_amd import ops

    for dtype in (BF, F32):
        c = to_gpu(tree_case(3, 2, 4, 4, 1, 900, dtype, mask="chain"))
        k, v, row0, n = c["segs"][0]
        k[:, :, row0 + n], v[:, :, row0 + n] = c["dk"][:, 0], c["dv"][:, 0]
        want = ops.DecodeAttention(2, 4, 4, n + 1, DEV).run(c["q"], [(k, v, row0, n + 1)])
        got = run_tree(c)
        assert (got.float() - want.float()).abs().max() <= (4 * 2.0 ** -8 if dtype == BF else 1e-5)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_tree_attention_of_values_nobody_sees(dtype):
    """Infinities and NaN in rows that a token does not see leave it as it is: drafted tokens of other branches and padding (keys
    and values), cached rows behind row_keys and outside the segments."""
    c = tree_case(5, 2, 2, 4, 40, 300, dtype, "dense", "tree")
    c["rk"] = torch.tensor([[300, 7], [0, 129]], dtype=torch.int32)
    c["dk"], c["dv"] = c["dk"].clone(), c["dv"].clone()
    want, tol = exact_tree(c)
    odd = [3, 17, 38]
    c["mask"][:, :, odd] = False            # nobody sees them ...
    want, tol = exact_tree(c)
    for i, bad in zip(odd, (float("nan"), float("inf"), float("-inf"))):
        c["dk"][:, i], c["dv"][:, i] = bad, bad
    for s in c["segs"]:
        for b in range(2):
            for j in range(2):
                end = s[2] + int(c["rk"][b, j])
                for x in s[:2]:
                    x[b, j, :s[2]], x[b, j, end:] = float("nan"), float("inf")
    check(run_tree(to_gpu(c)), want, tol)
    # ... and where some do, it is theirs alone
    c["dk"][:, odd] = 0.25
    c["mask"][:, 20, 17] = c["mask"][:, 30, 38] = c["mask"][:, 31, 3] = True
    got = run_tree(to_gpu(c)).cpu()
    rest = [i for i in range(40) if i not in (20, 30, 31)]
    clean = dict(c, dv=torch.where(torch.isfinite(c["dv"].float()), c["dv"], torch.zeros((), dtype=dtype)))
    want, tol = exact_tree(clean)
    check(got[:, rest], want[:, rest], tol[:, rest])
    assert (got[:, 20] == float("inf")).all() and (got[:, 30] == float("-inf")).all() and got[:, 31].isnan().all()


def test_tree_attention_of_extreme_scores():
    """Scores of +-10^4 and of 10^34 (fp32), equal scores, and a scale of its own."""
    for dtype, size in ((BF, 300.0), (F32, 300.0), (F32, 1e16)):
        c = tree_case(6, 1, 2, 4, 6, 200, dtype)
        c["q"] = (c["q"].float() * size).to(dtype)
        k, v, a, n = c["segs"][0]
        c["segs"] = [((k.float() * size).sign().to(dtype), v, a, n)]
        c["dk"] = c["dk"].float().sign().to(dtype)
        want, tol = exact_tree(c)
        top = tol.clone()
        if size > 1e6:  # one key's weight is 1, or equal scores share it: whichever the sums' rounding leaves on top
            got = run_tree(to_gpu(c)).double().cpu()
            assert torch.isfinite(got).all() and (got.abs() <= torch.cat([v.flatten(), c["dv"].flatten()]).abs().max()).all()
        else:
            check(run_tree(to_gpu(c)), want, top)
    c = tree_case(7, 2, 1, 4, 5, 77, BF, "index")
    want, tol = exact_tree(c, scale=0.31)
    check(run_tree(to_gpu(c), scale=0.31), want, tol)
    out = torch.full_like(to_gpu(c)["q"].contiguous(), 7)
    assert run_tree(to_gpu(c), out=out, scale=0.31) is out
    check(out, want, tol)


def test_tree_attention_clamps_wild_indices():
    c = tree_case(8, 1, 2, 4, 5, 64, BF, "index")
    c["segs"][1][4][0, 0, 3], c["segs"][1][4][0, 1, 5] = -9, 1 << 40
    check(run_tree(to_gpu(c)), *exact_tree(c))


def test_tree_attention_layouts():
    """Queries and drafted rows in other orders, a mask that is a slice, tensors that are not 16-byte aligned."""
    c = tree_case(9, 2, 2, 4, 6, 90, BF)
    want, tol = exact_tree(c)
    g = to_gpu(c)
    big = torch.zeros(2, 9, 13, dtype=torch.bool, device=DEV)
    big[:, 2:8, 5:11] = g["mask"]
    variants = [dict(g, mask=big[:, 2:8, 5:11]), dict(g, mask=g["mask"].transpose(1, 2).contiguous().transpose(1, 2)),
                dict(g, q=g["q"].permute(2, 0, 1, 3).contiguous().permute(1, 2, 0, 3)),
                dict(g, dk=g["dk"].transpose(1, 2).contiguous().transpose(1, 2), dv=g["dv"].transpose(0, 1).contiguous().transpose(0, 1))]
    for name in ("q", "dk", "dv"):
        flat = torch.zeros(g[name].numel() + 8, dtype=BF, device=DEV)
        flat[3:3 + g[name].numel()] = g[name].reshape(-1)
        variants.append(dict(g, **{name: flat[3:3 + g[name].numel()].view(g[name].shape)}))
    for x in variants:
        check(run_tree(x), want, tol)


def test_tree_attention_beyond_32_bits():
    """A K/V tensor of more than 2^32 bytes: the last (b, h) row, and the last rows of all."""
    bs, h, rows = 8, 8, 270000
    k = torch.zeros(bs, h, rows, D, dtype=BF, device=DEV)
    g = torch.Generator().manual_seed(1)
    tail = _randn(g, 500, D)
    k[-1, -1, -500:] = tail.to(DEV)
    c = tree_case(2, 1, 1, 4, 5, 500, BF)
    c["segs"] = [(tail.view(1, 1, 500, D), tail.view(1, 1, 500, D), 0, 500)]
    want, tol = exact_tree(c)
    x = {n: torch.zeros(bs, *c[n].shape[1:2], h * c[n].shape[2], D, dtype=BF, device=DEV) for n in ("q", "dk", "dv")}
    for n in x:
        x[n][-1, :, -c[n].shape[2]:] = c[n][0].to(DEV)
    mask = torch.zeros(bs, 5, 5, dtype=torch.bool, device=DEV)
    mask[-1] = c["mask"][0].to(DEV)
    got = run_tree(dict(x, segs=[(k, k, rows - 500, 500)], mask=mask, rk=None))
    check(got[-1:, :, -4:], want, tol)


def test_tree_attention_streams_and_graphs():
    """Two captured graphs, replayed in turn with eager calls between, on inputs that change; a call on a stream of its own."""
    cases = [to_gpu(tree_case(20 + i, 1, 2, 4, 5, 3000, BF)) for i in range(2)]
    outs, graphs = [], []
    for c in cases:
        run_tree(c)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(run_tree(c))
        graphs.append(graph)
    for turn in range(4):
        for c in cases:
            c["q"].mul_(-1.25)
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for c, out in zip(cases, outs):
            want = run_tree(c)
            torch.cuda.synchronize()
            assert torch.equal(out, want), turn
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [run_tree(c) for c in cases]
    both = [run_tree(c) for c in cases]
    torch.cuda.synchronize()
    for a, b in zip(got, both):
        assert torch.equal(a, b)


def test_tree_counts_may_change_between_replays():
    """A captured call deals its splits out by the counts of each replay, with a workspace of its own."""
    from pariskv_amd import ops

    c = tree_case(5, 3, 2, 4, 9, 4000, BF, mask="tree", ragged=True)
    g = to_gpu(c)
    att = ops.TreeAttention(3, 2, 4, 9, 4000, DEV)
    run = lambda rk: att.run(g["q"], g["segs"], g["dk"], g["dv"], mask=g["mask"], row_keys=rk)
    held = g["rk"].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(held)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run(held)
        graphs.append((graph, out))
    for counts in ([4000] * 6, [0, 4000, 0, 0, 0, 7], [1, 2, 3, 4, 5, 6], [-3, 100, 3999, 4001, 64, 0]):
        held.copy_(torch.tensor(counts, dtype=torch.int32).view(3, 2))
        eager = run(held)
        for graph, out in graphs:
            out.fill_(7.0)
            graph.replay()
        torch.cuda.synchronize()
        c["rk"] = held.cpu()
        check(eager, *exact_tree(c))
        assert all(torch.equal(out, eager) for _, out in graphs)


@pytest.mark.parametrize("bs,h,group,t,dtype", [(2, 2, 2, 5, BF), (1, 3, 7, 7, BF), (2, 2, 4, 40, BF), (1, 2, 3, 9, F32), (2, 1, 2, 4, F32)])
@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("sizes", [(300, 1, 40, 700), (3, 64, 64, 0), (1, 2, 3, 4), (0, 500, 0, 33)])
def test_tree_segments_in_any_tensors(bs, h, group, t, dtype, ragged, sizes):
    """Four segments in four tensors, two of them selected (one with numbers out of range: the nearest row), short ones side by side in a turn."""
    g = torch.Generator().manual_seed(sum(sizes) + t)
    c = tree_case(3, bs, h, group, t, 0, dtype, mask="tree")
    for i, n in enumerate(sizes):
        k, v = _randn(g, bs, h, 900, D, dtype=dtype), _randn(g, bs, h, 900, D, dtype=dtype)
        if i % 2:
            idx = torch.randint(-5 if i == 3 else 0, 1000 if i == 3 else 890, (bs, h, n + 2), generator=g)
            c["segs"].append((k, v, 7, n, idx))
        else:
            c["segs"].append((k, v, 11 * i, n))
    if ragged:
        c["rk"] = torch.randint(-1, sum(sizes) + 2, (bs, h), generator=g, dtype=torch.int32)
    check(run_tree(to_gpu(c)), *exact_tree(c))


@pytest.mark.parametrize("bs,h,group,t,dtype", [(1, 1, 2, 3, BF), (2, 4, 4, 3, BF), (8, 8, 2, 6, BF), (5, 13, 1, 9, BF), (3, 4, 7, 7, F32), (1, 3, 8, 20, BF)])
@pytest.mark.parametrize("counts", ["none", "all", "one", "ramp", "ones"])
def test_tree_key_counts(bs, h, group, t, dtype, counts):
    """Splits go to rows by their keys: all of them to one row, none, as many as there are turns, more rows than are dealt out that way."""
    rows = 5000 if bs * h < 20 else 700
    c = tree_case(9, bs, h, group, t, rows, dtype)
    n = torch.arange(bs * h, dtype=torch.int32)
    c["rk"] = {"none": -n, "all": n * 0 + rows + 5, "one": (n == bs * h // 2) * rows, "ramp": n * rows // (bs * h), "ones": n * 0 + 1}[counts].to(torch.int32).view(bs, h)
    want, tol = exact_tree(c)
    g = to_gpu(c)
    y = run_tree(g)
    check(y, want, tol)
    assert torch.equal(y, run_tree(g))


# ------------------------------------------------------------- 4-bit weights


def w4_case(seed, n, k, group):
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 16, (n, k), generator=g, dtype=torch.uint8)
    scales = (torch.rand(n, k // group, generator=g) * 0.05 + 0.001).to(BF)
    zeros = torch.randint(0, 16, (n, k // group), generator=g, dtype=torch.uint8)
    return codes, scales, zeros


def exact_w4(w):
    codes, scales, zeros = (t.double() for t in w)
    rep = codes.shape[1] // scales.shape[1]
    s, z = scales.repeat_interleave(rep, 1), zeros.repeat_interleave(rep, 1)
    return s * (codes - z), s * (32 + codes + z)


def handle(w):
    from pariskv_amd import ops

    return ops.W4Weight.from_codes(*(t.to(DEV) for t in w))


def exact_linear(x, w, bias, dtype):
    real, size = exact_w4(w)
    x = x.double()
    y = x @ real.T + (0 if bias is None else bias.double())
    k = x.shape[-1]
    return y, (148 + k / 128) * U * (x.abs() @ size.T) + HALF[dtype] * y.abs()


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("n", [1, 15, 16, 17, 100, 1000])
def test_w4_pack_and_unpack(group, n):
    for k in (group, 3 * group, 128 + group):
        if k % group:
            continue
        w = w4_case(n + k, n, k, group)
        real, _ = exact_w4(w)
        assert torch.equal(handle(w).dequantize().double().cpu(), real.float().double())


@pytest.mark.parametrize("m", [1, 2, 3, 8, 15, 16, 17, 31, 32, 33, 48, 50, 64, 65, 130])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_w4_linear_rows(m, group):
    from pariskv_amd import ops

    n, k = 203, 5 * group + (group if group != 128 else 0)
    w = w4_case(m, n, k, group)
    g = torch.Generator().manual_seed(m)
    x, bias = _randn(g, m, k), _randn(g, n)
    for b, dtype in ((None, BF), (bias, BF), (bias, F32)):
        y = ops.w4_linear(x.to(DEV), handle(w), None if b is None else b.to(DEV), dtype)
        assert y.dtype == dtype
        check(y, *exact_linear(x, w, b, dtype))


@pytest.mark.parametrize("n,k,group", [(1, 32, 32), (16, 128, 128), (17, 160, 32), (4096, 4096, 128), (1003, 1184, 32), (300, 12288, 64), (6144, 512, 64)])
@pytest.mark.parametrize("m", [1, 5, 40])
def test_w4_linear_sizes(n, k, group, m):
    from pariskv_amd import ops

    w = w4_case(n + k, n, k, group)
    x = _randn(torch.Generator().manual_seed(k), m, k)
    y = ops.w4_linear(x.to(DEV), handle(w), out_dtype=F32)
    want, tol = exact_linear(x, w, None, F32)
    check(y, want, tol)
    # and over all elements: a rounding of 2^-25 rms of partial sums of up to 31 sqrt(128) |x|, twice, against 4.6 sqrt(K) |x|: 6e-7
    if n * m > 100 and k > 500:
        assert (y.double().cpu() - want).norm() <= 2.0 ** -20 * want.norm()


# a few rows that stay in LDS: all of it, more than a workgroup's share of row tiles, tiles shared by fewer waves; rows that do not fit; columns
# split over workgroups, with an odd run of chunks at the end and with rows of the result that are not a multiple of four long; more rows that fit
@pytest.mark.parametrize("m,n,k,group", [(13, 50, 4096, 128), (3, 16500, 1024, 128), (2, 20011, 256, 32), (16, 5000, 640, 64), (5, 100, 16384, 128),
                                         (40, 64, 4224, 128), (20, 131, 8192, 32), (64, 4096, 2048, 64),
                                         (33, 5000, 896, 128), (100, 700, 160, 32), (64, 17000, 384, 64), (17, 90, 1920, 128), (32, 1003, 64, 32)])
def test_w4_ways(m, n, k, group):
    from pariskv_amd import ops

    a, b = w4_case(n + k, n, k, group), w4_case(n, n, k, group)
    g = torch.Generator().manual_seed(k)
    x, bias = _randn(g, m, k), _randn(g, n)
    gx, ha, hb = x.to(DEV), handle(a), handle(b)
    y = ops.w4_linear(gx, ha, bias.to(DEV), F32)
    check(y, *exact_linear(x, a, bias, F32))
    z = ops.w4_silu_mul(gx, ha, hb)
    (ya, ta), (yb, tb) = exact_linear(x, a, None, F32), exact_linear(x, b, None, F32)
    want = ya * torch.sigmoid(ya) * yb
    check(z, want, 1.1 * ta * (yb.abs() + tb) + ya.abs() * tb + 8 * U * want.abs() + HALF[BF] * want.abs() + 1e-37)
    for _ in range(2):
        assert torch.equal(y, ops.w4_linear(gx, ha, bias.to(DEV), F32)) and torch.equal(z, ops.w4_silu_mul(gx, ha, hb))


@pytest.mark.parametrize("m,n,k,group", [(3, 500, 1024, 128), (48, 500, 4096, 64), (40, 700, 640, 32)])
def test_w4_captured_calls_keep_their_own_shares(m, n, k, group):
    """Two captured graphs and eager calls in turn, on rows that change: every replay is the eager result."""
    from pariskv_amd import ops

    ha, hb = handle(w4_case(1, n, k, group)), handle(w4_case(2, n, k, group))
    g = torch.Generator().manual_seed(k)
    held = _randn(g, m, k).to(DEV)
    both = lambda: (ops.w4_linear(held, ha), ops.w4_silu_mul(held, ha, hb))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = both()
        graphs.append((graph, outs))
    for _ in range(4):
        held.copy_(_randn(g, m, k))
        want = both()
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for _, outs in graphs for x, y in zip(outs, want))


def test_w4_linear_layouts_and_odd_values():
    from pariskv_amd import ops

    w = w4_case(1, 77, 256, 64)
    h = handle(w)
    g = torch.Generator().manual_seed(2)
    x = _randn(g, 6, 300)
    want, tol = exact_linear(x[:, 8:264], w, None, BF)
    gx = x.to(DEV)
    check(ops.w4_linear(gx[:, 8:264], h), want, tol)                       # rows apart by 300: not a multiple of 8, copied
    padded = torch.zeros(6, 304, dtype=BF, device=DEV)
    padded[:, :300] = gx
    check(ops.w4_linear(padded[:, 8:264], h), want, tol)                   # read in place
    check(ops.w4_linear(padded[:, 8:264].t().contiguous().t(), h), want, tol)
    check(ops.w4_linear(gx[:, 8:264].reshape(2, 3, 256), h).view(6, 77), want, tol)
    check(ops.w4_linear(gx[0, 8:264], h), want[0], tol[0])
    one = gx[:1, 8:264].contiguous()
    assert torch.equal(ops.w4_linear(one.expand(6, 256), h), ops.w4_linear(one, h).expand(6, 77))
    assert ops.w4_linear(gx[:0, 8:264], h).shape == (0, 77)
    # a row with NaN or infinity is its own matter; a zero scale is a zero weight
    gx = padded[:, 8:264].clone()
    gx[2, 5], gx[4, 100] = float("nan"), float("inf")
    y = ops.w4_linear(gx, h)
    rest = [0, 1, 3, 5]
    check(y[rest], want[rest], tol[rest])
    assert y[2].isnan().all() and not torch.isfinite(y[4]).all()
    codes, scales, zeros = w4_case(3, 40, 128, 128)
    scales[::2] = 0
    y = ops.w4_linear(padded[:, :128], handle((codes, scales, zeros)))
    assert (y[:, ::2] == 0).all() and (y[:, 1::2] != 0).any()


@pytest.mark.parametrize("m", [1, 7, 16, 17, 40, 64, 70])
@pytest.mark.parametrize("n,k,group", [(1, 32, 32), (50, 384, 128), (501, 704, 64), (1500, 2048, 32)])
def test_w4_silu_mul(m, n, k, group):
    from pariskv_amd import ops

    a, b = w4_case(n, n, k, group), w4_case(n + 1, n, k, group)
    x = _randn(torch.Generator().manual_seed(m), m, k)
    y = ops.w4_silu_mul(x.to(DEV), handle(a), handle(b))
    (ya, ta), (yb, tb) = exact_linear(x, a, None, F32), exact_linear(x, b, None, F32)
    want = ya * torch.sigmoid(ya) * yb
    # |silu'| <= 1.1, |silu(a)| <= |a|; the exponential and the division: 8 u
    tol = 1.1 * ta * (yb.abs() + tb) + ya.abs() * tb + 8 * U * want.abs() + HALF[BF] * want.abs() + 1e-37
    check(y, want, tol)


def test_w4_silu_mul_saturates():
    from pariskv_amd import ops

    codes = torch.full((16, 32), 15, dtype=torch.uint8)
    up = (codes, torch.ones(16, 1, dtype=BF), torch.full((16, 1), 14, dtype=torch.uint8))     # weights of 1
    x = torch.zeros(4, 32, dtype=BF)
    x[:, 0] = torch.tensor([200.0, -200.0, 0.0, -30.0]).to(BF)
    y = ops.w4_silu_mul(x.to(DEV), handle(up), handle(up)).double().cpu()
    want = (x[:, :1].double() ** 2 * torch.sigmoid(x[:, :1].double())).expand(4, 16)
    assert (y - want).abs().max() <= 2.0 ** -8 * 40000 and (y[1] == 0).all() and (y[2] == 0).all()
    assert ((y[3] - want[3]).abs() <= 2.0 ** -7 * want[3].abs()).all()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("n,k,group", [(1, 32, 32), (33, 256, 64), (200, 1280, 128), (64, 96, 32)])
def test_w4_quantize(dtype, n, k, group):
    from pariskv_amd import ops

    g = torch.Generator().manual_seed(n)
    w = (torch.randn(n, k, generator=g) * torch.rand(n, 1, generator=g)).to(dtype)
    w[0, :group] = 0
    if n > 30:
        w[1], w[2], w[3, :group] = w[1].abs(), -w[2].abs(), 0.5
    wide = torch.zeros(n, k + 5, dtype=dtype, device=DEV)
    wide[:, :k] = w.to(DEV)
    for src in (w.to(DEV), wide[:, :k]):
        codes, scales, zeros = (t.cpu() for t in ops.w4_quantize(src, group))
        x = w.float().view(n, -1, group)
        lo, hi = x.amin(-1).clamp(max=0), x.amax(-1).clamp(min=0)
        want_s = ((hi - lo) / 15).to(BF)
        assert torch.equal(scales, want_s)
        s = want_s.float()
        z = torch.where(s > 0, (-lo / s).round().clamp(0, 15), torch.zeros(()))
        q = torch.where(s.unsqueeze(-1) > 0, ((x / s.unsqueeze(-1)).round() + z.unsqueeze(-1)).clamp(0, 15), torch.zeros(()))
        assert torch.equal(zeros, z.to(torch.uint8)) and torch.equal(codes.view(n, -1, group), q.to(torch.uint8))
    # a weight comes back within half a step, and a step more where the scale's own rounding clips the ends (15 * 2^-9 steps)
    real = ops.W4Weight.quantize(w.to(DEV), group).dequantize().cpu().view(n, -1, group)
    assert ((real - x).abs() <= (1.0 + 15 * 2.0 ** -8) * s.unsqueeze(-1)).all()


# ------------------------------------------------------------- the accepted path


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("norms", [False, True])
@pytest.mark.parametrize("layers,bs,h,t,n", [(1, 1, 1, 1, 1), (3, 2, 4, 7, 5), (5, 3, 2, 16, 16), (49, 1, 2, 3, 2)])
def test_path_append(dtype, norms, layers, bs, h, t, n):
    """Every row of the caches and norms is as an append token by token leaves it, to the bit."""
    from pariskv_amd import ops

    g = torch.Generator().manual_seed(layers)
    rows = n + 9
    draft = _randn(g, layers, bs, t, 2 * h, D, dtype=dtype).to(DEV)
    dk, dv = draft[:, :, :, :h], draft[:, :, :, h:]
    k, v = (_randn(g, layers, bs, h, rows, D, dtype=dtype).to(DEV) for _ in range(2))
    vn = torch.rand(layers, bs, h, rows, generator=g).to(DEV) if norms else None
    wk, wv, wn = k.clone(), v.clone(), None if vn is None else vn.clone()
    path = torch.rand(bs, t, generator=g).argsort(-1)[:, :n].contiguous()
    if t > 1:
        path[-1, -1], path[0, 0] = -1, t  # padding, and a token that does not exist
    slots = [i % 9 for i in range(layers)]
    for l, slot in enumerate(slots):
        for i in range(n):
            for b in range(bs):
                p = int(path[b, i])
                if 0 <= p < t:
                    ops.append_kv(dk[l, b:b + 1, p:p + 1], dv[l, b:b + 1, p:p + 1], wk[l, b:b + 1], wv[l, b:b + 1], slot + i,
                                  None if wn is None else wn[l, b:b + 1])
    for form in range(2):
        gk, gv, gn = k.clone(), v.clone(), None if vn is None else vn.clone()
        plan = ops.PathAppend(list(gk), list(gv), None if gn is None else list(gn))
        plan.launch(dk if form else list(dk), dv if form else [x.clone().contiguous() for x in dv], path.to(DEV), slots)
        assert torch.equal(gk, wk) and torch.equal(gv, wv) and (gn is None or torch.equal(gn, wn))
        plan.launch(dk, dv, path[:, :0].to(DEV), slots)
        assert torch.equal(gk, wk)
    # one slot for all, a path that is a slice of a wider one, captured and replayed on other tokens
    gk, gv = wk.clone(), wv.clone()
    plan = ops.PathAppend(list(gk), list(gv))
    wide = torch.zeros(bs, n + 3, dtype=torch.int64, device=DEV)
    plan.launch(dk, dv, wide[:, 1:1 + n], 2)
    torch.cuda.synchronize()
    assert torch.equal(gk[:, :, :, 2:2 + n], dk[:, :, :1].transpose(2, 3).expand(-1, -1, -1, n, -1)) and torch.equal(gv[:, :, :, 2 + n:], wv[:, :, :, 2 + n:])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan.launch(dk, dv, wide[:, 1:1 + n], 2)
    for p in (t - 1, 0, t - 1):
        wide.fill_(p)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(gv[:, :, :, 2:2 + n], dv[:, :, p:p + 1].transpose(2, 3).expand(-1, -1, -1, n, -1))


# ------------------------------------------------------------- 4-bit products at the ends of their range


@pytest.mark.parametrize("m", [1, 5, 16, 20, 40, 70])
@pytest.mark.parametrize("k,group", [(160, 32), (192, 64), (1056, 32), (16480, 32)])
def test_w4_large_rows_in_front_of_padded_columns(m, k, group):
    """A chunk that the columns do not fill is padded with nothing: x whose first columns add up to nearly the 10^37 that a group may have,
    from rows that stay in LDS and rows that are streamed."""
    from pariskv_amd import ops

    n = 77
    a, b = w4_case(k, n, k, group), w4_case(k + 1, n, k, group)
    x = _randn(torch.Generator().manual_seed(m), m, k)
    x[:, 8:group] = 0
    x[0::2, :8], x[1::2, :8] = 1.15e36, -1.15e36
    assert 8.9e36 < x[:, :group].double().abs().sum(1).max() < 1e37
    check(ops.w4_linear(x.to(DEV), handle(a), out_dtype=F32), *exact_linear(x, a, None, F32))
    small = lambda w: (w[0], (w[1].float() * 2.0 ** -110).to(BF), w[2])   # the product of both projections stays finite
    a, b = small(a), small(b)
    z = ops.w4_silu_mul(x.to(DEV), handle(a), handle(b))
    (ya, ta), (yb, tb) = exact_linear(x, a, None, F32), exact_linear(x, b, None, F32)
    want = ya * torch.sigmoid(ya) * yb
    check(z, want, 1.1 * ta * (yb.abs() + tb) + ya.abs() * tb + 8 * U * want.abs() + HALF[BF] * want.abs() + 1e-37)


@pytest.mark.parametrize("group", [32, 128])
def test_w4_quantize_of_the_largest_weights(group):
    """Weights of up to 10^38: scales, codes and what comes back stay finite, within a step and what the scale's rounding clips."""
    from pariskv_amd import ops

    w = torch.randn(8, 256, generator=torch.Generator().manual_seed(3)).clamp(-3, 3) / 3 * 1e38
    w[0, 0], w[0, 1], w[1], w[2] = 1e38, -1e38, w[1].abs(), -w[2].abs()
    w[1, 0], w[2, 0] = 1e38, -1e38
    real = ops.W4Weight.quantize(w.to(DEV), group).dequantize().cpu()
    scale = ops.w4_quantize(w.to(DEV), group)[1].cpu().float().repeat_interleave(group, 1)
    assert torch.isfinite(real).all() and ((real - w).abs() <= (1.0 + 15 * 2.0 ** -8) * scale).all()


# ------------------------------------------------------------- two row tiles a wave


def one_head(c, b, j):
    """The call of a case's (b, j) alone."""
    bs, _, hq, _ = c["q"].shape
    h = c["dk"].shape[2]
    g = hq // h
    at = lambda x: x[b:b + 1, j:j + 1]
    return dict(q=c["q"][b:b + 1, :, j * g:(j + 1) * g], dk=c["dk"][b:b + 1, :, j:j + 1], dv=c["dv"][b:b + 1, :, j:j + 1],
                segs=[(at(s[0]), at(s[1]), *s[2:4], *[at(i) for i in s[4:]]) for s in c["segs"]],
                mask=c["mask"] if c["mask"] is None or c["mask"].dim() == 2 else c["mask"][b:b + 1], rk=None if c["rk"] is None else at(c["rk"]))


def check_heads(c, got, heads, what=""):
    h = c["dk"].shape[2]
    g = c["q"].shape[2] // h
    for b, j in heads:
        want, tol = exact_tree(one_head(c, b, j))
        check(got[b:b + 1, :, j * g:(j + 1) * g], want, tol, (what, b, j))


# bf16, more than 64 query rows a KV head and at least 1024 keys to a split: a wave takes two tiles of 16 rows.  Row counts that leave the last of
# 128 rows' workgroups nearly empty, part full and full; one split to a head (and no join), and 8 or 16.
TWO_TILES = [(9, 15, 8, 9, 1130, 1), (2, 8, 8, 9, 16500, 16), (1, 8, 3, 43, 16500, 16), (1, 8, 7, 33, 17001, 16), (2, 4, 16, 25, 8300, 8), (1, 8, 16, 32, 8192, 8)]


def two_tiles_case(shape, form, mask, ragged):
    from pariskv_amd import _lib

    bs, h, group, t, rows, splits = shape
    n_rows = bs * h * group * t
    assert _lib.lib().pkv_tree_attention_ws_bytes(_lib.DTYPE_BF16, bs, h, group, t, rows) == (0 if splits == 1 else n_rows * splits * 130 * 4)
    return tree_case(rows + t, bs, h, group, t, rows, BF, form, mask, ragged)


@pytest.mark.parametrize("shape", TWO_TILES)
@pytest.mark.parametrize("form", ["dense", "two", "index", "index_two"])
@pytest.mark.parametrize("mask,ragged", [("tree", False), ("holes", True)])
def test_tree_two_row_tiles(shape, form, mask, ragged):
    c = two_tiles_case(shape, form, mask, ragged)
    g = to_gpu(c)
    got = run_tree(g)
    bs, h, group, t, _, _ = shape
    check_heads(c, got, [(0, 0), (bs - 1, h - 1)], (shape, form))
    assert torch.isfinite(got).all() and torch.equal(got, run_tree(g))
    if ragged:  # the last row has nothing in the cache: tokens whose mask is empty see nothing at all
        assert (got[-1, t // 2, -group:] == 0).all()


@pytest.mark.parametrize("shape", [TWO_TILES[0], TWO_TILES[3], TWO_TILES[4]])
def test_tree_two_row_tiles_of_values_nobody_sees(shape):
    """Infinities and NaN behind row_keys, outside the segments and in drafted tokens that no or one other token sees."""
    c = two_tiles_case(shape, "dense", "tree", True)
    bs, h, group, t, rows, _ = shape
    c["dk"], c["dv"] = c["dk"].clone(), c["dv"].clone()
    odd = [2, t // 2, t - 2]
    c["mask"][:, :, odd] = False
    heads = [(0, 0), (bs - 1, h - 1)]
    clean = dict(c, dk=c["dk"].clone(), dv=c["dv"].clone(), segs=[(s[0].clone(), s[1].clone(), *s[2:]) for s in c["segs"]])
    for i, bad in zip(odd, (float("nan"), float("inf"), float("-inf"))):
        c["dk"][:, i], c["dv"][:, i] = bad, bad
    for k, v, row0, _ in c["segs"]:
        for b in range(bs):
            for j in range(h):
                end = row0 + min(rows, max(0, int(c["rk"][b, j])))
                for x in (k, v):
                    x[b, j, :row0], x[b, j, end:] = float("nan"), float("inf")
    check_heads(clean, run_tree(to_gpu(c)), heads)
    c["dk"][:, odd] = 0.25
    c["mask"][:, t - 1, odd[1]], c["mask"][:, 1, odd[2]] = True, True
    got = run_tree(to_gpu(c)).cpu()
    clean["mask"] = c["mask"].clone()
    rest = [i for i in range(t) if i not in (1, t - 1)]
    for b, j in heads:
        want, tol = exact_tree(one_head(clean, b, j))
        check(got[b:b + 1, rest, j * group:(j + 1) * group], want[:, rest], tol[:, rest])
    assert (got[:, t - 1] == float("inf")).all() and (got[:, 1] == float("-inf")).all()


def test_tree_scores_beyond_10_to_the_16_pick_a_key_of_the_largest():
    """fp32 scores of some 10^16, apart by as much: the weight of one key is 1, or of those that lie closer to the largest than a score's rounding (twice
    130 u S, S the largest sum of |q| |k|) some share it.  The output lies between their values, up to the rounding of a weighted mean of n
    values, 2 (n + 200) u of the largest."""
    for mask in ("tree", "holes"):
        c = tree_case(6, 2, 2, 4, 6, 200, F32, "dense", mask)
        c["q"] = c["q"] * 1e16
        k, v, row0, n = c["segs"][0]
        c["segs"] = [(k.sign(), v, row0, n)]
        c["dk"] = c["dk"].sign()
        got = run_tree(to_gpu(c)).double().cpu()
        alone = 0
        for b in range(2):
            for j in range(2):
                for t in range(6):
                    see = c["mask"][b, t]
                    kk = torch.cat([c["segs"][0][0][b, j, row0:row0 + n], c["dk"][b, see, j]]).double()
                    vv = torch.cat([v[b, j, row0:row0 + n], c["dv"][b, see, j]]).double()
                    for i in range(4):
                        q = c["q"][b, t, 4 * j + i].double()
                        s, size = kk @ q / math.sqrt(D), (kk.abs() @ q.abs()).max() / math.sqrt(D)
                        top = vv[s >= s.max() - 2 * 130 * U * size]
                        slack = 2 * (len(vv) + 200) * U * top.abs().amax()
                        y = got[b, t, 4 * j + i]
                        assert (y >= top.amin(0) - slack).all() and (y <= top.amax(0) + slack).all(), (mask, b, j, t, i)
                        alone += len(top) == 1
        assert alone > 90   # of 96: that is one value for most rows
