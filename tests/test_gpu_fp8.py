"""Operators in eight bits on the GPU, each against its definition in 64 bits: rows written into a cache of e4m3 codes with power-of-two
scales and read back (ops.Fp8KVCache), attention over it (ops.Fp8Attention), rows and norms with a scale each (ops.fp8_rows,
ops.add_rmsnorm_fp8), products (ops.fp8_linear).

Tolerances.  u = 2^-24 is half a step of fp32, h half a step of the output's type (2^-8 bf16, 2^-24 fp32).
Written and read rows: none.  Dividing by a power of two is exact, a code is rounded once, and code times scale has four bits.
Norm: y = t inv w with inv = fp32(1 / sqrt(mean t^2 + eps)) out of 64 bits and two more roundings: off by at most 3 u |y|, so the code lies between
those of y (1 - 4 u) and y (1 + 4 u), and the scale is one of theirs.
Products (of few rows, or with fp32 results; see test_linear_blocks_rounded for the others): with B = sum |x| |w| a path through the sums of k exact products has at most 128 + k/128 + 20 additions, each off by at most a step
(2 u) of B, should an instruction cut off rather than round: 2 (148 + k/128) u B; two scales, 2 u |y|; the bias u (|y| + |bias|); h |y|.
Attention: with A = sum p |v| over the keys a row sees (p the exact weights) and S the largest sum of |q| |k| times the scale: a score is off by at
most 2 * 130 u S (128 exact products, their sum, two scales), which moves a weight by that much and the normaliser by as much again; the sum
over n keys is off by (n + 200) u A (3 n for fp32, whose weights go in three parts), twice with the normaliser.  bf16 weights are rounded by h each and summed up as
they are: h A + h |out|; scales that are no powers of two round them once more: 2 h A.  Together:
A (8 * 130 u S + 2 (n + 200) u + h [bf16]) + h |out| [bf16] + h |out|.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV, D = "cuda:0", 128
U = 2.0 ** -24
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
BF, F32, F64, F8, U8 = torch.bfloat16, torch.float32, torch.float64, torch.float8_e4m3fn, torch.uint8


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _exponent(top):
    """Least e >= -100 with top <= 448 * 2^e; top float64."""
    e = torch.full_like(top, -100.0)
    pos = top > 0
    e[pos] = torch.ceil(torch.log2(top[pos] / 448.0))
    e = torch.where(top > 448.0 * torch.exp2(e), e + 1, e)
    e = torch.where((top <= 448.0 * torch.exp2(e - 1)), e - 1, e)
    return e.clamp(min=-100.0)


def _top(x):
    mag = x.abs()
    return torch.where(torch.isfinite(mag), mag, torch.zeros_like(mag))


def _round(x):
    """Nearest e4m3 number, ties to even, of float64 x; past 448 it is 448, a NaN stays one."""
    y = x.clamp(-448.0, 448.0)
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.where(torch.isnan(x), x, torch.round(y / step) * step)


def same(a, b):
    """Equal, NaN where NaN."""
    a, b = a.to(F64).cpu(), b.to(F64).cpu()
    return a.shape == b.shape and bool(((a == b) | (a.isnan() & b.isnan())).all())


# ------------------------------------------------------------------ the cache


class CacheOracle:
    """A cache as float64 codes and scales on the host."""

    def __init__(self, bs, H, cap, block):
        self.block = block
        self.codes = [torch.zeros(bs, H, cap, D, dtype=F64) for _ in range(2)]
        self.scales = [torch.zeros(bs, H, cap // block, dtype=F64) for _ in range(2)]

    def store(self, k, v, start, lengths=None):
        bs, S = k.shape[:2]
        cap, block = self.codes[0].shape[2], self.block
        for x, codes, scales in zip((k, v), self.codes, self.scales):
            x = x.cpu().to(F64)
            for b in range(bs):
                p0, n = int(start[b]), S if lengths is None else min(int(lengths[b]), S)
                if not 0 <= p0 < cap or n <= 0:
                    continue
                end = min(p0 + n, cap)
                for i in range(p0 // block, (end - 1) // block + 1):
                    lo, hi = max(p0, i * block), min(end, (i + 1) * block)
                    new = x[b, lo - p0:hi - p0].transpose(0, 1)
                    need = torch.exp2(_exponent(_top(new).amax((1, 2))))
                    if lo > i * block:
                        was = scales[b, :, i].clone()
                        s = torch.maximum(was, need)
                        old = slice(i * block, lo)
                        codes[b, :, old] = _round(codes[b, :, old] * (was / s).view(-1, 1, 1))
                    else:
                        s = need
                    codes[b, :, lo:hi] = _round(new / s.view(-1, 1, 1))
                    scales[b, :, i] = s

    def values(self, which):
        return self.codes[which] * self.scales[which].repeat_interleave(self.block, -1).unsqueeze(-1)

    def check(self, cache):
        for codes, scales, want, want_s in zip((cache.k, cache.v), (cache.k_scale, cache.v_scale), self.codes, self.scales):
            assert same(scales, want_s)
            assert same(codes.float(), want)


def _ops():
    from pariskv_amd import ops

    return ops


def _rows(g, *shape, dtype=BF, spread=1.0):
    return (torch.randn(*shape, generator=g) * torch.exp(spread * torch.randn(*shape[:-1], 1, generator=g))).to(dtype)


@pytest.mark.parametrize("block", [16, 32, 64, 128])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_store_prompt_then_tokens(block, dtype):
    ops, g = _ops(), _gen(block)
    bs, H, S, cap = 2, 3, 150, 300
    cache = ops.Fp8KVCache(bs, H, cap, DEV, block=block)
    assert cache.capacity % block == 0 and cache.capacity - cap < block
    want = CacheOracle(bs, H, cache.capacity, block)
    x = _rows(g, bs, S, 2 * H + 5, D, dtype=dtype)
    k, v = x[:, :, 5:5 + H], x[:, :, 5 + H:]
    cache.store(k.to(DEV), v.to(DEV))
    want.store(k, v, [0] * bs)
    want.check(cache)
    at = S
    for t in range(12):  # some louder than all before, some with nothing in them
        x = _rows(g, bs, 1, 2 * H, D, dtype=dtype) * (0.0 if t == 5 else 3.0 ** (t % 4))
        x = x.to(DEV)
        cache.store(x[:, :, :H], x[:, :, H:], at + t)
        want.store(x[:, :, :H], x[:, :, H:], [at + t] * bs)
    want.check(cache)
    for d in (BF, F32):
        k, v = cache.read(0, S + 12, dtype=d)
        assert same(k, want.values(0)[:, :, :S + 12]) and same(v, want.values(1)[:, :, :S + 12])


@pytest.mark.parametrize("S", [1, 2, 17, 64, 65, 200])
def test_store_ragged(S):
    ops, g = _ops(), _gen(S)
    bs, H, cap, block = 6, 2, 256, 32
    cache = ops.Fp8KVCache(bs, H, cap, DEV, block=block)
    want = CacheOracle(bs, H, cap, block)
    first = _rows(g, bs, cap, 2 * H, D).to(DEV)
    cache.store(first[:, :, :H], first[:, :, H:])
    want.store(first[:, :, :H], first[:, :, H:], [0] * bs)
    starts = torch.tensor([0, 31, -1, cap - 1, cap, 45], dtype=torch.int32)
    lengths = torch.tensor([S, S // 2 + 1, S, S + 100, S, 0], dtype=torch.int32)
    x = _rows(g, bs, S, 2 * H, D, spread=2.0).to(DEV)
    for use in (None, lengths):
        cache.store(x[:, :, :H], x[:, :, H:], starts.to(DEV), lengths=None if use is None else use.to(DEV))
        want.store(x[:, :, :H], x[:, :, H:], starts, use)
        want.check(cache)


def test_store_extremes():
    """Infinities, NaN, zeros, the least and largest scales; a block's codes after its scale has grown twice."""
    ops, g = _ops(), _gen(1)
    bs, H, block = 1, 2, 16
    cache = ops.Fp8KVCache(bs, H, 64, DEV, block=block)
    want = CacheOracle(bs, H, 64, block)
    x = torch.randn(bs, 48, 2 * H, D, generator=g)
    x[0, 3, 0, 5], x[0, 4, 1, 6], x[0, 5, 2, 7] = math.inf, -math.inf, math.nan
    x[0, 6] = 0.0
    x[0, 16:32] = 0.0               # a block of nothing
    x[0, 32:40] *= 1e-37            # below the least scale
    x[0, 40:48] *= 2e36
    for a, b in ((0, 48),):
        cache.store(x[:, a:b, :H].to(DEV), x[:, a:b, H:].to(DEV), a)
        want.store(x[:, a:b, :H], x[:, a:b, H:], [a])
    want.check(cache)
    for t, loud in enumerate((0.01, 1.0, 1.0, 77.0, 0.1, 1e5)):
        y = torch.randn(bs, 1, 2 * H, D, generator=g).to(BF) * loud
        cache.store(y[:, :, :H].to(DEV), y[:, :, H:].to(DEV), 48 + t)
        want.store(y[:, :, :H], y[:, :, H:], [48 + t])
        want.check(cache)
    every = torch.cat([torch.arange(2 ** 15, dtype=torch.int32), torch.arange(2 ** 15, dtype=torch.int32) - 2 ** 15]).to(torch.int16).view(BF)
    every = every.view(1, 512, 1, D).expand(1, 512, 1, D)  # every bf16 number; those past 10^38 are not promised
    every = torch.where(every.abs() > 1e38, torch.where(every.isfinite(), torch.zeros((), dtype=BF), every), every).contiguous()
    cache, want = ops.Fp8KVCache(1, 1, 512, DEV, block=16), CacheOracle(1, 1, 512, 16)
    cache.store(every.to(DEV), every.to(DEV))
    want.store(every, every, [0])
    want.check(cache)


def test_store_leaves_the_rest():
    ops, g = _ops(), _gen(2)
    bs, H, cap, block = 2, 2, 128, 64
    cache = ops.Fp8KVCache(bs, H, cap, DEV, block=block)
    for t in (cache.k, cache.v):
        t.view(U8).fill_(0x7f)  # NaN: nothing may come of them
    cache.k_scale.fill_(3.0), cache.v_scale.fill_(5.0)
    x = _rows(g, bs, 10, 2 * H, D).to(DEV)
    cache.store(x[:, :, :H], x[:, :, H:], 64)
    for t, s, old in ((cache.k, cache.k_scale, 3.0), (cache.v, cache.v_scale, 5.0)):
        t = t.view(U8)
        assert bool((t[:, :, :64] == 0x7f).all()) and bool((t[:, :, 74:] == 0x7f).all()) and not bool((t[:, :, 64:74] == 0x7f).any())
        assert bool((s[:, :, 0] == old).all())


@pytest.mark.parametrize("what", ["odd", "misaligned", "transposed", "expanded"])
def test_store_layouts(what):
    ops, g = _ops(), _gen(3)
    bs, H, S, block = 2, 2, 33, 16
    if what == "odd":
        x = _rows(g, bs, S, H * D + 3).to(DEV)[:, :, :H * D].view(bs, S, H, D)
    elif what == "misaligned":
        x = _rows(g, bs * S * H * D + 1, 1).to(DEV).view(-1)[1:].view(bs, S, H, D)
    elif what == "transposed":
        x = _rows(g, bs, H, D, S).to(DEV).permute(0, 3, 1, 2)
    else:
        x = _rows(g, 1, S, 1, D).to(DEV).expand(bs, S, H, D)
    cache, want = ops.Fp8KVCache(bs, H, 64, DEV, block=block), CacheOracle(bs, H, 64, block)
    cache.store(x, x.flip(1), 7)
    want.store(x, x.flip(1), [7] * bs)
    want.check(cache)


def _filled(ops, g, bs, H, cap, block, n=None, spread=1.0, host=False):
    cache, want = ops.Fp8KVCache(bs, H, cap, DEV, block=block, host=host), CacheOracle(bs, H, -(-cap // block) * block, block)
    n = cap if n is None else n
    x = _rows(g, bs, n, 2 * H, D, spread=spread)
    cache.store(x[:, :, :H].to(DEV), x[:, :, H:].to(DEV))
    want.store(x[:, :, :H], x[:, :, H:], [0] * bs)
    return cache, want


@pytest.mark.parametrize("host", [False, True])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_read(dtype, host):
    ops, g = _ops(), _gen(4)
    bs, H, cap = 2, 3, 200
    cache, want = _filled(ops, g, bs, H, cap, 32, host=host)
    torch.cuda.synchronize()
    assert cache.host == host
    want.check(cache)
    k, v = want.values(0), want.values(1)
    for row0, n in ((0, None), (0, 1), (5, 130), (cache.capacity - 1, 1), (3, 0)):
        a, b = cache.read(row0, n, dtype=dtype)
        m = cache.capacity - row0 if n is None else n
        assert a.dtype == dtype and same(a, k[:, :, row0:row0 + m]) and same(b, v[:, :, row0:row0 + m])
    idx = torch.randint(0, cap, (bs, H, 77), generator=g)
    idx[0, 0, 3] = idx[0, 0, 4]  # twice
    a, b = cache.read(idx=idx.to(DEV), dtype=dtype)
    at = idx.unsqueeze(-1).expand(-1, -1, -1, D)
    assert same(a, k.gather(2, at)) and same(b, v.gather(2, at))
    bad = idx.clone()
    bad[0, 1, 5], bad[1, 2, 6], bad[1, 0, 0], bad[0, 0, 0] = -1, cache.capacity - 7, 2 ** 62, -2 ** 62
    a, b = cache.read(7, 50, idx=bad.to(DEV), dtype=dtype)
    off = (bad < 0) | (bad >= cache.capacity - 7)
    at = (bad.clamp(0, cache.capacity - 8) + 7).unsqueeze(-1).expand(-1, -1, -1, D)
    for x, y in ((a, k), (b, v)):
        assert same(x, torch.where(off.unsqueeze(-1), torch.zeros((), dtype=F64), y.gather(2, at))[:, :, :50])
    # behind the dense rows of a wider tensor, everything else left as it is
    wide = [torch.full((bs, H, 100, D), 9.0, dtype=dtype, device=DEV) for _ in range(2)]
    cache.read(2, 60, out=[t[:, :, 20:80] for t in wide], dtype=dtype)
    for t, y in zip(wide, (k, v)):
        assert same(t[:, :, 20:80], y[:, :, 2:62]) and bool((t[:, :, :20] == 9).all()) and bool((t[:, :, 80:] == 9).all())


def test_host_cache_grows():
    ops, g = _ops(), _gen(5)
    cache, want = _filled(ops, g, 1, 2, 96, 32, n=70, host=True)
    for t in range(8):
        x = _rows(g, 1, 1, 4, D) * 2.0 ** t
        cache.store(x[:, :, :2].to(DEV), x[:, :, 2:].to(DEV), 70 + t)
        want.store(x[:, :, :2], x[:, :, 2:], [70 + t])
    torch.cuda.synchronize()
    want.check(cache)


# ------------------------------------------------------------------ attention


def check_attention(out, q, want, segments, row_keys=None, scale=None, extra=0.0):
    """out against the definition in 64 bits; segments with host indices."""
    q = q.cpu()
    bs, T, Hq, _ = q.shape
    k, v = want.values(0), want.values(1)
    H, cap = k.shape[1], k.shape[2]
    G, dt = Hq // H, q.dtype
    scale = 1 / math.sqrt(D) if scale is None else scale
    out = out.cpu().to(F64)
    h = HALF[dt]
    for b in range(bs):
        for j in range(H):
            at = torch.cat([torch.zeros(0, dtype=torch.int64)] + [
                torch.arange(s[0], s[0] + s[1]) if len(s) < 3 else s[0] + s[2][b, j, :s[1]].cpu().clamp(0, cap - 1 - s[0]) for s in segments])
            L = len(at) if row_keys is None else max(0, min(len(at), int(row_keys[b, j])))
            kk, vv = k[b, j][at[:L]], v[b, j][at[:L]]
            for t in range(T):
                n = max(0, L - (T - 1 - t))
                got = out[b, t, j * G:(j + 1) * G]
                if n == 0:
                    assert bool((got == 0).all()), (b, j, t)
                    continue
                qq = q[b, t, j * G:(j + 1) * G].to(F64)
                z = qq @ kk[:n].t() * scale
                p = torch.softmax(z, 1)
                ref = p @ vv[:n]
                bad = ref.isnan()
                assert bool((got.isnan() == bad).all()), (b, j, t, "NaN")
                A = p @ vv[:n].abs()
                S = (qq.abs() @ kk[:n].abs().t() * abs(scale)).amax(1, keepdim=True)
                adds = n if dt == BF else 3 * n
                tol = A * (8 * 130 * U * S + 2 * (adds + 200) * U + (h if dt == BF else 0) + extra) + (2 if dt == BF else 1) * h * ref.abs() + 1e-30
                err = torch.where(bad, torch.zeros_like(ref), (got - ref).abs())
                worst = float((err / tol)[~bad].max()) if bool((~bad).any()) else 0.0
                assert worst <= 1.0, (b, j, t, worst)


def run_attention(ops, q, cache, segments, row_keys=None, **kw):
    segs = [s if len(s) < 3 else (s[0], s[1], s[2].to(DEV)) for s in segments]
    total = sum(s[1] for s in segments)
    plan = ops.Fp8Attention(q.shape[0], cache.n_kv_heads, q.shape[2] // cache.n_kv_heads, q.shape[1], max(total, 1), DEV)
    return plan.run(q.to(DEV), cache, segs, row_keys=None if row_keys is None else row_keys.to(DEV), **kw)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rows", [1, 2, 15, 16, 31, 33, 63, 64, 65, 255, 257, 1000, 5003])
def test_attention_lengths(rows, dtype):
    ops, g = _ops(), _gen(rows)
    bs, H, G = (2, 2, 4) if rows < 3000 else (1, 2, 4)
    cache, want = _filled(ops, g, bs, H, rows, 64, spread=0.5)
    q = torch.randn(bs, 1, H * G, D, generator=g).to(dtype)
    check_attention(run_attention(ops, q, cache, [(0, rows)]), q, want, [(0, rows)])


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("H,G,T", [(1, 1, 1), (2, 7, 5), (1, 16, 1), (1, 17, 1), (2, 8, 4), (1, 5, 13), (1, 2, 64), (2, 1, 33)])
def test_attention_heads_and_tokens(H, G, T, dtype):
    ops, g = _ops(), _gen(H * 100 + G * 10 + T)
    rows = 301
    cache, want = _filled(ops, g, 2, H, rows, 16, spread=0.5)
    q = torch.randn(2, T, H * G, D, generator=g).to(dtype)
    check_attention(run_attention(ops, q, cache, [(0, rows)]), q, want, [(0, rows)])
    few = [(3, 5)]  # fewer keys than tokens: the first ones see nothing
    check_attention(run_attention(ops, q, cache, few), q, want, few)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("block", [16, 32, 64, 128])
def test_attention_segments_and_counts(block, dtype):
    ops, g = _ops(), _gen(block + 1)
    bs, H, G, T, cap = 3, 2, 4, 3, 640
    cache, want = _filled(ops, g, bs, H, cap, block, spread=0.5)
    idx = torch.stack([torch.randperm(400, generator=g)[:150] for _ in range(bs * H)]).view(bs, H, 150)
    idx[0, 0, 7], idx[1, 1, 9] = -5, 2 ** 40  # clamped
    segments = [(0, 33), (64, 130, idx), (500, 77), (5, 20, idx)]
    total = sum(s[1] for s in segments)
    q = torch.randn(bs, T, H * G, D, generator=g).to(dtype)
    check_attention(run_attention(ops, q, cache, segments), q, want, segments)
    row_keys = torch.tensor([[0, 1], [2, total], [total + 100, -7]], dtype=torch.int32)
    check_attention(run_attention(ops, q, cache, segments, row_keys), q, want, segments, row_keys)
    row_keys = torch.tensor([[64, 65], [200, 128], [total - 1, 3]], dtype=torch.int32)
    check_attention(run_attention(ops, q, cache, segments, row_keys), q, want, segments, row_keys)
    empty = run_attention(ops, q, cache, [])
    assert bool((empty == 0).all())
    check_attention(run_attention(ops, q, cache, [(0, 0), (10, 40), (0, 0, idx)], scale=0.3), q, want, [(10, 40)], scale=0.3)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_attention_unseen_nan(dtype):
    """NaN among rows that are not attended to, or only by later tokens, reach no row that does not see them."""
    ops, g = _ops(), _gen(9)
    H, G, T, cap = 2, 4, 6, 192
    cache, want = _filled(ops, g, 1, H, cap, 64, spread=0.3)
    rows = 101
    for t, w in ((cache.k, want.codes[0]), (cache.v, want.codes[1])):
        t.view(U8)[:, :, rows:] = 0x7f
        w[:, :, rows:] = math.nan
    q = torch.randn(1, T, H * G, D, generator=g).to(dtype)
    check_attention(run_attention(ops, q, cache, [(0, rows)]), q, want, [(0, rows)])
    row_keys = torch.tensor([[rows, 70]], dtype=torch.int32)
    check_attention(run_attention(ops, q, cache, [(0, cap)], row_keys), q, want, [(0, cap)], row_keys)
    cache.v.view(U8)[0, 0, rows - 3, 17], want.codes[1][0, 0, rows - 3, 17] = 0xff, math.nan   # a value of the last but two
    cache.k.view(U8)[0, 1, rows - 2, 40], want.codes[0][0, 1, rows - 2, 40] = 0x7f, math.nan   # a key of the last but one
    check_attention(run_attention(ops, q, cache, [(0, rows)]), q, want, [(0, rows)])
    cache.v.view(U8)[0, 0, 5, 99], want.codes[1][0, 0, 5, 99] = 0x7f, math.nan                  # one that all see
    check_attention(run_attention(ops, q, cache, [(0, rows)]), q, want, [(0, rows)])


@pytest.mark.parametrize("dtype", [BF, F32])
def test_attention_scales_and_scores(dtype):
    """Scales of any size, among them none of two's powers, blocks that were never written, scores that climb late and steeply."""
    ops, g = _ops(), _gen(10)
    H, G, cap, block = 2, 4, 1024, 16
    cache, want = _filled(ops, g, 1, H, cap, block, spread=0.3)
    f = (torch.rand(1, H, cap // block, generator=g) + 0.5)
    for s, w, m in ((cache.k_scale, want.scales[0], f), (cache.v_scale, want.scales[1], f.flip(-1))):
        s.mul_(m.to(DEV))
        w.copy_(s.cpu().to(F64))
    cache.v_scale[0, 0, 3], want.scales[1][0, 0, 3] = 0.0, 0.0
    q = torch.randn(1, 1, H * G, D, generator=g).to(dtype)
    check_attention(run_attention(ops, q, cache, [(0, cap)]), q, want, [(0, cap)], extra=2 * 2.0 ** -8 if dtype == BF else 2 * U)
    cache, want = _filled(ops, g, 1, H, cap, block, spread=0.0)
    climb = torch.exp2(torch.arange(cap // block) // 8).to(F32)  # later keys ever larger
    cache.k_scale.mul_(climb.to(DEV))
    want.scales[0] = cache.k_scale.cpu().to(F64)
    check_attention(run_attention(ops, q, cache, [(0, cap)]), q, want, [(0, cap)])


def test_attention_layouts_streams_graph():
    ops, g = _ops(), _gen(11)
    bs, H, G, T, cap = 2, 2, 4, 2, 700
    cache, want = _filled(ops, g, bs, H, cap, 64, spread=0.3)
    wide = torch.randn(bs, T, H * G + 4, D, generator=g).to(BF).to(DEV)
    q = wide[:, :, :H * G]                     # a view into the fused projection
    plan = ops.Fp8Attention(bs, H, G, T, cap, DEV)
    ref = plan.run(q, cache, [(0, cap)])
    check_attention(ref, q, want, [(0, cap)])
    for other in (q.transpose(1, 2).contiguous().transpose(1, 2), torch.cat([q.reshape(-1).new_zeros(1), q.reshape(-1)])[1:].view(q.shape)):
        assert torch.equal(plan.run(other, cache, [(0, cap)]), ref)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = plan.run(q, cache, [(0, cap)])
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(there, ref)
    out = torch.empty(bs, T, H * G, D, dtype=BF, device=DEV)
    assert plan.run(q, cache, [(0, cap)], out=out) is out and torch.equal(out, ref)
    # two captured graphs that write a token, read it back and attend to it
    row = _rows(g, bs, 1, 2 * H, D).to(DEV)
    start = torch.tensor([500, 77], dtype=torch.int32, device=DEV)
    keys = torch.tensor([[501, 501], [78, 78]], dtype=torch.int32, device=DEV)
    q1 = q[:, :1].contiguous()

    def step():
        cache.store(row[:, :, :H], row[:, :, H:], start)
        return plan.run(q1, cache, [(0, cap)], row_keys=keys), *cache.read(0, cap)

    with torch.cuda.stream(side):
        step()
        side.synchronize()
        graphs = []
        for _ in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                outs = step()
            graphs.append((graph, outs))
    torch.cuda.synchronize()
    want.store(row[:, :, :H], row[:, :, H:], start)  # the call before the capture
    for i in range(4):
        row.copy_(_rows(g, bs, 1, 2 * H, D))
        q1.normal_(generator=torch.Generator(device=DEV).manual_seed(i))
        start.add_(1), keys.add_(1)
        for graph, outs in graphs:
            graph.replay()
            torch.cuda.synchronize()
            eager = step()
            torch.cuda.synchronize()
            for a, b in zip(outs, eager):
                assert torch.equal(a, b)
        want.store(row[:, :, :H], row[:, :, H:], start)
        check_attention(graphs[0][1][0], q1, want, [(0, cap)], keys.cpu())


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rows,H", [(4300, 1), (17000, 1), (33000, 2), (66000, 1)])
def test_attention_many_splits(rows, H, dtype):
    """Few heads and long rows: results joined from up to 256 parts, of which those past the row's last key have seen nothing."""
    ops, g = _ops(), _gen(rows)
    cache, want = _filled(ops, g, 1, H, -(-rows // 128) * 128, 128, spread=0.3)
    q = torch.randn(1, 2, H * 3, D, generator=g).to(dtype)
    check_attention(run_attention(ops, q, cache, [(0, rows)]), q, want, [(0, rows)])
    for n in (0, 1, 700, rows // 2):
        rk = torch.full((1, H), n, dtype=torch.int32)
        rk[0, -1] -= n % 2
        check_attention(run_attention(ops, q, cache, [(0, rows)], row_keys=rk), q, want, [(0, rows)], row_keys=rk)


def test_attention_far_rows():
    """Offsets past 2^32 bytes: a head's rows take 2 GiB."""
    ops, g = _ops(), _gen(12)
    H, cap, block = 3, 1 << 24, 128
    cache = ops.Fp8KVCache(1, H, cap, DEV, block=block)
    S = 300
    want = CacheOracle(1, H, 512, block)
    x = _rows(g, 1, S, 2 * H, D, spread=0.3)
    cache.store(x[:, :, :H].to(DEV), x[:, :, H:].to(DEV), cap - 512)
    want.store(x[:, :, :H], x[:, :, H:], [0])
    k, v = cache.read(cap - 512, 512)
    assert same(k, want.values(0)) and same(v, want.values(1))
    q = torch.randn(1, 2, H * 4, D, generator=g).to(BF)
    check_attention(run_attention(ops, q, cache, [(cap - 512, S)]), q, want, [(0, S)])
    idx = torch.randint(0, S, (1, H, 99), generator=g)
    check_attention(run_attention(ops, q, cache, [(0, 99, idx + cap - 512)]), q, want, [(0, 99, idx)])
    assert int(cache.k.view(U8)[:, :, :1 << 20].count_nonzero()) == 0


# ------------------------------------------------------------------ rows and norms


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rows,width", [(1, 1), (3, 7), (2, 128), (5, 129), (4, 1000), (1, 4096), (7, 5120), (2, 16384), (2, 16383), (0, 64)])
def test_rows(rows, width, dtype):
    ops, g = _ops(), _gen(rows * 17 + width)
    x = _rows(g, rows, width, dtype=dtype, spread=3.0)
    if rows > 2:
        x[1] = 0.0
        x[2, 0] = math.inf
        x[2, width - 1] = math.nan
    r = ops.fp8_rows(x.to(DEV))
    x = x.to(F64)
    e = _exponent(_top(x).amax(1)) if rows else x[:, 0]
    assert tuple(r.shape) == (rows, width) and r.codes.dtype == F8 and tuple(r.codes.shape) == (rows, width)
    assert same(r.scales, torch.exp2(e)) and same(r.codes.float(), _round(x / torch.exp2(e).unsqueeze(1)))
    assert not bool(r.padded.view(U8)[:, width:-(-width // 128) * 128].any())


def test_rows_layouts():
    ops, g = _ops(), _gen(20)
    x = _rows(g, 6, 300).to(DEV)
    for y in (x[:, 3:203], x[::2], x.t(), x.view(2, 3, 300), x[0], x[:, :256]):
        r = ops.fp8_rows(y)
        z = y.cpu().to(F64)
        s = torch.exp2(_exponent(z.abs().amax(-1)))
        assert tuple(r.codes.shape) == tuple(y.shape) and same(r.scales, s) and same(r.codes.float(), _round(z / s.unsqueeze(-1)))


@pytest.mark.parametrize("rows,width", [(1, 8), (2, 100), (3, 101), (1, 4096), (9, 4096), (2, 12288), (3, 16384), (2, 16381), (1, 1)])
@pytest.mark.parametrize("residual", [True, False])
def test_add_rmsnorm_fp8(rows, width, residual):
    ops, g = _ops(), _gen(rows + width)
    x, r, w = _rows(g, rows, width, spread=2.0), _rows(g, rows, width), (1 + 0.3 * torch.randn(width, generator=g)).to(BF)
    eps = 1e-6
    if rows > 1:
        x[1], r[1] = 0.0, 0.0
    total, q = ops.add_rmsnorm_fp8(x.to(DEV), r.to(DEV) if residual else None, w.to(DEV), eps)
    t = (x.float() + r.float()).to(BF) if residual else x
    assert torch.equal(total.cpu(), t)
    t = t.to(F64)
    y = t / torch.sqrt(t.square().mean(1, keepdim=True) + eps) * w.to(F64)
    lo, hi = torch.minimum(y * (1 - 4 * U), y * (1 + 4 * U)), torch.maximum(y * (1 - 4 * U), y * (1 + 4 * U))
    top = y.abs().amax(1)
    e0, e1, s = _exponent(top * (1 - 4 * U)), _exponent(top * (1 + 4 * U)), q.scales.cpu().to(F64)
    assert bool(((s == torch.exp2(e0)) | (s == torch.exp2(e1))).all())
    code = q.codes.float().cpu().to(F64)
    assert bool((code >= _round(lo / s.unsqueeze(1))).all()) and bool((code <= _round(hi / s.unsqueeze(1))).all())
    assert not bool(q.padded.view(U8)[:, width:-(-width // 128) * 128].any())


def test_add_rmsnorm_fp8_special():
    ops = _ops()
    x = torch.randn(3, 2, 256, generator=_gen(21)).to(BF)
    x[0, 1, 7], x[1, 0, 9] = math.nan, math.inf
    _, q = ops.add_rmsnorm_fp8(x.to(DEV), None, torch.ones(256, dtype=BF, device=DEV), 1e-6, want_sum=False)
    bad = q.codes.float().isnan().any(-1).cpu()
    assert tuple(q.scales.shape) == (3, 2)
    assert bool(bad[0, 1]) and bool(bad[1, 0]) and int(bad.sum()) == 2
    empty, q = ops.add_rmsnorm_fp8(x[:0].to(DEV), None, torch.ones(256, dtype=BF, device=DEV), 1e-6)
    assert tuple(q.codes.shape) == (0, 2, 256)


# ------------------------------------------------------------------ products


def check_linear(y, xc, sx, wc, sw, bias, out_dtype):
    """xc, wc float64 codes [m,k], [n,k]; sx, sw scales."""
    m, k = xc.shape
    ref = xc @ wc.t() * sx.unsqueeze(1) * sw
    B = xc.abs() @ wc.abs().t() * sx.abs().unsqueeze(1) * sw.abs()
    tol = 2 * (148 + k / 128) * U * B + 2 * U * ref.abs()
    if bias is not None:
        ref = ref + bias.to(F64)
        tol = tol + U * (ref.abs() + bias.to(F64).abs())
    tol = tol + HALF[out_dtype] * ref.abs() + 1e-30
    err = (y.cpu().to(F64) - ref).abs()
    assert bool((err <= tol).all()), float((err / tol).max())


@pytest.mark.parametrize("m", [1, 2, 15, 16, 17, 32, 33, 64, 65, 128, 129, 200, 257])
@pytest.mark.parametrize("n,k", [(64, 128), (100, 300), (16, 4096), (1003, 1185), (300, 129)])
def test_linear(m, n, k):
    ops, g = _ops(), _gen(m * 7 + n + k)
    x, w = _rows(g, m, k), _rows(g, n, k, dtype=F32) / math.sqrt(k)
    bias = torch.randn(n, generator=g).to(BF) if m % 2 else None
    weight, rows = ops.Fp8Weight.quantize(w.to(DEV)), ops.fp8_rows(x.to(DEV))
    sw, sx = torch.exp2(_exponent(w.to(F64).abs().amax(1))), torch.exp2(_exponent(x.to(F64).abs().amax(1)))
    wc, xc = _round(w.to(F64) / sw.unsqueeze(1)), _round(x.to(F64) / sx.unsqueeze(1))
    assert same(weight.dequantize(), wc * sw.unsqueeze(1))
    b = None if bias is None else bias.to(DEV)
    for dt in (BF, F32):
        y = ops.fp8_linear(rows, weight, bias=b, out_dtype=dt)
        assert y.dtype == dt and tuple(y.shape) == (m, n)
        check_linear(y, xc, sx, wc, sw, bias, dt)
    assert torch.equal(ops.fp8_linear(x.to(DEV), weight, bias=b), ops.fp8_linear(rows, weight, bias=b))


def test_linear_large():
    ops, g = _ops(), _gen(31)
    for m, n, k in ((300, 2000, 1000), (520, 1536, 4096), (8, 20000, 256)):
        x, w = _rows(g, m, k, dtype=F32), _rows(g, n, k)
        rows, weight = ops.fp8_rows(x.to(DEV)), ops.Fp8Weight.quantize(w.to(DEV))
        wd = weight.dequantize().cpu().to(F64)
        y = ops.fp8_linear(rows, weight, out_dtype=F32)
        check_linear(y, rows.codes.float().cpu().to(F64), rows.scales.cpu().to(F64), wd, torch.ones(n, dtype=F64), None, F32)


@pytest.mark.parametrize("m,n,k", [(64, 8192, 256), (65, 33000, 130), (130, 20000, 384), (300, 5000, 128), (520, 9001, 1000), (700, 12288, 640)])
@pytest.mark.parametrize("out_dtype", [BF, F32])
def test_linear_blocks(m, n, k, out_dtype):
    """Shapes that go through LDS.  Codes whose products are multiples of 2^-6 up to 2^2: nothing is below 2^-13 of the largest of eight, so the sums are
    exact in fp32 whatever instruction adds them up."""
    ops, g = _ops(), _gen(m + n)
    codes, wcodes = ((torch.randint(0x38, 0x48, (r, k), generator=g) + 128 * torch.randint(0, 2, (r, k), generator=g)).to(U8).to(DEV) for r in (m, n))
    sx, sw = (torch.rand(m, generator=g) + 0.1).to(DEV), (torch.rand(n, generator=g) - 0.5).to(DEV)
    bias = torch.randn(n, generator=g).to(BF).to(DEV) if m % 2 == 0 else None
    y = ops.fp8_linear(ops.Fp8Rows.from_codes(codes, sx), ops.Fp8Weight.from_codes(wcodes, sw), bias=bias, out_dtype=out_dtype)
    ref = codes.view(F8).to(F64) @ wcodes.view(F8).to(F64).t() * sx.to(F64).unsqueeze(1) * sw.to(F64)
    tol = 2 * U * ref.abs()
    if bias is not None:
        ref = ref + bias.to(F64)
        tol = tol + U * (ref.abs() + bias.to(F64).abs())
    err = (y.to(F64) - ref).abs()
    assert bool((err <= tol + HALF[out_dtype] * ref.abs() + 1e-30).all())


@pytest.mark.parametrize("m,n,k", [(145, 955, 12288), (40, 300, 8000), (300, 130, 9001), (78, 2452, 12288), (1000, 70, 12300), (65, 17, 16384), (129, 257, 8097)])
@pytest.mark.parametrize("out_dtype", [BF, F32])
def test_linear_splits(m, n, k, out_dtype):
    """Long rows and few results: sums in parts, joined by a second launch.  The codes of test_linear_blocks: sums of 16384 products of at most 2^4 are below 2^18,
    multiples of 2^-6, and exact in fp32 however they are parted."""
    ops, g = _ops(), _gen(m + n)
    codes, wcodes = ((torch.randint(0x38, 0x48, (r, k), generator=g) + 128 * torch.randint(0, 2, (r, k), generator=g)).to(U8).to(DEV) for r in (m, n))
    sx, sw = (torch.rand(m, generator=g) + 0.1).to(DEV), (torch.rand(n, generator=g) - 0.5).to(DEV)
    bias = torch.randn(n, generator=g).to(BF).to(DEV) if m % 2 == 0 else None
    weight = ops.Fp8Weight.from_codes(wcodes, sw)
    assert weight.ws_bytes(m, out_dtype) > 0
    y = ops.fp8_linear(ops.Fp8Rows.from_codes(codes, sx), weight, bias=bias, out_dtype=out_dtype)
    ref = codes.view(F8).to(F64) @ wcodes.view(F8).to(F64).t() * sx.to(F64).unsqueeze(1) * sw.to(F64)
    tol = 2 * U * ref.abs()
    if bias is not None:
        ref = ref + bias.to(F64)
        tol = tol + U * (ref.abs() + bias.to(F64).abs())
    err = (y.to(F64) - ref).abs()
    assert bool((err <= tol + HALF[out_dtype] * ref.abs() + 1e-30).all())


def test_linear_splits_streams_graphs():
    """Calls on two streams at once and in two captured graphs, whose sums are their own."""
    ops, g = _ops(), _gen(34)
    weight = ops.Fp8Weight.quantize(_rows(g, 300, 12288).to(DEV))
    x = [_rows(g, 70, 12288).to(DEV) for _ in range(2)]
    assert weight.ws_bytes(70) > 0
    want = [ops.fp8_linear(a, weight) for a in x]
    streams, got, graphs = [torch.cuda.Stream() for _ in x], [None, None], [torch.cuda.CUDAGraph() for _ in x]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = ops.fp8_linear(x[i], weight)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    for i, s in enumerate(streams):
        with torch.cuda.graph(graphs[i], stream=s):
            got[i] = ops.fp8_linear(x[i], weight)
    for _ in range(3):
        for a in x:
            a.copy_(_rows(g, 70, 12288))
        torch.cuda.synchronize()
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                graphs[i].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(b, ops.fp8_linear(a, weight)) for a, b in zip(x, got))


def test_linear_blocks_rounded():
    """bf16 results of many rows: the instructions for e4m3 codes cut each of eight neighbouring products off below 2^-13 of the largest of
    them, so every group of eight loses at most 7 * 2^-13 of its largest."""
    ops, g = _ops(), _gen(33)
    m, n, k = 130, 20000, 512
    x, w = _rows(g, m, k, dtype=F32), _rows(g, n, k, spread=2.0)
    rows, weight = ops.fp8_rows(x.to(DEV)), ops.Fp8Weight.quantize(w.to(DEV))
    xv, wv = rows.codes.to(F64) * rows.scales.to(F64).unsqueeze(1), weight.dequantize().to(F64)
    ref, B = xv @ wv.t(), xv.abs() @ wv.abs().t()
    lost = torch.zeros_like(ref)
    for i in range(0, k, 8):
        top = torch.zeros_like(ref)
        for e in range(i, i + 8):
            top = torch.maximum(top, (xv[:, e].unsqueeze(1) * wv[:, e]).abs())
        lost += 7 * 2.0 ** -13 * top
    err = (ops.fp8_linear(rows, weight).to(F64) - ref).abs()
    assert bool((err <= lost * (1 + 2.0 ** -7) + 2 * (148 + k / 128) * U * B + (2 * U + 2.0 ** -8) * ref.abs()).all())


def test_linear_codes_and_shapes():
    """Codes and scales of a checkpoint: any scales, NaN where they stand and nowhere else; leading dimensions; empty; other streams and graphs."""
    ops, g = _ops(), _gen(32)
    m, n, k = 5, 70, 200
    codes, wcodes = (torch.randint(0, 256, (r, k), generator=g, dtype=torch.int64).to(U8) for r in (m, n))
    for c in (codes, wcodes):
        c[(c & 0x7f) == 0x7f] = 0x38
    sx, sw = torch.rand(m, generator=g) + 0.1, torch.rand(n, generator=g) - 0.5
    weight, rows = ops.Fp8Weight.from_codes(wcodes.to(DEV), sw.to(DEV)), ops.Fp8Rows.from_codes(codes.to(DEV).view(F8), sx.to(DEV))
    xc, wc = codes.view(F8).float().to(F64), wcodes.view(F8).float().to(F64)
    y = ops.fp8_linear(rows, weight, out_dtype=F32)
    check_linear(y, xc, sx.to(F64), wc, sw.to(F64), None, F32)
    again = ops.Fp8Weight.from_codes(wcodes.to(DEV).t().contiguous().t(), sw.to(DEV))
    assert torch.equal(again.packed, weight.packed)
    codes[3, 9], wcodes[11, 4] = 0x7f, 0xff
    y2 = ops.fp8_linear(ops.Fp8Rows.from_codes(codes.to(DEV), sx.to(DEV)), ops.Fp8Weight.from_codes(wcodes.to(DEV), sw.to(DEV)), out_dtype=F32)
    bad = torch.zeros(m, n, dtype=torch.bool)
    bad[3], bad[:, 11] = True, True
    assert torch.equal(y2.isnan().cpu(), bad) and torch.equal(y2.cpu()[~bad], y.cpu()[~bad])
    x = torch.randn(2, 3, k, generator=g).to(BF).to(DEV)
    assert tuple(ops.fp8_linear(x, weight).shape) == (2, 3, n) and tuple(ops.fp8_linear(x[:, :0], weight).shape) == (2, 0, n)
    assert tuple(ops.fp8_linear(x[0, 0], weight).shape) == (n,)
    eager = ops.fp8_linear(x, weight)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(ops.fp8_linear(x, weight), eager)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            total, q = ops.add_rmsnorm_fp8(x, x, torch.ones(k, dtype=BF, device=DEV), 1e-6)
            out = ops.fp8_linear(q, weight)
    torch.cuda.synchronize()
    for i in range(3):
        x.copy_(torch.randn(2, 3, k, generator=g).to(BF))
        graph.replay()
        torch.cuda.synchronize()
        t, r = ops.add_rmsnorm_fp8(x, x, torch.ones(k, dtype=BF, device=DEV), 1e-6)
        assert torch.equal(t, total) and torch.equal(ops.fp8_linear(r, weight), out)
