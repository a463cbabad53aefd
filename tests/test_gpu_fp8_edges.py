"""Operators in eight bits where their arithmetic is at its limits: products that cancel, scales at both ends of fp32, and what else only a particular
input shows.  Inputs are made so that the definition's result is known to a few units in the last place; each bound stands at its test."""
import math

import pytest
import torch

from test_gpu_fp8 import BF, D, DEV, F8, F32, F64, HALF, U8, _exponent, _gen, _ops, _round, _top

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ the cache


@pytest.mark.parametrize("was", [-4.0, 4.0, -0.02, 0.02, -3.7, 2.9, -(2.0 ** -12), 2.0 ** -120, -1e30, 0.0])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_store_behind_any_scale(was, dtype):
    """Rows behind those of a block whose scale the caller set, negative or no power of two: the older rows stay.  The scale is the old one where that is the larger in
    magnitude; then older codes are untouched, and a new one is that of x times fp32(1 / scale), off by 2 u of itself before it is rounded.  Else it is
    the power of two that the new rows need, and an older code is rounded again, exactly as the oracle does where the old scale is a power of two, else after
    a product off by u."""
    ops, g = _ops(), _gen(17)
    old = torch.randint(0, 0x78, (1, 2, 32, 128), generator=g).to(U8)
    old[0, 0, 3:5] |= 0x80
    scale = torch.full((1, 2, 2), was)
    cache = ops.Fp8KVCache.from_codes(old.clone().to(DEV), scale.clone().to(DEV), old.clone().to(DEV), scale.clone().to(DEV), block=16)
    x = torch.randn(1, 2, 2, 128, generator=g).to(dtype)
    cache.store(x.to(DEV), x.to(DEV), 5)
    need = torch.exp2(_exponent(_top(x.to(F64)).amax((1, 3))))  # [1, heads]
    held = torch.tensor(was, dtype=F32).to(F64)
    for codes, scales in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        codes, scales = codes.float().cpu().to(F64), scales.cpu().to(F64)
        s = torch.where(held.abs() > need, held, need)
        assert torch.equal(scales[:, :, 0], s) and torch.equal(scales[:, :, 1], held.expand(1, 2))
        slack = torch.tensor([1 - 4 * 2.0 ** -24, 1 + 4 * 2.0 ** -24], dtype=F64).view(2, 1, 1, 1, 1)
        for got, exact in ((codes[:, :, :5], old.view(F8).float().to(F64)[:, :, :5] * (held / s).view(1, 2, 1, 1)), (codes[:, :, 5:7], x.to(F64).transpose(1, 2) / s.view(1, 2, 1, 1))):
            ends = _round(exact * slack)
            assert bool((got >= ends.amin(0)).all()) and bool((got <= ends.amax(0)).all())
        assert torch.equal(codes[:, :, 7:], old.view(F8).float().to(F64)[:, :, 7:])


# ------------------------------------------------------------------ attention in fp32


class Pinned:
    """Inputs of fp32 attention whose result is known to a few units in the last place: q [bs,T,H*G,128], codes and scales of K and V (blocks of 16), the result in
    64 bits and how far a number may be off, relative to itself.  ``cut(q)`` and ``cut(weights)`` stand for a kernel that holds fewer bits of them."""

    def result(self, cut_q=lambda x: x, cut_weights=lambda x: x):
        bs, H, n, _ = self.k.shape
        T, G = self.q.shape[1], self.q.shape[2] // H
        k, v = (c.view(F8).float().to(F64) for c in (self.k, self.v))
        ks, vs = (s.to(F64).repeat_interleave(16, -1)[:, :, :n] for s in (self.k_scale, self.v_scale))
        q = cut_q(self.q).to(F64).view(bs, T, H, G, D).permute(0, 2, 1, 3, 4)
        z = (q.reshape(bs, H, T * G, D) @ k.transpose(2, 3)) * ks.unsqueeze(2) * self.scale
        seen = torch.arange(n) < n - (T - 1 - torch.arange(T).repeat_interleave(G)).unsqueeze(1)
        p = torch.softmax(z.masked_fill(~seen, -math.inf), -1)
        top = p.amax(-1, keepdim=True)  # weights relative to the largest, as a kernel holds them
        o = (cut_weights((p / top * vs.unsqueeze(2)).to(F32)).to(F64) @ v) * top
        return o.view(bs, H, T, G, D).permute(0, 2, 1, 3, 4).reshape(bs, T, H * G, D)

    def holds(self, out):
        want = self.result()
        return bool(((out.cpu().to(F64) - want).abs() <= self.bound * want.abs() + 1e-18).all())


def pinned_weights(n, T, G, seed):
    """All scores 0: weights are 1 and their sum is a whole number, exactly.  A dim has one value other than 0 among all keys, whose scale has 24 bits: a number out is code * scale / keys,
    off by an addition of the parts' products, the division's two roundings and the joining of waves and splits: 8 steps, 16 u."""
    c, g, bs, H = Pinned(), _gen(seed), 2, 2
    blocks = -(-n // 16)
    c.q = torch.zeros(bs, T, H * G, D)
    c.k = torch.randint(0, 0x78, (bs, H, blocks * 16, D), generator=g).to(U8)[:, :, :n]
    c.v = torch.zeros(bs, H, n, D, dtype=U8)
    c.k_scale, c.v_scale = (torch.rand(bs, H, blocks, generator=g) + 1.0 for _ in range(2))
    c.v_scale *= torch.exp2(torch.randint(-20, 20, (bs, H, blocks), generator=g).float())
    for b in range(bs):
        for h in range(H):
            at = torch.randint(0, max(1, n - T + 1), (D,), generator=g)
            c.v[b, h, at, torch.arange(D)] = torch.randint(0x30, 0x78, (D,), generator=g).to(U8)
    c.scale, c.bound = 1 / math.sqrt(D), 16 * 2.0 ** -24
    return c


def pinned_scores(n, G, seed):
    """A head has two keys with one code 1 each, at two dims of q, all others are 0: the scores are two numbers of q, of 24 bits, 64 to 128 and at most 2 apart, and 0, whose weight is nothing (n 2^-64).
    A score in powers of two, S <= 186, is off by a rounding, u S, the base that a wave, and a split, subtracts by as much: 4 u S in a difference, which is as much of a weight times
    log 2, and twice that in the ratio's denominator; the scale's rounding moves the difference by 2 u 3; exponentials, sums and the division are some 40 u."""
    c, g, bs, H = Pinned(), _gen(seed), 2, 4
    blocks = -(-n // 16)
    a = 64 + torch.randint(0, 1 << 23, (bs, 1, H * G), generator=g).double() * 2.0 ** -17
    b = (a + torch.randint(-(1 << 18), 1 << 18, a.shape, generator=g).double() * 2.0 ** -17).clamp(64, 128 - 2.0 ** -17)
    c.q = torch.randn(bs, 1, H * G, D, generator=g)
    c.k, c.v = torch.zeros(bs, H, n, D, dtype=U8), torch.zeros(bs, H, n, D, dtype=U8)
    c.k_scale, c.v_scale = torch.ones(bs, H, blocks), torch.ones(bs, H, blocks)
    for i in range(bs):
        for h in range(H):
            dims, keys = torch.randperm(D, generator=g)[:2], torch.randperm(n, generator=g)[:2]
            c.q[i, 0, h * G:(h + 1) * G, dims[0]], c.q[i, 0, h * G:(h + 1) * G, dims[1]] = a[i, 0, h * G:(h + 1) * G].float(), b[i, 0, h * G:(h + 1) * G].float()
            c.k[i, h, keys, dims] = 0x38
            c.v[i, h, keys[0], :64], c.v[i, h, keys[1], 64:] = 0x38, 0x38
    c.scale, c.bound = 1.0, (8 * 186 + 6 + 40) * 2.0 ** -24
    return c


PINNED = [(pinned_weights, a) for a in ((1, 1, 4, 1), (40, 1, 4, 2), (301, 1, 1, 3), (301, 5, 7, 4), (1000, 1, 16, 5), (5003, 2, 8, 6))] + [
    (pinned_scores, a) for a in ((2, 4, 1), (33, 1, 2), (64, 16, 3), (300, 20, 4), (1000, 4, 5), (5003, 8, 6))]


@pytest.mark.parametrize("make,a", PINNED)
def test_attention_f32_holds_24_bits(make, a):
    """q and the weights in all of fp32's bits: with 16 of them, or 8, the bound is missed (tests/test_fp8_precision_host.py)."""
    ops, c = _ops(), make(*a)
    bs, H, n, _ = c.k.shape
    T, G, cap = c.q.shape[1], c.q.shape[2] // H, c.k_scale.shape[2] * 16
    k, v = (torch.cat([t, t.new_full((bs, H, cap - n, D), 0x7f)], 2).to(DEV) for t in (c.k, c.v))
    cache = ops.Fp8KVCache.from_codes(k, c.k_scale.to(DEV), v, c.v_scale.to(DEV), block=16)
    out = ops.Fp8Attention(bs, H, G, T, n, DEV).run(c.q.to(DEV), cache, [(0, n)], scale=c.scale)
    assert c.holds(out), float(((out.cpu().to(F64) - c.result()).abs() / c.result().abs().clamp(min=1e-18)).max() * 2.0 ** 24)


# ------------------------------------------------------------------ norms


@pytest.mark.parametrize("width", [8, 101, 256, 4096, 4099])
@pytest.mark.parametrize("residual", [True, False])
def test_norm_leaves_the_sum(width, residual):
    """The entry point's out_sum: x + residual, or x where there is no residual."""
    from pariskv_amd import _lib

    g, rows, wide = _gen(width), 3, -(-width // 128) * 128
    x, r, w = (torch.randn(n, width, generator=g).to(BF).to(DEV) for n in (rows, rows, 1))
    total, codes, scales = torch.full_like(x, 7.0), torch.zeros(rows, wide, dtype=U8, device=DEV), torch.zeros(rows, device=DEV)
    assert _lib.lib().pkv_add_rmsnorm_fp8(x.data_ptr(), r.data_ptr() if residual else None, w.data_ptr(), 1e-6, rows, width, total.data_ptr(), codes.data_ptr(), wide,
                                          scales.data_ptr(), torch.cuda.current_stream().cuda_stream) == 0
    assert torch.equal(total, (x.float() + r.float()).to(BF) if residual else x)


@pytest.mark.parametrize("width", [1, 100, 101, 1021, 4099])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_norm_padding(width, bad):
    """Zeros follow a row up to the next multiple of 128 columns, whatever is in it."""
    ops, g = _ops(), _gen(width)
    x = torch.randn(2, width, generator=g).to(BF)
    x[1, width // 2] = bad
    _, q = ops.add_rmsnorm_fp8(x.to(DEV), None, torch.ones(width, dtype=BF, device=DEV), 1e-6)
    assert bool(q.codes.float().isnan().any(1).cpu()[1]) and not bool(q.codes.float().isnan().any(1).cpu()[0])
    assert not bool(q.padded.view(U8)[:, width:].any())


def test_rows_more_than_2_to_26():
    """More rows than a launch has waves, which has fewer than 2^32 threads."""
    ops, g = _ops(), _gen(4)
    few, times, rest = 4096, 1 << 14, 5
    x = torch.randn(few, 8, generator=g).to(BF).to(DEV)
    want = ops.fp8_rows(x)
    q = ops.fp8_rows(torch.cat([x.repeat(times, 1), x[:rest]]))
    ones = torch.ones(8, dtype=BF, device=DEV)
    normed, norm = ops.add_rmsnorm_fp8(x, None, ones, 1e-6)[1], ops.add_rmsnorm_fp8(torch.cat([x.repeat(times, 1), x[:rest]]), None, ones, 1e-6)[1]
    for got, ref in ((q, want), (norm, normed)):
        codes, ref_codes, n = got.padded.view(U8), ref.padded.view(U8), few * times
        assert torch.equal(got.scales[:n].view(times, few), ref.scales.expand(times, few)) and torch.equal(got.scales[n:], ref.scales[:rest])
        for i in range(0, times, 1 << 12):
            part = codes[i * few:(i + (1 << 12)) * few].view(1 << 12, few, 128)
            assert bool((part == ref_codes).all())
        assert torch.equal(codes[n:], ref_codes[:rest])


# ------------------------------------------------------------------ products


def test_matrix_of_more_than_2_to_32():
    """A matrix of more elements than a launch has threads, there and back."""
    ops, n, k = _ops(), (1 << 16) + 3, 1 << 16
    row = torch.randint(0, 0x78, (1 << 10, k), generator=_gen(5)).to(U8).to(DEV)
    codes = row.repeat(-(-n // (1 << 10)), 1)[:n]
    scales = torch.exp2((torch.arange(n, device=DEV) % 7).float())
    w = ops.Fp8Weight.from_codes(codes, scales).dequantize()
    for i in range(0, n, 1 << 12):
        assert torch.equal(w[i:i + (1 << 12)], codes[i:i + (1 << 12)].view(F8).float() * scales[i:i + (1 << 12)].unsqueeze(1))



def _cancelling(g, rows, k, second):
    """Codes [rows,k]: 448 in columns 8 i, `second` in columns 8 i + 1, and 1, 1.5, 2 or 3 in the others."""
    codes = torch.tensor([0x38, 0x3c, 0x40, 0x44], dtype=U8)[torch.randint(0, 4, (rows, k), generator=g)]
    codes[:, 0::8], codes[:, 1::8] = 0x7e, second
    return codes.to(DEV)


@pytest.mark.parametrize("m,n,k", [(3, 100, 300), (16, 2000, 1000), (17, 2000, 1000), (130, 20000, 384), (520, 9001, 1000), (520, 1536, 4096), (256, 6144, 4096), (1024, 4096, 4096),
                                   (145, 955, 12288)])
@pytest.mark.parametrize("out_dtype", [BF, F32])
def test_linear_sums_cancel(m, n, k, out_dtype):
    """Of eight neighbouring products two are +-448^2 and cancel.  All products are multiples of 2^-2, those that are left add up to less than 2^17, and a path through the sum holds at
    most a few of the large ones (below 2^18 each) that have not met their opposites yet: every sum is a multiple of 2^-2 below 2^22, exact in
    fp32, and the scales are 1.  Only the rounding to bf16 is left."""
    ops, g = _ops(), _gen(m + n)
    codes, wcodes = _cancelling(g, m, k, 0x7e), _cancelling(g, n, k, 0xfe)
    one = lambda rows: torch.ones(rows, device=DEV)
    y = ops.fp8_linear(ops.Fp8Rows.from_codes(codes, one(m)), ops.Fp8Weight.from_codes(wcodes, one(n)), out_dtype=out_dtype)
    ref = codes.view(F8).to(F64) @ wcodes.view(F8).to(F64).t()
    assert float(ref.abs().max()) < 2.0 ** 17
    err = (y.to(F64) - ref).abs()
    assert bool((err <= (HALF[out_dtype] * ref.abs() if out_dtype == BF else 0.0)).all()), float((err / ref.abs()).max())


# (rows of x, rows of the matrix) a workgroup, split or not, workgroups at once to a compute unit: products that are dealt out so
PLANS = {
    (16, 16, False, 1): [(1, 17, 103), (15, 1003, 1185), (16, 512, 4096)],
    (16, 32, False, 1): [(1, 4103, 101), (13, 8000, 640)],
    (16, 64, False, 1): [(1, 8255, 101), (16, 20000, 256)],
    (32, 32, False, 1): [(17, 4285, 105), (32, 5000, 512)],
    (32, 64, False, 1): [(17, 8599, 101), (31, 12000, 384)],
    (64, 64, False, 1): [(33, 10297, 1431), (520, 1536, 4096)],
    (64, 64, True, 1): [(17, 17, 6173), (145, 955, 12288), (64, 512, 8192)],
    (64, 128, False, 1): [(35, 31537, 293), (256, 6144, 4096), (64, 24576, 4096)],
    (64, 128, True, 1): [(17, 8401, 5691), (256, 4096, 12288)],
    (128, 64, False, 1): [(97, 16229, 267), (110, 16000, 640)],
    (128, 64, True, 1): [(67, 1713, 6593), (78, 2448, 12288)],
    (128, 128, False, 1): [(65, 32199, 137), (1024, 4096, 4096)],
    (128, 128, True, 1): [(65, 9813, 6033), (68, 9360, 5760)],
    (128, 128, False, 2): [(67, 38391, 105), (520, 9001, 1000), (4096, 6144, 512)],
}


@pytest.mark.parametrize("plan,m,n,k", [(plan, *case) for plan, cases in PLANS.items() for case in cases])
def test_linear_every_kernel(plan, m, n, k):
    """Every kernel that the rule for shapes picks, bf16 and fp32 results, with and without a bias, odd and whole sizes; the case is one of the kernel it stands for.
    Codes 1 to 3.75 of either sign: products are multiples of 2^-6, sums below 2^18, exact in fp32; two roundings for the scales, one for the bias, one to
    the output's type."""
    ops, g = _ops(), _gen(m + n + k)
    codes, wcodes = ((torch.randint(0x38, 0x48, (r, k), generator=g) + 128 * torch.randint(0, 2, (r, k), generator=g)).to(U8).to(DEV) for r in (m, n))
    sx, sw = (torch.rand(m, generator=g) + 0.1).to(DEV), (torch.rand(n, generator=g) - 0.5).to(DEV)
    weight, rows = ops.Fp8Weight.from_codes(wcodes, sw), ops.Fp8Rows.from_codes(codes, sx)
    bm, bn, splits, at_once = weight.plan(m)
    assert (bm, bn, splits > 1, at_once) == plan
    ref = codes.view(F8).to(F64) @ wcodes.view(F8).to(F64).t() * sx.to(F64).unsqueeze(1) * sw.to(F64)
    for bias in (None, torch.randn(n, generator=g).to(BF).to(DEV)):
        want, tol = ref, 2 * 2.0 ** -24 * ref.abs()
        if bias is not None:
            want = ref + bias.to(F64)
            tol = tol + 2.0 ** -24 * (want.abs() + tol)
        for out_dtype in (BF, F32):
            y = ops.fp8_linear(rows, weight, bias=bias, out_dtype=out_dtype)
            assert y.dtype == out_dtype and (weight.ws_bytes(m, out_dtype) > 0) == (splits > 1)
            err = (y.to(F64) - want).abs()
            assert bool((err <= tol + (HALF[out_dtype] * (want.abs() + tol) if out_dtype == BF else 0.0) + 1e-30).all()), (out_dtype, float((err / want.abs()).max()))


@pytest.mark.parametrize("m,n,k", [(5, 100, 300), (60, 300, 300), (130, 20000, 384), (145, 955, 12288), (520, 1536, 4096)])
@pytest.mark.parametrize("out_dtype", [BF, F32])
@pytest.mark.parametrize("sx,sw", [(2.0 ** 107, 2.0 ** -25), (2.0 ** -25, 2.0 ** 118), (-3e36, 1e-37), (1e-42, 1.7e37), (3e-39, -3e38), (2.0 ** -100, 2.0 ** 100)])
def test_linear_scales(m, n, k, sx, sw, out_dtype):
    """Scales of both ends of fp32, subnormal ones among them, whose results are in the middle of it.  Codes 1 to 3.75 of either sign: products are multiples of 2^-6, sums below 2^18,
    exact; then two roundings for the scales, 2 u |y|, and that to the output's type."""
    ops, g = _ops(), _gen(m + n)
    codes, wcodes = ((torch.randint(0x38, 0x48, (r, k), generator=g) + 128 * torch.randint(0, 2, (r, k), generator=g)).to(U8).to(DEV) for r in (m, n))
    sx, sw = torch.full((m,), sx, device=DEV), torch.full((n,), sw, device=DEV)
    y = ops.fp8_linear(ops.Fp8Rows.from_codes(codes, sx), ops.Fp8Weight.from_codes(wcodes, sw), out_dtype=out_dtype)
    ref = codes.view(F8).to(F64) @ wcodes.view(F8).to(F64).t() * (sx.to(F64).unsqueeze(1) * sw.to(F64))
    err = (y.to(F64) - ref).abs()
    assert bool((err <= (2 * 2.0 ** -24 + HALF[out_dtype]) * ref.abs()).all()), float((err / ref.abs()).max())


# ------------------------------------------------------------------ the dense cache


def test_dense_cache_lengths():
    """Attention over sequences whose prompts differ in length is refused, as their next rows are: there is one length for all."""
    from pariskv_amd.cache_hub.fp8_cache import fp8_cache

    g, bs = _gen(3), 2
    cache = fp8_cache(0, 2, bs, 40, 2, 4, D, BF, {"0": DEV, "1": DEV})
    k, q = torch.randn(bs, 30, 2, D, generator=g).to(BF).to(DEV), torch.randn(bs, 1, 4, D, generator=g).to(BF).to(DEV)
    cache.prefill_update_kv_cache(None, k[:1, :20], k[:1, :20], 0, 0)
    for n in (None, 23):  # the other sample without a prompt, and with a longer one
        if n:
            cache.prefill_update_kv_cache(None, k[1:, :n], k[1:, :n], 0, 1)
        with pytest.raises(RuntimeError, match="several lengths"):
            cache.compute(q, 0)
        with pytest.raises(RuntimeError, match="several lengths"):
            cache.decode_update_kv_cache(k[:, :1], k[:, :1], 0)
    cache.prefill_update_kv_cache(None, k[1:, :20], k[1:, :20], 0, 1)
    want = cache.compute(q, 0)
    cache.prefill_update_kv_cache(None, k[:, :20], k[:, :20], 1, 0)
    assert torch.equal(cache.compute(q, 1), want)
