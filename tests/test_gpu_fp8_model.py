"""A decode step in eight bits as a user runs it: ``fp8_cache`` (rows written, attended to) under ``QwenModel(fp8=True)`` (norms that write eight-bit
rows, products that read them).  Every call that the step makes of an operator is compared with the operator's definition in 64 bits on that call's own inputs
(tolerances: tests/test_gpu_fp8.py), and the step as a whole with the same model in plain torch operations."""
import math

import pytest
import torch

from test_gpu_fp8 import BF, DEV, F32, F64, U, CacheOracle, _exponent, _gen, _round, _rows, check_attention, check_linear

pytestmark = pytest.mark.gpu


def _cache(layers, bs, length, heads, group, dtype=BF, block=64, valid_start=0):
    from pariskv_amd.cache_hub.fp8_cache import fp8_cache

    return fp8_cache(valid_start, layers, bs, length, heads, heads * group, 128, dtype, {str(i): DEV for i in range(layers)}, block=block)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("together", [True, False])
def test_cache(dtype, together):
    """A prompt of all samples or one by one, then tokens one by one and several at once, into two layers; then another prompt in the same cache."""
    g, bs, heads, group, block = _gen(5), 3, 2, 4, 32
    cache = _cache(2, bs, 300, heads, group, dtype, block, valid_start=[2] * bs)
    for n in (150, 41):
        oracles = [CacheOracle(bs, heads, cache.layers[0].capacity, block) for _ in range(2)]
        for layer, oracle in enumerate(oracles):
            k, v = _rows(g, bs, n + 2, heads, 128, dtype=dtype), _rows(g, bs, n + 2, heads, 128, dtype=dtype)
            oracle.store(k[:, 2:], v[:, 2:], [0] * bs)
            kd, vd = k.to(DEV), v.to(DEV)
            if together:
                for b in range(bs):  # the calls of a loop over samples: the first does it
                    back = cache.prefill_update_kv_cache(None, kd, vd, layer, b)
                assert torch.equal(back[0], kd[:, 2:])
            else:
                for b in range(bs):
                    cache.prefill_update_kv_cache(None, kd[b:b + 1], vd[b:b + 1], layer, b)
        assert cache.context == n
        at = n
        for T in (1, 1, 7, 1):
            for layer, oracle in enumerate(oracles):
                k, v = _rows(g, bs, T, heads, 128, dtype=dtype), _rows(g, bs, T, heads, 128, dtype=dtype)
                q = torch.randn(bs, T, heads * group, 128, generator=g).to(dtype)
                oracle.store(k, v, [at] * bs)
                cache.decode_update_kv_cache(k.to(DEV), v.to(DEV), layer)
                out = cache.compute(q.to(DEV), layer)
                check_attention(out, q, oracle, [(0, at + T)])
            at += T
            assert cache.context == at and cache.current_seq_len == [at, at]
        for layer, oracle in enumerate(oracles):
            for codes, scales, want, want_s in zip((cache.layers[layer].k, cache.layers[layer].v), (cache.layers[layer].k_scale, cache.layers[layer].v_scale),
                                                   oracle.codes, oracle.scales):
                assert torch.equal(codes[:, :, :at].float().cpu().to(F64), want[:, :, :at])
                assert torch.equal(scales[:, :, :-(-at // block)].cpu().to(F64), want_s[:, :, :-(-at // block)])


def test_cache_refuses():
    g = _gen(6)
    cache = _cache(1, 2, 40, 2, 2, valid_start=[0, 3])
    k = _rows(g, 2, 41, 2, 128).to(DEV)
    for states, batch_idx in ((k[:, :20], 0), (k[:1], 0), (k[:1, :20], 2), (k[1:, :3], 1), (torch.cat([k, k])[:3], 0)):
        with pytest.raises(RuntimeError):  # two starts at once; longer than the cache; no such sample; nothing left; other samples than the cache's
            cache.prefill_update_kv_cache(None, states, states, 0, batch_idx)
    cache.prefill_update_kv_cache(None, k[:1, :20], k[:1, :20], 0, 0)
    with pytest.raises(RuntimeError, match="several lengths"):
        cache.decode_update_kv_cache(k[:, :1], k[:, :1], 0)
    cache.prefill_update_kv_cache(None, k[1:, :23], k[1:, :23], 0, 1)
    cache.decode_update_kv_cache(k[:, :20], k[:, :20], 0)
    with pytest.raises(RuntimeError):
        cache.decode_update_kv_cache(k[:, :1], k[:, :1], 0)
    with pytest.raises(RuntimeError, match="drafted"):
        cache.draft_attend(None, None, None, 0)


def _model(cache, **kw):
    from pariskv_amd.model_hub import QwenConfig, QwenModel

    cfg = QwenConfig(hidden_size=520, num_layers=2, num_heads=8, num_key_value_heads=2, intermediate_size=1000, vocab_size=1111)
    return QwenModel(cfg, cache, device=DEV, max_positions=600, seed=4, **kw)


def _decoded(monkeypatch=None, steps=3, fp8=True):
    """Logits of a few tokens behind a prompt, and every call made of an operator."""
    from pariskv_amd import ops

    g, bs, n = _gen(8), 2, 100
    cache = _cache(2, bs, 200, 2, 4)
    model = _model(cache, fp8=fp8)
    for layer in range(2):
        k, v = (torch.randn(bs, n, 2, 128, generator=g).to(BF).to(DEV) for _ in range(2))
        cache.prefill_update_kv_cache(None, k, v, layer, 0)
    calls = []
    if monkeypatch is not None:
        def watch(owner, name):
            real = getattr(owner, name)

            def seen(*a, **kw):
                out = real(*a, **kw)
                calls.append((name, a, kw, out))
                return out

            monkeypatch.setattr(owner, name, seen)

        watch(ops, "fp8_linear"), watch(ops, "add_rmsnorm_fp8"), watch(ops.Fp8KVCache, "store"), watch(ops.Fp8Attention, "run")
    logits = [model.decode_forward(torch.randint(0, 1111, (bs, 1), generator=g).to(DEV)) for _ in range(steps)]
    return model, logits, calls


def test_decode_step_calls(monkeypatch):
    """The step runs on the operators, and each result is what its definition says of the call's inputs."""
    model, _, calls = _decoded(monkeypatch, steps=1)
    names = [c[0] for c in calls]
    layer = ["add_rmsnorm_fp8", "fp8_linear", "store", "run", "fp8_linear", "add_rmsnorm_fp8", "fp8_linear", "fp8_linear"]
    assert names == layer * 2 + ["add_rmsnorm_fp8", "fp8_linear"]
    for name, a, kw, out in calls:
        if name == "fp8_linear":
            from pariskv_amd import ops

            x, weight = a[:2]
            rows = x if isinstance(x, ops.Fp8Rows) else ops.fp8_rows(x)
            xc, sx = rows.codes.float().cpu().to(F64).reshape(-1, rows.k), rows.scales.cpu().to(F64).reshape(-1)
            if x is not rows:
                v = x.cpu().to(F64).reshape(-1, rows.k)
                assert torch.equal(sx, torch.exp2(_exponent(v.abs().amax(1)))) and torch.equal(xc, _round(v / sx.unsqueeze(1)))
            check_linear(out.reshape(-1, weight.n), xc, sx, weight.dequantize().cpu().to(F64), torch.ones(weight.n, dtype=F64), None, out.dtype)
        elif name == "add_rmsnorm_fp8":
            x, residual, weight, eps = a
            total, q = out
            t = x if residual is None else (x.float() + residual.float()).to(BF)
            assert torch.equal(total, t) or kw.get("want_sum") is False
            t = t.cpu().to(F64)
            y = t / torch.sqrt(t.square().mean(-1, keepdim=True) + eps) * weight.cpu().to(F64)
            s, code = q.scales.cpu().to(F64).unsqueeze(-1), q.codes.float().cpu().to(F64)
            lo, hi = torch.minimum(y * (1 - 4 * U), y * (1 + 4 * U)), torch.maximum(y * (1 - 4 * U), y * (1 + 4 * U))
            assert bool((code >= _round(lo / s)).all()) and bool((code <= _round(hi / s)).all())
        elif name == "run":
            _, q, cache, segments = a[:4]
            want = CacheOracle(cache.bs, cache.n_kv_heads, cache.capacity, cache.block)  # its own codes, as the step left them
            want.codes = [t.float().cpu().to(F64) for t in (cache.k, cache.v)]
            want.scales = [t.cpu().to(F64) for t in (cache.k_scale, cache.v_scale)]
            check_attention(out, q, want, segments)


def test_decode_step_whole():
    """Against the step in plain operations on the weights' own values and bf16 rows: what is left is the rounding of activations and cached rows to e4m3.  A number is off
    by at most 2^-4 of itself, uniformly over a step: 2^-4 / sqrt(3) = 3.6 % a product's operand at the most.  Two layers have eight products of rounded
    rows and two attentions over rounded keys and values, and the logits one more; errors of different numbers are independent: sqrt(13) * 3.6 % = 13 % of the logits'
    norm.  Wrong wiring leaves nothing in common: 140 %.  A third is the line."""
    model, logits, _ = _decoded()
    model.lm_head = model.lm_head.dequantize().to(BF)  # a code has four bits and its scale is a power of two: nothing is rounded
    for layer in model.layers:
        for name in ("wqkv", "wo", "gate_up_proj", "down_proj"):
            setattr(layer, name, getattr(layer, name).dequantize().to(BF))
    model.fp8 = False
    g, cache = _gen(8), model.kv_cache

    class Plain:
        def __init__(self):
            self.context, self.rows = 100, [[torch.randn(2, 100, 2, 128, generator=g).to(BF).to(DEV) for _ in range(2)] for _ in range(2)]

        def decode_update_kv_cache(self, k, v, layer):
            self.rows[layer] = [torch.cat([a, b], 1) for a, b in zip(self.rows[layer], (k, v))]
            self.context += layer == 0
            return None, None

        def compute(self, q, layer):
            k, v = (t.float().repeat_interleave(4, 2).transpose(1, 2).contiguous() for t in self.rows[layer])
            p = torch.softmax((q.float().transpose(1, 2).unsqueeze(3) * k.unsqueeze(2)).sum(-1) / math.sqrt(128), -1)
            return (p.unsqueeze(-1) * v.unsqueeze(2)).sum(3).transpose(1, 2).to(BF)

    model.kv_cache = Plain()
    for got in logits:
        want = model.decode_forward(torch.randint(0, 1111, (2, 1), generator=g).to(DEV))
        assert got.shape == want.shape and got.dtype == F32
        assert float((got - want).norm() / want.norm()) < 1 / 3
    assert cache.context == 103


def test_decode_step_repeats():
    """The same tokens give the same logits bit for bit."""
    for a, b in zip(_decoded()[1], _decoded()[1]):
        assert torch.equal(a, b)


def test_drafted_products():
    """A step over drafted tokens with eight-bit products (its norms are plain): on the cache that attends to them."""
    from pariskv_amd.cache_hub.polar_cache import polar_cache

    g = _gen(9)
    cache = polar_cache(valid_start=0, layer_num=2, batch_size=2, max_length=600, num_key_value_heads=2, num_heads=8, head_dim=128, dtype=BF,
                        layer_mapping={str(i): DEV for i in range(2)}, max_new_length=100, sink_size=16, local_size=64, enable_offload=False)
    model = _model(cache, fp8=True)
    for layer in range(2):
        k, v = (torch.randn(2, 50, 2, 128, generator=g).to(BF).to(DEV) for _ in range(2))
        cache.prefill_update_kv_cache(None, k, v, layer, 0)
    ids = torch.randint(0, 1111, (2, 3), generator=g).to(DEV)
    drafted = model.draft_forward(ids)
    model.accept_draft([[], []])
    one = model.decode_forward(ids[:, :1])
    # the norm of a decoded token goes to e4m3 unrounded, of a drafted one by way of bf16, which moves a code by one step where it is near a tie
    assert float((drafted[:, :1] - one).norm() / one.norm()) < 1 / 3
    with pytest.raises(ValueError, match="fp8"):
        _model(cache, fp8=True, weight_bits=4)
    with pytest.raises(ValueError, match="fp8"):
        _model(cache, fp8=True, dtype=F32)
