"""A step over drafted tokens through the cache and the model: ``polar_cache.draft_attend`` / ``commit_draft`` and
``QwenModel.draft_forward`` / ``accept_draft``, with 16- and 4-bit weights.

Attention is checked against its definition in 64 bits over the rows the cache reports as selected (tolerance of test_gpu_drafts.py);
what a committed path leaves behind is compared with what the same tokens leave behind that are decoded one by one, bit for bit; the
fp32 model's logits over a tree with those of its paths decoded one by one.  Their tolerance is 2^-7 of a row's largest logit: three layers
of some ten sums of at most 1024 terms, each sum off by at most 1024 * 2^-24 of its terms' sum, are off by 30 * 2^-14 = 2^-9 of the
values' size at each step, four times for the normalisations that pass it on."""
import math

import pytest
import torch

from test_gpu_drafts import BF, D, DEV, F32, check, exact_tree, _randn

pytestmark = pytest.mark.gpu


def make_cache(offload, bs, hkv, hq, layers, rows, sink, local, interval, topk, thr=100, dtype=BF, kind="polar_cache", **kw):
    import importlib

    cls = importlib.import_module(f"pariskv_amd.cache_hub.{kind}").polar_cache
    if offload == "mixed":   # a host budget that holds one layer: the others stay in HBM
        es = torch.empty((), dtype=dtype).element_size()
        offload, kw["host_kv_budget_bytes"] = True, int(1.5 * 2 * bs * hkv * (rows - sink - local) * D * es)
    return cls(valid_start=[0] * bs, layer_num=layers, batch_size=bs, max_length=rows, num_key_value_heads=hkv, num_heads=hq,
               head_dim=D, dtype=dtype, layer_mapping={i: DEV for i in range(layers)}, max_new_length=100, sink_size=sink,
               local_size=local, core=1, nprobe=1, cache_unit_size=1, cache_cluster_num=1, num_gpus=1, model_size=7, final_topk=topk,
               dynamic_update_interval=interval, full_attention_threshold=thr, enable_offload=offload, **kw)


def prefill(caches, seed, bs, s, hkv, layers, dtype=BF):
    """The same prompt into several caches; returns its K and V, [layers,bs,S,Hkv,128] on the CPU."""
    g = torch.Generator().manual_seed(seed)
    k, v = _randn(g, layers, bs, s, hkv, D), _randn(g, layers, bs, s, hkv, D)
    k[..., [7, 31, 64, 101]] *= 3.0
    k, v = k.to(dtype), v.to(dtype)
    for cache in caches:
        for l in range(layers):
            cache.prefill_update_kv_cache(None, k[l].to(DEV), v[l].to(DEV), l, 0)
    torch.cuda.synchronize()
    return k, v


def attended(cache, l, k, v):
    """[bs,Hkv] lists of the rows of k, v [bs,S,Hkv,128] that the last retrieval of layer l left to attend to."""
    z, ids = cache._zones[l], cache.last_topk_indices.cpu()
    bs, hkv = ids.shape[:2]
    rows = [[torch.cat([torch.arange(cache.sink_size), cache.sink_size + ids[b, h], torch.arange(z.local_start, z.seq_len)])
             for h in range(hkv)] for b in range(bs)]
    pick = lambda t: torch.stack([torch.stack([t[b, rows[b][h], h] for h in range(hkv)]) for b in range(bs)])
    return pick(k), pick(v)


@pytest.mark.parametrize("offload", [False, True, "mixed"])
@pytest.mark.parametrize("bs,hkv,group,t,dtype", [(1, 2, 4, 1, BF), (2, 2, 4, 7, BF), (2, 1, 7, 33, BF), (1, 2, 2, 64, F32)])
def test_draft_attend_retrieves(offload, bs, hkv, group, t, dtype):
    from pariskv_amd import ops

    layers, s, sink, local, interval, topk = 2, 1500, 4, 64, 32, 100
    cache = make_cache(offload, bs, hkv, hkv * group, layers, s + 200, sink, local, interval, topk, dtype=dtype)
    other = make_cache(offload, bs, hkv, hkv * group, layers, s + 200, sink, local, interval, topk, dtype=dtype)
    k, v = prefill((cache, other), 1, bs, s, hkv, layers, dtype)
    g = torch.Generator().manual_seed(2)
    parents = [-1] + [int(torch.randint(-1, i, (), generator=g)) for i in range(1, t)]
    mask = ops.tree_mask(parents)
    for l in range(layers):
        q, dk, dv = (_randn(g, bs, t, h * D, dtype=dtype).view(bs, t, h, D) for h in (hkv * group, hkv, hkv))
        out = cache.draft_attend(q.to(DEV), dk.to(DEV), dv.to(DEV), l, mask.to(DEV))
        ak, av = attended(cache, l, k[l], v[l])
        want, tol = exact_tree(dict(q=q, segs=[(ak, av, 0, ak.shape[2])], dk=dk, dv=dv, mask=mask, rk=None))
        check(out, want, tol)
        if t == 1:  # what a decode step selects
            ids = cache.last_topk_indices.sort(-1).values
            other.decode_update_kv_cache(dk.to(DEV), dv.to(DEV), l)
            step = other.compute(q.to(DEV), l)
            assert torch.equal(ids, other.last_topk_indices.sort(-1).values)
            check(step, want, 4 * tol)   # the same keys in other kernels: the same bound, for either, and a margin for theirs


@pytest.mark.parametrize("offload", [False, True, "mixed"])
@pytest.mark.parametrize("s", [1, 40, 90, 300])
def test_draft_attend_to_everything(offload, s):
    """Below the threshold: prompts without and with a retrieval zone, whose rows are read from where they are."""
    bs, hkv, group, t, layers = 2, 2, 4, 5, 2
    cache = make_cache(offload, bs, hkv, hkv * group, layers, 1000, 4, 64, 32, 50, thr=600)
    k, v = prefill((cache,), s, bs, s, hkv, layers)
    g = torch.Generator().manual_seed(3)
    for l in range(layers):
        q, dk, dv = (_randn(g, bs, t, h, D) for h in (hkv * group, hkv, hkv))
        out = cache.draft_attend(q.to(DEV), dk.to(DEV), dv.to(DEV), l)
        rows = [x[l].transpose(1, 2).contiguous() for x in (k, v)]
        want, tol = exact_tree(dict(q=q, segs=[(*rows, 0, s)], dk=dk, dv=dv, mask=None, rk=None))
        check(out, want, tol)


def state(cache):
    out = []
    for l, z in enumerate(cache._zones):
        n = z.gpu_prefix_rows if cache._layer_offload[l] else z.seq_len
        out += [cache.unified_keys_gpu[l][:, :, :n], cache.unified_values_gpu[l][:, :, :n], cache.cluster_key_counts_gpu[l],
                cache._codes_km[l][:, :, 4:4 + z.encoded], cache._nib_km[l][:, :, 4:4 + z.encoded]]
        if cache._layer_offload[l]:
            out += [cache.unified_keys_cpu[l][:, :, :z.encoded], cache.unified_values_cpu[l][:, :, :z.encoded]]
        if hasattr(cache, "_sl_vnorm_cache"):
            out += [cache._sl_vnorm_cache[l][:, :, :n], cache.value_norm_gpu[l][:, :, 4:4 + z.encoded]]
    return out


@pytest.mark.parametrize("kind,offload", [("polar_cache", False), ("polar_cache", True), ("polar_cache", "mixed"),
                                          ("polar_cache_adaptivek_varlen", True),
                                          ("polar_cache_atten_value_indices_adaptive_k", False)])
@pytest.mark.parametrize("s", [3, 60, 500])
@pytest.mark.parametrize("stacked", [False, True])
def test_commit_equals_decoding_one_by_one(kind, offload, s, stacked):
    bs, hkv, group, t, layers = 2, 2, 2, 12, 2
    kw = {} if kind == "polar_cache" else dict(collision_ratio=0.3, candidate_ratio=0.05)
    a, b = (make_cache(offload, bs, hkv, hkv * group, layers, 800, 4, 64, 8, 20, kind=kind, **kw) for _ in range(2))
    prefill((a, b), s, bs, s, hkv, layers)
    g = torch.Generator().manual_seed(5)
    for n in (1, 12, 5, 0, 7, 3, 9, 12, 12):   # 61 tokens: the refresh interval of 8 is crossed within paths and met at their ends
        dk, dv = _randn(g, layers, bs, t, hkv, D).to(DEV), _randn(g, layers, bs, t, hkv, D).to(DEV)
        path = torch.stack([torch.randperm(t, generator=g)[:n] for _ in range(bs)])
        a.commit_draft(*((dk, dv) if stacked else (list(dk), list(dv))), path.tolist())
        for i in range(n):
            for l in range(layers):
                row = lambda x: torch.stack([x[l, j, path[j, i]] for j in range(bs)])[:, None]
                b.decode_update_kv_cache(row(dk), row(dv), l)
        torch.cuda.synchronize()
        assert a.context == b.context and a.current_seq_len == b.current_seq_len and a._zones == b._zones
        for x, y in zip(state(a), state(b)):
            assert torch.equal(x, y)
    if s == 500:   # and both go on alike
        q, k1, v1 = (_randn(g, bs, 1, h, D).to(DEV) for h in (hkv * group, hkv, hkv))
        for l in range(layers):
            a.decode_update_kv_cache(k1, v1, l), b.decode_update_kv_cache(k1, v1, l)
            assert torch.equal(a.compute(q, l), b.compute(q, l))


def test_refusals():
    bs, hkv, group, layers = 2, 2, 2, 2
    cache = make_cache(False, bs, hkv, hkv * group, layers, 800, 4, 64, 8, 20)
    prefill((cache,), 1, bs, 500, hkv, layers)
    g = torch.Generator().manual_seed(5)
    dk = _randn(g, layers, bs, 5, hkv, D).to(DEV)
    before = [x.clone() for x in state(cache)]
    for path in ([[0], [5]], [[0], [-1]], [[0]], [0, 1], [[0], [0, 1]], [[0.5], [1]], torch.zeros(2, 1, dtype=torch.int64, device=DEV)):
        with pytest.raises(RuntimeError, match="path"):
            cache.commit_draft(dk, dk, path)
    with pytest.raises(RuntimeError, match="a layer"):
        cache.commit_draft(dk[:1], dk[:1], [[0], [0]])
    with pytest.raises(RuntimeError, match="fit"):
        cache.commit_draft(dk, dk, [[0] * 301] * 2)
    q, k1 = _randn(g, bs, 0, hkv * group, D).to(DEV), _randn(g, bs, 0, hkv, D).to(DEV)
    with pytest.raises(RuntimeError, match="queries"):
        cache.draft_attend(q, k1, k1, 0)
    with pytest.raises(RuntimeError, match="queries"):
        cache.draft_attend(dk[0], dk[0], dk[0], 0)
    assert all(torch.equal(x, y) for x, y in zip(before, state(cache)))
    chooses = make_cache(True, bs, hkv, hkv * group, layers, 800, 4, 64, 8, 20, kind="polar_cache_adaptivek_varlen")
    prefill((chooses,), 1, bs, 500, hkv, layers)
    with pytest.raises(RuntimeError, match="token by token"):
        chooses.draft_attend(_randn(g, bs, 3, hkv * group, D).to(DEV), dk[0, :, :3], dk[0, :, :3], 0)


# ------------------------------------------------------------- the model


def models(dtype, s, thr, n=2, **kw):
    from pariskv_amd.model_hub import QwenConfig, QwenModel

    cfg = QwenConfig(hidden_size=256, num_layers=3, num_heads=8, num_key_value_heads=2, head_dim=D, intermediate_size=512, vocab_size=500)
    caches = [make_cache(False, 2, 2, 8, 3, s + 100, 4, 64, 8, 40, thr=thr, dtype=dtype) for _ in range(n)]
    prefill(caches, 7, 2, s, 2, 3, dtype)
    return [QwenModel(cfg, c, device=DEV, dtype=dtype, max_positions=s + 100, seed=3, **kw) for c in caches]


def close(a, b, share):
    off, most = (a - b).abs().amax().item(), b.abs().amax().item()
    assert off <= share * most


def test_tree_logits_equal_those_of_its_paths():
    """fp32, every token attended to: each node of the tree against its path decoded one by one; then a path is accepted and both go on."""
    draft, *rest = models(F32, 300, 2000, n=4)
    g = torch.Generator().manual_seed(1)
    parents = [-1, 0, 0, 2, 1, -1, 3]
    paths = [[0, 1, 4], [5], [0, 2, 3, 6]]
    ids = torch.randint(0, 500, (2, 7), generator=g).to(DEV)
    logits = draft.draft_forward(ids, parents)
    assert logits.shape == (2, 7, 500) and logits.dtype == F32 and draft.kv_cache.context == 300
    for model, path in zip(rest, paths):
        for t in path:
            close(logits[:, t:t + 1], model.decode_forward(ids[:, t:t + 1]), 2.0 ** -7)
    draft.accept_draft([paths[2], paths[2]])
    one = rest[2]
    assert draft.kv_cache.context == one.kv_cache.context == 304
    following = torch.randint(0, 500, (2, 3), generator=g).to(DEV)
    logits = draft.draft_forward(following)   # a chain
    for t in range(3):
        close(logits[:, t:t + 1], one.decode_forward(following[:, t:t + 1]), 2.0 ** -7)
    draft.accept_draft([[0, 1], [0, 1]])
    nxt = torch.randint(0, 500, (2, 1), generator=g).to(DEV)
    first = draft.decode_forward(following[:, 2:])
    close(first, logits[:, 2:], 2.0 ** -7)
    close(draft.decode_forward(nxt), one.decode_forward(nxt), 2.0 ** -7)


def test_one_drafted_token_equals_a_decode_step_that_retrieves():
    draft, one = models(F32, 900, 100)
    ids = torch.tensor([[3], [77]], device=DEV)
    for _ in range(20):   # over index refreshes
        logits = draft.draft_forward(ids)
        refreshes = draft.kv_cache._zones[0].next_append_refreshes()
        want = one.decode_forward(ids)
        if refreshes:   # the decode step attends with the new index, and its rows of the next layers are of that: decoded here too
            draft.accept_draft([[], []])
            close(draft.decode_forward(ids), want, 2.0 ** -7)
        else:
            close(logits, want, 2.0 ** -7)
            draft.accept_draft([[0], [0]])
        assert draft.kv_cache._zones == one.kv_cache._zones
        ids = want.argmax(-1)


def test_batch_paths_differ():
    """Sequences of a batch accept different tokens, as many each."""
    draft, one = models(F32, 200, 2000)
    g = torch.Generator().manual_seed(2)
    ids = torch.randint(0, 500, (2, 4), generator=g).to(DEV)
    draft.draft_forward(ids, [-1, 0, 0, -1])
    draft.accept_draft([[0, 2], [0, 1]])
    for at in ([0, 0], [2, 1]):
        one.decode_forward(torch.stack([ids[b, t] for b, t in enumerate(at)])[:, None])
    nxt = torch.randint(0, 500, (2, 1), generator=g).to(DEV)
    close(draft.decode_forward(nxt), one.decode_forward(nxt), 2.0 ** -7)


@pytest.mark.parametrize("group", [32, 128])
def test_four_bit_weights(group):
    """The 4-bit model against the fp32 model of the weights it holds.  bf16 rounds some 12 values of each layer's way by 2^-8, 36 in all and the
    logits': at most 37 * 2^-8 < 0.15 of the values' size if all of them added up; a quarter bounds it with the normalisations."""
    model, other = models(BF, 300, 2000, weight_bits=4, weight_group=group)
    exact = models(F32, 300, 2000, n=1)[0]
    exact.kv_cache.unified_keys_gpu = [t.float() for t in model.kv_cache.unified_keys_gpu]
    exact.kv_cache.unified_values_gpu = [t.float() for t in model.kv_cache.unified_values_gpu]
    for ly, src in zip(exact.layers, model.layers):
        for name in ("wqkv", "wo", "down_proj"):
            setattr(ly, name, getattr(src, name).dequantize())
        ly.gate_up_proj = torch.cat([src.gate_proj.dequantize(), src.up_proj.dequantize()])
    exact.lm_head, exact.embed_tokens = model.lm_head.dequantize(), model.embed_tokens.float()
    exact.cos_cache, exact.sin_cache = model.cos_cache.float(), model.sin_cache.float()
    g = torch.Generator().manual_seed(4)
    ids = torch.randint(0, 500, (2, 20), generator=g).to(DEV)
    parents = [-1] + [int(torch.randint(-1, i, (), generator=g)) for i in range(1, 20)]
    want = exact.draft_forward(ids, parents)
    got = model.draft_forward(ids, parents)
    close(got, want, 0.25)
    assert torch.equal(got, other.draft_forward(ids, parents))
    roots = [t for t in range(20) if parents[t] < 0]
    close(model.decode_forward(ids[:, roots[0]:roots[0] + 1]), want[:, roots[0]:roots[0] + 1], 0.25)
    close(other.lm(other.layernorm(other.word_embedding(ids), 1e-6, other.norm_weight)),
          exact.lm(exact.layernorm(exact.word_embedding(ids), 1e-6, exact.norm_weight)), 2.0 ** -6)


def test_model_refusals():
    model = models(BF, 50, 2000, n=1)[0]
    with pytest.raises(ValueError, match="weight_bits"):
        models(F32, 50, 2000, n=1, weight_bits=4)
    with pytest.raises(ValueError, match="weight_bits"):
        models(BF, 50, 2000, n=1, weight_bits=8)
    ids = torch.zeros(2, 3, dtype=torch.int64, device=DEV)
    with pytest.raises(RuntimeError, match="draft_forward first"):
        model.accept_draft([[0], [0]])
    for parents in ([-1, 0], [-1, 1, 0], [0, 0, 0], [-2, 0, 0], []):
        with pytest.raises(RuntimeError, match="parents"):
            model.draft_forward(ids, parents)
    with pytest.raises(RuntimeError, match="max_positions"):
        model.draft_forward(torch.zeros(2, 101, dtype=torch.int64, device=DEV))
    model.draft_forward(ids, [-1, 0, 0])
    for path in ([[1], [0]], [[0, 1, 2], [0, 1, 2]], [[0, 1], [0]], [[0]], [[0], [3]], [[0], [-1]]):
        with pytest.raises(RuntimeError, match="path"):
            model.accept_draft(path)
    model.decode_forward(ids[:, :1])
    with pytest.raises(RuntimeError, match="grown"):
        model.accept_draft([[0], [0]])
    model.draft_forward(ids, [-1, 0, 0])
    model.accept_draft([[], []])   # nothing accepted: dropped
    assert model.kv_cache.context == 51
    with pytest.raises(RuntimeError, match="draft_forward first"):
        model.accept_draft([[0], [0]])


@pytest.mark.parametrize("layout", ["transposed", "expanded", "strided", "int32"])
def test_commit_takes_paths_of_any_layout(layout):
    """A path as a host tensor, whatever its strides: what the same numbers as lists leave."""
    bs, hkv, group, t, layers, n = 3, 2, 2, 12, 2, 5
    a, b = (make_cache(False, bs, hkv, hkv * group, layers, 800, 4, 64, 8, 20) for _ in range(2))
    prefill((a, b), 4, bs, 500, hkv, layers)
    g = torch.Generator().manual_seed(9)
    dk, dv = _randn(g, layers, bs, t, hkv, D).to(DEV), _randn(g, layers, bs, t, hkv, D).to(DEV)
    path = torch.stack([torch.randperm(t, generator=g)[:n] for _ in range(bs)])
    if layout == "expanded":
        path = path[:1].expand(bs, n)
    given = {"transposed": lambda: path.t().contiguous().t(), "expanded": lambda: path, "int32": lambda: path.t().contiguous().t().to(torch.int32),
             "strided": lambda: path.repeat_interleave(2, 1)[:, ::2]}[layout]()
    a.commit_draft(dk, dv, given)
    b.commit_draft(dk, dv, path.tolist())
    assert a._zones == b._zones and all(torch.equal(x, y) for x, y in zip(state(a), state(b)))
    one = given[:, :1].t().contiguous().t()   # one token each: a column
    a.commit_draft(dk, dv, one)
    b.commit_draft(dk, dv, path[:, :1].tolist())
    assert a._zones == b._zones and all(torch.equal(x, y) for x, y in zip(state(a), state(b)))


@pytest.mark.parametrize("kinds", [(torch.Tensor, torch.Tensor), (list, torch.Tensor), (torch.Tensor, list), (list, list)])
def test_commit_converts_rows_of_another_type(kinds):
    """Drafted rows of a model in another type enter the cache in its own, stacked or a layer at a time, as a decoded token's rows do."""
    bs, hkv, group, t, layers = 2, 2, 2, 6, 2
    a, b = (make_cache(False, bs, hkv, hkv * group, layers, 800, 4, 64, 8, 20) for _ in range(2))
    prefill((a, b), 4, bs, 500, hkv, layers)
    g = torch.Generator().manual_seed(9)
    dk, dv = _randn(g, layers, bs, t, hkv, D, dtype=F32).to(DEV), _randn(g, layers, bs, t, hkv, D, dtype=F32).to(DEV)
    path = [[0, 3, 5], [1, 2, 4]]
    a.commit_draft(*(x if kind is torch.Tensor else list(x) for x, kind in zip((dk, dv), kinds)), path)
    b.commit_draft(dk.to(BF), dv.to(BF), path)
    assert a._zones == b._zones and all(torch.equal(x, y) for x, y in zip(state(a), state(b)))


@pytest.mark.parametrize("kind,offload", [("polar_cache_adaptivek_varlen", True), ("polar_cache_atten_value_indices_adaptive_k", False)])
@pytest.mark.parametrize("s", [40, 300])
def test_draft_attend_to_everything_in_adaptive_caches(kind, offload, s):
    """Below the length at which they retrieve these caches take drafts as the other does, and a committed path is attended to afterwards."""
    bs, hkv, group, t, layers = 2, 2, 4, 5, 2
    cache = make_cache(offload, bs, hkv, hkv * group, layers, 1000, 4, 64, 32, 50, thr=600, kind=kind, collision_ratio=0.3, candidate_ratio=0.05)
    k, v = prefill((cache,), s, bs, s, hkv, layers)
    g = torch.Generator().manual_seed(3)
    path = torch.tensor([[0, 3], [1, 4]])
    for step in range(2):
        drafts = []
        for l in range(layers):
            q, dk, dv = (_randn(g, bs, t, h, D) for h in (hkv * group, hkv, hkv))
            drafts.append((dk, dv))
            out = cache.draft_attend(q.to(DEV), dk.to(DEV), dv.to(DEV), l)
            rows = [x[l].transpose(1, 2).contiguous() for x in (k, v)]
            check(out, *exact_tree(dict(q=q, segs=[(*rows, 0, s + 2 * step)], dk=dk, dv=dv, mask=None, rk=None)))
        cache.commit_draft([d[0].to(DEV) for d in drafts], [d[1].to(DEV) for d in drafts], path)
        kept = lambda x: torch.stack([x[b, path[b]] for b in range(bs)])
        k, v = (torch.cat([x, torch.stack([kept(d[i]) for d in drafts])], 2) for i, x in enumerate((k, v)))
