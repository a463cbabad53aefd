"""What the operators of a step over several drafted tokens refuse, and their host-side rules: no GPU, nothing is launched (host
tensors that say they are on a GPU stand in for device tensors; every call ends in the checks or at a null pointer)."""
import contextlib
import ctypes

import pytest
import torch

from pariskv_amd import _lib, ops

BF, F32 = torch.bfloat16, torch.float32


@pytest.fixture(autouse=True)
def no_stream(monkeypatch):
    """Calls reach the library's checks: looking up a stream raises without a GPU."""
    monkeypatch.setattr(ops, "_stream", lambda t: None)


@contextlib.contextmanager
def refuses():
    """A refusal by a check, and not the error of a launch, or of a stream's lookup, on a machine without a GPU."""
    with pytest.raises(RuntimeError) as e:
        yield
    assert not any(words in str(e.value) for words in ("HIP error", "launch of", "No HIP")), str(e.value)


class On:
    """A host tensor that says it is on a GPU."""

    def __init__(self, t, device="cuda:0"):
        self._t, self.device, self.is_cuda = t, torch.device(device), True

    def get_device(self):
        return self.device.index

    def __getattr__(self, name):
        return getattr(self._t, name)


def _tree(**change):
    bs, t, h, g, rows = 2, 5, 2, 4, 40
    a = dict(q=torch.zeros(bs, t, h * g, 128, dtype=BF), k=torch.zeros(bs, h, rows, 128, dtype=BF), v=torch.zeros(bs, h, rows, 128, dtype=BF),
             dk=torch.zeros(bs, t, h, 128, dtype=BF), dv=torch.zeros(bs, t, h, 128, dtype=BF), mask=torch.zeros(bs, t, t, dtype=torch.bool),
             rk=torch.zeros(bs, h, dtype=torch.int32), idx=torch.zeros(bs, h, 9, dtype=torch.int64), out=torch.zeros(bs, t, h * g, 128, dtype=BF))
    where = change.pop("where", {})
    a.update(change)
    return {n: On(x, where.get(n, "cuda:0")) for n, x in a.items()}


def _run(o, row0=0, n=20, segments=None, max_keys=1000):
    att = ops.TreeAttention(2, 2, 4, 6, max_keys, "cuda:0")
    segs = [(o["k"], o["v"], row0, n), (o["k"], o["v"], 3, 9, o["idx"])] if segments is None else segments
    return att.run(o["q"], segs, o["dk"], o["dv"], mask=o["mask"], row_keys=o["rk"], out=o["out"])


def test_tree_attention_refuses_other_devices():
    for name in ("k", "v", "dk", "dv", "mask", "rk", "idx", "out"):
        with pytest.raises(RuntimeError, match="tensors of one launch"):
            _run(_tree(where={name: "cuda:1"}))
    host = _tree()
    host["dk"] = host["dk"]._t
    with pytest.raises(RuntimeError, match="must be on the GPU"):
        _run(host)


@pytest.mark.parametrize("change,words", [
    (dict(q=torch.zeros(2, 7, 8, 128, dtype=BF)), "max_draft"), (dict(q=torch.zeros(2, 0, 8, 128, dtype=BF)), "max_draft"),
    (dict(q=torch.zeros(2, 5, 7, 128, dtype=BF)), "queries"), (dict(q=torch.zeros(2, 5, 8, 64, dtype=BF)), "queries"),
    (dict(q=torch.zeros(2, 5, 8, 128, dtype=F32)), "queries' type"), (dict(dk=torch.zeros(2, 4, 2, 128, dtype=BF)), "draft_k"),
    (dict(dv=torch.zeros(2, 5, 2, 128, dtype=F32)), "draft_k"), (dict(k=torch.zeros(2, 2, 40, 128, dtype=F32)), "share a dtype"),
    (dict(k=torch.zeros(2, 2, 39, 128, dtype=BF)), "contiguous rows"), (dict(mask=torch.zeros(2, 5, 5)), "mask"),
    (dict(mask=torch.zeros(3, 5, 5, dtype=torch.bool)), "mask"), (dict(mask=torch.zeros(5, 4, dtype=torch.bool)), "mask"),
    (dict(rk=torch.zeros(2, 2)), "row_keys"), (dict(rk=torch.zeros(2, 3, dtype=torch.int32)), "row_keys"),
    (dict(idx=torch.zeros(2, 2, 8, dtype=torch.int64)), "indices"), (dict(idx=torch.zeros(2, 2, 9, dtype=torch.int32)), "indices"),
    (dict(out=torch.zeros(2, 5, 8, 128)), "out"), (dict(out=torch.zeros(2, 8, 5, 128, dtype=BF).transpose(1, 2)), "out")])
def test_tree_attention_refuses(change, words):
    with pytest.raises(RuntimeError, match=words):
        _run(_tree(**change))


def test_tree_attention_refuses_rows_and_counts():
    o = _tree()
    for row0, n in ((30, 11), (-1, 5), (0, 41)):
        with pytest.raises(RuntimeError, match="out of range"):
            _run(o, row0, n)
    with pytest.raises(RuntimeError, match="max_keys"):
        _run(o, max_keys=28)
    with pytest.raises(RuntimeError, match="0..4"):
        _run(o, segments=[(o["k"], o["v"], 0, 1)] * 5)
    for bad in ((0, 2, 4, 6), (2, 0, 4, 6), (2, 2, 0, 6), (2, 2, 4, 0), (2, 2, 4, 1025), (1, 1, 33, 256)):
        with pytest.raises(RuntimeError, match="drafted tokens"):
            ops.TreeAttention(*bad, 100, "cuda:0")


def test_tree_attention_entry_point_checks_its_arguments():
    L = _lib.lib()
    assert L.pkv_tree_attention(None, None) == _lib.EINVAL

    def args(**change):
        a = _lib.TreeArgs()
        a.q, a.out, a.draft_k, a.draft_v, a.dtype = 1 << 20, 2 << 20, 3 << 20, 4 << 20, _lib.DTYPE_BF16
        a.bs, a.n_kv_heads, a.group, a.n_draft, a.q_stride_t, a.scale = 1, 2, 4, 5, 1024, 0.1
        a.segments[0] = _lib.AttnSegment(5 << 20, 6 << 20, 0, 1 << 20, 0, 5000, None, 0, 0)
        a.n_segments = 1
        for n, x in change.items():
            setattr(a, n, x)
        return a

    for change, code, words in ((dict(), _lib.ENOMEM, b"workspace"), (dict(ws=1 << 30, ws_bytes=100), _lib.ENOMEM, b"workspace"),
                                (dict(q=None), _lib.EINVAL, b"null"), (dict(draft_v=None), _lib.EINVAL, b"null"), (dict(dtype=7), _lib.EINVAL, b"dtype"),
                                (dict(n_draft=1025), _lib.EINVAL, b"shape"), (dict(group=3000), _lib.EINVAL, b"shape"), (dict(bs=0), _lib.EINVAL, b"shape"),
                                (dict(bs=65536), _lib.EINVAL, b"shape"), (dict(n_segments=5), _lib.EINVAL, b"segments"), (dict(q=(1 << 20) + 8), _lib.EINVAL, b"aligned"),
                                (dict(q_stride_t=1028), _lib.EINVAL, b"strides"), (dict(dk_stride_b=-8), _lib.EINVAL, b"strides"),
                                (dict(mask=8, mask_stride_t=-5), _lib.EINVAL, b"mask"), (dict(row_keys=6), _lib.EINVAL, b"row_keys")):
        a = args(**change)
        assert L.pkv_tree_attention(ctypes.byref(a), None) == code and words in L.pkv_last_error(), (change, L.pkv_last_error())
    a = args()
    a.segments[0].n_rows = 1 << 23
    assert L.pkv_tree_attention(ctypes.byref(a), None) == _lib.EINVAL and b"2^23" in L.pkv_last_error()
    a.segments[0].n_rows, a.segments[0].stride_h = 5000, 4
    assert L.pkv_tree_attention(ctypes.byref(a), None) == _lib.EINVAL
    assert L.pkv_tree_attention_ws_bytes(1, 1, 1, 1, 1, 0) == 0 and L.pkv_tree_attention_ws_bytes(1, 0, 1, 1, 1, 100) == 0
    assert L.pkv_tree_attention_ws_bytes(1, 1, 8, 4, 5, 100000) > 0


def test_tree_mask():
    def walk(parents):
        t = len(parents)
        m = torch.zeros(t, t, dtype=torch.bool)
        for i in range(t):
            at = i
            while at >= 0:
                m[i, at], at = True, parents[at]
        return m

    g = torch.Generator().manual_seed(0)
    for t in (1, 2, 3, 8, 33, 64):
        p = (torch.rand(3, t, generator=g) * (torch.arange(t) + 1)).long() - 1
        want = torch.stack([walk(row) for row in p.tolist()])
        assert torch.equal(ops.tree_mask(p), want) and torch.equal(ops.tree_mask(p[1].tolist()), want[1])
        assert torch.equal(ops.tree_mask(list(range(-1, t - 1))), torch.ones(t, t, dtype=torch.bool).tril())
    for bad in ([0], [-1, 1], [-1, 2, 0], [-2]):
        with pytest.raises(RuntimeError, match="parents"):
            ops.tree_mask(bad)


# ------------------------------------------------------------- 4-bit weights


def _codes(n=20, k=256, g=64):
    return On(torch.zeros(n, k, dtype=torch.uint8)), On(torch.zeros(n, k // g, dtype=BF)), On(torch.zeros(n, k // g, dtype=torch.uint8))


def test_w4_bytes():
    size = _lib.lib().pkv_w4_bytes
    assert size(16, 128, 128) == 1024 + 64 and size(1, 32, 32) == 1024 + 256 and size(17, 129 * 32, 32) == 2 * 33 * (1024 + 256)
    for bad in ((0, 128, 128), (16, 0, 32), (16, 100, 32), (16, 128, 16), (16, 96, 64), (16, 128, 256), (1 << 31, 128, 128), (-4, 128, 128)):
        assert size(*bad) == 0, bad


def test_w4_refusals():
    c, s, z = _codes()
    for bad in ((c, s, On(z._t[:, :3])), (On(c._t[:19]), s, z), (On(c._t[:, :250]), s, z), (On(c._t.int()), s, z), (c, On(s._t.float()), z),
                (On(torch.zeros(20, 64, dtype=torch.uint8)), s, z), (c, s, On(z._t, "cuda:1")), (c._t, s, z)):
        with refuses():
            ops.W4Weight.from_codes(*bad)
    w = ops.W4Weight(On(torch.zeros(_lib.lib().pkv_w4_bytes(20, 256, 64), dtype=torch.uint8)), 20, 256, 64)
    other = ops.W4Weight(On(torch.zeros(_lib.lib().pkv_w4_bytes(20, 256, 32), dtype=torch.uint8)), 20, 256, 32)
    with pytest.raises(RuntimeError, match="packed"):
        ops.W4Weight(On(torch.zeros(100, dtype=torch.uint8)), 20, 256, 64)
    x = On(torch.zeros(3, 256, dtype=BF))
    for bad in (On(torch.zeros(3, 255, dtype=BF)), On(torch.zeros(3, 256)), torch.zeros(3, 256, dtype=BF), On(torch.zeros(3, 256, dtype=BF), "cuda:1")):
        with refuses():
            ops.w4_linear(bad, w)
        with refuses():
            ops.w4_silu_mul(bad, w, w)
    for bad in (On(torch.zeros(19, dtype=BF)), On(torch.zeros(20)), On(torch.zeros(40, dtype=BF)[::2]), On(torch.zeros(20, dtype=BF), "cuda:1")):
        with refuses():
            ops.w4_linear(x, w, bad)
    with pytest.raises(RuntimeError, match="one shape"):
        ops.w4_silu_mul(x, w, other)
    for m, g in ((On(torch.zeros(4, 100)), 32), (On(torch.zeros(4, 128)), 16), (torch.zeros(4, 128), 32), (On(torch.zeros(4, 128, dtype=torch.float16)), 32),
                 (On(torch.zeros(128)), 32)):
        with refuses():
            ops.w4_quantize(m, g)
    L = _lib.lib()
    A = 1 << 20
    for args, words in (((A, 128, 4, None, 16, 128, 128, None, A, 1, None, 0, None), b"weights"), ((A, 128, 4, A, 16, 100, 32, None, A, 1, None, 0, None), b"groups"),
                        ((A, 128, 4, A, 16, 128, 128, None, A, 5, None, 0, None), b"dtype"), ((A, 128, 0, A, 16, 128, 128, None, A, 1, None, 0, None), b"row count"),
                        ((A, 120, 4, A, 16, 128, 128, None, A, 1, None, 0, None), b"overlap"), ((A, 129, 4, A, 16, 128, 128, None, A, 1, None, 0, None), b"aligned"),
                        ((A + 2, 128, 4, A, 16, 128, 128, None, A, 1, None, 0, None), b"aligned"), ((None, 128, 4, A, 16, 128, 128, None, A, 1, None, 0, None), b"null")):
        assert L.pkv_w4_linear(*args) == _lib.EINVAL and words in L.pkv_last_error(), (args, L.pkv_last_error())
    assert L.pkv_w4_silu_mul(A, 128, 4, A, None, 16, 128, 128, A, None, 0, None) == _lib.EINVAL
    assert L.pkv_w4_pack(A, A, A, 16, 128, 48, A, None) == _lib.EINVAL and L.pkv_w4_unpack(A, 16, 128, 128, None, None) == _lib.EINVAL
    assert L.pkv_w4_quantize(A, 0, 100, 16, 128, 128, A, A, A, None) == _lib.EINVAL


# ------------------------------------------------------------- the accepted path


def _path(layers=3, bs=2, h=2, rows=20, t=5, dtype=BF):
    return ([On(torch.zeros(bs, h, rows, 128, dtype=dtype)) for _ in range(layers)], [On(torch.zeros(bs, h, rows, 128, dtype=dtype)) for _ in range(layers)],
            [On(torch.zeros(bs, t, h, 128, dtype=dtype)) for _ in range(layers)], [On(torch.zeros(bs, t, h, 128, dtype=dtype)) for _ in range(layers)],
            [On(torch.zeros(bs, h, rows)) for _ in range(layers)])


def test_path_append_refusals():
    k, v, dk, dv, vn = _path()
    for bad in ((k, v[:2]), ([], []), (k, v[:2] + [On(torch.zeros(2, 2, 21, 128, dtype=BF))]), (k, v[:2] + [On(v[2]._t, "cuda:1")]),
                (k, v[:2] + [v[2]._t]), (k, v[:2] + [On(v[2]._t.float())]), (k, v, vn[:2]), (k, v, vn[:2] + [On(torch.zeros(2, 2, 20, dtype=BF))])):
        with refuses():
            ops.PathAppend(*bad)
    plan = ops.PathAppend(k, v)
    path = On(torch.zeros(2, 3, dtype=torch.int64))
    for a, b, p, slots in ((dk[:2], dv, path, 0), (dk, dv, On(torch.zeros(2, 3, dtype=torch.int32)), 0), (dk, dv, On(torch.zeros(3, 3, dtype=torch.int64)), 0),
                           (dk, dv, On(torch.zeros(2, 3, dtype=torch.int64), "cuda:1"), 0), (dk, dv, On(torch.zeros(3, 2, dtype=torch.int64).t()), 0),
                           (dk, dv[:2] + [On(dv[2]._t, "cuda:1")], path, 0), (dk, dv[:2] + [On(torch.zeros(2, 6, 2, 128, dtype=BF))], path, 0),
                           (dk, [On(torch.zeros(2, 6, 2, 128, dtype=BF))] * 3, path, 0), ([On(x._t.float()) for x in dk], dv, path, 0),
                           (dk, dv, path, 18), (dk, dv, path, -1), (dk, dv, path, [0, 0, 18]), (dk, dv, path._t, 0)):
        with refuses():
            plan.launch(a, b, p, slots)
    for slot in (2**62, 2**63 - 1, 2**63 - 3):  # slot + rows passes 64 bits
        with pytest.raises(RuntimeError, match="do not fit"):
            plan.launch(dk, dv, path, slot)
    with pytest.raises(ValueError):
        plan.launch(dk, dv, path, [0, 1])
    L = _lib.lib()
    assert L.pkv_append_path(None, None, None, 0, None) == _lib.EINVAL


def test_new_struct_mirrors_have_the_library_sizes():
    for which, mirror in ((7, _lib.PathLayer), (8, _lib.PathArgs), (9, _lib.TreeArgs)):
        assert _lib.lib().pkv_struct_bytes(which) == ctypes.sizeof(mirror) > 0


def test_tokens_to_refresh():
    from pariskv_amd.cache_hub.zones import LayerZones

    for offload in (False, True):
        for prompt in (0, 1, 5, 11, 12, 13, 40):
            z = LayerZones(4, 8, 3, offload)
            z.prefill(prompt)
            for _ in range(30):
                due, slot, steps = z.tokens_to_refresh(), z.append_slot(), 0
                while True:
                    assert z.append_slot() == slot + steps   # the rows of a run follow one another
                    steps += 1
                    if z.appended() is not None:
                        break
                assert steps == due


@pytest.mark.parametrize("dim,dtype", [(64, F32), (128, torch.float16), (256, BF), (256, torch.float16)])
def test_norms_of_other_rows_are_refused(dim, dtype):
    """The launches tell bf16 rows of 128 elements from fp32 ones by their bytes: rows of as many bytes that are neither would get norms of
    something else."""
    rows = lambda *shape: On(torch.zeros(*shape, dim, dtype=dtype))
    k, v, vn = rows(2, 2, 20), rows(2, 2, 20), On(torch.zeros(2, 2, 20))
    for call in (lambda: ops.PathAppend([k], [v], [vn]), lambda: ops.BoundAppend(k, v, vn), lambda: ops.append_kv(rows(2, 1, 2), rows(2, 1, 2), k, v, 3, vn)):
        with pytest.raises(RuntimeError, match="128 bf16 or fp32"):
            call()
    ops.PathAppend([k], [v]), ops.BoundAppend(k, v)   # without norms any rows are moved
