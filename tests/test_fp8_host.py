"""What the operators in eight bits refuse, and their host-side rules: no GPU, nothing is launched (host tensors that say they are on a GPU stand in
for device tensors; every call ends in the checks, at a null pointer or at a recorder in front of the entry points)."""
import contextlib
import ctypes

import pytest
import torch

from pariskv_amd import _lib, ops
from test_drafts_host import On

BF, F32, U8, I32, I64 = torch.bfloat16, torch.float32, torch.uint8, torch.int32, torch.int64
REAL_LAUNCH = ops._launch


@pytest.fixture(autouse=True)
def launches(monkeypatch):
    """(device, entry point) of every launch, in place of it."""
    seen = []
    monkeypatch.setattr(ops, "_stream", lambda t: None)
    monkeypatch.setattr(ops, "_launch", lambda at, entry, *args: seen.append((at, entry.__name__)))
    return seen


class Gpu(On):
    """A host tensor on a GPU, whose views and allocations are there too."""

    def __init__(self, t, device="cuda:0"):
        super().__init__(t, device)
        self.dtype, self.shape = t.dtype, t.shape

    def __getattr__(self, name):
        got = getattr(self._t, name)
        if name in ("view", "reshape", "contiguous", "new_empty", "clone"):
            return lambda *a, **kw: Gpu(got(*a, **kw), self.device)
        return got


def gpu(*shape, dtype=BF, device="cuda:0"):
    return Gpu(torch.zeros(*shape, dtype=dtype), device)


def _cache(bs=2, h=2, cap=64, block=16, device="cuda:0", **change):
    a = dict(k=gpu(bs, h, cap, 128, dtype=U8, device=device), k_scale=gpu(bs, h, cap // block, dtype=F32, device=device),
             v=gpu(bs, h, cap, 128, dtype=U8, device=device), v_scale=gpu(bs, h, cap // block, dtype=F32, device=device))
    a.update(change)
    return ops.Fp8KVCache.from_codes(a["k"], a["k_scale"], a["v"], a["v_scale"], block=change.get("block", block))


@pytest.mark.parametrize("change", [
    dict(k=gpu(2, 2, 64, 64, dtype=U8)), dict(k=gpu(2, 2, 48, 128, dtype=U8)), dict(k=gpu(2, 2, 64, 128)), dict(v=gpu(2, 2, 64, 128, dtype=I32)),
    dict(k=Gpu(torch.zeros(2, 64, 2, 128, dtype=U8).transpose(1, 2))), dict(k_scale=gpu(2, 2, 4)), dict(v_scale=gpu(2, 2, 3, dtype=F32)),
    dict(v_scale=Gpu(torch.zeros(2, 4, 2).transpose(1, 2))), dict(k=gpu(2, 2, 64, 128, dtype=U8, device="cuda:1")),
    dict(k_scale=gpu(2, 2, 4, dtype=F32, device="cuda:1")), dict(k_scale=torch.zeros(2, 2, 4)), dict(k=torch.zeros(2, 2, 64, 128, dtype=U8)),
    dict(block=8), dict(block=48), dict(block=256), dict(k=Gpu(torch.zeros(2 * 2 * 64 * 128 + 8, dtype=U8)[8:].view(2, 2, 64, 128)))])
def test_cache_refuses(change):
    with pytest.raises(RuntimeError):
        _cache(**change)


def test_cache_shapes():
    for bad in ((0, 2, 64), (2, 0, 64), (2, 2, 0)):
        with pytest.raises(RuntimeError):
            ops.Fp8KVCache(*bad, "cuda:0")
    with pytest.raises(RuntimeError, match="16, 32, 64 or 128"):
        ops.Fp8KVCache(1, 1, 64, "cuda:0", block=24)


def _kv(n=3, dtype=BF, device="cuda:0", bs=2, h=2):
    return gpu(bs, n, h, 128, dtype=dtype, device=device)


def test_store_refuses(launches):
    c = _cache()
    c.store(_kv(), _kv(), 4)
    c.store(_kv(0), _kv(0), 4)  # nothing to do
    c.store(_kv(), _kv(), gpu(2, dtype=I32), gpu(2, dtype=I32))
    assert launches == [(0, "pkv_fp8_store")] * 2
    for k, v, kw in ((_kv(), _kv(4), {}), (_kv(), _kv(dtype=F32), {}), (_kv(dtype=torch.float16), _kv(dtype=torch.float16), {}), (_kv(bs=1), _kv(bs=1), {}),
                     (_kv(h=4), _kv(h=4), {}), (gpu(2, 3, 2, 64), gpu(2, 3, 2, 64), {}), (_kv(device="cuda:1"), _kv(), {}), (_kv(), _kv(device="cuda:1"), {}),
                     (_kv()._t, _kv(), {}), (_kv(), _kv()._t, {}), (_kv(), _kv(), dict(start=gpu(2, dtype=I64))), (_kv(), _kv(), dict(start=gpu(3, dtype=I32))),
                     (_kv(), _kv(), dict(start=gpu(2, dtype=I32, device="cuda:1"))), (_kv(), _kv(), dict(lengths=gpu(2, dtype=F32))),
                     (_kv(), _kv(), dict(lengths=Gpu(torch.zeros(4, dtype=I32)[::2]))), (_kv(), _kv(), dict(lengths=gpu(2, 1, dtype=I32)))):
        with pytest.raises(RuntimeError):
            c.store(k, v, **kw)
    assert len(launches) == 2


def test_read_refuses(launches):
    c = _cache()
    out = lambda n=5, **kw: (gpu(2, 2, n, 128, **kw), gpu(2, 2, n, 128, **kw))
    c.read(3, 5, out=out())
    c.read(3, idx=gpu(2, 2, 5, dtype=I64), out=out())
    c.read(3, 0, out=out(0))
    assert launches == [(0, "pkv_fp8_read")] * 2
    for a, kw in (((60, 5), {}), ((-1, 5), {}), ((0, 65), {}), ((3, -1), dict(out=out())), ((64, 1), dict(idx=gpu(2, 2, 5, dtype=I64))),
                  ((-1, 1), dict(idx=gpu(2, 2, 5, dtype=I64))), ((0, 6), dict(idx=gpu(2, 2, 5, dtype=I64))), ((0, 5), dict(idx=gpu(2, 2, 5, dtype=I32))),
                  ((0, 5), dict(idx=gpu(2, 1, 5, dtype=I64))), ((0, 5), dict(idx=gpu(2, 2, 5, dtype=I64, device="cuda:1"))), ((0, 5), dict(idx=torch.zeros(2, 2, 5, dtype=I64))),
                  ((0, 5), dict(out=out(4))), ((0, 5), dict(out=out(dtype=F32))), ((0, 5), dict(out=out(device="cuda:1"))), ((0, 5), dict(dtype=torch.float16)),
                  ((0, 5), dict(out=(Gpu(torch.zeros(2, 2, 5, 132, dtype=BF)[..., :128]),) * 2)), ((0, 5), dict(out=(Gpu(torch.zeros(2, 2, 128, 5, dtype=BF).mT),) * 2))):
        with pytest.raises(RuntimeError):
            c.read(*a, **kw)
    assert len(launches) == 2


def test_attention_refuses(launches):
    c, plan = _cache(), ops.Fp8Attention(2, 2, 4, 6, 60, "cuda:0")
    q, idx = gpu(2, 5, 8, 128), gpu(2, 2, 9, dtype=I64)
    plan.run(q, c, [(0, 20), (30, 9, idx)], row_keys=gpu(2, 2, dtype=I32), out=gpu(2, 5, 8, 128))
    assert launches == [(0, "pkv_fp8_attention")]
    whole = [(0, 20)]
    for queries, segments, kw in (
            (gpu(2, 7, 8, 128), whole, {}), (gpu(2, 0, 8, 128), whole, {}), (gpu(2, 5, 7, 128), whole, {}), (gpu(2, 5, 8, 64), whole, {}), (gpu(1, 5, 8, 128), whole, {}),
            (gpu(2, 8, 128), whole, {}), (gpu(2, 5, 8, 128, dtype=torch.float16), whole, {}), (gpu(2, 5, 8, 128, device="cuda:1"), whole, {}), (q._t, whole, {}),
            (q, [(0, 1)] * 5, {}), (q, [(0, 61)], {}), (q, [(60, 5)], {}), (q, [(-1, 5)], {}), (q, [(0, -1)], {}), (q, [(0, 40), (0, 30)], {}), (q, [(64, 1, idx)], {}),
            (q, [(0, 10, idx)], {}), (q, [(0, 9, gpu(2, 2, 9, dtype=I32))], {}), (q, [(0, 9, gpu(2, 1, 9, dtype=I64))], {}), (q, [(0, 9, gpu(2, 2, 9, dtype=I64, device="cuda:1"))], {}),
            (q, [(0, 4, Gpu(torch.zeros(2, 2, 9, dtype=I64)[..., ::2]))], {}), (q, whole, dict(row_keys=gpu(2, 2))), (q, whole, dict(row_keys=gpu(2, dtype=I32))),
            (q, whole, dict(row_keys=gpu(2, 2, dtype=I32, device="cuda:1"))), (q, whole, dict(out=gpu(2, 5, 8, 128, dtype=F32))), (q, whole, dict(out=gpu(2, 4, 8, 128))),
            (q, whole, dict(out=gpu(2, 5, 8, 128, device="cuda:1"))), (q, whole, dict(out=Gpu(torch.zeros(2, 8, 5, 128, dtype=BF).transpose(1, 2))))):
        with pytest.raises(RuntimeError):
            plan.run(queries, c, segments, **kw)
    for other in (_cache(bs=1), _cache(h=4), _cache(device="cuda:1")):
        with pytest.raises(RuntimeError):
            plan.run(q, other, whole)
    for bad in ((0, 2, 4, 6), (2, 0, 4, 6), (2, 2, 0, 6), (2, 2, 4, 0), (2, 2, 4, 1025), (1, 1, 33, 256)):
        with pytest.raises(RuntimeError, match="query"):
            ops.Fp8Attention(*bad, 100, "cuda:0")
    assert len(launches) == 1


def _weight(n=20, k=200, device="cuda:0"):
    return ops.Fp8Weight(gpu(_lib.lib().pkv_fp8_bytes(n, k), dtype=U8, device=device), n, k)


def test_rows_norms_and_products_refuse(launches):
    ops.fp8_rows(gpu(3, 200))
    for bad in (gpu(3, 200, dtype=torch.float16), gpu(3, 0), torch.zeros(3, 200, dtype=BF), Gpu(torch.zeros((), dtype=BF))):
        with pytest.raises(RuntimeError):
            ops.fp8_rows(bad)
    x, w = gpu(3, 200), gpu(200)
    ops.add_rmsnorm_fp8(x, gpu(3, 200), w, 1e-6, want_sum=False)
    for a in ((gpu(3, 200, dtype=F32), None, w), (x._t, None, w), (Gpu(torch.zeros(200, 3, dtype=BF).t()), None, w), (x, None, gpu(199)), (x, None, gpu(200, dtype=F32)),
              (x, None, Gpu(torch.zeros(400, dtype=BF)[::2])), (x, None, gpu(200, device="cuda:1")), (x, gpu(3, 199), w), (x, gpu(3, 200, dtype=F32), w),
              (x, gpu(3, 200, device="cuda:1"), w), (x, Gpu(torch.zeros(200, 3, dtype=BF).t()), w), (gpu(3, 0), None, gpu(0))):
        with pytest.raises(RuntimeError):
            ops.add_rmsnorm_fp8(*a, 1e-6)
    weight, rows = _weight(), ops.Fp8Rows(gpu(3, 256, dtype=ops.FP8), gpu(3, dtype=F32), (3, 200))
    ops.fp8_linear(rows, weight, bias=gpu(20))
    assert launches == [(0, "pkv_fp8_rows"), (0, "pkv_add_rmsnorm_fp8"), (0, "pkv_fp8_linear")]
    other = ops.Fp8Rows(gpu(3, 256, dtype=ops.FP8, device="cuda:1"), gpu(3, dtype=F32, device="cuda:1"), (3, 200))
    for a, kw in (((rows, _weight(k=201)), {}), ((other, weight), {}), ((rows, weight), dict(bias=gpu(19))), ((rows, weight), dict(bias=gpu(20, dtype=F32))),
                  ((rows, weight), dict(bias=gpu(20, device="cuda:1"))), ((rows, weight), dict(bias=Gpu(torch.zeros(40, dtype=BF)[::2]))),
                  ((rows, weight), dict(out_dtype=torch.float16))):
        with pytest.raises(RuntimeError):
            ops.fp8_linear(*a, **kw)
    for bad in ((gpu(100, dtype=U8), 20, 200), (gpu(_lib.lib().pkv_fp8_bytes(20, 200)), 20, 200), (gpu(0, dtype=U8), 0, 200)):
        with pytest.raises(RuntimeError, match="packed"):
            ops.Fp8Weight(*bad)
    for codes, scales in ((gpu(20, 200, dtype=U8), gpu(19, dtype=F32)), (gpu(20, 200, dtype=U8), gpu(20)), (gpu(20, 200), gpu(20, dtype=F32)),
                          (gpu(20, 200, dtype=U8), gpu(20, dtype=F32, device="cuda:1")), (gpu(20, 200, dtype=U8)._t, gpu(20, dtype=F32))):
        with pytest.raises(RuntimeError):
            ops.Fp8Weight.from_codes(codes, scales)
        with pytest.raises(RuntimeError):
            ops.Fp8Rows.from_codes(codes, scales)
    with pytest.raises(RuntimeError):
        ops.Fp8Weight.quantize(gpu(0, 200))
    assert len(launches) == 3


def test_launches_go_to_the_tensors_gpu(launches, monkeypatch):
    """Each entry point is called with the tensors' GPU as the current device, whichever was."""
    at = "cuda:1"
    c = _cache(device=at)
    c.store(_kv(device=at), _kv(device=at))
    c.read(0, 5, out=(gpu(2, 2, 5, 128, device=at), gpu(2, 2, 5, 128, device=at)))
    ops.Fp8Attention(2, 2, 4, 6, 60, at).run(gpu(2, 5, 8, 128, device=at), c, [(0, 20)])
    rows = ops.fp8_rows(gpu(3, 200, device=at))
    ops.add_rmsnorm_fp8(gpu(3, 200, device=at), None, gpu(200, device=at), 1e-6)
    ops.fp8_linear(rows, _weight(device=at))
    assert launches == [(1, "pkv_" + n) for n in ("fp8_store", "fp8_read", "fp8_attention", "fp8_rows", "add_rmsnorm_fp8", "fp8_linear")]
    here, seen = [0], []

    @contextlib.contextmanager
    def device(index):
        was, here[0] = here[0], index
        yield
        here[0] = was

    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(ops, "_this_device", lambda: here[0])
    for index in (0, 1):
        REAL_LAUNCH(index, lambda *a: seen.append((here[0], a)) or 0, 5, None)
    assert seen == [(0, (5, None)), (1, (5, None))] and here == [0]
    monkeypatch.setattr(ops._lib, "check", lambda rc: (_ for _ in ()).throw(RuntimeError(str(rc))))
    with pytest.raises(RuntimeError, match="-7"):
        REAL_LAUNCH(0, lambda: -7)


# ------------------------------------------------------------------ the entry points


def _kv_args(**change):
    a = dict(k=1 << 20, v=2 << 20, k_scale=3 << 20, v_scale=4 << 20, bs=1, n_kv_heads=2, capacity=640, block=64)
    a.update(change)
    return _lib.Fp8Kv(*(a[n] for n, _ in _lib.Fp8Kv._fields_))


BAD_CACHES = (dict(k=None), dict(v_scale=None), dict(bs=0), dict(n_kv_heads=0), dict(bs=65536), dict(capacity=0), dict(capacity=(1 << 24) + 64), dict(capacity=650),
              dict(block=0), dict(block=8), dict(block=256), dict(k=(1 << 20) + 8), dict(k_scale=(3 << 20) + 2), dict(capacity=-64))


def test_store_and_read_entry_points():
    L = _lib.lib()

    def store(cache=None, **change):
        a = dict(k=5 << 20, v=6 << 20, dtype=_lib.DTYPE_BF16, n=5, kb=1280, kt=256, kh=128, vb=1280, vt=256, vh=128, start=0, starts=None, lengths=None)
        a.update(change)
        return L.pkv_fp8_store(ctypes.byref(cache if cache is not None else _kv_args()), *a.values(), None)

    def read(cache=None, **change):
        a = dict(row0=0, n=5, idx=None, idx_stride=0, dtype=_lib.DTYPE_BF16, k=5 << 20, v=6 << 20, kb=1280, kh=640, kr=128, vb=1280, vh=640, vr=128)
        a.update(change)
        return L.pkv_fp8_read(ctypes.byref(cache if cache is not None else _kv_args()), *a.values(), None)

    assert L.pkv_fp8_store(None, *[None] * 2, 1, *[0] * 8, None, None, None) == _lib.EINVAL
    for change in BAD_CACHES:
        assert store(_kv_args(**change)) == _lib.EINVAL and read(_kv_args(**change)) == _lib.EINVAL, change
    for change in (dict(k=None), dict(v=None), dict(dtype=7), dict(n=0), dict(n=-1), dict(n=641), dict(start=-1), dict(start=636), dict(start=(1 << 63) - 1), dict(k=(5 << 20) + 8),
                   dict(kb=1284), dict(kt=4), dict(vh=2), dict(starts=2), dict(lengths=6), dict(n=(1 << 63) - 1)):
        assert store(**change) == _lib.EINVAL, change
    for change in (dict(k=None), dict(v=None), dict(dtype=7), dict(n=0), dict(n=-1), dict(n=641), dict(row0=636), dict(row0=-1), dict(row0=640, idx=8, idx_stride=9), dict(idx=8, idx_stride=4),
                   dict(idx=4, idx_stride=9), dict(n=1 << 31, idx=8, idx_stride=1 << 31), dict(row0=(1 << 63) - 1), dict(v=(6 << 20) + 4), dict(kr=4), dict(vb=1),
                   dict(n=1 << 40, idx=8, idx_stride=1 << 40)):
        assert read(**change) == _lib.EINVAL, change


def test_attention_entry_point():
    L = _lib.lib()
    assert L.pkv_fp8_attention(None, None) == _lib.EINVAL

    def args(cache=None, segment=None, **change):
        a = _lib.Fp8AttnArgs()
        a.q, a.out, a.dtype, a.group, a.n_tokens, a.scale = 1 << 20, 2 << 20, _lib.DTYPE_BF16, 4, 5, 0.1
        a.q_stride_b, a.q_stride_t, a.n_segments, a.cache = 5120, 1024, 1, cache or _kv_args()
        a.segments[0] = segment or _lib.Fp8Segment(0, 600, None, 0)
        for n, x in change.items():
            setattr(a, n, x)
        return a

    run = lambda *a, **kw: L.pkv_fp8_attention(ctypes.byref(args(*a, **kw)), None)
    for change in BAD_CACHES:
        assert run(_kv_args(**change)) == _lib.EINVAL, change
    assert run() == _lib.ENOMEM and b"workspace" in L.pkv_last_error()
    need = L.pkv_fp8_attention_ws_bytes(_lib.DTYPE_BF16, 1, 2, 4, 5, 600)
    for change, code in ((dict(ws=1 << 30, ws_bytes=need - 1), _lib.ENOMEM), (dict(ws=(1 << 30) + 8, ws_bytes=need), _lib.ENOMEM), (dict(q=None), _lib.EINVAL), (dict(out=None), _lib.EINVAL),
                         (dict(dtype=7), _lib.EINVAL), (dict(group=0), _lib.EINVAL), (dict(n_tokens=0), _lib.EINVAL), (dict(n_tokens=1025), _lib.EINVAL), (dict(group=1639), _lib.EINVAL),
                         (dict(n_segments=5), _lib.EINVAL), (dict(n_segments=-1), _lib.EINVAL), (dict(q=(1 << 20) + 8), _lib.EINVAL), (dict(out=(2 << 20) + 4), _lib.EINVAL),
                         (dict(q_stride_t=1028), _lib.EINVAL), (dict(q_stride_b=5121), _lib.EINVAL), (dict(row_keys=6), _lib.EINVAL)):
        assert run(**change) == code, (change, L.pkv_last_error())
    most = (1 << 63) - 1
    for segment in ((0, 641, None, 0), (600, 41, None, 0), (641, 0, None, 0), (-1, 5, None, 0), (0, -1, None, 0), (0, 9, 8, 8), (640, 9, 8, 9), (0, 9, 4, 9), (1, most, None, 0),
                    (0, (1 << 24) + 1, 8, 1 << 25), (0, most, 8, most)):
        assert run(segment=_lib.Fp8Segment(*segment)) == _lib.EINVAL, segment
    a = args(_kv_args(capacity=1 << 24), _lib.Fp8Segment(0, 1 << 24, None, 0))
    a.segments[1], a.n_segments = _lib.Fp8Segment(0, 1, None, 0), 2
    assert L.pkv_fp8_attention(ctypes.byref(a), None) == _lib.EINVAL and b"keys" in L.pkv_last_error()
    size = L.pkv_fp8_attention_ws_bytes
    assert size(1, 1, 8, 4, 1, 100000) > 0 and size(1, 1, 8, 4, 1, 0) == 0 and size(1, 1, 8, 4, 1, 64) == 0
    for bad in ((1, 0, 8, 4, 1, 100000), (1, 1, 8, 4, 0, 100000), (1, 1, 8, 4, 1, -1), (1, 70000, 8, 4, 1, 100000)):
        assert size(*bad) == 0, bad


def test_rows_and_product_entry_points():
    L, B = _lib.lib(), 1 << 20
    rows = lambda x=B, dtype=_lib.DTYPE_BF16, step=200, n=3, width=200, codes=2 * B, wide=256, scales=3 * B: L.pkv_fp8_rows(x, dtype, step, n, width, codes, wide, scales, None)
    norm = lambda x=B, res=None, weight=4 * B, n=3, width=200, total=None, codes=2 * B, wide=256, scales=3 * B: L.pkv_add_rmsnorm_fp8(
        x, res, weight, 1e-6, n, width, total, codes, wide, scales, None)
    for bad in (dict(x=None), dict(codes=None), dict(scales=None), dict(n=0), dict(n=-1), dict(n=1 << 31), dict(width=0), dict(width=16385, wide=16512), dict(wide=255), dict(wide=128), dict(wide=264),
                dict(codes=2 * B + 8), dict(scales=3 * B + 2), dict(x=B + 1)):
        assert rows(**bad) == _lib.EINVAL and norm(**bad) == _lib.EINVAL, bad
    assert rows(dtype=7) == _lib.EINVAL and rows(step=-1) == _lib.EINVAL and rows(x=B + 2, dtype=_lib.DTYPE_F32) == _lib.EINVAL
    assert norm(weight=None) == _lib.EINVAL and norm(res=B + 1) == _lib.EINVAL and norm(total=B + 1) == _lib.EINVAL and norm(weight=B + 1) == _lib.EINVAL
    linear = lambda x=B, step=256, xs=2 * B, m=3, packed=3 * B, n=20, k=200, bias=None, y=4 * B, out=_lib.DTYPE_F32: L.pkv_fp8_linear(
        x, step, xs, m, packed, n, k, bias, y, out, None, 0, None)
    for bad in (dict(x=None), dict(xs=None), dict(packed=None), dict(y=None), dict(out=7), dict(m=0), dict(m=(1 << 22) + 1), dict(n=0), dict(k=0), dict(k=(1 << 20) + 1, step=1 << 21), dict(n=1 << 31), dict(m=1 << 22, n=(1 << 18) + 1),
                dict(step=128), dict(step=264), dict(x=B + 8), dict(xs=2 * B + 2), dict(packed=3 * B + 8), dict(bias=B + 1), dict(y=4 * B + 8)):
        assert linear(**bad) == _lib.EINVAL, bad
    need = L.pkv_fp8_linear_ws_bytes(145, 955, 12288, _lib.DTYPE_F32)
    assert need > 0 and need % (145 * 956 * 4) == 0 and L.pkv_fp8_linear_ws_bytes(3, 20, 200, _lib.DTYPE_BF16) == 0
    for ws, size in ((None, 0), (None, need), (5 * B, need - 1), (5 * B + 8, need)):
        assert L.pkv_fp8_linear(B, 12288, 2 * B, 145, 3 * B, 955, 12288, None, 4 * B, _lib.DTYPE_F32, ws, size, None) == _lib.ENOMEM and b"workspace" in L.pkv_last_error()
    for bad in ((0, 955, 12288), (145, 0, 12288), (145, 955, 0), ((1 << 22) + 1, 955, 12288)):
        assert L.pkv_fp8_linear_ws_bytes(*bad, _lib.DTYPE_BF16) == 0, bad
    assert L.pkv_fp8_pack(None, 200, B, 20, 200, B, None) == _lib.EINVAL and L.pkv_fp8_pack(B, 199, B, 20, 200, B, None) == _lib.EINVAL
    assert L.pkv_fp8_pack(B, 200, B, 20, 200, B + 8, None) == _lib.EINVAL and L.pkv_fp8_pack(B, 200, B + 2, 20, 200, B, None) == _lib.EINVAL
    assert L.pkv_fp8_unpack(None, 20, 200, B, None) == _lib.EINVAL and L.pkv_fp8_unpack(B + 8, 20, 200, B, None) == _lib.EINVAL
    size = L.pkv_fp8_bytes
    assert size(16, 128) == 2048 + 64 and size(1, 1) == 2048 + 64 and size(17, 129) == 4 * 2048 + 128
    for bad in ((0, 128), (16, 0), (-1, 128), (16, (1 << 20) + 1), (1 << 31, 128)):
        assert size(*bad) == 0, bad


def test_fp8_cache_refuses():
    from pariskv_amd.cache_hub.fp8_cache import fp8_cache

    def make(heads=2, group=4, dim=128, dtype=BF, device="cuda:0", **kw):
        return fp8_cache(0, 1, 2, 100, heads, heads * group, dim, dtype, {"0": device}, **kw)

    for kw, kind in ((dict(dim=64), ValueError), (dict(dtype=torch.float16), ValueError), (dict(device="cpu"), RuntimeError), (dict(block=48), RuntimeError)):
        with pytest.raises(kind) as e:
            make(**kw)
        assert "HIP" not in str(e.value)
    with pytest.raises(ValueError, match="multiple"):
        fp8_cache(0, 1, 2, 100, 3, 8, 128, BF, {"0": "cuda:0"})


def test_struct_mirrors():
    for which, mirror in ((10, _lib.Fp8Kv), (11, _lib.Fp8AttnArgs)):
        assert _lib.lib().pkv_struct_bytes(which) == ctypes.sizeof(mirror) > 0
    assert ops._FP8_ATTN_BLOCK.size == ctypes.sizeof(_lib.Fp8AttnArgs)


def test_product_plan():
    L, plan = _lib.lib(), (ctypes.c_int * 4)()
    for bad in ((0, 955, 12288), (145, 0, 12288), (145, 955, 0), ((1 << 22) + 1, 955, 12288), (145, 1 << 31, 128)):
        assert L.pkv_fp8_linear_plan(*bad, plan) == _lib.EINVAL, bad
    assert L.pkv_fp8_linear_plan(145, 955, 12288, None) == _lib.EINVAL
    for m, n, k in ((1, 1, 1), (16, 4096, 4096), (17, 4096, 4096), (145, 955, 12288), (4096, 6144, 4096), (1 << 22, 16, 128), (1 << 22, 1 << 15, 128), (1, 1 << 28, 128)):
        assert L.pkv_fp8_linear_plan(m, n, k, plan) == 0
        bm, bn, splits, at_once = plan
        assert bm in (16, 32, 64, 128) and bn in (16, 32, 64, 128) and at_once in (1, 2) and 1 <= splits <= 16 and splits <= -(-k // 128)
        # the workspace is that of these splits, and a launch's workgroups and threads are within its limits
        for dtype in (_lib.DTYPE_BF16, _lib.DTYPE_F32):
            assert L.pkv_fp8_linear_ws_bytes(m, n, k, dtype) == (0 if splits == 1 else splits * m * (-(-n // 4) * 4) * 4)
        down, across, threads = -(-m // bm), -(-n // bn), 512 if bm * bn <= 2048 else 256
        assert (down <= 65535 and across * threads < 1 << 32) if threads == 512 else down * across * threads < 1 << 32
    weight = _weight()
    assert weight.plan(3) == (16, 16, 1, 1)
    with pytest.raises(RuntimeError):
        weight.plan(0)


def test_layer_takes_any_packing():
    """A layer whose weights are packed to 4 bits has the two matrices that the gated product takes; any other packing goes to both as one."""
    from pariskv_amd.model_hub.qwen import QwenConfig, QwenLayer

    cfg = QwenConfig(hidden_size=16, num_layers=1, num_heads=2, num_key_value_heads=1, intermediate_size=8, vocab_size=5)
    layer = lambda pack: QwenLayer(cfg, "cpu", F32, torch.Generator().manual_seed(1), pack)
    four = layer(lambda w: ops.W4Weight.__new__(ops.W4Weight))
    assert four.gate_up_proj is None and isinstance(four.gate_proj, ops.W4Weight) and isinstance(four.up_proj, ops.W4Weight)
    shapes = []
    eight = layer(lambda w: shapes.append(tuple(w.shape)) or ops.Fp8Weight.__new__(ops.Fp8Weight))
    assert isinstance(eight.gate_up_proj, ops.Fp8Weight) and (16, 16) in shapes and not hasattr(eight, "gate_proj")
    assert tuple(layer(None).gate_up_proj.shape) == (16, 16)
