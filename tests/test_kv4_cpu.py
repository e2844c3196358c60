"""Refusals of the 4-bit cache and of sampling that need no GPU: null arguments in the C ABI, and
tensors of another type, shape or device in the Python classes (a stand-in context; nothing of the
library runs).  The numpy definitions are checked against plain loops."""
import ctypes as C

import numpy as np
import pytest

from oracle import kv4 as ok
from oracle import sampling as osm


class _Ctx:
    h, device = None, 0


def test_null_arguments_are_refused():
    from voxcpm_rs_b200 import _lib
    L = _lib.lib()
    c = _lib.Kv4C(None, None, None, None, None, None, 1, 1, 32, 64)
    ref = C.addressof(c)
    assert L.vx_kv4_append(None, ref, None, None, 0, 0, 1, None, None, None, None) == _lib.VX_ERR_ARG
    assert L.vx_kv4_read(None, ref, 1, None, None, None, None, None) == _lib.VX_ERR_ARG
    assert L.vx_kv4_attend(None, ref, None, 0, 1, None, 1, 1.0, 0, None, 0, None, 0, None) == _lib.VX_ERR_ARG
    assert L.vx_kv4_evict(None, ref, None, None, 1, 1, 0, 0, None, None, None, None) == _lib.VX_ERR_ARG
    assert L.vx_lm_sample(None, None, 1, 1, 1, None, None, None, None, None, None) == _lib.VX_ERR_ARG
    assert L.vx_sample(None, None, 1, 1, 1, None, None, None, None, None, None, None, None) == _lib.VX_ERR_ARG


def test_attend_workspace():
    """0 for arguments that a call refuses and for short sequences; else it grows with the length,
    and a tracking call's holds a score of 8 query heads for each row."""
    from voxcpm_rs_b200 import _lib
    f = _lib.lib().vx_kv4_attend_workspace
    c = _lib.Kv4C(None, None, None, None, None, None, 2, 2, 131072, 128)
    ref = C.addressof(c)
    assert f(None, 8, 10, 0) == 0 and f(ref, 0, 10, 0) == 0 and f(ref, 3, 10, 0) == 0 and f(ref, 16, -1, 0) == 0
    assert [f(ref, 16, n, t) for n in (0, 1, 500, 4096) for t in (0, 1)] == [0] * 8
    assert f(ref, 16, 131072, 0) > f(ref, 16, 8192, 0) > 0
    for n in (5000, 131072):
        assert f(ref, 16, n, 1) >= f(ref, 16, n, 0) + 2 * 2 * n * 8 * 4
    assert f(ref, 32, 100, 1) >= 2 * 2 * 2 * 100 * 8 * 4  # 16 query heads share a KV head: two blocks of them


def _bufs(b=1, nkv=2, cap=64, d=64):
    import torch
    codes = lambda: torch.zeros(b, nkv, cap, d // 2, dtype=torch.uint8)  # noqa: E731
    scales = lambda: torch.zeros(b, nkv, cap, d // 16, dtype=torch.uint8).view(torch.float8_e4m3fn)  # noqa: E731
    return [codes(), scales(), codes(), scales()]


def test_buffers_of_another_device_are_refused():
    from voxcpm_rs_b200._lib import VX_ERR_ARG, VxError
    from voxcpm_rs_b200.kv4 import Kv4Cache
    with pytest.raises(VxError) as e:
        Kv4Cache.from_buffers(_Ctx(), *_bufs())  # host tensors, a context of cuda:0
    assert e.value.code == VX_ERR_ARG and "cuda:0" in str(e.value)


@pytest.fixture
def host_cache(monkeypatch):
    """A cache over host tensors (whose device index is -1): the classes' own checks alone."""
    import torch
    from voxcpm_rs_b200 import kv4

    class Lib:
        def __getattr__(self, n):
            return (lambda *a: 0) if n.endswith("workspace") else (lambda *a: pytest.fail(n + " was called"))

    class Torch:
        def __getattr__(self, n):
            return (lambda *a: torch.device("cpu")) if n == "device" else getattr(torch, n)

    monkeypatch.setattr(kv4, "lib", Lib)
    monkeypatch.setattr(kv4, "_torch", Torch)
    monkeypatch.setattr(_Ctx, "device", -1)
    w, p = torch.zeros(1, 2, 64), torch.zeros(1, 2, 64, dtype=torch.int64)
    return kv4.Kv4Cache.from_buffers(_Ctx(), *_bufs(), weights=w, positions=p)


def test_cache_arguments_are_checked(host_cache):
    import torch
    from voxcpm_rs_b200._lib import VxError
    from voxcpm_rs_b200.kv4 import Kv4Cache
    c = host_cache
    i = torch.zeros(1, dtype=torch.int32)
    x = torch.zeros(1, 3, 2, 64)
    q = torch.zeros(1, 4 * 64)
    bad = [
        lambda: c.append(x.double(), x, i), lambda: c.append(x, x[:, :2], i), lambda: c.append(x, x, i.long()),
        lambda: c.append(x, x, torch.zeros(2, dtype=torch.int32)), lambda: c.append(x, x, i, i.float()),
        lambda: c.append(torch.zeros(1, 3, 64, 2).transpose(2, 3), torch.zeros(1, 3, 64, 2).transpose(2, 3), i),
        lambda: c.append(x, torch.zeros(1, 6, 2, 64)[:, ::2], i), lambda: c.append(x[0], x[0], i),
        lambda: c.read(-1), lambda: c.read(1, i.long()), lambda: c.read(1, counts=torch.zeros(2, dtype=torch.int32)),
        lambda: c.attend(q.half(), i), lambda: c.attend(q[0], i), lambda: c.attend(torch.zeros(2, 256), i),
        lambda: c.attend(torch.zeros(1, 100), i), lambda: c.evict(i, i, 8, weights_out=torch.zeros(1, 2, 32)),
        lambda: c.evict(i, i, 8, positions_out=torch.zeros(1, 2, 64)),
        lambda: Kv4Cache.from_buffers(_Ctx(), *_bufs()).evict(i, i, 8),
        lambda: Kv4Cache.from_buffers(_Ctx(), *_bufs()[:3], _bufs(cap=32)[3]),
        lambda: Kv4Cache.from_buffers(_Ctx(), *_bufs(), weights=torch.zeros(1, 2, 63)),
        lambda: Kv4Cache.from_buffers(_Ctx(), *_bufs(), positions=torch.zeros(1, 2, 64, dtype=torch.int32)),
    ]
    for n, call in enumerate(bad):
        with pytest.raises(VxError):
            call()
            raise AssertionError(f"call {n} was not refused")


def test_strides_of_one_token_or_sequence_do_not_matter(host_cache, monkeypatch):
    """A dimension of size 1 has no stride: rows that lie alike are not refused for it."""
    import torch
    got = []
    lib = type("Lib", (), {"vx_kv4_append": lambda self, *a: got.append(a[4:7]) or 0})()
    monkeypatch.setattr(host_cache, "_L", lib)
    monkeypatch.setattr(host_cache, "_raw_stream", lambda i: 0)
    i = torch.zeros(1, dtype=torch.int32)
    dense, fused = torch.zeros(1, 1, 2, 64), torch.zeros(400).as_strided((1, 1, 2, 64), (390, 3, 64, 1))
    assert dense.stride() != fused.stride()
    host_cache.append(dense, fused, i)
    host_cache.append(torch.zeros(1, 3, 2, 64), torch.zeros(5, 3, 2, 64)[2:3], i)
    assert got == [(0, 0, 1), (0, 128, 3)]


def test_outputs_are_f32_whatever_the_default_type(host_cache, monkeypatch):
    import torch
    from voxcpm_rs_b200.kv4 import Kv4Cache
    before = torch.get_default_dtype()
    try:
        torch.set_default_dtype(torch.bfloat16)
        c = Kv4Cache.from_buffers(_Ctx(), *_bufs())
        monkeypatch.setattr(c, "_L", type("Lib", (), {"vx_kv4_read": lambda self, *a: 0})())
        monkeypatch.setattr(c, "_raw_stream", lambda i: 0)
        assert [t.dtype for t in c.read(3)] == [torch.float32] * 2
        own = Kv4Cache(_Ctx(), 1, 2, 64, 64)
        assert own.weights.dtype is torch.float32
    finally:
        torch.set_default_dtype(before)


def test_plans_do_not_grow_without_end(host_cache, monkeypatch):
    import torch
    monkeypatch.setattr(host_cache, "_L", type("Lib", (), {"vx_kv4_attend_workspace": lambda self, *a: 0,
                                                           "vx_kv4_attend": lambda self, *a: 0})())
    monkeypatch.setattr(host_cache, "_raw_stream", lambda i: 0)
    for n in range(3000):
        host_cache.attend(torch.zeros(1, 256), torch.zeros(1, dtype=torch.int32), n)
    assert len(host_cache._plans) <= 1024


def test_sample_arguments_are_checked():
    import torch
    from voxcpm_rs_b200._lib import VxError
    from voxcpm_rs_b200.sampling import sample
    with pytest.raises(VxError):
        sample(_Ctx(), torch.zeros(2, 10), torch.zeros(2))  # host tensors


# ------------------------------------------------------------------------- the definitions

def test_quantise_definition():
    """Nearest by brute force over all code and scale values, ties to the even pattern."""
    rng = np.random.default_rng(0)
    x = np.concatenate([rng.standard_normal((40, 64)) * 10.0 ** rng.uniform(-4, 3, (40, 1)),
                        rng.integers(-12, 13, (20, 64)) * 0.25]).astype(np.float32)
    codes, s8 = ok.quantise(x)
    table = ok.e4m3_values()
    assert table[-1] == 448 and np.all(np.diff(table) > 0)
    for row, c, s in zip(x.astype(np.float64), codes, s8):
        for g in range(4):
            part = row[g * 16:g * 16 + 16]
            t = min(np.abs(part).max() / 6, 448)
            best = min(range(127), key=lambda i: (abs(table[i] - t), i % 2))
            assert s[g] == best
            for j, v in enumerate(part):
                nib = (c[(g * 16 + j) // 2] >> (4 * (j % 2))) & 15
                want = 0 if table[best] == 0 else min(range(8), key=lambda i: (abs(ok.CODE_VALUES[i] - abs(v) / table[best]), i % 2))
                assert nib & 7 == want and bool(nib & 8) == bool(np.signbit(v))
    back = ok.values(codes, s8)
    assert np.abs(back - x).max() <= np.abs(x).max() / 6 * 1.07


def test_evict_definition():
    w = np.array([5.0, 1.0, 3.0, 3.0, 9.0, 0.0, 3.0], np.float32)
    pos = np.arange(7)
    assert ok.evict(w, pos, 7, 7, 4, 0, 0).tolist() == [0, 4, 2, 3]          # 1 goes, 4 takes its slot; 6 loses the tie
    assert ok.evict(w, pos, 7, 7, 4, 0, 1).tolist() == [0, 4, 2, 6]          # the newest stays, so slot 3 goes
    assert ok.evict(w, pos, 7, 7, 3, 2, 1).tolist() == [0, 1, 6]
    assert ok.evict(w, pos, 3, 3, 4, 0, 0).tolist() == [0, 1, 2]
    assert ok.evict(w, pos, 7, 7, 0, 0, 0).tolist() == []


def test_sample_definition():
    x = np.log(np.array([0.1, 0.4, 0.2, 0.3], np.float32))
    pick = lambda u, **k: osm.sample_row(x, u, **k)[0]  # noqa: E731
    assert [pick(u) for u in (0.0, 0.05, 0.15, 0.55, 0.75, 0.99)] == [0, 0, 1, 2, 3, 3]
    assert [pick(u, top_k=2) for u in (0.0, 0.5, 0.6, 0.99)] == [1, 1, 3, 3]
    assert [pick(u, top_p=0.65) for u in (0.0, 0.5, 0.6, 0.99)] == [1, 1, 3, 3]
    assert [pick(u, min_p=0.6) for u in (0.0, 0.6, 0.99)] == [1, 3, 3]
    assert pick(0.9, temperature=0.0) == 1 and osm.sample_row(x, 0.9, temperature=0.0)[1] == 0.0
