"""Refusals of ragged attention, shared-prefix attention and the cache read-back: by the C
entry points before a device is touched, and the oracle of their tests against hand-made
answers (no GPU)."""
import ctypes

import numpy as np
import pytest

from gollek_b200 import _lib
from tests import paged_ref as R


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


D = ctypes.c_void_p(16)


def varlen(lib, **kw):
    a = dict(out=D, q=D, k=D, v=D, ks=None, vs=None, bt=D, cu=D, ctx=D, slopes=None, prefix=None, starts=None, S=2,
             total=4, hq=8, hkv=2, d=128, bs=16, maxb=4, nb=0, stride=0, qd=_lib.BF16, kd=_lib.BF16, s0=0, s1=0, s2=0,
             scale=0.1, cap=0.0, window=0, causal=1, ws=None, wsb=0, stream=None)
    a.update(kw)
    return lib.gollek_paged_attention_varlen(*a.values())


def shared(lib, **kw):
    a = dict(out=D, q=D, k=D, v=D, ks=None, vs=None, pt=D, pl=D, gs=D, bt=D, ctx=D, groups=1, maxp=4, S=2, hq=8, hkv=2,
             d=128, bs=16, maxb=4, nb=0, stride=0, qd=_lib.BF16, kd=_lib.BF16, s0=0, s1=0, s2=0, scale=0.1, cap=0.0,
             ws=None, wsb=0, stream=None)
    a.update(kw)
    return lib.gollek_paged_attention_shared_prefix(*a.values())


def gather(lib, **kw):
    a = dict(key=D, value=D, out=_lib.F32, seq=None, pos=D, bt=D, S=2, maxb=4, nb=0, k=D, v=D, ks=None, vs=None,
             kd=_lib.BF16, T=3, hkv=2, d=128, bs=16, stride=0, s0=0, s1=0, s2=0, stream=None)
    a.update(kw)
    return lib.gollek_kv_gather(*a.values())


INVALID, UNSUPPORTED = _lib.ERR_INVALID_ARGUMENT, _lib.ERR_UNSUPPORTED


@pytest.mark.parametrize("call", [varlen, shared])
@pytest.mark.parametrize("kw,code", [
    ({"q": None}, INVALID), ({"out": None}, INVALID), ({"k": None}, INVALID), ({"bt": None}, INVALID),
    ({"ctx": None}, INVALID), ({"hq": 6, "hkv": 4}, INVALID), ({"hq": 0}, INVALID), ({"hkv": 0}, INVALID),
    ({"d": 0}, INVALID), ({"bs": 0}, INVALID), ({"maxb": 0}, INVALID), ({"S": -1}, INVALID), ({"nb": -1}, INVALID),
    ({"stride": 100}, INVALID), ({"stride": -4096}, INVALID), ({"kd": _lib.I8}, INVALID),
    ({"maxb": 1 << 28, "bs": 64}, INVALID), ({"d": 257}, UNSUPPORTED), ({"qd": _lib.I8}, UNSUPPORTED),
    ({"kd": 9}, UNSUPPORTED), ({"kd": _lib.I4, "ks": D, "vs": D, "d": 63}, UNSUPPORTED)])
def test_attention_refusals(lib, call, kw, code):
    assert call(lib, **kw) == code
    assert lib.gollek_last_error_string() != b""


def test_varlen_refusals(lib):
    assert varlen(lib, cu=None) == INVALID
    assert varlen(lib, total=-1) == INVALID
    assert varlen(lib, window=5, causal=0) == UNSUPPORTED
    assert b"causal" in lib.gollek_last_error_string()
    assert varlen(lib, S=0) == 0 and varlen(lib, total=0) == 0  # nothing to do


def test_shared_refusals(lib):
    for name in ("pt", "pl", "gs"):
        assert shared(lib, **{name: None}) == INVALID
    assert shared(lib, groups=0) == INVALID and shared(lib, maxp=0) == INVALID
    assert shared(lib, maxp=1 << 28, bs=64, maxb=1) == INVALID
    assert shared(lib, S=0) == 0


@pytest.mark.parametrize("kw,code", [
    ({"key": None}, INVALID), ({"value": None}, INVALID), ({"pos": None}, INVALID), ({"bt": None}, INVALID),
    ({"k": None}, INVALID), ({"T": -1}, INVALID), ({"S": -1}, INVALID), ({"hkv": 0}, INVALID), ({"d": 0}, INVALID),
    ({"bs": 0}, INVALID), ({"maxb": 0}, INVALID), ({"nb": -2}, INVALID), ({"stride": 5}, INVALID),
    ({"kd": _lib.I8}, INVALID), ({"out": _lib.I8}, UNSUPPORTED), ({"kd": 7}, UNSUPPORTED),
    ({"kd": _lib.I4, "ks": D, "vs": D, "d": 63}, UNSUPPORTED)])
def test_gather_refusals(lib, kw, code):
    assert gather(lib, **kw) == code
    assert lib.gollek_last_error_string() != b""


def test_gather_of_nothing(lib):
    assert gather(lib, T=0) == 0


def test_python_refusals():
    torch = pytest.importorskip("torch")
    from gollek_b200 import ops
    q = torch.zeros((4, 8, 128))
    with pytest.raises(ValueError, match="CUDA"):
        ops.paged_attention_varlen(q, q, q, q, q, q, num_kv_heads=2, block_size=16)
    with pytest.raises(ValueError, match="CUDA"):
        ops.paged_attention_shared_prefix(q, q, q, q, q, q, q, q, num_kv_heads=2, block_size=16)
    with pytest.raises(ValueError, match="CUDA"):
        ops.kv_gather(q, q, torch.zeros(3, dtype=torch.int32), q, num_kv_heads=2, head_dim=128, block_size=16)


def test_gather_cache_refuses_missing_blocks():
    from gollek_b200 import engine
    from gollek_b200.kv_cache import IllegalStateError
    bm = engine.BlockManager(device="cpu")
    s = engine.KVCacheSession(64, bm)
    s.allocate(1, 2, 8)
    with pytest.raises(IllegalStateError):
        engine.gather_cache(s, 0, 0, 17)
    with pytest.raises(ValueError):
        engine.gather_cache(s, 0, -1, 4)


def test_reference_known_answers():
    """The tests' definition on cases small enough to do by hand."""
    pool = R.Pool("f32", np.zeros((2, 1, 2, 2)), np.arange(8.0).reshape(2, 1, 2, 2))
    tables = np.array([[1, 0]])
    q = np.ones((2, 1, 2))
    # scores 0: means of the visible rows; positions are page 1's rows [4,5],[6,7], then page 0's [0,1],[2,3]
    out = R.varlen(q, pool, tables, [0, 2], [3], 1.0)
    assert np.allclose(out[0, 0], [5, 6]) and np.allclose(out[1, 0], [10 / 3, 13 / 3])
    out = R.varlen(q, pool, tables, [0, 2], [3], 1.0, window=1)
    assert np.allclose(out[:, 0], [[6, 7], [0, 1]])
    out = R.varlen(q, pool, tables, [0, 2], [3], 1.0, starts=np.array([2, 2]))
    assert np.allclose(out[:, 0], [[0, 0], [0, 1]])
    out = R.varlen(q, pool, tables, [0, 2], [3], 1.0, prefix=[3])
    assert np.allclose(out[0], out[1])
    # bias ln 2 per step of distance: weights 1/4, 1/2, 1
    out = R.varlen(q[:1], pool, tables, [0, 1], [3], 1.0, slopes=np.array([np.log(2.0)]))
    assert np.allclose(out[0, 0], (np.array([4, 5]) / 4 + np.array([6, 7]) / 2 + np.array([0, 1])) / 1.75)
    out = R.shared_prefix(q[:1], pool, np.array([[1]]), [2], [0, 1], np.array([[0]]), [1], 1.0)
    assert np.allclose(out[0, 0], [10 / 3, 13 / 3])


@pytest.mark.parametrize("hq,hkv,d", [(32, 8, 128), (8, 8, 64), (64, 2, 128), (20, 4, 96)])
def test_a_workspace_for_more_is_enough_for_less(hq, hkv, d):
    """Callers keep the workspace of their largest batch, whichever kernels smaller ones go to."""
    from gollek_b200 import ops
    seqs, tokens = [1, 2, 31, 32, 33, 64, 300], [1, 2, 64, 65, 500, 1024, 5000, 40000]
    size = {(s, t): ops.varlen_workspace_size(s, t, hq, hkv, d) for s in seqs for t in tokens}
    for (s, t), n in size.items():
        assert n > 0
        assert all(n <= size[s2, t2] for s2 in seqs for t2 in tokens if s2 >= s and t2 >= t)
    size = {(g, s): ops.shared_prefix_workspace_size(g, s, hq, hkv, d) for g in (1, 2, 40) for s in seqs}
    for (g, s), n in size.items():
        assert n > 0
        assert all(n <= size[g2, s2] for g2 in (1, 2, 40) for s2 in seqs if g2 >= g and s2 >= s)
