"""Every position that a query sees counts once, and no other: ragged and shared-prefix attention over pools whose
outputs count positions, and the norms of the error over long contexts (tests/paged_rows.py)."""
import numpy as np
import pytest

from tests import paged_ref as R
from tests import paged_rows as P
from tests.helpers import make_tables
from tests.test_gpu_varlen import SLOPES, run_shared, run_varlen, shared_case, varlen_case

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

KINDS = [("bf16", "bf16"), ("f16", "f16"), ("i8", "bf16"), ("f32", "f32"), ("i4", "bf16"), ("bf16", "f32")]


def counting_case(ctx, new, hq, hkv, d, bs, kind, seed):
    rng = np.random.default_rng(seed)
    ctx = np.asarray(ctx, np.int32)
    nb = sum((int(c) + bs - 1) // bs for c in ctx) + 3
    tables = make_tables(ctx, bs, nb, rng)
    cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    return np.zeros((int(cu[-1]), hq, d)), P.counting_pool(kind, tables, ctx, hkv, d, bs, nb, rng, dead=0.0), tables, cu, ctx


def check_counts(dev, case, qkind, **kw):
    from gollek_b200 import ops
    got = run_varlen(dev, *case, qkind, **kw).double().cpu().numpy()
    want = R.varlen(*case, 1 / np.sqrt(case[0].shape[2]), **kw)
    assert ops.device_status(dev.index or 0) == 0
    assert P.counts_agree(got, want, qkind)


def masks(what, ctx, new, hq, rng):
    if what == "bias":
        return {"slopes": np.zeros(hq, np.float32)}  # the kernels with a bias, and weights that stay equal
    if what == "cap":
        return {"cap": 5.0}
    if what == "window":
        return {"window": 129, "cap": 5.0}
    if what == "prefix":
        return {"prefix": rng.integers(0, np.asarray(ctx) + 50).astype(np.int32)}
    if what == "docs":
        return {"starts": np.concatenate([np.maximum(0, c - n + np.arange(n) - rng.integers(-2, max(3, c), n))
                                          for c, n in zip(ctx, new)]).astype(np.int32), "slopes": np.zeros(hq, np.float32)}
    return {"causal": False} if what == "full" else {}


@pytest.mark.parametrize("kind,qkind", KINDS)
@pytest.mark.parametrize("what", ["plain", "bias", "cap", "window", "prefix", "docs", "full"])
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (6, 2, 64)])
def test_counts_of_chunks_beside_decode_steps(cuda_device, kind, qkind, what, hq, hkv, d):
    ctx, new = [900, 37, 128, 5, 1500, 257, 640, 16], [200, 1, 128, 1, 130, 3, 1, 16]
    kw = masks(what, ctx, new, hq, np.random.default_rng(100))
    check_counts(cuda_device, counting_case(ctx, new, hq, hkv, d, 16, kind, 101), qkind, **kw)


@pytest.mark.parametrize("kind,qkind", KINDS)
@pytest.mark.parametrize("ctx,new", [([6000], [1]), ([8000, 1, 3000, 17], [1] * 4), ([4500, 900], [300, 900])])
@pytest.mark.parametrize("d,bs", [(128, 16), (128, 8), (64, 32)])
def test_counts_of_units_cut_over_the_gpu(cuda_device, kind, qkind, ctx, new, d, bs):
    check_counts(cuda_device, counting_case(ctx, new, 4, 2, d, bs, kind, 102), qkind)


@pytest.mark.parametrize("kind", ["bf16", "i8"])
@pytest.mark.parametrize("hq,hkv,bs,d", [(4, 4, 16, 128), (32, 8, 8, 128), (16, 2, 48, 128), (8, 8, 16, 64)])
def test_counts_of_many_sequences_in_turn(cuda_device, kind, hq, hkv, bs, d):
    rng = np.random.default_rng(103)
    n = 70
    ctx = np.where(rng.random(n) < 0.5, rng.integers(1, 140, n), rng.integers(128, 2500, n))
    new = np.where(rng.random(n) < 0.7, 1, np.minimum(ctx, rng.integers(1, 60, n)))
    check_counts(cuda_device, counting_case(ctx, np.ones(n, int), hq, hkv, d, bs, kind, 104), "bf16")
    check_counts(cuda_device, counting_case(ctx, new, hq, hkv, d, bs, kind, 105), "bf16", window=700)


@pytest.mark.parametrize("kind,qkind", KINDS)
@pytest.mark.parametrize("seqs,plens,starts,hq,hkv,d", [
    (70, [2100], [0, 70], 8, 2, 128), (43, [130, 50, 0, 1700], [2, 9, 9, 14, 40], 8, 2, 128), (9, [5000], [0, 9], 6, 2, 64),
    (64, [900, 16], [0, 30, 64], 16, 4, 128), (130, [900, 16, 0], [3, 60, 100, 128], 16, 4, 128)])
def test_counts_behind_shared_prefixes(cuda_device, kind, qkind, seqs, plens, starts, hq, hkv, d):
    rng = np.random.default_rng(106)
    ctx = np.where(rng.random(seqs) < 0.2, 0, rng.integers(1, 500, seqs)).astype(np.int32)
    both = np.concatenate([plens, ctx]).astype(np.int32)
    nb = sum((int(c) + 15) // 16 for c in both) + 2
    tables = make_tables(both, 16, nb, rng)
    pool = P.counting_pool(kind, tables, both, hkv, d, 16, nb, rng, dead=0.0)
    g = len(plens)
    case = (np.zeros((seqs, hq, d)), pool, tables[:g], np.asarray(plens, np.int32), np.asarray(starts, np.int32),
            tables[g:], ctx)
    got = run_shared(cuda_device, case, qkind).double().cpu().numpy()
    want = R.shared_prefix(*case, 1 / np.sqrt(d))
    assert P.counts_agree(got, want, qkind)


# ------------------------------------------------------------------------ norms

def check_norms(dev, case, qkind, **kw):
    q, pool, tables, cu, ctx = case
    scale = 1 / np.sqrt(q.shape[2])
    got = run_varlen(dev, *case, qkind, **kw).double().cpu().numpy()
    want = R.varlen(*case, scale, **kw)
    most = float(np.max(np.abs(kw["slopes"]))) * float(np.max(ctx)) if kw.get("slopes") is not None else 0.0
    assert np.isfinite(got).all()
    assert P.norms_agree(got, want, q, pool, scale, qkind, p_kind=None if qkind == "f32" else qkind, most_bias=most,
                         cap=kw.get("cap", 0.0))


@pytest.mark.parametrize("ctx,new", [([6000], [1]), ([5000, 3000, 17], [1, 1, 1]), ([2500, 900], [700, 900]), ([4096], [512])])
@pytest.mark.parametrize("kind,qkind", [("bf16", "bf16"), ("f16", "f16"), ("i8", "bf16"), ("f32", "f32")])
@pytest.mark.parametrize("what", ["plain", "bias", "cap", "window"])
def test_norms_over_long_contexts(cuda_device, ctx, new, kind, qkind, what):
    kw = {"bias": {"slopes": SLOPES(8) / 64}, "cap": {"cap": 20.0}, "window": {"window": 2000}}.get(what, {})
    check_norms(cuda_device, varlen_case(ctx, new, 8, 2, 128, 16, kind, qkind, 110, window=kw.get("window", 0)), qkind, **kw)


@pytest.mark.parametrize("kind,qkind", [("bf16", "bf16"), ("f16", "f16"), ("i8", "bf16"), ("f32", "f32")])
@pytest.mark.parametrize("seqs,plen,hq,hkv,d", [(1, 5000, 8, 2, 128), (70, 2100, 8, 2, 128), (33, 640, 8, 2, 64),
                                                 (50, 1500, 16, 8, 128), (130, 700, 32, 4, 128)])
def test_norms_behind_a_shared_prefix(cuda_device, kind, qkind, seqs, plen, hq, hkv, d):
    rng = np.random.default_rng(111)
    case = shared_case([plen], [0, seqs], rng.integers(0, 300, seqs), hq, hkv, d, 16, kind, qkind, 112)
    q, pool = case[:2]
    got = run_shared(cuda_device, case, qkind).double().cpu().numpy()
    want = R.shared_prefix(*case, 1 / np.sqrt(d))
    assert P.norms_agree(got, want, q, pool, 1 / np.sqrt(d), qkind, p_kind=None if qkind == "f32" else qkind)
