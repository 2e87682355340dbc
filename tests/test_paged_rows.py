"""The sharper checks of paged attention's tests see what they are for (definitions only, no GPU)."""
import numpy as np
import pytest

from tests import paged_ref as R
from tests import paged_rows as P
from tests.helpers import make_tables


def case(kind, ctx, counting, d=128, bs=16, hq=4, hkv=2, seed=0):
    rng = np.random.default_rng(seed)
    nb = (ctx + bs - 1) // bs + 2
    tables = make_tables([ctx], bs, nb, rng)
    if counting:
        return np.zeros((1, hq, d)), P.counting_pool(kind, tables, [ctx], hkv, d, bs, nb, rng), tables
    k, v = rng.standard_normal((2, nb, hkv, bs, d))
    return rng.standard_normal((1, hq, d)), R.Pool(kind, k, v), tables


def without(pool, tables, ctx, gone, q, twice=False):
    """The definition with some positions left out (or taken twice)."""
    pos = np.setdiff1d(np.arange(ctx), gone) if not twice else np.concatenate([np.arange(ctx), gone])
    k, v = (pool.rows(w, tables[0], ctx)[pos] for w in "kv")
    return R.attend(q, k, v, np.ones((1, len(pos)), bool), q.shape[2] ** -0.5)


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16", "i8", "i4"])
@pytest.mark.parametrize("ctx", [1, 40, 6000, 16000])
def test_counting_pools_see_one_position(kind, ctx):
    q, pool, tables = case(kind, ctx, True)
    want = R.varlen(q, pool, tables, [0, 1], [ctx], 128 ** -0.5)
    assert np.isfinite(want).all() and np.allclose(want.sum(-1), P.ONE.get(kind, 1.0))
    for qkind in ("bf16", "f16", "f32"):
        assert P.counts_agree(want, want, qkind)
        for gone in {0, ctx // 2, ctx - 1}:
            if ctx > 1:
                assert not P.counts_agree(without(pool, tables, ctx, [gone], q), want, qkind)
                assert not P.counts_agree(without(pool, tables, ctx, [gone], q, twice=True), want, qkind)


@pytest.mark.parametrize("kind,qkind", [("bf16", "bf16"), ("f16", "f16"), ("i8", "bf16"), ("f32", "f32")])
@pytest.mark.parametrize("ctx", [700, 2400, 6000])
def test_norms_see_one_page(kind, qkind, ctx):
    q, pool, tables = case(kind, ctx, False, seed=ctx)
    scale = 128 ** -0.5
    want = R.varlen(q, pool, tables, [0, 1], [ctx], scale)
    kw = dict(p_kind=None if qkind == "f32" else qkind)
    assert P.norms_agree(want, want, q, pool, scale, qkind, **kw)
    for first in (0, ctx // 2 // 16 * 16, (ctx - 1) // 16 * 16):
        gone = np.arange(first, min(first + 16, ctx))
        for twice in (False, True):
            assert not P.norms_agree(without(pool, tables, ctx, gone, q, twice), want, q, pool, scale, qkind, **kw)
