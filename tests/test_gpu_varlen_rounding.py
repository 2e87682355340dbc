"""Rounding of ragged attention's tensor-core kernels: what small probabilities lose, and what a result's bits
depend on."""
import numpy as np
import pytest

from tests import paged_ref as R
from tests.test_gpu_varlen import check_varlen, run_varlen, spoil, up, varlen_case

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


# ------------------------------------------------------------------------ small probabilities

@pytest.mark.parametrize("d,new", [(128, 1), (64, 1), (64, 200), (128, 40)])
@pytest.mark.parametrize("sink", [3990, 3700, 3685, 2000, 3])
@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_a_long_tail_behind_one_large_score(cuda_device, kind, d, new, sink):
    """One position takes all but 2^-13.5 of the weight, and its value is 0: the output is the tail's, 4,000 positions
    of weight 2^-25.5 each.

    Tolerance: every tail probability is rounded to the cache's type, by half a step of the value (h) where the type has
    its full precision there, else (f16) by half of 2^-24 in a scale where the largest probability is 2^7 or more: 2^-32
    of it, twice if the column is scaled after it was stored.  The scores' own error: 18 products' sizes at 2^-24, 25.5
    binary orders at 2^-23, exp2 2^-21: below 2^-16.  Then half a step of the output."""
    hkv, grp, n, seqs, bs = 8, 2, 4000, 8, 16
    rng = np.random.default_rng(91)
    pages = n // bs
    table = rng.permutation(pages + 2)[:pages].astype(np.int32)
    k = np.zeros((pages + 2, hkv, bs, d))
    v = np.full((pages + 2, hkv, bs, d), 1000.0)
    at = table[sink // bs], slice(None), sink % bs
    k[at + (0,)] = 25.5 * np.log(2) * np.sqrt(d)
    v[at] = 0.0
    pool = R.Pool(kind, k, v)
    q = np.zeros((seqs * new, hkv * grp, d))
    q[..., 0] = 1.0
    tables = np.repeat(table[None], seqs, axis=0)
    cu = (np.arange(seqs + 1) * new).astype(np.int32)
    ctx = np.full(seqs, n, np.int32)
    got = run_varlen(cuda_device, q, pool, tables, cu, ctx, kind, causal=False).double().cpu().numpy()
    want = R.varlen(q[:1], pool, tables[:1], np.array([0, 1]), ctx[:1], 1 / np.sqrt(d), causal=False)[0, 0]
    assert want[0] > 0.05
    tol = (2 * R.HALF_STEP[kind] + 2.0 ** -15) * want + (2 * n * 2.0 ** -32 * 1000 if kind == "f16" else 0)
    assert (np.abs(got - want) <= tol).all(), f"{got.min()} .. {got.max()}, not {want[0]}"


# ------------------------------------------------------------------------ same bits

def unseen_filled(k, v, tables, ctx, bs, value):
    """K and V with `value` wherever spoil() says that no query looks."""
    k, v = k.copy(), v.copy()
    spoil(k, v, tables, ctx, bs)
    return np.nan_to_num(k, nan=value), np.nan_to_num(v, nan=value)


@pytest.mark.parametrize("kind,qkind", [("bf16", "bf16"), ("f16", "f16"), ("i8", "bf16")])
@pytest.mark.parametrize("ctx,new", [([300, 45, 129, 1000, 8] * 8, [1] * 40), ([300, 45, 203, 1000], [90, 30, 203, 7])])
@pytest.mark.parametrize("cap", [30.0, 0.0])
def test_bits_do_not_depend_on_what_nobody_attends(cuda_device, kind, qkind, ctx, new, cap):
    """Whatever slots behind a sequence hold, and whatever calls ran before."""
    d, bs, hq, hkv = 128, 16, 8, 2
    ctx = np.array(ctx, np.int32)
    rng = np.random.default_rng(92)
    q, pool, tables, cu, ctx = varlen_case(ctx, new, hq, hkv, d, bs, "f32", qkind, 93, plant=False)
    k, v = pool.k.double().numpy(), pool.v.double().numpy()
    outs = []
    for value in (0.25, 3000.0):
        a = R.Pool(kind, *unseen_filled(k, v, tables, ctx, bs, value))
        outs.append(run_varlen(cuda_device, q, a, tables, cu, ctx, qkind, cap=cap))
        # scores of some hundreds behind it: what they leave in shared memory is there for the next call
        loud = R.Pool(kind, k * 40, v)
        run_varlen(cuda_device, q * 4, loud, tables, cu, ctx, qkind, cap=cap)
        outs.append(run_varlen(cuda_device, q, a, tables, cu, ctx, qkind, cap=cap))
    assert all(torch.equal(outs[0], o) for o in outs[1:])


@pytest.mark.parametrize("kind,qkind", [("bf16", "bf16"), ("i8", "bf16")])
@pytest.mark.parametrize("ctx,new", [([300, 45, 129] * 14, [1] * 42), ([300, 45, 203], [90, 30, 203])])
def test_capped_bits_of_a_head_are_its_own(cuda_device, kind, qkind, ctx, new):
    """A head's rows come out the same whatever the scores of the other heads of its group are."""
    case = varlen_case(ctx, new, 8, 2, 128, 16, kind, qkind, 94)
    a = run_varlen(cuda_device, *case, qkind, cap=30.0)
    q = case[0].copy()
    q[:, 3] *= 64
    b = run_varlen(cuda_device, q, *case[1:], qkind, cap=30.0)
    others = [0, 1, 2, 4, 5, 6, 7]
    assert torch.equal(a[:, others], b[:, others]) and not torch.equal(a[:, 3], b[:, 3])


@pytest.mark.parametrize("kind,qkind", [("bf16", "bf16"), ("f16", "f16"), ("i8", "bf16")])
@pytest.mark.parametrize("cap", [0.3, 1.0, 30.0])
def test_capped_scores_on_both_sides_of_a_half(cuda_device, kind, qkind, cap):
    """Scores far below, around and far above half the cap, beside one another in one tile."""
    for ctx, new in (([300, 45, 129] * 14, [1] * 42), ([300, 45, 203], [90, 30, 203])):
        q, pool, tables, cu, ctx = varlen_case(ctx, new, 8, 2, 128, 16, kind, qkind, 95)
        q = torch.from_numpy(q * np.array([0.01, 0.3, 1, 1, 3, 8, 0.5, 20])[None, :, None])
        q = q.to({"bf16": torch.bfloat16, "f16": torch.float16}[qkind]).double().numpy()
        check_varlen(cuda_device, (q, pool, tables, cu, ctx), qkind, cap=cap)
