"""Rounding of ragged attention's tensor-core kernels: what small probabilities lose, and what a result's bits
depend on."""
import numpy as np
import pytest

from tests import paged_ref as R
from tests.test_gpu_varlen import check_varlen, run_varlen, spoil, up, varlen_case

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


# ------------------------------------------------------------------------ same bits

def unseen_filled(k, v, tables, ctx, bs, value):
    """K and V with `value` wherever spoil() says that no query looks."""
    k, v = k.copy(), v.copy()
    spoil(k, v, tables, ctx, bs)
    return np.nan_to_num(k, nan=value), np.nan_to_num(v, nan=value)


@pytest.mark.parametrize("kind,qkind", [("bf16", "bf16"), ("f16", "f16"), ("i8", "bf16")])
@pytest.mark.parametrize("ctx,new", [([300, 45, 129, 1000, 8] * 8, [1] * 40), ([300, 45, 203, 1000], [90, 30, 203, 7])])
def test_capped_bits_do_not_depend_on_what_nobody_attends(cuda_device, kind, qkind, ctx, new):
    """With a soft-cap, whatever slots behind a sequence hold, and whatever calls ran before."""
    d, bs, hq, hkv, cap = 128, 16, 8, 2, 30.0
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
