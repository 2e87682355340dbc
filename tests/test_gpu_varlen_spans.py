"""Rows and whole blocks of ragged attention that see nothing, and limits at the ends of their type, in every kernel."""
import numpy as np
import pytest

from tests.test_gpu_varlen import SLOPES, check_varlen, varlen_case

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

# outside the tensor-core kernels (blocked where a sequence has rows enough) and inside them
OTHERS = [("f32", "f32", 8, 2, 128, 16), ("i4", "bf16", 8, 2, 64, 16), ("bf16", "f32", 5, 1, 96, 16), ("f16", "f16", 6, 6, 10, 7)]
TILES = [("bf16", "bf16", 8, 2, 128, 16), ("f16", "f16", 8, 2, 64, 32), ("i8", "bf16", 8, 2, 128, 16)]


@pytest.mark.parametrize("kind,qkind,hq,hkv,d,bs", OTHERS + TILES)
def test_blocks_that_see_nothing(cuda_device, kind, qkind, hq, hkv, d, bs):
    """No context yet, more queries than context by several blocks, and every row starting behind its end."""
    case = varlen_case([0, 40, 0, 300, 90], [200, 240, 64, 1, 90], hq, hkv, d, bs, kind, qkind, 120)
    got = check_varlen(cuda_device, case, qkind, slopes=SLOPES(hq))
    assert (got[:400] == 0).all() and (got[400:440] != 0).any() and (got[440:504] == 0).all()
    case = varlen_case([300, 90], [150, 90], hq, hkv, d, bs, kind, qkind, 121)
    starts = np.concatenate([np.full(150, 301), np.arange(90) + 1]).astype(np.int32)
    assert (check_varlen(cuda_device, case, qkind, starts=starts) == 0).all()
    # one row in a block of nothing
    starts[100] = 10
    got = check_varlen(cuda_device, case, qkind, starts=starts)
    assert (got[100] != 0).any() and (np.delete(got, 100, axis=0) == 0).all()


INT_MAX, INT_MIN = 2 ** 31 - 1, -2 ** 31


@pytest.mark.parametrize("kind,qkind,hq,hkv,d,bs", OTHERS + TILES)
@pytest.mark.parametrize("ctx,new", [([300, 45, 7, 0, 129] * 8, [1] * 40), ([300, 90, 40], [150, 1, 40])])
def test_starts_and_prefixes_at_the_ends_of_their_type(cuda_device, kind, qkind, hq, hkv, d, bs, ctx, new):
    """First positions up to the largest integer (rows that see nothing) and down to the smallest, windows and prefixes
    likewise, in decode steps and in prompts."""
    case = varlen_case(ctx, new, hq, hkv, d, bs, kind, qkind, 122)
    n = sum(new)
    starts = np.resize(np.array([0, INT_MAX, 3, INT_MAX - 1, INT_MIN, INT_MAX - 7, INT_MAX - 27, INT_MAX - 200, -1], np.int64), n)
    got = check_varlen(cuda_device, case, qkind, starts=starts.astype(np.int32), slopes=SLOPES(hq))
    assert (got[starts > 2 ** 20] == 0).all()
    check_varlen(cuda_device, case, qkind, starts=starts.astype(np.int32), causal=False)
    prefix = np.resize(np.array([INT_MAX, INT_MIN, -1, 20], np.int64), len(ctx)).astype(np.int32)
    check_varlen(cuda_device, case, qkind, prefix=prefix, window=INT_MAX)
    assert (check_varlen(cuda_device, case, qkind, starts=np.full(n, INT_MAX, np.int32)) == 0).all()
