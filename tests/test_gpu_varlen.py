"""Ragged attention, shared-prefix attention and the cache read-back on the device, against
their definitions in 64 bits (tests/paged_ref.py says how far outputs may be off)."""
import math

import numpy as np
import pytest

from tests import paged_ref as R
from tests.helpers import make_tables

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def rounded(x, kind):
    return torch.from_numpy(x).to(DT[kind]).double().numpy()


def spoil(k, v, tables, lens, bs, seen_from=None):
    """NaN wherever no query looks: pages of nobody, slots behind a sequence's last token and
    before the first position any of its queries sees."""
    dead = np.ones((k.shape[0], bs), bool)
    for s, c in enumerate(lens):
        pos = np.arange(0 if seen_from is None else seen_from[s], int(c))
        dead[np.asarray(tables[s])[pos // bs], pos % bs] = False
    k.transpose(0, 2, 1, 3)[dead] = np.nan
    v.transpose(0, 2, 1, 3)[dead] = np.nan


def varlen_case(ctx, new, hq, hkv, d, bs, kind, qkind, seed, scales="token", plant=True, window=0, starts=None,
                std=1.0, gap=0):
    rng = np.random.default_rng(seed)
    ctx = np.asarray(ctx, np.int32)
    nb = sum((int(c) + bs - 1) // bs for c in ctx) + 3
    tables = make_tables(ctx, bs, nb, rng)
    k = rng.standard_normal((nb, hkv, bs, d)) * std
    v = rng.standard_normal((nb, hkv, bs, d)) * std
    cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32) + gap
    if plant and kind not in ("i8", "i4"):
        first = [max(0, int(c) - n - window + 1) if window else 0 for c, n in zip(ctx, new)]
        spoil(k, v, tables, ctx, bs, first)
    pool = R.Pool(kind, k, v, scales)
    q = rounded(rng.standard_normal((int(cu[-1]) + gap, hq, d)), qkind)
    return q, pool, tables, cu, ctx


def up(x, dev, dt=None):
    t = torch.from_numpy(np.ascontiguousarray(x)).to(dev)
    return t if dt is None else t.to(dt)


def run_varlen(dev, q, pool, tables, cu, ctx, qkind, out=None, **kw):
    from gollek_b200 import ops
    conv = {"slopes": ("alibi_slopes", torch.float32), "prefix": ("prefix_lens", torch.int32),
            "starts": ("token_starts", torch.int32)}
    more = {conv[n][0]: up(kw[n], dev, conv[n][1]) for n in conv if kw.get(n) is not None}
    return ops.paged_attention_varlen(up(q, dev, DT[qkind]), block_tables=up(tables, dev),
                                      cu_seqlens_q=up(cu, dev), context_lens=up(ctx, dev),
                                      causal=kw.get("causal", True), soft_cap=kw.get("cap", 0.0),
                                      sliding_window=kw.get("window", 0), out=out, **more, **pool.args(dev))


def check_varlen(dev, case, qkind, **kw):
    from gollek_b200 import ops
    q, pool, tables, cu, ctx = case
    scale = 1 / math.sqrt(q.shape[2])
    out = torch.full(q.shape, 7.0, dtype=DT[qkind], device=dev)
    got = run_varlen(dev, q, pool, tables, cu, ctx, qkind, out=out, **kw).double().cpu().numpy()
    want = R.varlen(q, pool, tables, cu, ctx, scale, **kw)
    assert ops.device_status(dev.index or 0) == 0
    outside = np.isnan(want).any(axis=(1, 2))
    assert (got[outside] == 7.0).all(), "rows in no sequence were written"
    most = float(np.max(np.abs(kw["slopes"]))) * float(ctx.max()) if kw.get("slopes") is not None else 0.0
    tol = R.bound(want[~outside], q, pool, scale, qkind, p_kind=None if qkind == "f32" else qkind,
                  most_bias=most, cap=kw.get("cap", 0.0))
    err = np.abs(got[~outside] - want[~outside])
    assert np.isfinite(got[~outside]).all()
    assert (err <= tol).all(), f"{(err - tol).max()} over the bound, worst {err.max()}"
    return got


SLOPES = lambda hq: (2.0 ** (-8.0 * np.arange(1, hq + 1) / hq)).astype(np.float32)


@pytest.mark.parametrize("kind,qkind", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("i8", "bf16"),
                                        ("i4", "bf16"), ("f32", "bf16"), ("bf16", "f32"), ("i8", "f32"),
                                        ("i8", "f16"), ("f16", "bf16")])
@pytest.mark.parametrize("hq,hkv,d,bs", [(8, 2, 128, 16), (6, 2, 64, 32), (5, 1, 96, 16)])
def test_decode_types(cuda_device, kind, qkind, hq, hkv, d, bs):
    case = varlen_case([1, 37, 128, 300, 129], [1] * 5, hq, hkv, d, bs, kind, qkind, 1)
    check_varlen(cuda_device, case, qkind, slopes=SLOPES(hq))


@pytest.mark.parametrize("kind,qkind", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("i8", "bf16"), ("i4", "bf16")])
@pytest.mark.parametrize("hq,hkv,d,bs", [(8, 2, 128, 16), (3, 1, 64, 32), (16, 1, 128, 64)])
def test_ragged_prompts(cuda_device, kind, qkind, hq, hkv, d, bs):
    """Chunks of every length beside decode steps, sequences without queries, empty contexts."""
    case = varlen_case([300, 5, 64, 0, 257, 131, 500], [300, 1, 0, 0, 130, 3, 77], hq, hkv, d, bs, kind, qkind, 2)
    check_varlen(cuda_device, case, qkind)


@pytest.mark.parametrize("kind,qkind", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("i8", "bf16")])
@pytest.mark.parametrize("what", ["bias", "cap", "window", "prefix", "docs", "all", "full", "full_bias"])
def test_masks_and_bias(cuda_device, kind, qkind, what):
    ctx, new = [200, 333, 129, 40, 700], [150, 1, 129, 40, 90]
    rng = np.random.default_rng(5)
    kw = {}
    if what in ("bias", "all", "full_bias"):
        kw["slopes"] = SLOPES(8)
    if what in ("cap", "all"):
        kw["cap"] = 4.0
    if what in ("window", "all"):
        kw["window"] = 37
    if what in ("prefix", "all"):
        kw["prefix"] = np.array([180, 500, 0, 17, 650], np.int32)
    if what in ("docs", "all"):
        # the start of each query's document; some rows start behind themselves (nothing to see)
        kw["starts"] = np.concatenate([np.maximum(0, c - n + np.arange(n) - rng.integers(-2, 60, n))
                                       for c, n in zip(ctx, new)]).astype(np.int32)
    if what.startswith("full"):
        kw["causal"] = False
    case = varlen_case(ctx, new, 8, 2, 128, 16, kind, qkind, 3)
    check_varlen(cuda_device, case, qkind, **kw)


@pytest.mark.parametrize("kind,qkind", [("f32", "f32"), ("i4", "bf16"), ("i8", "f32"), ("bf16", "f32"), ("f16", "bf16")])
@pytest.mark.parametrize("hq,hkv,d,bs", [(5, 1, 96, 16), (6, 6, 10, 7), (4, 2, 256, 8), (20, 4, 128, 24), (64, 1, 34, 16),
                                         (65, 1, 16, 16)])
def test_ragged_prompts_of_odd_shapes(cuda_device, kind, qkind, hq, hkv, d, bs):
    """Prompts outside the tensor-core kernels: blocks of 64 rows that end anywhere in a sequence, 64 heads and more."""
    case = varlen_case([90, 0, 33, 1, 70, 41], [33, 0, 33, 1, 12, 40], hq, hkv, d, bs, kind, qkind, 75, gap=2)
    check_varlen(cuda_device, case, qkind, slopes=SLOPES(hq), window=50, cap=3.0)
    check_varlen(cuda_device, case, qkind, prefix=np.array([80, 0, 5, 1, 70, 9], np.int32))


def test_rows_with_nothing_to_see_are_zero(cuda_device):
    q, pool, tables, cu, ctx = varlen_case([70, 20], [70, 20], 8, 2, 128, 16, "bf16", "bf16", 4)
    starts = np.concatenate([np.arange(70) + 1, np.full(20, 10 ** 9)]).astype(np.int32)
    got = check_varlen(cuda_device, (q, pool, tables, cu, ctx), "bf16", starts=starts)
    assert (got == 0).all()


def test_more_queries_than_context(cuda_device):
    """Queries before position 0 attend nothing; the others are not disturbed."""
    q, pool, tables, cu, ctx = varlen_case([10, 33], [14, 40], 4, 1, 64, 16, "bf16", "bf16", 6)
    got = check_varlen(cuda_device, (q, pool, tables, cu, ctx), "bf16")
    assert (got[:4] == 0).all() and (got[14:21] == 0).all() and (got[4:14] != 0).any()


def test_rows_outside_every_sequence_stay(cuda_device):
    case = varlen_case([90, 40], [64, 1], 8, 2, 128, 16, "bf16", "bf16", 7, gap=5)
    check_varlen(cuda_device, case, "bf16", slopes=SLOPES(8))


@pytest.mark.parametrize("kind,qkind", [("bf16", "bf16"), ("i8", "bf16"), ("f32", "f32")])
def test_large_scores_and_one_hot_rows(cuda_device, kind, qkind):
    """Scores of some hundreds: the running maximum moves often and softmax is one-hot."""
    case = varlen_case([400, 260], [60, 260], 4, 2, 128, 16, kind, qkind, 8, std=8.0)
    check_varlen(cuda_device, case, qkind)


@pytest.mark.parametrize("kind", ["i8", "i4"])
def test_scale_per_page(cuda_device, kind):
    case = varlen_case([200, 75], [100, 1], 8, 2, 128, 16, kind, "bf16", 9, scales="page")
    check_varlen(cuda_device, case, "bf16", slopes=SLOPES(8))


@pytest.mark.parametrize("bs", [1, 7, 8, 24, 128, 256])
def test_page_sizes(cuda_device, bs):
    for kind, qkind in (("bf16", "bf16"), ("i8", "bf16")):
        case = varlen_case([300, 45, 8], [100, 1, 8], 8, 2, 128, bs, kind, qkind, 10)
        check_varlen(cuda_device, case, qkind)


@pytest.mark.parametrize("ctx,new", [([5000, 3000, 17], [1, 1, 1]), ([6000], [1]), ([2500, 900], [700, 900]),
                                     ([4096], [4096 // 8]), ([1500] * 9, [1, 2, 3, 4, 5, 6, 7, 8, 9])])
@pytest.mark.parametrize("kind,qkind", [("bf16", "bf16"), ("i8", "bf16")])
def test_long_contexts_split_over_the_gpu(cuda_device, ctx, new, kind, qkind):
    case = varlen_case(ctx, new, 8, 2, 128, 16, kind, qkind, 11)
    check_varlen(cuda_device, case, qkind, slopes=SLOPES(8) / 64)


@pytest.mark.parametrize("kind,qkind", [("bf16", "bf16"), ("f16", "f16"), ("i8", "bf16")])
@pytest.mark.parametrize("what", ["bias", "cap", "window", "prefix", "docs", "all", "full_bias", "plain"])
def test_few_rows(cuda_device, kind, qkind, what):
    """Batches of a few queries each (at most 16 rows), one sequence with many among them, one with none."""
    ctx = [200, 333, 129, 40, 700, 1, 128, 0, 127, 256, 1025, 64] + [31 * i % 190 + 1 for i in range(28)]
    new = [5, 1, 30, 1, 2, 1, 4, 0, 1, 3, 1, 1] + [1] * 28
    rng = np.random.default_rng(70)
    kw = {}
    if what in ("bias", "all", "full_bias"):
        kw["slopes"] = SLOPES(32)
    if what in ("cap", "all"):
        kw["cap"] = 2.0
    if what in ("window", "all"):
        kw["window"] = 37
    if what in ("prefix", "all"):
        kw["prefix"] = np.arange(40, dtype=np.int32) * 11
    if what in ("docs", "all"):
        kw["starts"] = np.concatenate([np.maximum(0, c - n + np.arange(n) - rng.integers(-2, 60, n))
                                       for c, n in zip(ctx, new)]).astype(np.int32)
    if what == "full_bias":
        kw["causal"] = False
    case = varlen_case(ctx, new, 32, 8, 128, 16, kind, qkind, 71)
    check_varlen(cuda_device, case, qkind, **kw)


@pytest.mark.parametrize("kind,qkind", [("bf16", "bf16"), ("i8", "bf16")])
def test_many_rows_in_blocks_of_few(cuda_device, kind, qkind):
    """No more tokens than sequences, but most of them in one: its rows go in blocks of 16."""
    new = [1, 30, 0, 3, 1] + [0] * 33
    ctx = [400, 1300, 50, 3, 129] + [7] * 33
    case = varlen_case(ctx, new, 10, 2, 128, 16, kind, qkind, 81)
    check_varlen(cuda_device, case, qkind, slopes=SLOPES(10), cap=2.0, prefix=np.array([0, 1290, 0, 0, 0] + [0] * 33, np.int32))
    check_varlen(cuda_device, case, qkind, window=300)


@pytest.mark.parametrize("hq,hkv,bs,scales", [(4, 4, 16, "token"), (32, 8, 8, "token"), (16, 2, 48, "page"),
                                              (16, 1, 64, "token"), (24, 2, 8, "page")])
@pytest.mark.parametrize("kind", ["bf16", "i8"])
def test_few_rows_in_turn(cuda_device, hq, hkv, bs, scales, kind):
    """Runs of one tile and of many behind one another, cut anywhere by the ends of the SMs' shares."""
    rng = np.random.default_rng(72)
    for rep in range(2):
        n = 70
        ctx = np.where(rng.random(n) < 0.5, rng.integers(1, 140, n), rng.integers(128, 2500, n))
        case = varlen_case(ctx, [1] * n, hq, hkv, 128, bs, kind, "bf16", 73 + rep, scales=scales)
        check_varlen(cuda_device, case, "bf16", slopes=SLOPES(hq) / 32 if rep else None)


@pytest.mark.parametrize("hq,hkv", [(10, 2), (12, 4), (7, 1), (45, 9)])
@pytest.mark.parametrize("kind", ["bf16", "i8"])
def test_few_rows_cut_inside_a_token(cuda_device, hq, hkv, kind):
    """Groups that do not divide 16: blocks end between the heads of one query token."""
    new = [1, 2, 3, 5, 9, 1, 1, 2, 1, 1] + [1] * 20
    ctx = [13 * i + n for i, n in enumerate(new)]
    case = varlen_case(ctx, new, hq, hkv, 128, 16, kind, "bf16", 76)
    check_varlen(cuda_device, case, "bf16", slopes=SLOPES(hq), window=200)


@pytest.mark.parametrize("kind,qkind", [("bf16", "bf16"), ("f16", "f16"), ("i8", "bf16")])
@pytest.mark.parametrize("what", ["plain", "bias", "cap", "window", "docs"])
def test_few_rows_beside_many(cuda_device, kind, qkind, what):
    """Decode steps, short drafts and prompt chunks in one call: each goes to the kernel for its rows, and a call
    has parts that both cut over the ends of their shares."""
    rng = np.random.default_rng(79)
    new = np.array([1, 1, 200, 1, 4, 0, 1, 5, 1, 33, 1, 1, 3, 1, 90] + [1] * 25)
    ctx = new + rng.integers(0, 900, len(new))
    kw = {"slopes": SLOPES(32)} if what == "bias" else {"cap": 3.0} if what == "cap" else {"window": 70} if what == "window" else {}
    if what == "docs":
        kw["starts"] = np.concatenate([np.maximum(0, c - n + np.arange(n) - rng.integers(-2, 400, n))
                                       for c, n in zip(ctx, new)]).astype(np.int32)
    case = varlen_case(ctx, new, 32, 8, 128, 16, kind, qkind, 80, window=kw.get("window", 0))
    check_varlen(cuda_device, case, qkind, **kw)


def test_documents_of_more_blocks_than_plan_threads(cuda_device):
    """token_starts over more than 1,024 blocks, the last ones of a few rows."""
    rng = np.random.default_rng(77)
    n = 1100
    new = rng.integers(1, 5, n)
    ctx = new + rng.integers(0, 40, n)
    starts = np.concatenate([rng.integers(0, c, k) for c, k in zip(ctx, new)]).astype(np.int32)
    case = varlen_case(ctx, new, 16, 2, 128, 16, "bf16", "bf16", 78)
    check_varlen(cuda_device, case, "bf16", starts=starts)
    case = varlen_case(ctx, new, 16, 2, 64, 16, "bf16", "bf16", 78)
    check_varlen(cuda_device, case, "bf16", starts=starts)


@pytest.mark.parametrize("kind,qkind", [("bf16", "bf16"), ("f16", "f16"), ("i8", "bf16")])
def test_few_rows_large_scores(cuda_device, kind, qkind):
    """Maxima that keep rising from tile to tile: the references of all warps of a group move together."""
    q, pool, tables, cu, ctx = varlen_case([1500, 700, 2000, 129], [1] * 4, 8, 2, 128, 16, kind, qkind, 74)
    check_varlen(cuda_device, (rounded(q * 12, qkind), pool, tables, cu, ctx), qkind)


@pytest.mark.parametrize("hq,hkv,window,cap", [(32, 8, 1024, 30.0), (8, 8, 0, 0.0), (12, 4, 200, 0.0), (64, 2, 0, 4.0)])
def test_large_and_small_blocks_in_turn(cuda_device, hq, hkv, window, cap):
    """Blocks of more and of fewer than 128 rows, of many tiles and of one, behind one another in every order: what the
    warps of a block hand each other may not be mistaken for the next block's."""
    rng = np.random.default_rng(60)
    for rep in range(3):
        n = 24
        ctx = np.where(rng.random(n) < 0.5, rng.integers(1, 128, n), rng.integers(128, 2000, n))
        new = np.where(rng.random(n) < 0.5, 1, np.minimum(ctx, rng.integers(1, 300, n)))
        case = varlen_case(ctx, new, hq, hkv, 128, 16, "bf16", "bf16", 61 + rep, window=window)
        check_varlen(cuda_device, case, "bf16", window=window, cap=cap)


def test_one_layer_of_a_pool(cuda_device):
    """page_stride: a layer of a [block][layer][...] pool, through a view of it."""
    from gollek_b200 import ops
    q, pool, tables, cu, ctx = varlen_case([150, 60], [30, 1], 8, 2, 128, 16, "bf16", "bf16", 12)
    nb, L = pool.nb, 3
    big = torch.zeros((2, nb, L, 2, 16, 128), dtype=torch.bfloat16, device=cuda_device)
    big[0, :, 1] = pool.k.to(cuda_device)
    big[1, :, 1] = pool.v.to(cuda_device)
    args = pool.args(cuda_device)
    args.update(k_cache=big[0, :, 1], v_cache=big[1, :, 1], page_stride=L * 2 * 16 * 128)
    got = ops.paged_attention_varlen(up(q, cuda_device, torch.bfloat16), block_tables=up(tables, cuda_device),
                                     cu_seqlens_q=up(cu, cuda_device), context_lens=up(ctx, cuda_device), **args)
    want = run_varlen(cuda_device, q, pool, tables, cu, ctx, "bf16")
    assert torch.equal(got, want)


def test_varlen_reports_bad_ids_and_lengths(cuda_device):
    from gollek_b200 import _lib, ops
    q, pool, tables, cu, ctx = varlen_case([150, 60], [30, 1], 8, 2, 128, 16, "bf16", "bf16", 13, plant=False)
    ops.device_status(cuda_device.index or 0)
    bad = tables.copy()
    bad[0, 2] = pool.nb + 5
    run_varlen(cuda_device, q, pool, bad, cu, ctx, "bf16")
    assert ops.device_status(cuda_device.index or 0) == _lib.STATUS_BAD_BLOCK_ID
    run_varlen(cuda_device, q, pool, tables, cu, np.array([150, 10 ** 6], np.int32), "bf16")
    assert ops.device_status(cuda_device.index or 0) & _lib.STATUS_BAD_POSITION
    # a cu_seqlens_q that runs backwards or past the rows: those sequences write nothing
    out = torch.full(q.shape, 7.0, dtype=torch.bfloat16, device=cuda_device)
    run_varlen(cuda_device, q, pool, tables, np.array([0, 30, 10 ** 6], np.int32), ctx, "bf16", out=out)
    assert ops.device_status(cuda_device.index or 0) & _lib.STATUS_BAD_POSITION
    assert (out[30:] == 7.0).all()
    run_varlen(cuda_device, q, pool, tables, np.array([20, 10, 31], np.int32), ctx, "bf16")
    assert ops.device_status(cuda_device.index or 0) & _lib.STATUS_BAD_POSITION
    check_varlen(cuda_device, (q, pool, tables, cu, ctx), "bf16")
    assert ops.device_status(cuda_device.index or 0) == 0


# ------------------------------------------------------------------------ shared prefixes

def shared_case(plens, starts, ctx, hq, hkv, d, bs, kind, qkind, seed, scales="token", std=1.0):
    rng = np.random.default_rng(seed)
    both = np.concatenate([plens, ctx]).astype(np.int32)
    nb = sum((int(c) + bs - 1) // bs for c in both) + 2
    tables = make_tables(both, bs, nb, rng)
    k = rng.standard_normal((nb, hkv, bs, d)) * std
    v = rng.standard_normal((nb, hkv, bs, d)) * std
    if kind not in ("i8", "i4"):
        spoil(k, v, tables, both, bs)
    g = len(plens)
    wide = lambda t, lens: t[:, :max(1, max((int(c) + bs - 1) // bs for c in lens))]
    return (rounded(rng.standard_normal((len(ctx), hq, d)), qkind), R.Pool(kind, k, v, scales),
            wide(tables[:g], plens), np.asarray(plens, np.int32), np.asarray(starts, np.int32),
            wide(tables[g:], ctx), np.asarray(ctx, np.int32))


def run_shared(dev, case, qkind, cap=0.0, **kw):
    from gollek_b200 import ops
    q, pool, pt, plens, starts, t, ctx = case
    return ops.paged_attention_shared_prefix(up(q, dev, DT[qkind]), prefix_tables=up(pt, dev),
                                             prefix_lens=up(plens, dev), group_starts=up(starts, dev),
                                             block_tables=up(t, dev), context_lens=up(ctx, dev), soft_cap=cap,
                                             **kw, **pool.args(dev))


def check_shared(dev, case, qkind, cap=0.0):
    from gollek_b200 import ops
    q, pool, pt, plens, starts, t, ctx = case
    scale = 1 / math.sqrt(q.shape[2])
    got = run_shared(dev, case, qkind, cap).double().cpu().numpy()
    want = R.shared_prefix(q, pool, pt, plens, starts, t, ctx, scale, cap)
    assert ops.device_status(dev.index or 0) == 0
    tol = R.bound(want, q, pool, scale, qkind, p_kind=None if qkind == "f32" else qkind, cap=cap)
    err = np.abs(got - want)
    assert np.isfinite(got).all()
    assert (err <= tol).all(), f"{(err - tol).max()} over the bound, worst {err.max()}"
    return got


@pytest.mark.parametrize("kind,qkind", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("i8", "bf16"),
                                        ("i4", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("hq,hkv,d,bs", [(8, 2, 128, 16), (6, 2, 64, 32), (12, 1, 96, 16)])
def test_shared_prefix(cuda_device, kind, qkind, hq, hkv, d, bs):
    case = shared_case([300], [0, 6], [1, 40, 17, 0, 129, 260], hq, hkv, d, bs, kind, qkind, 20)
    check_shared(cuda_device, case, qkind)


@pytest.mark.parametrize("kind,qkind", [("bf16", "bf16"), ("i8", "bf16"), ("f32", "f32")])
def test_shared_prefix_groups(cuda_device, kind, qkind):
    """Several groups: an empty group, a group without a prefix, sequences outside every group."""
    case = shared_case([130, 50, 0, 700], [2, 9, 9, 14, 40], [(7 * i) % 97 for i in range(43)], 8, 2, 128, 16,
                       kind, qkind, 21)
    got = check_shared(cuda_device, case, qkind, cap=3.0)
    assert (got[0] == 0).all()  # no prefix, no context


@pytest.mark.parametrize("seqs,plen,hq,hkv", [(1, 5000, 8, 2), (70, 2100, 8, 2), (90, 640, 16, 1), (33, 16, 32, 8)])
def test_shared_prefix_many_sequences(cuda_device, seqs, plen, hq, hkv):
    rng = np.random.default_rng(22)
    case = shared_case([plen], [0, seqs], rng.integers(0, 300, seqs), hq, hkv, 128, 16, "bf16", "bf16", 22)
    check_shared(cuda_device, case, "bf16")


@pytest.mark.parametrize("kind,qkind", [("bf16", "bf16"), ("f16", "f16"), ("i8", "bf16")])
@pytest.mark.parametrize("hq,hkv,seqs", [(16, 4, 64), (32, 2, 130), (8, 8, 40), (34, 2, 130)])
def test_shared_prefix_own_tokens_apart(cuda_device, kind, qkind, hq, hkv, seqs):
    """Batches whose own tokens alone fill the device (16 rows at most per sequence and kv head: a kernel of their
    own; 17: the same kernel for all), in groups of every size and outside them."""
    rng = np.random.default_rng(24)
    ctx = np.where(rng.random(seqs) < 0.2, 0, rng.integers(1, 500, seqs))
    case = shared_case([0, 900, 130, 1], [1, 5, seqs // 2, seqs // 2, seqs - 3], ctx, hq, hkv, 128, 16, kind, qkind, 25)
    got = check_shared(cuda_device, case, qkind, cap=0.0 if kind == "f16" else 5.0)
    if ctx[0] == 0:
        assert (got[0] == 0).all()


def test_shared_prefix_equals_the_prefix_in_every_table(cuda_device):
    """One definition, two calls: the shared form, and decode over tables that repeat the prefix."""
    from gollek_b200 import ops
    case = shared_case([256], [0, 5], [30, 1, 64, 99, 200], 8, 2, 128, 16, "bf16", "bf16", 23)
    q, pool, pt, plens, starts, t, ctx = case
    got = run_shared(cuda_device, case, "bf16")
    full = np.concatenate([np.repeat(pt, 5, axis=0), t], axis=1)
    a = pool.args(cuda_device)
    dense = ops.paged_attention(up(q, cuda_device, torch.bfloat16), a["k_cache"], a["v_cache"],
                                up(full, cuda_device), up(ctx + 256, cuda_device), num_kv_heads=2, block_size=16,
                                num_blocks=pool.nb)
    tol = 2 * R.bound(got.double().cpu().numpy(), q, pool, 1 / math.sqrt(128), "bf16", p_kind="bf16")
    assert (np.abs((got.double() - dense.double()).cpu().numpy()) <= tol).all()


def test_shared_prefix_reports_bad_groups(cuda_device):
    from gollek_b200 import _lib, ops
    case = shared_case([64, 64], [0, 3, 6], [20] * 6, 8, 2, 128, 16, "bf16", "bf16", 24)
    ops.device_status(cuda_device.index or 0)
    for starts in ([0, 5, 3], [0, 3, 99], [-4, 3, 6]):
        run_shared(cuda_device, case[:4] + (np.array(starts, np.int32),) + case[5:], "bf16")
        assert ops.device_status(cuda_device.index or 0) & _lib.STATUS_BAD_POSITION
    check_shared(cuda_device, case, "bf16")
    assert ops.device_status(cuda_device.index or 0) == 0


# ------------------------------------------------------------------------ read-back

@pytest.mark.parametrize("kind", ["f32", "bf16", "f16", "i8", "i4"])
@pytest.mark.parametrize("to", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("hkv,d,bs,scales", [(2, 128, 16, "token"), (3, 64, 32, "page"), (1, 10, 7, "token"),
                                             (12, 96, 16, "token")])
def test_gather(cuda_device, kind, to, hkv, d, bs, scales):
    """Bit for bit: one fp32 product and one rounding; any order, the same row twice, bad rows zero."""
    from gollek_b200 import _lib, ops
    rng = np.random.default_rng(30)
    ctx = np.array([5, 1, 70, 33], np.int32)
    nb = sum((int(c) + bs - 1) // bs for c in ctx) + 2
    tables = make_tables(ctx, bs, nb, rng)
    pool = R.Pool(kind, rng.standard_normal((nb, hkv, bs, d)), rng.standard_normal((nb, hkv, bs, d)), scales)
    seq = rng.integers(0, 4, 301).astype(np.int32)
    pos = (rng.integers(0, 10 ** 6, 301) % ctx[seq]).astype(np.int32)
    seq[7], pos[7] = seq[8], pos[8]
    pos[11], pos[12], seq[13], pos[14], seq[15] = -1, 10 ** 6, 4, tables.shape[1] * bs, -1
    bad = [11, 12, 13, 14, 15]
    ops.device_status(cuda_device.index or 0)
    got = ops.kv_gather(token_pos=up(pos, cuda_device), block_tables=up(tables, cuda_device),
                        token_seq=up(seq, cuda_device), head_dim=d, dtype=DT[to], **pool.args(cuda_device))
    assert ops.device_status(cuda_device.index or 0) == _lib.STATUS_BAD_POSITION
    ok = np.setdiff1d(np.arange(301), bad)
    page = tables[seq[ok], pos[ok] // bs]
    for g, full in zip(got, (pool.fk, pool.fv)):
        g = g.cpu()
        # products of an integer below 2^8 and an fp32 scale, rounded to fp32, then to the output type
        want = torch.from_numpy(full[page, :, pos[ok] % bs]).float().to(DT[to])
        assert torch.equal(g[torch.from_numpy(ok)], want)
        assert (g[bad] == 0).all()


def test_gather_reports_bad_pages(cuda_device):
    from gollek_b200 import _lib, ops
    pool = R.Pool("bf16", np.ones((4, 2, 16, 128)), np.ones((4, 2, 16, 128)))
    tables = np.array([[0, 9, -1, 1]], np.int32)
    ops.device_status(cuda_device.index or 0)
    pos = np.array([0, 20, 40, 50], np.int32)
    k, v = ops.kv_gather(token_pos=up(pos, cuda_device), token_seq=up(np.zeros(4, np.int32), cuda_device),
                         block_tables=up(tables, cuda_device), head_dim=128, **pool.args(cuda_device))
    assert ops.device_status(cuda_device.index or 0) == _lib.STATUS_BAD_BLOCK_ID
    assert (k[[0, 3]] == 1).all() and (k[[1, 2]] == 0).all() and (v[[1, 2]] == 0).all()


# ------------------------------------------------------------------------ streams and graphs

def test_on_another_stream(cuda_device):
    case = varlen_case([900, 500, 33], [300, 1, 20], 8, 2, 128, 16, "bf16", "bf16", 40)
    q, pool, tables, cu, ctx = case
    want = run_varlen(cuda_device, q, pool, tables, cu, ctx, "bf16")
    from gollek_b200 import ops
    side = torch.cuda.Stream(cuda_device)
    args = pool.args(cuda_device)
    ins = [up(q, cuda_device, torch.bfloat16), up(tables, cuda_device), up(cu, cuda_device), up(ctx, cuda_device)]
    side.wait_stream(torch.cuda.current_stream(cuda_device))
    got = [ops.paged_attention_varlen(ins[0], block_tables=ins[1], cu_seqlens_q=ins[2], context_lens=ins[3],
                                      stream=s, **args) for s in (side, side.cuda_stream)]
    side.synchronize()
    assert torch.equal(got[0], want) and torch.equal(got[1], want)


def test_two_graphs_replayed_at_once(cuda_device):
    """Two captured calls have scratch of their own: replayed on two streams at once, and again
    with other contents, they give what an eager call gives."""
    from gollek_b200 import ops
    cases = [varlen_case([3000, 700], [40, 1], 8, 2, 128, 16, "bf16", "bf16", 41 + i, plant=False) for i in range(2)]
    want = [run_varlen(cuda_device, *c, "bf16") for c in cases]
    held, graphs, outs = [], [], []
    for q, pool, tables, cu, ctx in cases:
        t = [up(q, cuda_device, torch.bfloat16), up(tables, cuda_device), up(cu, cuda_device), up(ctx, cuda_device)]
        args = pool.args(cuda_device)
        call = lambda: ops.paged_attention_varlen(t[0], block_tables=t[1], cu_seqlens_q=t[2], context_lens=t[3], **args)
        call()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call())
        graphs.append(g)
        held.append((t, args))
    streams = [torch.cuda.Stream(cuda_device) for _ in graphs]
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(outs, want))
    held[0][0][0].mul_(2)
    graphs[0].replay()
    torch.cuda.synchronize()
    q, pool, tables, cu, ctx = cases[0]
    assert torch.equal(outs[0], run_varlen(cuda_device, 2 * q, pool, tables, cu, ctx, "bf16"))


def test_same_call_same_bits(cuda_device):
    case = varlen_case([5000, 1200, 300], [1, 200, 300], 8, 2, 128, 16, "bf16", "bf16", 43)
    a = run_varlen(cuda_device, *case, "bf16")
    assert all(torch.equal(a, run_varlen(cuda_device, *case, "bf16")) for _ in range(3))
    sc = shared_case([3000], [0, 40], [200] * 40, 8, 2, 128, 16, "bf16", "bf16", 44)
    b = run_shared(cuda_device, sc, "bf16")
    assert all(torch.equal(b, run_shared(cuda_device, sc, "bf16")) for _ in range(3))


def test_callers_workspace(cuda_device):
    """A workspace of the documented size with any contents; a smaller one is refused."""
    from gollek_b200 import _lib, ops
    case = varlen_case([3000, 100], [50, 1], 8, 2, 128, 16, "bf16", "bf16", 45)
    q, pool, tables, cu, ctx = case
    want = run_varlen(cuda_device, q, pool, tables, cu, ctx, "bf16")
    n = ops.varlen_workspace_size(2, q.shape[0], 8, 2, 128)
    args = pool.args(cuda_device)
    call = lambda ws: ops.paged_attention_varlen(
        up(q, cuda_device, torch.bfloat16), block_tables=up(tables, cuda_device), cu_seqlens_q=up(cu, cuda_device),
        context_lens=up(ctx, cuda_device), workspace=ws, **args)
    for fill in (0, 255, 77):
        assert torch.equal(call(torch.full((max(n, 1),), fill, dtype=torch.uint8, device=cuda_device)), want)
    if n:
        with pytest.raises(_lib.GollekError) as e:
            call(torch.empty(n - 1, dtype=torch.uint8, device=cuda_device))
        assert e.value.code == _lib.ERR_WORKSPACE


# ------------------------------------------------------------------------ together

@pytest.mark.parametrize("storage", ["BF16", "INT8"])
def test_append_prompt_decode_and_read_back(cuda_device, storage):
    """A serving step as the engine runs it: a prompt and two conversations behind it are appended, the prompt's
    chunk attends ragged, the conversations decode behind the shared prompt, and the rows come back."""
    from gollek_b200 import engine, ops
    dev, hq, hkv, d, P = cuda_device, 8, 2, 128, 200
    rng = np.random.default_rng(50)
    own = [60, 9]
    bm = engine.BlockManager(device=dev)
    sess = engine.KVCacheSession(1024, bm)
    sess.allocate(1, hkv, d, engine.KvStorageType[storage])
    rows = {n: [rng.standard_normal((c, hkv, d)).astype(np.float32) for _ in range(2)] for n, c in enumerate([P] + own)}
    engine.update_cache(up(rows[0][0], dev), up(rows[0][1], dev), sess, 0, 0, P)
    blocks = [[bm.allocate_block() for _ in range((c + 15) // 16)] for c in own]
    width = max(map(len, blocks))
    t = torch.tensor([b + [-1] * (width - len(b)) for b in blocks], dtype=torch.int32, device=dev)
    ctx = torch.tensor(own, dtype=torch.int32, device=dev)
    pool = engine._kv_args(bm)
    seq = torch.repeat_interleave(torch.arange(2, device=dev), ctx.long()).int()
    pos = torch.cat([torch.arange(c, device=dev) for c in own]).int()
    ops.kv_append(up(np.concatenate([rows[1][0], rows[2][0]]), dev), up(np.concatenate([rows[1][1], rows[2][1]]), dev),
                  pos, t, bm.k_slab, bm.v_slab, block_size=16, num_blocks=bm.max_blocks, token_seq=seq, **pool)
    key, value = engine.gather_cache(sess, 0, 0, P)
    k2, v2 = ops.kv_gather(bm.k_slab, bm.v_slab, pos, t, num_kv_heads=hkv, head_dim=d, block_size=16,
                           num_blocks=bm.max_blocks, token_seq=seq, **pool)
    # rows come back as they were stored: half a step of bf16, or of the row's int8 scale
    for got, src in ((key, rows[0][0]), (value, rows[0][1]), (k2[:60], rows[1][0]), (v2[60:], rows[2][1])):
        err = np.abs(got.double().cpu().numpy() - src)
        step = 2.0 ** -8 * np.abs(src) if storage == "BF16" else np.abs(src).max(-1, keepdims=True) / 127 * 0.5001
        assert (err <= step).all()
    # attention over the stored rows, from the read-back values
    f64 = lambda x: x.double().cpu().numpy()
    q = rounded(rng.standard_normal((P + 2, hq, d)), "bf16")
    common = dict(num_kv_heads=hkv, block_size=16, num_blocks=bm.max_blocks, **pool)
    ptab = sess.block_table_tensor(0)
    got = ops.paged_attention_varlen(up(q[:P], dev, torch.bfloat16), bm.k_slab, bm.v_slab, ptab,
                                     torch.tensor([0, P], dtype=torch.int32, device=dev),
                                     torch.tensor([P], dtype=torch.int32, device=dev), **common)
    scale = 1 / math.sqrt(d)
    seen = np.tril(np.ones((P, P), bool))
    want = R.attend(q[:P], f64(key), f64(value), seen, scale)
    class Values:
        fk, fv = f64(key), f64(value)
    tol = R.bound(want, q, Values, scale, "bf16", p_kind="bf16")
    assert (np.abs(f64(got) - want) <= tol).all()
    got = ops.paged_attention_shared_prefix(
        up(q[P:], dev, torch.bfloat16), bm.k_slab, bm.v_slab, ptab, torch.tensor([P], dtype=torch.int32, device=dev),
        torch.tensor([0, 2], dtype=torch.int32, device=dev), t, ctx, **common)
    at = 0
    for i, c in enumerate(own):
        k = np.concatenate([f64(key), f64(k2[at:at + c])])
        v = np.concatenate([f64(value), f64(v2[at:at + c])])
        want = R.attend(q[P + i:P + i + 1], k, v, np.ones((1, P + c), bool), scale)
        class Values:
            fk, fv = k, v
        assert (np.abs(f64(got[i:i + 1]) - want) <= R.bound(want, q, Values, scale, "bf16", p_kind="bf16")).all()
        at += c
