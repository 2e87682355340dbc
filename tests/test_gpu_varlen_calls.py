"""Calls of ragged attention that its documentation allows beside the usual ones: pools whose size is not given,
tensors at odd addresses, one sequence's pages in several tables, two calls at once."""
import numpy as np
import pytest

from tests import paged_ref as R
from tests import paged_rows as P
from tests.test_gpu_varlen import DT, SLOPES, run_varlen, up, varlen_case

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

KINDS = [("bf16", "bf16"), ("f16", "f16"), ("i8", "bf16"), ("f32", "f32")]


def case_of(kind, qkind, d=128, seed=140):
    return varlen_case([900, 37, 5, 300], [200, 1, 5, 3], 8, 2, d, 16, kind, qkind, seed, plant=False)


def agrees(case, got, qkind, **kw):
    q, pool = case[:2]
    scale = 1 / np.sqrt(q.shape[2])
    want = R.varlen(*case, scale, **kw)
    return P.norms_agree(got.double().cpu().numpy(), want, q, pool, scale, qkind, p_kind=None if qkind == "f32" else qkind,
                         most_bias=900.0 if kw.get("slopes") is not None else 0.0)


def call(dev, case, qkind, q=None, **kw):
    from gollek_b200 import ops
    args = dict(block_tables=up(case[2], dev), cu_seqlens_q=up(case[3], dev), context_lens=up(case[4], dev),
                **case[1].args(dev))
    args.update(kw)
    return ops.paged_attention_varlen(up(case[0], dev, DT[qkind]) if q is None else q, **args)


@pytest.mark.parametrize("kind,qkind", KINDS)
@pytest.mark.parametrize("d", [64, 128])
def test_a_pool_of_unknown_size(cuda_device, kind, qkind, d):
    """num_blocks = 0, the default: ids are not checked against a size."""
    case = case_of(kind, qkind, d)
    got = call(cuda_device, case, qkind, num_blocks=0)
    assert agrees(case, got, qkind)
    assert torch.equal(got, run_varlen(cuda_device, *case, qkind))


@pytest.mark.parametrize("kind,qkind", KINDS)
@pytest.mark.parametrize("which", ["q", "out", "k_cache"])
def test_tensors_at_odd_addresses(cuda_device, kind, qkind, which):
    """One element off an aligned address: the calls that the vector and tensor-core kernels leave."""
    case = case_of(kind, qkind)
    def off(t):
        room = torch.empty(t.numel() + 1, dtype=t.dtype, device=cuda_device)
        room[1:] = t.flatten()
        return room[1:].view(t.shape)
    if which == "k_cache":
        args = case[1].args(cuda_device)
        got = call(cuda_device, case, qkind, k_cache=off(args["k_cache"]))
    elif which == "q":
        got = call(cuda_device, case, qkind, q=off(up(case[0], cuda_device, DT[qkind])))
    else:
        got = call(cuda_device, case, qkind, out=off(torch.zeros(case[0].shape, dtype=DT[qkind], device=cuda_device)))
    assert agrees(case, got, qkind)


@pytest.mark.parametrize("kind,qkind", KINDS)
def test_sequences_that_share_pages(cuda_device, kind, qkind):
    """The same table for every sequence, as prompts that came from one cache have it, and one page twice in a table."""
    q, pool, tables, cu, ctx = case_of(kind, qkind)
    tables = np.repeat(tables[:1], 4, axis=0)
    tables[1, 1] = tables[1, 0]
    case = (q, pool, tables, cu, np.array([900, 37, 800, 900], np.int32))
    assert agrees(case, call(cuda_device, case, qkind, alibi_slopes=up(SLOPES(8), cuda_device)), qkind, slopes=SLOPES(8))


def test_two_calls_at_once(cuda_device):
    """On two streams, each with scratch from the allocator, many times over."""
    cases = [varlen_case([3000, 700, 90], [40, 1, 90], 8, 2, 128, 16, k, "bf16", 141 + i, plant=False)
             for i, k in enumerate(("bf16", "i8"))]
    want = [run_varlen(cuda_device, *c, "bf16") for c in cases]
    ready = [(up(c[0], cuda_device, torch.bfloat16),
              dict(block_tables=up(c[2], cuda_device), cu_seqlens_q=up(c[3], cuda_device),
                   context_lens=up(c[4], cuda_device), **c[1].args(cuda_device))) for c in cases]
    from gollek_b200 import ops
    streams = [torch.cuda.Stream(cuda_device) for _ in cases]
    torch.cuda.synchronize()
    got = []
    for _ in range(20):
        for (q, kw), s in zip(ready, streams):
            got.append(ops.paged_attention_varlen(q, stream=s, **kw))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i % 2]) for i, g in enumerate(got))
    assert ops.device_status(cuda_device.index or 0) == 0
