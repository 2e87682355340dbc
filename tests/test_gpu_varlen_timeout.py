"""Failure detection in ragged and shared-prefix attention, without a GPU fault: waits that give up.

GOLLEK_TEST_SKIP_GROUP stops CTA 0's producers behind so many tiles of their first run, so that whoever waits for the
next copy runs out of the bound that GOLLEK_TEST_WAIT_LIMIT makes short.  Nothing faults: the copy is simply never
made.  Every warp of the CTA leaves, the status says TIMEOUT, and the next call, in the same workspace, is right."""
import numpy as np
import pytest

from tests.test_gpu_varlen import run_shared, shared_case, varlen_case

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

DECODE = ([6000, 3000, 5000, 2000], [1] * 4)
PROMPTS = ([2500, 900], [700, 900])
CHUNKS = ([6000, 5000, 8000], [20, 31, 17])  # blocks of fewer than 128 rows
HQ, HKV = 32, 8                              # CTA 0 has 5 tiles and more in every case


@pytest.mark.parametrize("kind", ["bf16", "i8"])
@pytest.mark.parametrize("ctx,new,d", [(*DECODE, 128), (*DECODE, 64), (*PROMPTS, 128), (*CHUNKS, 128), (*PROMPTS, 64)])
@pytest.mark.parametrize("stop_at", [0, 1, 4])
def test_a_wait_gives_up_then_the_next_call_is_right(cuda_device, monkeypatch, kind, ctx, new, d, stop_at):
    from gollek_b200 import _lib, ops
    q, pool, tables, cu, ctx = varlen_case(ctx, new, HQ, HKV, d, 16, kind, "bf16", 130, plant=False)
    ws = torch.zeros(ops.varlen_workspace_size(len(ctx), len(q), HQ, HKV, d), dtype=torch.uint8, device=cuda_device)
    up = lambda x, dt=None: torch.from_numpy(np.ascontiguousarray(x)).to(cuda_device, dt)
    args = dict(block_tables=up(tables), cu_seqlens_q=up(cu), context_lens=up(ctx), workspace=ws, **pool.args(cuda_device))
    call = lambda: ops.paged_attention_varlen(up(q, torch.bfloat16), **args)
    ops.device_status(cuda_device.index or 0)
    want = call()
    assert ops.device_status(cuda_device.index or 0) == 0
    monkeypatch.setenv("GOLLEK_TEST_WAIT_LIMIT", "20000")
    monkeypatch.setenv("GOLLEK_TEST_SKIP_GROUP", str(stop_at))
    call()
    assert ops.device_status(cuda_device.index or 0) == _lib.STATUS_TIMEOUT
    monkeypatch.delenv("GOLLEK_TEST_WAIT_LIMIT")
    monkeypatch.delenv("GOLLEK_TEST_SKIP_GROUP")
    for _ in range(2):
        assert torch.equal(call(), want)
        assert ops.device_status(cuda_device.index or 0) == 0


def test_a_wait_behind_a_shared_prefix_gives_up(cuda_device, monkeypatch):
    """Two kernels in a row (the prefix's and the own tokens'): both stop, both leave."""
    from gollek_b200 import _lib, ops
    case = shared_case([30000], [0, 64], [400] * 64, 32, 8, 128, 16, "bf16", "bf16", 131)
    ops.device_status(cuda_device.index or 0)
    want = run_shared(cuda_device, case, "bf16")
    monkeypatch.setenv("GOLLEK_TEST_WAIT_LIMIT", "20000")
    monkeypatch.setenv("GOLLEK_TEST_SKIP_GROUP", "2")
    run_shared(cuda_device, case, "bf16")
    assert ops.device_status(cuda_device.index or 0) == _lib.STATUS_TIMEOUT
    monkeypatch.delenv("GOLLEK_TEST_WAIT_LIMIT")
    monkeypatch.delenv("GOLLEK_TEST_SKIP_GROUP")
    assert torch.equal(run_shared(cuda_device, case, "bf16"), want)
    assert ops.device_status(cuda_device.index or 0) == 0
