"""The scratch of ragged and shared-prefix attention: the library's own (a NULL workspace, as C and Java
callers pass it) beside the split-K scratch of the other attention entry points on one stream."""
import ctypes
import itertools
import math

import numpy as np
import pytest

from tests import paged_ref as R
from tests.helpers import make_tables

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

HQ, HKV, D, BS = 32, 8, 128, 16


class Calls:
    """C calls with NULL workspaces over one pool: a decode step whose sequences are cut over many SMs, a
    multi-query step, a prompt, and a decode step behind a shared prefix."""

    def __init__(self, dev):
        from gollek_b200 import _lib
        rng = np.random.default_rng(90)
        self.lib, self.dev, self.code = _lib.load(), dev, _lib
        self.ctx = np.array([8000, 7000, 6000, 9000], np.int32)
        nb = sum((int(c) + BS - 1) // BS for c in self.ctx) + 3
        up = lambda x, dt=None: torch.from_numpy(np.ascontiguousarray(x)).to(dev, dt)
        self.nb, self.tables = nb, make_tables(self.ctx, BS, nb, rng)
        self.t, self.c = up(self.tables), up(self.ctx)
        self.k, self.v = (up(rng.standard_normal((nb, HKV, BS, D)) * 0.5, torch.bfloat16) for _ in range(2))
        self.q1 = up(rng.standard_normal((4, HQ, D)), torch.bfloat16)
        self.q16 = up(rng.standard_normal((4, 16, HQ, D)), torch.bfloat16)
        self.qp = up(rng.standard_normal((700, HQ, D)), torch.bfloat16)
        self.cu = up(np.array([0, 300, 301, 500, 700], np.int32))
        self.gs, self.pl = up(np.array([0, 4], np.int32)), up(np.array([5000], np.int32))
        self.own = up(np.array([100, 1, 2000, 37], np.int32))

    def pool(self):
        return self.k.data_ptr(), self.v.data_ptr(), None, None

    def check(self, rc):
        self.code.check(rc)

    def decode(self, stream):
        out = torch.full_like(self.q1, 7.0)
        self.check(self.lib.gollek_paged_attention_v2(
            out.data_ptr(), self.q1.data_ptr(), *self.pool(), self.t.data_ptr(), self.c.data_ptr(), 4, HQ, HKV, D, BS,
            self.t.shape[1], self.nb, 0, self.code.BF16, self.code.BF16, 0, 0, 0, 1 / math.sqrt(D), 0.0, 0, None, 0, stream))
        return out

    def multi(self, stream):
        out = torch.full_like(self.q16, 7.0)
        self.check(self.lib.gollek_paged_attention_prefill(
            out.data_ptr(), self.q16.data_ptr(), *self.pool(), self.t.data_ptr(), self.c.data_ptr(), 4, 16, HQ, HKV, D, BS,
            self.t.shape[1], self.nb, 0, self.code.BF16, self.code.BF16, 0, 0, 0, 1 / math.sqrt(D), 0.0, 0, 1, None, 0, stream))
        return out

    def varlen(self, stream):
        out = torch.full_like(self.qp, 7.0)
        self.check(self.lib.gollek_paged_attention_varlen(
            out.data_ptr(), self.qp.data_ptr(), *self.pool(), self.t.data_ptr(), self.cu.data_ptr(), self.c.data_ptr(),
            None, None, None, 4, 700, HQ, HKV, D, BS, self.t.shape[1], self.nb, 0, self.code.BF16, self.code.BF16, 0, 0, 0,
            1 / math.sqrt(D), 0.0, 0, 1, None, 0, stream))
        return out

    def shared(self, stream):
        out = torch.full_like(self.q1, 7.0)
        self.check(self.lib.gollek_paged_attention_shared_prefix(
            out.data_ptr(), self.q1.data_ptr(), *self.pool(), self.t[:1].data_ptr(), self.pl.data_ptr(), self.gs.data_ptr(),
            self.t.data_ptr(), self.own.data_ptr(), 1, self.t.shape[1], 4, HQ, HKV, D, BS, self.t.shape[1], self.nb, 0,
            self.code.BF16, self.code.BF16, 0, 0, 0, 1 / math.sqrt(D), 0.0, None, 0, stream))
        return out


def test_null_workspaces_of_all_entry_points_on_one_stream(cuda_device):
    """Every order of the calls, each order on a stream of its own, gives what each call gives alone."""
    calls = Calls(cuda_device)
    names = ("decode", "multi", "varlen", "shared")
    alone = {}
    for n in names:
        s = torch.cuda.Stream(cuda_device)
        with torch.cuda.stream(s):
            alone[n] = getattr(calls, n)(s.cuda_stream)
        s.synchronize()
    f64 = lambda x: x.double().cpu().numpy()
    pool = R.Pool("bf16", f64(calls.k), f64(calls.v))
    want = R.varlen(f64(calls.q1), pool, calls.tables, np.arange(5), calls.ctx, 1 / math.sqrt(D))
    assert np.abs(f64(alone["decode"]) - want).max() < 2e-2  # written, and the right rows
    for order in itertools.permutations(names):
        s = torch.cuda.Stream(cuda_device)
        with torch.cuda.stream(s):
            got = [(n, getattr(calls, n)(s.cuda_stream)) for n in order + order]
        s.synchronize()
        for n, out in got:
            # the split-K kernel joins partials in the order of their arrival: bits may move, rows may not
            same = torch.equal(out, alone[n]) if n in ("varlen", "shared") else torch.allclose(
                out.float(), alone[n].float(), atol=2e-3, rtol=0)
            assert same, f"{n} in the order {order}"


def test_a_captured_call_needs_its_own_workspace(cuda_device):
    """NULL is refused under capture, where the library's scratch could be freed or shared behind the graph; the
    capture goes on, and a graph with a workspace gives the eager call's rows."""
    from gollek_b200 import _lib
    calls = Calls(cuda_device)
    want = [calls.varlen(0), calls.shared(0)]  # the default stream's scratch is large enough from here on
    torch.cuda.synchronize()
    graph, s = torch.cuda.CUDAGraph(), torch.cuda.Stream(cuda_device)
    with torch.cuda.stream(s):
        eager = [calls.varlen(s.cuda_stream), calls.shared(s.cuda_stream)]
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(eager, want))
    n = _lib.load().gollek_paged_attention_varlen_workspace_size(4, 700, HQ, HKV, D)
    ws, out = torch.empty(n, dtype=torch.uint8, device=cuda_device), torch.zeros_like(calls.qp)
    with torch.cuda.graph(graph, stream=s):
        for call in (calls.varlen, calls.shared):
            with pytest.raises(_lib.GollekError) as e:
                call(s.cuda_stream)
            assert e.value.code == _lib.ERR_WORKSPACE and "captured" in str(e.value)
        _lib.check(_lib.load().gollek_paged_attention_varlen(
            out.data_ptr(), calls.qp.data_ptr(), *calls.pool(), calls.t.data_ptr(), calls.cu.data_ptr(), calls.c.data_ptr(),
            None, None, None, 4, 700, HQ, HKV, D, BS, calls.t.shape[1], calls.nb, 0, _lib.BF16, _lib.BF16, 0, 0, 0,
            1 / math.sqrt(D), 0.0, 0, 1, ws.data_ptr(), n, s.cuda_stream))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want[0])
    del graph


def test_two_host_threads_on_one_stream(cuda_device):
    """Calls with NULL workspaces from two threads: each call's kernels follow one another in the stream."""
    import threading
    calls = Calls(cuda_device)
    s = torch.cuda.Stream(cuda_device)
    want, wrong = {}, []
    with torch.cuda.stream(s):
        for n in ("varlen", "shared"):
            want[n] = getattr(calls, n)(s.cuda_stream)
    s.synchronize()

    def work(name):
        try:
            with torch.cuda.stream(s):
                for _ in range(100):
                    if not torch.equal(getattr(calls, name)(s.cuda_stream), want[name]):
                        wrong.append(name)
        except Exception as e:  # noqa: BLE001 -- reported by the main thread
            wrong.append(repr(e))

    threads = [threading.Thread(target=work, args=(n,)) for n in ("varlen", "shared", "varlen")]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not wrong, wrong[:3]
