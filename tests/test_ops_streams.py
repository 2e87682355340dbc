"""Streams that the tensor-level calls refuse (no GPU)."""
from types import SimpleNamespace

import pytest

torch = pytest.importorskip("torch")


def test_a_stream_of_another_device_is_refused():
    """The kernels would run on the stream's device, on tensors of another."""
    from gollek_b200 import ops
    elsewhere = SimpleNamespace(cuda_stream=16, device=torch.device("cuda", 1))
    with pytest.raises(ValueError, match="stream is on cuda:1, not cuda:0"):
        ops._on(torch.device("cuda", 0), elsewhere).__enter__()
