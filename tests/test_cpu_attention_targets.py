"""Targets of the attention block, candidates say, on the CPU path: each takes from its sequence what it takes alone."""
import pytest
import torch

import tensornet_b200 as tn


@pytest.fixture(autouse=True)
def _cpu_runtime():
    tn.core.shutdown()
    tn.core.config.force_cpu = True
    tn.core.init()
    yield
    tn.core.shutdown()


@pytest.mark.parametrize("shape", [(0, 16), (0, 3, 16), (2, 0, 16)])
def test_no_targets(shape):
    layer = tn.layers.SequenceAttention(16, heads=2, distance_bias=True)
    t = torch.randn(shape)
    lengths = torch.zeros(shape[0], dtype=torch.int64)
    assert layer(torch.randn(shape[0], 5, 16), lengths, t).shape == shape
    assert layer(torch.randn(shape[0], 0, 16), None, t).shape == shape
