"""Targets of the attention block on the GPU: each takes from its sequence what it takes alone."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads, kv_heads, n, T", [(2, 2, 5, 12), (4, 2, 33, 12), (4, 1, 70, 300), (2, 2, 129, 40), (8, 8, 3, 2000)])
def test_targets_do_not_depend_on_their_neighbours(tn_gpu, status_ok, heads, kv_heads, n, T):
    from test_cpu_attention_targets import one_by_one

    dev = tn_gpu.core.runtime().device
    torch.manual_seed(n)
    layer = tn_gpu.layers.SequenceAttention(16 * heads, heads=heads, kv_heads=kv_heads, distance_bias=True, cap=20.0).to(dev)
    x, lengths = torch.randn(3, T, 16 * heads, device=dev), torch.tensor([T, 0, T // 3], device=dev)
    target = torch.randn(3, n, 16 * heads, device=dev).requires_grad_()
    together, alone, off = one_by_one(layer, x, lengths, target)
    assert bool(((together - alone).abs() <= off).all())
    g = torch.randn_like(together)
    a, b = [torch.autograd.grad(y, target, g)[0] for y in (together, alone)]
    assert float((a - b).norm()) <= 2.0 ** -6 * float(b.norm())


def test_captured(tn_gpu, status_ok):
    dev = tn_gpu.core.runtime().device
    torch.manual_seed(0)
    layer = tn_gpu.layers.SequenceAttention(32, heads=4, distance_bias=True).to(dev)
    x, target = torch.randn(4, 50, 32, device=dev), torch.randn(4, 70, 32, device=dev)
    lengths = torch.tensor([50, 1, 0, 33], dtype=torch.int32, device=dev)
    with torch.no_grad():
        layer(x, lengths, target)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = layer(x, lengths, target)
        target.copy_(target.flip(1))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, layer(x, lengths, target))
