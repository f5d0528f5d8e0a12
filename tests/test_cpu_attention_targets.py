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


def one_by_one(layer, x, lengths, target):
    """What each target gathers alone, how far bf16 may put that off what it gathers beside others, and the gradients of both."""
    D = layer.heads * layer.head_dim
    with torch.no_grad():                       # the block's output product hands the attention's results out as they are
        layer.output.copy_(torch.eye(layer.output.shape[0], layer.output.shape[1], device=layer.output.device))
    assert layer.dim == D
    together = layer(x, lengths, target)
    alone = torch.stack([layer(x, lengths, target[:, i]) for i in range(target.shape[1])], 1)
    with torch.no_grad():
        # a result is a mean of values with weights off by half a step each time, rounded by another, and rounded again by the product
        w = layer.key_value[layer.kv_heads * layer.head_dim:, :layer.dim]
        size = (layer.norm(x) @ w.t()).abs().amax(1).unflatten(-1, (layer.kv_heads, -1)).repeat_interleave(layer.heads // layer.kv_heads, 1)
        off = (2 * 2.0 ** -8 + 2 * 2.0 ** -7) * size.flatten(1).unsqueeze(1)
    return together, alone, off


@pytest.mark.parametrize("heads, kv_heads, n", [(2, 2, 5), (4, 2, 33), (4, 1, 2), (2, 2, 66)])
def test_targets_do_not_depend_on_their_neighbours(heads, kv_heads, n):
    torch.manual_seed(n)
    layer = tn.layers.SequenceAttention(8 * heads, heads=heads, kv_heads=kv_heads, distance_bias=True, causal=True, cap=20.0)
    x, lengths, target = torch.randn(3, 12, 8 * heads), torch.tensor([12, 0, 5]), torch.randn(3, n, 8 * heads).requires_grad_()
    together, alone, off = one_by_one(layer, x, lengths, target)
    assert bool(((together - alone).abs() <= off).all())
    same = layer(x, lengths, target[:, :1].expand(3, n, 8 * heads))
    assert bool(((same - same[:, :1]).abs() <= off).all())
    g = torch.randn_like(together)
    a, b = [torch.autograd.grad(y, target, g)[0] for y in (together, alone)]
    assert float((a - b).norm()) <= 2.0 ** -6 * float(b.norm())


@pytest.mark.parametrize("nq, nk", [(1, 4), (5, 9), (9, 5)])
def test_newest_queries_stand_at_the_last_key(nq, nk):
    from tensornet_b200.ops import functional as F

    g = torch.Generator().manual_seed(nq)
    q, k, v = [torch.randn((2, n, 2, 8), generator=g).bfloat16() for n in (nq, nk, nk)]
    slopes = torch.tensor([0.5, 0.1])
    got = F.attention(q, k, v, slopes=slopes, newest=True)
    s = torch.einsum("bihd,bjhd->bhij", q.double(), k.double()) * 8 ** -0.5 - slopes.double().view(1, 2, 1, 1) * (nk - 1 - torch.arange(nk))
    want = torch.einsum("bhij,bjhd->bihd", torch.softmax(s, -1), v.double())
    assert bool(((got.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -18 * v.double().abs().max()).all())      # fp32, rounded once
    with pytest.raises(ValueError, match="newest"):
        F.attention(q, k, v, causal=True, newest=True)


@pytest.mark.parametrize("causal", [False, True])
def test_a_prefix_does_not_go_with_targets(causal):
    layer = tn.layers.SequenceAttention(16, heads=2, causal=causal)
    prefix = torch.ones(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="targets see all"):
        layer(torch.zeros(2, 5, 16), None, torch.zeros(2, 16), prefix=prefix)
    if causal:
        assert layer(torch.zeros(2, 5, 16), prefix=prefix).shape == (2, 5, 16)
