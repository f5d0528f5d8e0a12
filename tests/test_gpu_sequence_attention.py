"""The attention block on the GPU: against the CPU path, and in a model that trains, captured, from a table's sequences."""
import copy

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kw", [dict(heads=4), dict(heads=4, kv_heads=1, head_dim=24, causal=True, distance_bias=True, cap=5.0)])
@pytest.mark.parametrize("shape", [None, (7, 64), (7, 3, 64)])
def test_like_the_cpu_path(tn_gpu, status_ok, kw, shape):
    dev = tn_gpu.core.runtime().device
    torch.manual_seed(0)
    cpu = tn_gpu.layers.SequenceAttention(64, **kw)
    gpu = copy.deepcopy(cpu).to(dev)
    x, lengths = torch.randn(7, 50, 64), torch.tensor([50, 0, 1, 17, 49, 33, 16])
    target = None if shape is None else torch.randn(shape)
    out, grads = [], []
    for layer, d in ((cpu, "cpu"), (gpu, dev)):
        leaves = [t.to(d).requires_grad_() for t in ([x.clone()] if target is None else [x.clone(), target.clone()])]
        y = layer(leaves[0], lengths.to(d), *leaves[1:])
        torch.manual_seed(1)
        y.backward(torch.randn(y.shape).to(d))
        out.append(y.detach().cpu())
        grads.append([t.grad.cpu() for t in leaves] + [p.grad.cpu() for p in layer.parameters()])
    assert torch.allclose(out[0], out[1], atol=0.06)                # both round operands to bf16, at slightly different sums
    for a, b in zip(*grads):
        # what one rounding of an operand moves (2^-8 of it) enters four products in a row, and the CPU path rounds its gradients nowhere
        assert float((a - b).norm()) <= 4 * 2.0 ** -8 * 2 * float(a.norm()) + 1e-5


def test_trains_and_scores_in_a_model(tn_gpu, status_ok):
    from test_cpu_sequence_attention import _Behaviour, behaviour_batch

    tn = tn_gpu
    torch.manual_seed(0)
    m = _Behaviour()
    m.compile(optimizer=tn.optimizer.Optimizer(tn.core.Adam(learning_rate=1e-3)))
    batches = [behaviour_batch(seed=s) for s in range(12)]
    before = m.encode.query.detach().clone()
    losses = [float(m.train_on_batch(f, y)) for f, y in batches]
    assert all(l == l for l in losses) and not torch.equal(before, m.encode.query)
    p = torch.as_tensor(m.predict_on_batch(batches[0][0])).reshape(-1)
    assert p.shape == (32,) and bool(((p > 0) & (p < 1)).all())


def test_a_run_of_the_operators_in_a_graph(tn_gpu, status_ok):
    """Norm, projections, attention and the backward pass of two blocks, captured and replayed on other inputs."""
    dev = tn_gpu.core.runtime().device
    torch.manual_seed(0)
    blocks = [tn_gpu.layers.SequenceAttention(64, heads=4, causal=True, distance_bias=True).to(dev), tn_gpu.layers.SequenceAttention(64, heads=4).to(dev)]
    x, target, g = torch.randn(9, 70, 64, device=dev), torch.randn(9, 64, device=dev), torch.randn(9, 64, device=dev)
    lengths = torch.tensor([70, 3, 0, 64, 65, 1, 30, 16, 17], dtype=torch.int32, device=dev)
    params = [p for b in blocks for p in b.parameters()]
    for p in params:
        p.grad = torch.zeros_like(p)

    def go():
        for p in params:
            p.grad.zero_()
        xs = x.detach().requires_grad_()
        y = blocks[1](blocks[0](xs, lengths), lengths, target)
        y.backward(g)
        return [y.detach(), xs.grad, *[p.grad for p in params]]

    stream = torch.cuda.Stream(dev)
    stream.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(stream):
        for _ in range(2):
            go()
    torch.cuda.current_stream(dev).wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = go()
    x.copy_(torch.randn_like(x))
    lengths.copy_(lengths.flip(0))
    graph.replay()
    torch.cuda.synchronize()
    got = [t.clone() for t in captured]
    for a, b in zip(got, go()):
        assert torch.allclose(a, b, rtol=1e-5, atol=1e-5 * float(b.abs().max()))       # (weight gradients are added by split products)
