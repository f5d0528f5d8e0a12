"""Attention whose queries all stand at their sequence's last key, through each of the kernels, against the definition in 64 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu

#       B, queries, keys, H, G, columns, backward too
SHAPES = {"few, keys over a block": (2, 5, 500, 4, 2, 64, True), "few, a warp each": (300, 3, 400, 4, 4, 64, False), "few, splits": (2, 16, 20011, 4, 2, 32, False),
          "few, 128 columns": (3, 20, 300, 2, 2, 128, True), "one": (2, 1, 90, 2, 2, 16, True), "short 16": (3, 100, 60, 4, 2, 16, True),
          "short 32": (2, 150, 200, 2, 2, 32, True), "short 64": (2, 70, 90, 4, 4, 64, True), "long 64": (1, 600, 700, 2, 1, 64, True),
          "long 80": (2, 333, 150, 2, 2, 80, True), "long 128, two tiles": (1, 2100, 2100, 20, 20, 128, False)}


@pytest.mark.parametrize("cap", [None, 20.0, 1e6])
@pytest.mark.parametrize("shape", SHAPES)
def test_newest(tn_gpu, status_ok, shape, cap):
    from tensornet_b200.ops import functional as F
    from test_gpu_attention_caps import definition

    dev = tn_gpu.core.runtime().device
    B, nq, nk, H, G, D, train = SHAPES[shape]
    gen = torch.Generator(device=dev).manual_seed(nk)
    q, go = [torch.randn((B, nq, H, D), generator=gen, device=dev).bfloat16() for _ in range(2)]
    k, v = [torch.randn((B, nk, G, D), generator=gen, device=dev).bfloat16() for _ in range(2)]
    slopes = torch.tensor([0.3 / (3 * h + 1) for h in range(H)], device=dev)
    lengths, kv_lengths = [nq - b % 2 for b in range(B)], [nk - (nk // 3 * b) % (nk + 1) for b in range(B)]
    ints = [torch.tensor(n, dtype=torch.int32, device=dev) for n in (lengths, kv_lengths)]
    leaves = [t.requires_grad_(train) for t in (q, k, v)]
    out = F.attention(*leaves, lengths=ints[0], kv_lengths=ints[1], cap=cap, slopes=slopes, newest=True)
    got = [out.detach(), *(torch.autograd.grad(out, leaves, go) if train else ())]
    want, tol = definition(q, k, v, go, lengths, kv_lengths, False, cap, slopes, newest=True)
    for name, a, b, t in zip(("out", "gq", "gk", "gv"), got, want, tol):
        off = (a.cpu().double() - b).abs() - t
        assert bool((off <= 1e-30).all()), (name, float(off.max()), float(b.abs().max()), int((off > 0).sum()))


def test_without_slopes_it_does_not_matter(tn_gpu, status_ok):
    from tensornet_b200.ops import functional as F

    dev = tn_gpu.core.runtime().device
    q, k, v = [torch.randn((2, 40, 2, 32), device=dev).bfloat16() for _ in range(3)]
    assert torch.equal(F.attention(q, k, v, newest=True), F.attention(q, k, v))
    with pytest.raises(ValueError, match="newest"):
        F.attention(q, k, v, newest=True, causal=True)
