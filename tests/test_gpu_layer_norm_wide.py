"""Layer normalisation of few very wide rows: what the backward pass takes of memory, and its sums."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [1, 2, 64, 65])
def test_workspace_goes_by_the_rows(tn_gpu, status_ok, rows):
    from tensornet_b200.ops import functional as F

    dev, columns = tn_gpu.core.runtime().device, 1 << 18
    gen = torch.Generator(device=dev).manual_seed(rows)
    x, dy = [torch.randn((rows, columns), generator=gen, device=dev) for _ in range(2)]
    gamma, beta = [torch.randn(columns, generator=gen, device=dev).requires_grad_() for _ in range(2)]
    x.requires_grad_()
    y = F.layer_norm(x, gamma, beta)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats(dev)
    before = torch.cuda.memory_allocated(dev)
    gx, gg, gb = torch.autograd.grad(y, (x, gamma, beta), dy)
    torch.cuda.synchronize()
    # three results, and two sums per column of each row or of 64 shares of the rows
    assert torch.cuda.max_memory_allocated(dev) - before <= 4 * columns * (rows + 2 + 2 * min(rows, 64)) + (1 << 20)
    d, xd = dy.double(), x.detach().double()
    c = xd - xd.mean(1, keepdim=True)
    xhat = c / torch.sqrt((c * c).mean(1, keepdim=True) + 1e-5)
    # fp32 sums of up to two terms, then fp64; a normalised value is off by its rounding, that of the mean's 256 terms per thread and the tree's
    off = 300 * 2.0 ** -24
    assert torch.all((gb.double() - d.sum(0)).abs() <= 2.0 ** -22 * d.abs().sum(0))
    assert torch.all((gg.double() - (d * xhat).sum(0)).abs() <= off * (d.abs() * (1 + xhat.abs())).sum(0))
