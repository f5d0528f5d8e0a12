"""What comes of layer normalisation may be changed in place, with and without a graph."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape, dtype", [((5, 24), torch.float32), ((2, 3, 1000), torch.bfloat16), ((40,), torch.float32)])
def test_results_are_changed_in_place(tn_gpu, status_ok, shape, dtype):
    from tensornet_b200.ops import functional as F

    dev = tn_gpu.core.runtime().device
    gen = torch.Generator(device=dev).manual_seed(1)
    x = torch.randn(shape, generator=gen, device=dev).to(dtype).requires_grad_()
    dy = torch.randn(shape, generator=gen, device=dev).to(dtype)
    want = F.layer_norm(x)
    (gx,) = torch.autograd.grad(want, x, dy)
    y = F.layer_norm(x)
    y.mul_(2.0)
    assert torch.equal(y, 2 * want) and torch.equal(torch.autograd.grad(y, x, dy)[0], torch.autograd.grad(F.layer_norm(x), x, 2 * dy)[0])
    with torch.no_grad():
        assert torch.equal(F.layer_norm(x).add_(1.0), want + 1.0)
