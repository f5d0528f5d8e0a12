"""Layer normalisation on the CPU path, and what it refuses."""
import pytest
import torch

import tensornet_b200 as tn
from tensornet_b200.ops import functional as F


def test_matches_its_formula_and_differences():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(5, 3, 7, generator=g).requires_grad_()
    gamma, beta = torch.randn(7, generator=g).requires_grad_(), torch.randn(7, generator=g).requires_grad_()
    y = F.layer_norm(x, gamma, beta, eps=1e-3)
    xd = x.detach().double()
    c = xd - xd.mean(-1, keepdim=True)
    ref = c / torch.sqrt((c * c).mean(-1, keepdim=True) + 1e-3) * gamma.detach().double() + beta.detach().double()
    assert torch.allclose(y.detach().double(), ref, rtol=0, atol=64 * 2.0 ** -24 * float(ref.abs().max()))
    dy = torch.randn(y.shape, generator=g)
    grads = torch.autograd.grad(y, (x, gamma, beta), dy)
    x64, g64, b64 = [t.detach().double().requires_grad_() for t in (x, gamma, beta)]
    c = x64 - x64.mean(-1, keepdim=True)
    want = torch.autograd.grad(c / torch.sqrt((c * c).mean(-1, keepdim=True) + 1e-3) * g64 + b64, (x64, g64, b64), dy.double())
    for a, b in zip(grads, want):
        assert torch.allclose(a.double(), b, rtol=0, atol=512 * 2.0 ** -24 * float(b.abs().max()))


def test_layer_has_its_configuration_and_parameters():
    layer = tn.layers.LayerNormalization(6, center=False, epsilon=1e-3, name="ln")
    assert layer.beta is None and layer.gamma.shape == (6,)
    again = tn.layers.LayerNormalization(**layer.get_config())
    assert again.get_config() == layer.get_config()
    x = torch.randn(4, 6)
    assert torch.equal(layer(x), F.layer_norm(x, torch.ones(6), None, 1e-3))
    with pytest.raises(ValueError, match="rows of 6 columns"):
        layer(torch.randn(4, 5))


@pytest.mark.parametrize("kw, text", [
    (dict(x=torch.zeros(3, 4, dtype=torch.float64)), "fp32, bf16 or fp16"),
    (dict(x=torch.zeros(3, 4, dtype=torch.int32)), "fp32, bf16 or fp16"),
    (dict(x=torch.zeros(3, 0)), "one column"),
    (dict(x=torch.zeros(())), "one column"),
    (dict(x=torch.zeros(3, 4), gamma=torch.ones(5)), "gamma"),
    (dict(x=torch.zeros(3, 4), gamma=torch.ones(1, 4)), "gamma"),
    (dict(x=torch.zeros(3, 4), beta=torch.ones(4, dtype=torch.bfloat16)), "beta"),
    (dict(x=torch.zeros(3, 4), eps=0.0), "eps"),
    (dict(x=torch.zeros(3, 4), eps=1e-40), "eps"),
    (dict(x=torch.zeros(3, 4), eps=float("nan")), "eps"),
])
def test_refusals(kw, text):
    with pytest.raises(ValueError, match=text):
        F.layer_norm(**kw)


def test_no_rows():
    x = torch.zeros(0, 4, requires_grad=True)
    assert F.layer_norm(x).shape == (0, 4)
