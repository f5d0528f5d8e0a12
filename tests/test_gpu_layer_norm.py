"""Layer normalisation kernels against the formula in 64 bits.

Tolerances: a result is rounded to its type once (half a step, eps / 2 of it).  In fp32, a thread adds 16 elements and the group adds
in a tree of at most 5 + 16 steps, so a sum of C terms is off by at most 40 steps of 2^-24 of the sum of their magnitudes; a mean
is then off by 40 * 2^-24 * max|x|, which the division by the spread turns into 40 * 2^-24 * max|x| * rstd of a normalised value,
and the variance, the square root, the division and the products add less than 60 more.  ``_K`` is their sum."""
import pytest
import torch

pytestmark = pytest.mark.gpu

_K = 100 * 2.0 ** -24


def _formula(x, gamma, beta, eps):
    c = x - x.mean(-1, keepdim=True)
    return c / torch.sqrt((c * c).mean(-1, keepdim=True) + eps) * (1.0 if gamma is None else gamma) + (0.0 if beta is None else beta)


def _check(x, gamma, beta, eps, dy):
    from tensornet_b200.ops import functional as F

    half = torch.finfo(x.dtype).eps / 2
    wrt = [t for t in (x, gamma, beta) if t is not None and t.requires_grad]
    y = F.layer_norm(x, gamma, beta, eps)
    assert y.shape == x.shape and y.dtype == x.dtype
    grads = dict(zip(map(id, wrt), torch.autograd.grad(y, wrt, dy) if wrt else ()))
    copies = [None if t is None else t.detach().double().requires_grad_() for t in (x, gamma, beta)]
    ref = _formula(*copies, eps)
    there = [c for c in copies if c is not None]
    want = dict(zip(map(id, there), torch.autograd.grad(ref, there, dy.double())))
    xd, ref, dyd = x.detach().double(), ref.detach(), dy.double()
    C = x.shape[-1]
    c = xd - xd.mean(-1, keepdim=True)
    rstd = 1.0 / torch.sqrt((c * c).mean(-1, keepdim=True) + eps)
    xhat = c * rstd
    off = _K * (1.0 + xd.abs().amax(-1, keepdim=True) * rstd)            # of a normalised value
    g = torch.ones(C, dtype=torch.float64, device=x.device) if gamma is None else gamma.detach().double().abs()
    b = 0.0 if beta is None else beta.detach().double().abs()
    assert torch.all((y.double() - ref).abs() <= half * ref.abs() + off * (g * (1 + xhat.abs()) + b) + 2.0 ** -24)
    if id(x) in grads:
        gd = dyd.abs() * g
        size = rstd * (gd + gd.mean(-1, keepdim=True) + (1 + xhat.abs()) * (gd * (1 + xhat.abs())).mean(-1, keepdim=True))
        dx = want[id(copies[0])]
        tiny = torch.finfo(x.dtype).smallest_normal * half if x.dtype == torch.float16 else 0.0
        assert torch.all((grads[id(x)].double() - dx).abs() <= half * dx.abs() + 4 * off * size + tiny)
    lead = tuple(range(x.dim() - 1))
    if gamma is not None and id(gamma) in grads:
        size = (dyd.abs() * (xhat.abs() * 2.0 ** -17 + 2 * off * (1 + xhat.abs()))).sum(lead)      # up to 128 terms one after another
        assert torch.all((grads[id(gamma)].double() - want[id(copies[1])]).abs() <= size)
    if beta is not None and id(beta) in grads:
        assert torch.all((grads[id(beta)].double() - want[id(copies[2])]).abs() <= (dyd.abs() * 2.0 ** -17).sum(lead))
    return y, grads


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows, C", [(1, 1), (3, 2), (200, 64), (1, 8192), (37, 7), (1000, 8), (65, 9), (513, 33), (129, 429), (31, 500),
                                     (50, 512), (17, 513), (24, 1000), (40, 6413), (9, 8191), (3, 8192), (5, 8193), (2, 20000), (4097, 16)])
def test_forward_backward(tn_gpu, status_ok, dtype, rows, C):
    dev = tn_gpu.core.runtime().device
    gen = torch.Generator(device=dev).manual_seed(rows * 10007 + C)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=dev)

    x = (normal(rows, C) * (0.2 + normal(rows, 1).abs()) + normal(rows, 1)).to(dtype).requires_grad_()
    gamma, beta = (1 + 0.3 * normal(C)).requires_grad_(), normal(C).requires_grad_()
    _check(x, gamma, beta, 1e-5, (normal(rows, C) * 0.1).to(dtype))


def _made(dev, *shape, dtype=torch.float32, seed=1):
    return torch.randn(shape, generator=torch.Generator(device=dev).manual_seed(seed), device=dev).to(dtype)


@pytest.mark.parametrize("which", ["none", "gamma", "beta", "x only", "parameters only", "gamma only"])
def test_what_is_left_out_or_frozen(tn_gpu, status_ok, which):
    dev = tn_gpu.core.runtime().device
    x, dy = _made(dev, 70, 45).requires_grad_(which not in ("parameters only", "gamma only")), _made(dev, 70, 45, seed=2)
    gamma = _made(dev, 45, seed=3).requires_grad_(which != "x only") if which not in ("none", "beta") else None
    beta = _made(dev, 45, seed=4).requires_grad_(which in ("beta", "parameters only")) if which not in ("none", "gamma") else None
    _check(x, gamma, beta, 1e-3, dy)


@pytest.mark.parametrize("form", ["transposed", "slice", "off a boundary", "4-d", "broadcast gradient", "gamma of stride 2"])
def test_layouts(tn_gpu, status_ok, form):
    dev = tn_gpu.core.runtime().device
    dtype = torch.bfloat16
    gamma, beta = _made(dev, 40, seed=3), _made(dev, 40, seed=4)
    dy = _made(dev, 33, 40, dtype=dtype, seed=2)
    x = _made(dev, 33, 40, dtype=dtype)
    if form == "transposed":
        x, dy = _made(dev, 40, 33, dtype=dtype).t(), _made(dev, 40, 33, dtype=dtype).t()
    elif form == "slice":
        x = _made(dev, 33, 100, dtype=dtype)[:, 13:53]
    elif form == "off a boundary":
        x, dy = _made(dev, 33 * 40 + 3, dtype=dtype)[3:].view(33, 40), _made(dev, 33 * 40 + 1, dtype=dtype)[1:].view(33, 40)
    elif form == "4-d":
        x, dy = x.view(3, 11, 2, 20), dy.view(3, 11, 2, 20)
        gamma, beta = gamma[:20], beta[:20]
    elif form == "broadcast gradient":
        dy = _made(dev, 1, 40, dtype=dtype).expand(33, 40)
    elif form == "gamma of stride 2":
        gamma = _made(dev, 80)[::2]
    _check(x.detach().requires_grad_(), gamma.detach().requires_grad_(), beta.detach().requires_grad_(), 1e-5, dy)


def test_rows_without_spread_far_from_zero_and_not_finite(tn_gpu, status_ok):
    from tensornet_b200.ops import functional as F

    dev = tn_gpu.core.runtime().device
    x = _made(dev, 6, 100)
    x[0] = 0.0
    x[1] = 7.5
    x[2] = x[2] * 1e-3 + 1000.0
    x[3] = x[3] * 1e4 - 1e6
    good = x.clone().requires_grad_()
    _check(good, None, None, 1e-5, _made(dev, 6, 100, seed=2))
    clean = F.layer_norm(x)
    x[4, 17], x[5, 99] = float("nan"), float("inf")
    y = F.layer_norm(x)
    assert torch.equal(y[:4], clean[:4]) and bool(y[4:].isnan().all())


def test_no_rows(tn_gpu, status_ok):
    from tensornet_b200.ops import functional as F

    dev = tn_gpu.core.runtime().device
    x, gamma, beta = torch.zeros(0, 3, 12, device=dev, requires_grad=True), _made(dev, 12).requires_grad_(), _made(dev, 12).requires_grad_()
    y = F.layer_norm(x, gamma, beta)
    gx, gg, gb = torch.autograd.grad(y.sum(), (x, gamma, beta))
    assert y.shape == x.shape and gx.shape == x.shape and not gg.any() and not gb.any()


def test_same_bits_each_time_on_other_streams_and_from_a_graph(tn_gpu, status_ok):
    from tensornet_b200.ops import functional as F

    dev = tn_gpu.core.runtime().device
    x, gamma, beta = _made(dev, 5000, 77).requires_grad_(), _made(dev, 77, seed=2).requires_grad_(), _made(dev, 77, seed=3).requires_grad_()
    dy = _made(dev, 5000, 77, seed=4)

    def go():
        y = F.layer_norm(x, gamma, beta)
        return [y.detach(), *torch.autograd.grad(y, (x, gamma, beta), dy)]

    want = go()
    assert all(torch.equal(a, b) for a, b in zip(go(), want))
    streams = [torch.cuda.Stream(dev) for _ in range(2)]
    got = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream(dev))
        with torch.cuda.stream(s):
            got.append(go())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g in got for a, b in zip(g, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = go()
    with torch.no_grad():
        dy.mul_(2.0)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out[0], want[0]) and all(torch.equal(a, 2 * b) for a, b in zip(out[1:], want[1:]))


def test_layer_trains(tn_gpu, status_ok):
    dev = tn_gpu.core.runtime().device
    layer = tn_gpu.layers.LayerNormalization(24).to(dev)
    x = _made(dev, 4, 9, 24)
    layer(x).square().sum().backward()
    assert layer.gamma.grad.shape == (24,) and bool(layer.beta.grad.isfinite().all())
    with torch.no_grad():
        assert layer(x).shape == x.shape


def test_second_derivatives_are_refused(tn_gpu, status_ok):
    from tensornet_b200.ops import functional as F

    x = _made(tn_gpu.core.runtime().device, 4, 8).requires_grad_()
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(F.layer_norm(x).square().sum(), x, create_graph=True)
