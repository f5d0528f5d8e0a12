"""Attention with caps far above its scores, which then leave them as they are, and beside scores that a cap cuts, through each of the kernels.

Tolerances: a kernel's score ``cap tanh(x / cap)`` may be off by 2^-18 of the magnitudes that it is made of (products, bias), whatever the
cap: the fp32 sum of its products and the tanh are off relative to their own values, the latter by less than 2^-20, or by 2^-22 of a cap of up
to 256.  A weight is then off by ``e`` = 2^-12 + 2^-18 size of itself (2^-12 for such caps, the exponentials and fp32 sums of up to 2^15
terms), and the sum that it is divided by by the mean of ``e`` under the weights.  bf16 weights, score gradients and results add half a step,
``u`` = 2^-8, each where they are rounded."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def definition(q, k, v, go, lengths, kv_lengths, causal, cap, slopes, newest=False):
    """``[out, gq, gk, gv]`` in 64 bits and how far each may be off, ``[B, T, heads, columns]``."""
    u, f, g18 = 2.0 ** -8, 2.0 ** -12, 2.0 ** -18
    q64, k64, v64, g64 = [t.detach().cpu().double() for t in (q, k, v, go)]
    H, G, scale = q.shape[2], k.shape[2], q.shape[3] ** -0.5
    R = H // G
    want, tol = [[torch.zeros_like(t) for t in (q64, q64, k64, v64)] for _ in range(2)]
    for b in range(q.shape[0]):
        nq, nk = int(lengths[b]), int(kv_lengths[b])
        if not nq or not nk:
            continue
        qb, gb = [t[b, :nq].transpose(0, 1) for t in (q64, g64)]
        kb, vb = [t[b, :nk].transpose(0, 1).repeat_interleave(R, dim=0) for t in (k64, v64)]
        x = qb @ kb.transpose(1, 2) * scale
        size = qb.abs() @ kb.abs().transpose(1, 2) * scale
        th = torch.tanh(x / cap) if cap else torch.zeros_like(x)
        place = torch.full((nq, 1), nk - 1) if newest else torch.arange(nq).view(-1, 1) + nk - nq
        j = torch.arange(nk).view(1, -1)
        bias = slopes.cpu().double().view(-1, 1, 1) * (place - j).abs()
        x, size = (cap * th if cap else x) - bias, size + bias
        if causal:
            x = x.masked_fill(j > place, -torch.inf)
        p = torch.softmax(x, dim=-1).nan_to_num()          # rows that see nothing
        o = p @ vb
        e = f + g18 * size
        e = e + (p * e).sum(-1, keepdim=True)
        off_o = (((u + e) * p) @ vb.abs()) + u * o.abs()
        dp, dpa = gb @ vb.transpose(1, 2), gb.abs() @ vb.abs().transpose(1, 2)
        delta = (gb * o).sum(-1, keepdim=True)
        slope = (1 - th * th) * scale
        ds = p * (dp - delta) * slope
        off_delta = (gb.abs() * off_o).sum(-1, keepdim=True) + f * (gb * o).abs().sum(-1, keepdim=True)
        off_ds = (u + e) * ds.abs() + p * slope * (off_delta + f * dpa) + p * (dp - delta).abs() * scale * g18

        def shared(t):
            return t.unflatten(0, (G, R)).sum(1).transpose(0, 1)

        gq, gk, gv = ds @ kb, shared(ds.transpose(1, 2) @ qb), shared(p.transpose(1, 2) @ gb)
        for to, t in zip(want, (o.transpose(0, 1), gq.transpose(0, 1), gk, gv)):
            to[b, :t.shape[0]] = t
        off = (off_o.transpose(0, 1), ((off_ds + f * ds.abs()) @ kb.abs() + u * gq.abs()).transpose(0, 1),
               shared((off_ds + f * ds.abs()).transpose(1, 2) @ qb.abs()) + u * gk.abs(), shared(((u + e) * p).transpose(1, 2) @ gb.abs()) + u * gv.abs())
        for to, t in zip(tol, off):
            to[b, :t.shape[0]] = t
    return want, tol


#       B, queries, keys, H, G, columns, causal, train
SHAPES = {"few, keys over a block": (2, 1, 500, 4, 2, 64, False, True), "few, a warp each": (300, 2, 400, 4, 4, 64, True, False),
          "few, splits": (2, 1, 20011, 4, 2, 128, False, False), "few, 16 columns": (3, 3, 300, 2, 2, 16, True, True),
          "short 16": (3, 50, 50, 4, 2, 16, True, True), "short 32": (2, 150, 150, 2, 2, 32, False, True),
          "short 64": (2, 90, 90, 4, 4, 64, True, True), "long 64": (1, 600, 600, 2, 1, 64, True, True),
          "long 80": (2, 333, 333, 2, 2, 80, False, True), "long 128, two tiles": (1, 2100, 2100, 20, 20, 128, True, False)}


def _check(dev, shape, cap, cut):
    from tensornet_b200.ops import functional as F

    B, nq, nk, H, G, D, causal, train = SHAPES[shape]
    gen = torch.Generator(device=dev).manual_seed(nk)
    q, go = [torch.randn((B, nq, H, D), generator=gen, device=dev) for _ in range(2)]
    k, v = [torch.randn((B, nk, G, D), generator=gen, device=dev) for _ in range(2)]
    if cut:                     # of 16 keys one has a score of -3 cap with every query, and so no weight: it decides nothing but how the rest is made
        q[..., 0] = 1.0
        k[:, 3::16] = 0.0
        k[:, 3::16, :, 0] = -3.0 * cap * D ** 0.5
    q, k, v, go = [t.bfloat16() for t in (q, k, v, go)]
    slopes = torch.tensor([0.02 / (h + 1) for h in range(H)], device=dev)
    kv_lengths = [nk - (7 * b) % nk for b in range(B)]
    lengths = kv_lengths if nq == nk else [nq] * B
    leaves = [t.requires_grad_(train) for t in (q, k, v)]
    out = F.attention(*leaves, lengths=torch.tensor(lengths, dtype=torch.int32, device=dev), causal=causal, cap=cap, slopes=slopes,
                      kv_lengths=torch.tensor(kv_lengths, dtype=torch.int32, device=dev))
    got = [out.detach(), *(torch.autograd.grad(out, leaves, go) if train else ())]
    want, tol = definition(q, k, v, go, lengths, kv_lengths, causal, cap, slopes)
    for name, a, b, t in zip(("out", "gq", "gk", "gv"), got, want, tol):
        off = (a.cpu().double() - b).abs() - t
        assert bool((off <= 1e-30).all()), (name, float(off.max()), float(b.abs().max()), int((off > 0).sum()))


@pytest.mark.parametrize("cap", [50.0, 256.0, 257.0, 1e4, 1e6, 1e9, 1e28])
@pytest.mark.parametrize("shape", SHAPES)
def test_caps_above_the_scores(tn_gpu, status_ok, shape, cap):
    _check(tn_gpu.core.runtime().device, shape, cap, False)


@pytest.mark.parametrize("cap", [20.0, 1e6])
@pytest.mark.parametrize("shape", SHAPES)
def test_caps_that_cut_some_scores(tn_gpu, status_ok, shape, cap):
    _check(tn_gpu.core.runtime().device, shape, cap, True)
