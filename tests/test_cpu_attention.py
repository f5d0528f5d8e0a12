"""Attention on the CPU path against its definition, and what it refuses."""
import pytest
import torch

from seq_oracle import attention as oracle
from tensornet_b200.ops import functional as F


def bf(*shape, seed=0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).bfloat16()


def ints(*v):
    return torch.tensor(v, dtype=torch.int32)


@pytest.mark.parametrize("kw", [
    dict(),
    dict(causal=True, cap=5.0, slopes=torch.tensor([0.5, 0.25, 0.1, 0.0]), scale=0.7),
    dict(causal=True, prefix=ints(0, 3, 9), lengths=ints(7, 0, 5), kv_lengths=ints(7, 4, 0)),
])
def test_padded(kw):
    q, k, v, go = bf(3, 7, 4, 8), bf(3, 9, 2, 8, seed=1), bf(3, 9, 2, 8, seed=2), bf(3, 7, 4, 8, seed=3)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    out = F.attention(q, k, v, **kw)
    got = [out.detach(), *torch.autograd.grad(out, leaves, go)]
    kw = {{"lengths": "q_rows", "kv_lengths": "kv_rows"}.get(n, n): x for n, x in kw.items()}
    want, bounds = oracle(q, k, v, go=go, **kw)
    for a, b, tol in zip(got, want, bounds):
        assert torch.all((a.double() - b).abs() <= tol + 1e-30)


def test_packed_queries_padded_keys():
    q, k, v = bf(11, 2, 16), bf(3, 6, 1, 16, seed=1), bf(3, 6, 1, 16, seed=2)
    off, ln = ints(1, 4, 4, 9), ints(6, 2, 3)
    out = F.attention(q, k, v, offsets=off, kv_lengths=ln, causal=True)
    want, tol = oracle(q, k, v, off, ln, causal=True)
    assert torch.all((out.double() - want).abs() <= tol + 1e-30)
    assert not out[0].any() and not out[9:].any()


OK = dict(q=bf(2, 3, 4, 8), k=bf(2, 3, 2, 8), v=bf(2, 3, 2, 8))


@pytest.mark.parametrize("kw, text", [
    (dict(q=OK["q"].float()), "q must be bf16"),
    (dict(v=OK["v"].half()), "v must be bf16"),
    (dict(q=OK["q"][0, 0]), "q must be bf16"),
    (dict(k=bf(2, 3, 2, 16)), "alike"),
    (dict(v=bf(2, 4, 2, 8)), "alike"),
    (dict(q=bf(2, 3, 4, 12), k=bf(2, 3, 2, 12), v=bf(2, 3, 2, 12)), "multiple of 8"),
    (dict(q=bf(2, 3, 4, 136), k=bf(2, 3, 2, 136), v=bf(2, 3, 2, 136)), "multiple of 8"),
    (dict(q=bf(2, 3, 3, 8)), "no multiple"),
    (dict(q=bf(3, 3, 4, 8)), "numbers of sequences"),
    (dict(lengths=ints(1, 2, 3)), "numbers of sequences"),
    (dict(lengths=torch.tensor([1, 2])), "lengths must be int32"),
    (dict(offsets=ints(0, 3, 6)), "padded operands go with"),
    (dict(kv_offsets=ints(0, 3, 6)), "padded operands go with kv_"),
    (dict(q=bf(6, 4, 8)), "packed operands go with offsets"),
    (dict(q=bf(6, 4, 8), offsets=ints(0, 6)), "numbers of sequences"),
    (dict(q=bf(6, 4, 8), offsets=ints(0, 3, 6), lengths=ints(3, 3)), "packed operands go with offsets"),
    (dict(k=bf(6, 2, 8), v=bf(6, 2, 8), kv_offsets=torch.zeros(0, dtype=torch.int32)), "kv_offsets must be int32"),
    (dict(prefix=ints(1, 1)), "prefix"),
    (dict(prefix=ints(1, 1, 1), causal=True), "prefix"),
    (dict(slopes=torch.ones(2)), "slopes"),
    (dict(slopes=torch.ones(4, requires_grad=True)), "no gradient"),
    (dict(cap=-1.0), "above zero"),
    (dict(cap=-0.5), "above zero"),
    (dict(cap=float("inf")), "above zero"),
    (dict(scale=0.0), "above zero"),
    (dict(scale=1e-40), "above zero"),
    (dict(scale=1e20, cap=1e-20), "above zero"),
    (dict(cap=float("nan")), "above zero"),
    (dict(scale=float("nan")), "above zero"),
])
def test_refusals(kw, text):
    with pytest.raises(ValueError, match=text):
        F.attention(**{**OK, **kw})


def test_nothing_there():
    assert F.attention(bf(0, 3, 4, 8), bf(0, 3, 2, 8), bf(0, 3, 2, 8)).shape == (0, 3, 4, 8)
    assert not F.attention(OK["q"], bf(2, 0, 2, 8), bf(2, 0, 2, 8)).any()
    assert F.attention(bf(0, 4, 8), bf(0, 2, 8), bf(0, 2, 8), offsets=ints(0), kv_offsets=ints(0)).shape == (0, 4, 8)
