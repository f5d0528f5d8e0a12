"""Attention kernels against the definition in 64 bits; ``seq_oracle.attention`` derives the tolerances."""
import pytest
import torch

from seq_oracle import attention as oracle

pytestmark = pytest.mark.gpu


def ints(dev, *v):
    return torch.tensor(v, dtype=torch.int32, device=dev)


def normal(dev, *shape, seed=0, by=1.0):
    return (torch.randn(shape, generator=torch.Generator(device=dev).manual_seed(seed), device=dev) * by).bfloat16()


def check(q, k, v, go=None, lengths=None, kv_lengths=None, offsets=None, kv_offsets=None, leaves=None, **kw):
    from tensornet_b200.ops import functional as F

    train = go is not None
    q, k, v = [t.detach().requires_grad_(train) for t in (q, k, v)]
    out = F.attention(q, k, v, lengths=lengths, kv_lengths=kv_lengths, offsets=offsets, kv_offsets=kv_offsets, **kw)
    got = [out.detach(), *(torch.autograd.grad(out, (q, k, v), go) if train else ())]
    want, tol = oracle(q, k, v, offsets if q.dim() == 3 else lengths, kv_offsets if k.dim() == 3 else kv_lengths, go=go, **kw)
    if not train:
        want, tol = [want], [tol]
    for name, a, b, t in zip(("out", "gq", "gk", "gv"), got, want, tol):
        off = (a.cpu().double() - b).abs() - t
        assert not bool(a.isnan().any()), name
        assert bool((off <= 1e-30).all()), (name, float(off.max()), float(b.abs().max()), int((off > 0).sum()))
    return got


def slopes_of(dev, H):
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / H) for h in range(H)], device=dev)


LENGTHS = [1, 2, 7, 31, 63, 64, 65, 127, 128, 129, 255, 256, 257, 300, 511, 640]


@pytest.mark.parametrize("T", LENGTHS)
@pytest.mark.parametrize("D", [16, 64, 128])
def test_self_causal(tn_gpu, status_ok, T, D):
    dev = tn_gpu.core.runtime().device
    q, k, v, go = [normal(dev, 2, T, 2, D, seed=s) for s in range(4)]
    check(q, k, v, go, causal=True)


@pytest.mark.parametrize("D", [8, 24, 32, 40, 48, 56, 72, 80, 96, 104, 120])
def test_columns(tn_gpu, status_ok, D):
    dev = tn_gpu.core.runtime().device
    q, go = [normal(dev, 1, 200, 4, D, seed=s) for s in range(2)]
    k, v = [normal(dev, 1, 200, 2, D, seed=s) for s in (2, 3)]
    check(q, k, v, go)


@pytest.mark.parametrize("H, G", [(1, 1), (3, 1), (4, 2), (6, 3), (16, 2), (5, 5)])
def test_shared_key_heads(tn_gpu, status_ok, H, G):
    dev = tn_gpu.core.runtime().device
    q, go = [normal(dev, 2, 150, H, 32, seed=s) for s in range(2)]
    k, v = [normal(dev, 2, 150, G, 32, seed=s) for s in (2, 3)]
    check(q, k, v, go, causal=True, slopes=slopes_of(dev, H))


@pytest.mark.parametrize("nq, nk", [(1, 1), (1, 500), (3, 129), (5, 4), (130, 7), (128, 128), (200, 333), (333, 200), (16, 1000), (17, 70)])
@pytest.mark.parametrize("causal", [False, True])
def test_cross(tn_gpu, status_ok, nq, nk, causal):
    """Queries at the end of their keys; where there are more queries than keys the first ones see nothing."""
    dev = tn_gpu.core.runtime().device
    q, go = [normal(dev, 3, nq, 4, 64, seed=s) for s in range(2)]
    k, v = [normal(dev, 3, nk, 2, 64, seed=s) for s in (2, 3)]
    got = check(q, k, v, go, causal=causal, slopes=slopes_of(dev, 4), cap=20.0)
    if causal and nq > nk:
        assert not got[0][:, :nq - nk].any() and not got[1][:, :nq - nk].any()
    check(q, k, v, causal=causal)


@pytest.mark.parametrize("cap", [None, 1.5, 30.0])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("mask", ["full", "causal", "prefix"])
def test_scores(tn_gpu, status_ok, cap, bias, mask):
    dev = tn_gpu.core.runtime().device
    q, k, v, go = [normal(dev, 3, 300, 2, 80, seed=s, by=1.5) for s in range(4)]
    prefix = ints(dev, 0, 140, 1000) if mask == "prefix" else None
    check(q, k, v, go, causal=mask != "full", prefix=prefix, cap=cap, slopes=slopes_of(dev, 2) if bias else None, scale=0.2,
          lengths=ints(dev, 300, 251, 200), kv_lengths=ints(dev, 300, 251, 200))


def test_padding_is_not_looked_at_and_comes_back_zero(tn_gpu, status_ok):
    """Rows behind a length hold NaN, infinities and the type's lowest value."""
    dev = tn_gpu.core.runtime().device
    ql, kl = [300, 0, 5, 129, 128], [299, 17, 0, 260, 128]
    q, go = [normal(dev, 5, 300, 4, 64, seed=s) for s in range(2)]
    k, v = [normal(dev, 5, 300, 2, 64, seed=s) for s in (2, 3)]
    dirt = torch.tensor([float("nan"), float("inf"), float("-inf"), torch.finfo(torch.bfloat16).min], device=dev).bfloat16()
    for t, ln in ((q, ql), (go, ql), (k, kl), (v, kl)):
        for b, n in enumerate(ln):
            t[b, n:] = dirt[torch.arange(300 - n, device=dev) % 4].view(-1, 1, 1)
    for causal in (False, True):
        got = check(q, k, v, go, lengths=ints(dev, *ql), kv_lengths=ints(dev, *kl), causal=causal, slopes=slopes_of(dev, 4))
        for t, ln in zip(got, (ql, ql, kl, kl)):
            for b, n in enumerate(ln):
                assert not t[b, n:].any()


@pytest.mark.parametrize("D, H, G", [(16, 4, 4), (64, 2, 1), (128, 2, 2)])
def test_packed(tn_gpu, status_ok, D, H, G):
    """Ragged sequences one after another, some empty, one row or exactly a tile, with dirt in front of the first and behind the last."""
    dev = tn_gpu.core.runtime().device
    lens = [1, 0, 128, 3, 256, 0, 0, 127, 129, 50, 383, 1]
    off = [5]
    for n in lens:
        off.append(off[-1] + n)
    N = off[-1] + 140
    q, go = [normal(dev, N, H, D, seed=s) for s in range(2)]
    k, v = [normal(dev, N, G, D, seed=s) for s in (2, 3)]
    for t in (q, go, k, v):
        t[:5] = float("nan")
        t[off[-1]:] = float("inf")
    o = ints(dev, *off)
    for kw in (dict(causal=True), dict(causal=True, cap=10.0, slopes=slopes_of(dev, H), prefix=ints(dev, *[n // 3 for n in lens])), dict()):
        got = check(q, k, v, go, offsets=o, kv_offsets=o, **kw)
        for t in got:
            assert not t[:5].any() and not t[off[-1]:].any()


def test_packed_with_padded_and_offsets_beyond_the_rows(tn_gpu, status_ok):
    dev = tn_gpu.core.runtime().device
    q, go = [normal(dev, 3, 9, 2, 32, seed=s) for s in range(2)]
    k, v = [normal(dev, 400, 2, 32, seed=s) for s in (2, 3)]
    check(q, k, v, go, lengths=ints(dev, 9, 1, 4), kv_offsets=ints(dev, 0, 200, 230, 400), causal=True)
    check(q, k, v, go, lengths=ints(dev, 9, -3, 400), kv_offsets=ints(dev, -7, 200, 230, 9999))
    check(k, q, q, v, offsets=ints(dev, 0, 200, 230, 400), kv_lengths=ints(dev, 9, 0, 4))


def test_very_ragged_batches(tn_gpu, status_ok):
    dev = tn_gpu.core.runtime().device
    g = torch.Generator().manual_seed(5)
    lens = torch.randint(0, 60, (300,), generator=g)
    lens[17] = 1000
    off = torch.cat([torch.zeros(1, dtype=torch.int64), lens.cumsum(0)]).int().to(dev)
    N = int(lens.sum())
    q, k, v, go = [normal(dev, N, 2, 16, seed=s) for s in range(4)]
    check(q, k, v, go, offsets=off, kv_offsets=off, causal=True, slopes=slopes_of(dev, 2))


@pytest.mark.parametrize("form", ["fused projection", "heads first", "odd row", "off a boundary", "columns apart", "broadcast heads",
                                  "broadcast gradient"])
def test_layouts(tn_gpu, status_ok, form):
    dev = tn_gpu.core.runtime().device
    B, T, H, D = 2, 140, 4, 32
    q, k, v, go = [normal(dev, B, T, H, D, seed=s) for s in range(4)]
    if form == "fused projection":
        rows = normal(dev, B * T, 3 * H * D + 8)
        q, k, v = [rows[:, i * H * D:(i + 1) * H * D].unflatten(0, (B, T)).unflatten(2, (H, D)) for i in range(3)]
    elif form == "heads first":
        q, k, v, go = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v, go)]
    elif form == "odd row":
        q, k, v, go = [normal(dev, B, T, H * D + 3, seed=s)[..., :H * D].unflatten(2, (H, D)) for s in range(4)]
    elif form == "off a boundary":
        q, k, v, go = [normal(dev, B * T * H * D + 1, seed=s)[1:].view(B, T, H, D) for s in range(4)]
    elif form == "columns apart":
        q, k, v, go = [normal(dev, B, T, H, 2 * D, seed=s)[..., ::2] for s in range(4)]
    elif form == "broadcast heads":
        k, v = [normal(dev, B, T, 1, D, seed=s).expand(B, T, H, D) for s in (2, 3)]
    else:
        go = normal(dev, 1, 1, 1, D).expand(B, T, H, D)
    check(q, k, v, go, causal=True)


def test_long_rows_of_few_queries(tn_gpu, status_ok):
    dev = tn_gpu.core.runtime().device
    for nq, H, G, D, nk in ((1, 8, 1, 128, 20011), (1, 2, 2, 64, 33000), (4, 4, 2, 32, 9000), (16, 1, 1, 16, 12345), (2, 16, 1, 64, 5000)):
        q = normal(dev, 2, nq, H, D)
        k, v = normal(dev, 2, nk, G, D, seed=1), normal(dev, 2, nk, G, D, seed=2)
        check(q, k, v, kv_lengths=ints(dev, nk, nk // 3), causal=True, slopes=slopes_of(dev, H) * 0.01, cap=30.0)


def test_large_scores(tn_gpu, status_ok):
    """Weights that are all but one on a single key, and maxima that grow from tile to tile."""
    dev = tn_gpu.core.runtime().device
    T = 700
    q, k, v, go = [normal(dev, 1, T, 2, 64, seed=s) for s in range(4)]
    ramp = torch.linspace(0.1, 8.0, T, device=dev).view(1, T, 1, 1)
    check(q * 4, (k * ramp).bfloat16(), v, go, causal=True)
    check((q.abs() * 3).bfloat16(), (k.abs() * ramp).bfloat16(), v, go)
    check((q.abs() * 3).bfloat16(), (k.abs() * ramp.flip(1)).bfloat16(), v, go)
    check((-q.abs() * 3).bfloat16(), (k.abs() * ramp).bfloat16(), v, go, causal=True)


def test_gradients_are_those_of_differences(tn_gpu, status_ok):
    """The change of a weighted sum of the results along a direction, from the definition in 64 bits."""
    from tensornet_b200.ops import functional as F

    dev = tn_gpu.core.runtime().device
    T, H, D = 70, 2, 16
    q, k, v, go = [normal(dev, 1, T, H, D, seed=s) for s in range(4)]
    kw = dict(causal=True, cap=8.0, slopes=slopes_of(dev, H))
    leaves = [t.requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(F.attention(*leaves, **kw), leaves, go)
    for i in range(3):
        step = torch.randn(leaves[i].shape, generator=torch.Generator().manual_seed(i), dtype=torch.float64)
        ends = []
        for sign in (1, -1):
            moved = [t.detach().cpu().double() for t in leaves]
            moved[i] = moved[i] + sign * 1e-5 * step
            ends.append((oracle(*moved, **kw)[0] * go.cpu().double()).sum())
        change = (ends[0] - ends[1]) / 2e-5
        _, bounds = oracle(q, k, v, go=go, **kw)
        assert abs((grads[i].cpu().double() * step).sum() - change) <= (bounds[i + 1] * step.abs()).sum() + 1e-6 * abs(change)


def test_one_tensor_as_all_operands(tn_gpu, status_ok):
    from tensornet_b200.ops import functional as F

    dev = tn_gpu.core.runtime().device
    x, go = normal(dev, 2, 90, 2, 32).requires_grad_(), normal(dev, 2, 90, 2, 32, seed=1)
    (g,) = torch.autograd.grad(F.attention(x, x, x, causal=True), x, go)
    want, tol = oracle(x, x, x, causal=True, go=go)
    total, bound = sum(want[1:]), sum(tol[1:])
    assert torch.all((g.cpu().double() - total).abs() <= 2 * bound + 2 * 2.0 ** -8 * sum(t.abs() for t in want[1:]))


def test_operands_without_gradients(tn_gpu, status_ok):
    from tensornet_b200.ops import functional as F

    dev = tn_gpu.core.runtime().device
    q, k, v, go = [normal(dev, 1, 40, 2, 16, seed=s) for s in range(4)]
    v.requires_grad_()
    want, tol = oracle(q, k, v, go=go)
    (gv,) = torch.autograd.grad(F.attention(q, k, v), v, go)
    assert torch.all((gv.cpu().double() - want[3]).abs() <= tol[3])
    with torch.no_grad():
        assert F.attention(q, k, v).grad_fn is None


def test_same_bits_each_time_on_other_streams_and_from_graphs(tn_gpu, status_ok):
    from tensornet_b200.ops import functional as F

    dev = tn_gpu.core.runtime().device
    off = ints(dev, 0, 300, 310, 600)
    q, go = [normal(dev, 600, 4, 64, seed=s) for s in range(2)]
    k, v = [normal(dev, 600, 2, 64, seed=s) for s in (2, 3)]
    few, long_k, long_v = normal(dev, 2, 1, 4, 64), normal(dev, 2, 5000, 2, 64, seed=5), normal(dev, 2, 5000, 2, 64, seed=6)
    q, k, v = [t.requires_grad_() for t in (q, k, v)]

    def go_once():
        out = F.attention(q, k, v, offsets=off, kv_offsets=off, causal=True)
        return [out.detach(), *torch.autograd.grad(out, (q, k, v), go), F.attention(few, long_k, long_v)]

    want = go_once()
    assert all(torch.equal(a, b) for a, b in zip(go_once(), want))
    streams, got = [torch.cuda.Stream(dev) for _ in range(3)], []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream(dev))
        with torch.cuda.stream(s):
            got.append(go_once())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g in got for a, b in zip(g, want))
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = go_once()
        graphs.append((graph, out))
    off.copy_(ints(dev, 0, 10, 10, 599))          # replays read what the offsets are then
    for (graph, out), s in zip(graphs, streams):
        s.wait_stream(torch.cuda.current_stream(dev))
        with torch.cuda.stream(s):
            graph.replay()
    torch.cuda.synchronize()
    want = go_once()
    assert all(torch.equal(a, b) for _, out in graphs for a, b in zip(out, want))


def test_nothing_there(tn_gpu, status_ok):
    from tensornet_b200.ops import functional as F

    dev = tn_gpu.core.runtime().device
    e = normal(dev, 2, 0, 2, 16).requires_grad_()
    q = normal(dev, 2, 3, 2, 16).requires_grad_()
    out = F.attention(q, e, e)
    assert not out.any()
    gq, ge = torch.autograd.grad(out.sum(), (q, e))
    assert not gq.any() and ge.shape == e.shape
    assert F.attention(e, q, q).shape == e.shape
    p = normal(dev, 0, 2, 16)
    assert F.attention(p, p, p, offsets=ints(dev, 0), kv_offsets=ints(dev, 0)).shape == p.shape
    n = normal(dev, 7, 2, 16)
    assert not F.attention(n, n, n, offsets=ints(dev, 3), kv_offsets=ints(dev, 3)).any()
    z = ints(dev, 0, 0, 0)
    assert not F.attention(n, n, n, offsets=z, kv_offsets=z, causal=True).any()


def test_second_derivatives_are_refused(tn_gpu, status_ok):
    from tensornet_b200.ops import functional as F

    q = normal(tn_gpu.core.runtime().device, 1, 5, 1, 8).requires_grad_()
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(F.attention(q, q, q).float().sum(), q, create_graph=True)


@pytest.mark.parametrize("D", [16, 64, 80])
@pytest.mark.parametrize("cap", [None, 5.0])
@pytest.mark.parametrize("L, causal", [(50, True), (290, True), (290, False), (1100, False)])
def test_bits_do_not_depend_on_what_lies_behind_a_sequence(tn_gpu, status_ok, D, cap, L, causal):
    """Nor on what another call has left on the chip: one with far larger scores runs between two that have to agree."""
    from tensornet_b200.ops import functional as F

    dev = tn_gpu.core.runtime().device
    n = ints(dev, L, L - 13, 1, 0, L // 2 + 5)
    q, k, v, go = [normal(dev, 5, L + 30, 4, D, seed=s) for s in range(4)]
    big = normal(dev, 3, 700, 4, D, seed=9, by=300.0)
    behind = torch.arange(L + 30, device=dev) >= n[:, None]

    def once(fill):
        a = [t.masked_fill(behind[:, :, None, None], fill).requires_grad_() for t in (q, k, v)]
        out = F.attention(*a, lengths=n, kv_lengths=n, causal=causal, cap=cap, slopes=slopes_of(dev, 4))
        return [out.detach(), *torch.autograd.grad(out, a, go.masked_fill(behind[:, :, None, None], fill))]

    want = once(0.0)
    for fill in (0.0, 1.0, 200.0, float("inf"), float("nan"), 0.0):
        x = big.requires_grad_()
        F.attention(x, x, x, cap=cap).sum().backward()
        assert all(torch.equal(a, b) for a, b in zip(once(fill), want)), fill


def test_forward_mode_derivatives_are_refused(tn_gpu, status_ok):
    import torch.autograd.forward_ad as fwd

    from tensornet_b200.ops import functional as F

    dev = tn_gpu.core.runtime().device
    q, rows = normal(dev, 1, 20, 2, 16), normal(dev, 5, 16)
    with fwd.dual_level():
        for call in (lambda: F.attention(fwd.make_dual(q, q), q, q), lambda: F.layer_norm(fwd.make_dual(rows, rows))):
            with pytest.raises((RuntimeError, NotImplementedError)):
                call()
            with torch.no_grad(), pytest.raises((RuntimeError, NotImplementedError)):
                call()


@pytest.mark.parametrize("D", [16, 32, 56, 128])
@pytest.mark.parametrize("G, lens", [(1, [40001]), (2, [70000, 1]), (1, [0, 38000, 40, 70000])])
def test_one_query_and_keys_in_many_splits(tn_gpu, status_ok, D, G, lens):
    dev = tn_gpu.core.runtime().device
    B, T = len(lens), max(lens)
    q, k, v = normal(dev, B, 1, 2 * G, D), normal(dev, B, T, G, D, seed=1), normal(dev, B, T, G, D, seed=2)
    check(q, k, v, kv_lengths=ints(dev, *lens), slopes=slopes_of(dev, 2 * G) * 1e-3)


@pytest.mark.parametrize("D, H, G", [(16, 4, 4), (64, 8, 4), (128, 4, 4)])
def test_many_histories_some_of_them_long(tn_gpu, status_ok, D, H, G):
    """A warp per history and key head, or per 512 keys of it."""
    dev = tn_gpu.core.runtime().device
    lens = [(b * 37) % 1200 for b in range(300)]
    lens[:6] = [0, 1, 512, 513, 1024, 1200]
    q = normal(dev, 300, 2, H, D)
    k, v = normal(dev, 300, 1200, G, D, seed=1), normal(dev, 300, 1200, G, D, seed=2)
    check(q, k, v, kv_lengths=ints(dev, *lens), causal=True, slopes=slopes_of(dev, H) * 0.01)
    go = normal(dev, 300, 2, H, D, seed=3)
    check(q[:, :1], k, v, go[:, :1], kv_lengths=ints(dev, *lens))
