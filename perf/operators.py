"""Operators over behaviour sequences: layer normalisation and attention, forward and backward, what a program has in hand
before a call and the call itself.

* ``norm``    layer normalisation of rows, alone or with the gradients of its input, gain and shift;
* ``attend``  attention within sequences (packed or padded, causal, with a visible prefix, scores capped by a tanh, a bias
  that falls with the distance), with the gradients of its three operands where the case trains, and of few queries against
  long histories, as scoring runs it.

Lengths of sequences are the quantiles of a logarithmic spread, in an order that the seed draws, so that a case's work does
not depend on its seed; the first of eight or more is empty.
"""
import math

import torch

own = False

_DEV = "cuda"
_TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_EPS = 1e-5
_BLOCK = 1 << 28          # scores that the plain form holds at one time


# ------------------------------------------------------------------------------------------------------------- cases
def listed():
    """``norm``: ``rows`` of ``width``.  ``attend``: ``batch`` sequences of up to ``length`` keys; ``shortest``: the shortest of
    them (0: all have ``length``); ``queries``: queries per sequence (0: its keys' tokens); ``packed``: tokens of all sequences
    behind one another with offsets, else ``[batch, length]`` with lengths."""
    return [
        # one request's history between two layers of an encoder: latency is everything
        dict(name="norm request", do="norm", rows=200, width=64, type="bf16", train=False),
        # a training batch of 8192 histories of 50
        dict(name="norm histories", do="norm", rows=409600, width=64, type="fp32", train=True),
        # the input of the headline job's tower, 26 x 16 + 13 columns
        dict(name="norm 429", do="norm", rows=8192, width=429, type="fp32", train=True),
        # the width of the cross network of the largest job, 100 x 64 + 13 columns
        dict(name="norm 6413", do="norm", rows=8192, width=6413, type="bf16", train=True),
        # one request: a candidate against one user's history
        _attend("score one", batch=1, length=200, queries=1, heads=4, kv_heads=4, dim=32),
        # a request batch of 512 users, histories of 20 to 2000
        _attend("score 512", batch=512, length=2000, shortest=20, queries=1, heads=8, kv_heads=8, dim=64, bias=True),
        # the newest token of four lifelong histories, shared key heads
        _attend("score lifelong", batch=4, length=131072, queries=1, heads=16, kv_heads=2, dim=128),
        # scoring with an encoder over fixed histories, every token sees all
        _attend("encode 512", batch=64, length=512, heads=8, kv_heads=8, dim=64),
        # a training batch of short ragged histories, recency bias
        _attend("train histories", batch=4096, length=200, shortest=1, packed=True, heads=4, kv_heads=4, dim=16, causal=True, bias=True,
                train=True),
        # documents of very different lengths in one row of tokens
        _attend("train documents", batch=24, length=8000, shortest=60, packed=True, heads=8, kv_heads=8, dim=64, causal=True, train=True),
        # odd sizes: padded, a visible prefix, capped, biased
        _attend("train prefix odd", batch=6, length=1999, shortest=333, heads=6, kv_heads=3, dim=80, causal=True, prefix=True, cap=30.0,
                bias=True, train=True),
        # long sequences, shared key heads, capped: products are everything
        _attend("train long", batch=1, length=8192, heads=16, kv_heads=4, dim=128, causal=True, cap=50.0, train=True),
    ]


def _attend(name=None, **kw):
    case = dict(do="attend", batch=1, length=1, shortest=0, queries=0, packed=False, heads=1, kv_heads=1, dim=64, causal=False,
                prefix=False, cap=0.0, bias=False, train=False)
    case.update(kw)
    return case if name is None else dict(name=name, **case)


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case: rows of 1 to 8192 columns; sequences of 1 to 8192 tokens, up to 4096 of them; 1 to 16 queries against up to
    131072 keys; 1 to 16 heads of 8 to 128 columns, any sharing of key heads."""
    kind = rng.choice(["norm", "norm", "self", "self", "self", "few"])
    if kind == "norm":
        width = _log(rng, 1, 8192)
        return dict(do="norm", rows=_log(rng, 1, min(409600, 52_000_000 // width)), width=width, type=rng.choice(["fp32", "bf16", "fp16"]),
                    train=rng.random() < 0.6)
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    heads = kv_heads * rng.choice([g for g in (1, 1, 2, 4, 8) if g * kv_heads <= 16])
    dim = rng.choice([8, 16, 24, 32, 40, 64, 64, 80, 96, 128, 128])
    cap = rng.choice([0.0, 0.0, 0.0, 30.0, 50.0])
    if kind == "few":
        length = _log(rng, 1, 131072)
        batch = _log(rng, 1, max(1, min(2048, (1 << 28) // (length * kv_heads * dim))))
        return _attend(batch=batch, length=length, shortest=rng.choice([0, 1, max(1, length // 50)]), queries=rng.choice([1, 1, 1, 2, 5, 16]),
                       heads=heads, kv_heads=kv_heads, dim=dim, cap=cap, bias=rng.random() < 0.4)
    length = _log(rng, 1, 8192)
    batch = _log(rng, 1, max(1, min(4096, 1_000_000_000 // (length * length * heads), 60_000_000 // (length * heads * dim))))
    causal = rng.random() < 0.7
    return _attend(batch=batch, length=length, shortest=rng.choice([0, 1, max(1, length // 30)]), packed=rng.random() < 0.6, heads=heads,
                   kv_heads=kv_heads, dim=dim, causal=causal, prefix=causal and rng.random() < 0.3, cap=cap, bias=rng.random() < 0.4,
                   train=rng.random() < 0.7)


# ------------------------------------------------------------------------------------------------------------- inputs
def _lengths(case):
    """Lengths of the sequences, before the seed orders them."""
    n, lo, hi = case["batch"], case["shortest"], case["length"]
    if not lo:
        return [hi] * n
    out = [int(round(lo * (hi / lo) ** ((i + 0.5) / n))) for i in range(n)]
    out[-1] = hi
    if n >= 8:
        out[0] = 0
    return out


def _slopes(heads):
    """One slope per head, halving every ``heads / 8`` heads."""
    return [2.0 ** (-8.0 * (h + 1) / heads) for h in range(heads)]


class _State:
    pass


def prepare(case, seed):
    s = _State()
    s.case = case
    gen = torch.Generator(device=_DEV).manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=_DEV)

    if case["do"] == "norm":
        rows, width, kind = case["rows"], case["width"], _TYPES[case["type"]]
        # rows as layers hand them over: each with a level and a spread of its own
        s.x = (normal(rows, width) * (0.2 + normal(rows, 1).abs()) + 0.5 * normal(rows, 1)).to(kind)
        s.gamma, s.beta = 1.0 + 0.1 * normal(width), 0.1 * normal(width)
        if case["train"]:
            s.dy = (normal(rows, width) * 1e-2).to(kind)
            s.x, s.gamma, s.beta = s.x.requires_grad_(), s.gamma.requires_grad_(), s.beta.requires_grad_()
        return s
    H, G, D, B, T = case["heads"], case["kv_heads"], case["dim"], case["batch"], case["length"]
    lengths = torch.tensor(_lengths(case), dtype=torch.int64)
    order = torch.randperm(B, generator=torch.Generator().manual_seed(seed))
    lengths = lengths[order]
    s.host_lengths = lengths.tolist()
    s.lengths = lengths.to(torch.int32).to(_DEV)
    s.offsets = torch.cat([torch.zeros(1, dtype=torch.int64), lengths.cumsum(0)]).to(torch.int32).to(_DEV) if case["packed"] else None
    lead = (int(lengths.sum()),) if case["packed"] else (B, T)

    def heads_of(n_tokens, n_heads):      # side by side in one product's padded rows
        cols = sum(n_heads) * D
        rows = (normal(n_tokens, (cols + 8) // 8 * 8) * 1.2).to(torch.bfloat16)
        parts = rows[:, :cols].split([h * D for h in n_heads], dim=1)
        return [p.unflatten(1, (h, D)) for p, h in zip(parts, n_heads)]

    if case["queries"]:
        (s.q,) = heads_of(B * case["queries"], [H])
        s.k, s.v = heads_of(math.prod(lead), [G, G])
        s.q = s.q.unflatten(0, (B, case["queries"]))
    else:
        s.q, s.k, s.v = heads_of(math.prod(lead), [H, G, G])
        s.q = s.q.unflatten(0, lead)
    s.k, s.v = s.k.unflatten(0, lead), s.v.unflatten(0, lead)
    s.prefix = (s.lengths * torch.rand(B, generator=gen, device=_DEV)).to(torch.int32) if case["prefix"] else None
    s.slopes = torch.tensor(_slopes(H), dtype=torch.float32, device=_DEV) if case["bias"] else None
    s.scale = 1.0 / math.sqrt(D)
    s.plan = [(torch.tensor(seqs, device=_DEV), longest) for seqs, longest in _plan(case, s.host_lengths)]
    if case["train"]:
        s.do = (normal(*s.q.shape) * 1e-2).to(torch.bfloat16)
        s.q, s.k, s.v = s.q.requires_grad_(), s.k.requires_grad_(), s.v.requires_grad_()
    return s


def _plan(case, lengths):
    """What the plain form has side by side: sequences of like lengths, as many as :data:`_BLOCK` scores allow."""
    order = sorted((i for i in range(len(lengths)) if lengths[i]), key=lambda i: -lengths[i])
    out = []
    while order:
        longest = lengths[order[0]]
        n = max(1, min(len(order), _BLOCK // (case["heads"] * (case["queries"] or longest) * longest)))
        while lengths[order[n - 1]] * 2 < longest:
            n -= 1
        out.append((order[:n], longest))
        order = order[n:]
    return out


# ------------------------------------------------------------------------------------------------------------- passes
def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return _plain_norm(state) if state.case["do"] == "norm" else _plain_attend(state)


def _run_own(s):
    from tensornet_b200.ops import functional as F

    case = s.case
    if case["do"] == "norm":
        if not case["train"]:
            return F.layer_norm(s.x, s.gamma, s.beta, eps=_EPS)
        y = F.layer_norm(s.x, s.gamma, s.beta, eps=_EPS)
        return [y.detach(), *torch.autograd.grad(y, (s.x, s.gamma, s.beta), s.dy)]
    own_keys = case["queries"] > 0
    out = F.attention(s.q, s.k, s.v, lengths=None if case["packed"] or own_keys else s.lengths, kv_lengths=None if case["packed"] else s.lengths,
                      offsets=s.offsets, kv_offsets=s.offsets, causal=case["causal"], prefix=s.prefix, cap=case["cap"] or None,
                      slopes=s.slopes, scale=s.scale)
    if not case["train"]:
        return out
    return [out.detach(), *torch.autograd.grad(out, (s.q, s.k, s.v), s.do)]


# ------------------------------------------------------------------------------------------------------------- plain forms
def _plain_norm(s):
    x = s.x.float()
    mean = x.mean(dim=1, keepdim=True)
    rstd = 1.0 / torch.sqrt(((x - mean) ** 2).mean(dim=1, keepdim=True) + _EPS)
    xhat = (x - mean) * rstd
    y = (xhat * s.gamma + s.beta).to(s.x.dtype)
    if not s.case["train"]:
        return y
    dy = s.dy.float()
    dgamma = (dy * xhat).sum(dim=0, dtype=torch.float64).float()
    dbeta = dy.sum(dim=0, dtype=torch.float64).float()
    g = dy * s.gamma
    dx = rstd * (g - g.mean(dim=1, keepdim=True) - xhat * (g * xhat).mean(dim=1, keepdim=True))
    return [y, dx.to(s.x.dtype), dgamma, dbeta]


def _plain_attend(s):
    """Sequences of like lengths side by side, padded; a row behind the last takes what padding leaves."""
    case = s.case
    H, G, D, B = case["heads"], case["kv_heads"], case["dim"], case["batch"]
    R, few, train = H // G, case["queries"], case["train"]
    begin = s.offsets[:-1].long() if case["packed"] else torch.arange(B, device=_DEV) * case["length"]
    q, k, v = [t.reshape(-1, *t.shape[-2:]) for t in (s.q, s.k, s.v)]

    def result(like):
        return torch.zeros((like.shape[0] + 1, *like.shape[1:]), dtype=torch.bfloat16, device=_DEV)

    out = result(q)
    if train:
        do = s.do.reshape(-1, H, D)
        dq, dk, dv = result(q), result(k), result(v)
    for seqs, Lk in s.plan:
        n, Lq = seqs.numel(), few or Lk
        lens = s.lengths[seqs].long()
        kpos, qpos = torch.arange(Lk, device=_DEV), torch.arange(Lq, device=_DEV)
        kthere = kpos < lens[:, None]                                            # [n, Lk]
        krow = begin[seqs][:, None] + kpos
        kinto, krow = torch.where(kthere, krow, k.shape[0]), torch.where(kthere, krow, 0)
        if few:
            qlens, qthere = torch.full_like(lens, few), torch.ones((n, Lq), dtype=torch.bool, device=_DEV)
            qrow = qinto = seqs[:, None] * few + qpos
        else:
            qlens, qthere, qrow, qinto = lens, kthere, krow, kinto
        place = qpos + (lens - qlens)[:, None]                                   # of a query among the keys, [n, Lq]
        mask = (kthere[:, None, :] & qthere[:, :, None])
        if case["causal"]:
            seen = kpos <= place[:, :, None]
            if s.prefix is not None:
                seen |= kpos < s.prefix[seqs][:, None, None]
            mask = mask & seen
        mask = mask[:, None, None]                                               # [n, 1, 1, Lq, Lk]
        away = (place[:, :, None] - kpos).abs().float()[:, None, None] if s.slopes is not None else None
        step = max(1, min(G, _BLOCK // (n * R * Lq * Lk)))
        for g0 in range(0, G, step):
            g1 = min(G, g0 + step)
            hs = slice(g0 * R, g1 * R)
            qf = q[qrow, hs].float().unflatten(2, (g1 - g0, R)).permute(0, 2, 3, 1, 4)     # [n, g, R, Lq, D]
            kf = k[krow, g0:g1].float().permute(0, 2, 1, 3)[:, :, None]                    # [n, g, 1, Lk, D]
            vf = v[krow, g0:g1].float().permute(0, 2, 1, 3)[:, :, None]
            sc = qf @ kf.transpose(-1, -2) * s.scale
            th = None
            if case["cap"]:
                th = torch.tanh(sc / case["cap"])
                sc = case["cap"] * th
            if away is not None:
                sc = sc - s.slopes[hs].view(1, g1 - g0, R, 1, 1) * away
            sc = sc.masked_fill(~mask, -math.inf)
            top = sc.amax(dim=-1, keepdim=True)
            p = torch.exp(sc - torch.where(top == -math.inf, 0.0, top))
            p = p / p.sum(dim=-1, keepdim=True).clamp(min=1e-30)
            del sc
            o = p @ vf
            out[qinto, hs] = o.permute(0, 3, 1, 2, 4).flatten(2, 3).to(torch.bfloat16)
            if not train:
                continue
            dof = do[qrow, hs].float().unflatten(2, (g1 - g0, R)).permute(0, 2, 3, 1, 4)
            dof = dof * qthere[:, None, None, :, None]
            dvf = (p.transpose(-1, -2) @ dof).sum(dim=2)                                    # [n, g, Lk, D]
            ds = p * (dof @ vf.transpose(-1, -2) - (o * dof).sum(dim=-1, keepdim=True))
            if th is not None:
                ds = ds * (1.0 - th * th)
            ds = ds * s.scale
            dqf = ds @ kf
            dkf = (ds.transpose(-1, -2) @ qf).sum(dim=2)
            dq[qinto, hs] = dqf.permute(0, 3, 1, 2, 4).flatten(2, 3).to(torch.bfloat16)
            dk[kinto, g0:g1] = dkf.transpose(1, 2).to(torch.bfloat16)
            dv[kinto, g0:g1] = dvf.transpose(1, 2).to(torch.bfloat16)
    out = out[:-1].view(s.q.shape)
    return [out, dq[:-1].view(s.q.shape), dk[:-1].view(s.k.shape), dv[:-1].view(s.v.shape)] if train else out


# ------------------------------------------------------------------------------------------------------------- definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return _exact_norm(s) if case["do"] == "norm" else _exact_attend(s)


def _exact_norm(s):
    # in pieces of rows: the widest cases have 52 M elements
    train, n = s.case["train"], s.x.shape[0]
    gamma, beta = [t.detach().double().requires_grad_(train) for t in (s.gamma, s.beta)]
    dgamma, dbeta = torch.zeros_like(gamma), torch.zeros_like(beta)
    ys, dxs = [], []
    for lo in range(0, n, 1 << 16):
        x = s.x.detach()[lo:lo + (1 << 16)].double().requires_grad_(train)
        centred = x - x.sum(dim=1, keepdim=True) / x.shape[1]
        var = (centred * centred).sum(dim=1, keepdim=True) / x.shape[1]
        y = gamma * centred / torch.sqrt(var + _EPS) + beta
        ys.append(y.detach())
        if train:
            dx, dg, db = torch.autograd.grad(y, (x, gamma, beta), s.dy[lo:lo + (1 << 16)].double())
            dxs.append(dx)
            dgamma, dbeta = dgamma.detach() + dg, dbeta.detach() + db
    if not train:
        return torch.cat(ys)
    return [torch.cat(ys), torch.cat(dxs), dgamma.detach(), dbeta.detach()]


def _exact_attend(s):
    """Sequence by sequence and key head by key head."""
    case = s.case
    G, R, few, train = case["kv_heads"], case["heads"] // case["kv_heads"], case["queries"], case["train"]
    out = torch.zeros(s.q.shape, dtype=torch.float64, device=_DEV)
    grads = [torch.zeros(t.shape, dtype=torch.float64, device=_DEV) for t in (s.q, s.k, s.v)] if train else []
    start = 0
    for b, L in enumerate(s.host_lengths):
        where_k = slice(start, start + L) if case["packed"] else (b, slice(0, L))
        where_q = (b, slice(0, few)) if few else where_k
        start += L
        if L == 0:
            continue
        for g in range(G):
            q = s.q.detach()[where_q][:, g * R:(g + 1) * R].transpose(0, 1).double().requires_grad_(train)      # [R, Lq, D]
            k, v = [t.detach()[where_k][:, g].double().requires_grad_(train) for t in (s.k, s.v)]
            score = torch.einsum("rid,jd->rij", q, k) * s.scale
            if case["cap"]:
                score = case["cap"] * torch.tanh(score / case["cap"])
            i = torch.arange(L - q.shape[1], L, device=_DEV).view(1, -1, 1)
            j = torch.arange(L, device=_DEV).view(1, 1, -1)
            if s.slopes is not None:
                score = score - s.slopes[g * R:(g + 1) * R].double().view(R, 1, 1) * (i - j).abs()
            if case["causal"]:
                hidden = j > i
                if s.prefix is not None:
                    hidden = hidden & (j >= s.prefix[b])
                score = score.masked_fill(hidden, -math.inf)
            o = torch.einsum("rij,jd->rid", torch.softmax(score, dim=-1), v)
            out[where_q][:, g * R:(g + 1) * R] = o.detach().transpose(0, 1)
            if train:
                do = s.do[where_q][:, g * R:(g + 1) * R].transpose(0, 1).double()
                dq, dk, dv = torch.autograd.grad(o, (q, k, v), do)
                grads[0][where_q][:, g * R:(g + 1) * R] = dq.transpose(0, 1)
                grads[1][where_k][:, g] = dk
                grads[2][where_k][:, g] = dv
            del score, o
    return [out, *grads] if train else out


# ------------------------------------------------------------------------------------------------------------- work
def work(case):
    """What sequences hold of each operand read and each result written once, padding (zeros) included.  Flops of ``attend``: two products of the pairs that see one another forward,
    five backward (the prefix, whose length the seed draws, is counted at half of its sequence)."""
    if case["do"] == "norm":
        size = 4 if case["type"] == "fp32" else 2
        n, w = case["rows"] * case["width"], case["width"]
        if not case["train"]:
            return {"bytes": 2 * n * size + 8 * w, "flops": 8 * n}
        return {"bytes": 4 * n * size + 16 * w, "flops": 20 * n}
    H, G, D, few = case["heads"], case["kv_heads"], case["dim"], case["queries"]
    lens = _lengths(case)
    keys = sum(lens)
    queries = few * case["batch"] if few else keys
    pairs = 0.0
    for L in lens:
        Lq = few or L
        full = float(Lq) * L
        if not case["causal"]:
            pairs += full
        else:
            hidden = L * (L - 1) / 2.0
            pairs += full - hidden * (0.75 if case["prefix"] else 1.0)
    places = keys if case["packed"] else case["batch"] * case["length"]          # of tokens, padding among them
    result = 2 * D * H * (queries if few else places)
    operands = 2 * D * (H * queries + 2 * G * keys)
    if not case["train"]:
        return {"bytes": operands + result, "flops": 4 * pairs * H * D}
    grads = result + 2 * D * 2 * G * places
    return {"bytes": operands + result + 2 * D * H * queries + grads, "flops": 14 * pairs * H * D}
