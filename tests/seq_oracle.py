"""Attention within sequences from its definition, in 64 bits, sequence by sequence."""
import math

import torch


def spans(t, rows, B):
    """Per sequence the index of its rows in ``t`` (padded or packed)."""
    out = []
    for b in range(B):
        if t.dim() == 3:
            lo = min(max(int(rows[b]), 0), t.shape[0])
            out.append(slice(lo, min(max(int(rows[b + 1]), lo), t.shape[0])))
        else:
            out.append((b, slice(0, t.shape[1] if rows is None else min(max(int(rows[b]), 0), t.shape[1]))))
    return out


def attention(q, k, v, q_rows=None, kv_rows=None, causal=False, prefix=None, cap=None, slopes=None, scale=None, go=None):
    """``(out, bound)`` or with ``go`` ``([out, gq, gk, gv], bounds)``, on the CPU in fp64.

    ``bounds`` are how far kernels may be off that multiply bf16 operands, with the weights ``p`` and the score gradients ``ds``
    rounded to bf16, the forward result that the backward pass reads rounded too, and fp32 in between.  With u = 2^-8, half a
    step of bf16 relative to the value:

    * out = sum p v: rounding p costs u sum p |v|; rounding the result u |out|.
    * gv likewise from p and go.
    * delta = sum go out is off by u sum |go| |out| from the rounded result; ds = p (dp - delta) dscore is off by that, times p dscore,
      and by u |ds| from its rounding; gq = sum ds k and gk = sum ds q carry those.

    fp32 sums of up to 2^16 terms in blocks, and scores off by 2^-18 of the products' magnitude, are covered by a further
    ``f`` = 2^-12 of each sum of magnitudes and of each weight."""
    u, f = 2.0 ** -8, 2.0 ** -12
    q64, k64, v64 = [t.detach().cpu().double() for t in (q, k, v)]
    H, D = q.shape[-2:]
    G = k.shape[-2]
    R = H // G
    scale = D ** -0.5 if scale is None else scale
    B = len(q_rows) - 1 if q.dim() == 3 else q.shape[0]
    out, bo = torch.zeros_like(q64), torch.zeros_like(q64)
    train = go is not None
    if train:
        g64 = go.detach().cpu().double()
        gq, gk, gv = [torch.zeros_like(t) for t in (q64, k64, v64)]
        bq, bk, bv = [torch.zeros_like(t) for t in (q64, k64, v64)]
    for b, (wq, wk) in enumerate(zip(spans(q, q_rows, B), spans(k, kv_rows, B))):
        qb = q64[wq].transpose(0, 1)                                            # [H, nq, D]
        kb, vb = [t[wk].transpose(0, 1).repeat_interleave(R, dim=0) for t in (k64, v64)]
        nq, nk = qb.shape[1], kb.shape[1]
        if nq == 0 or nk == 0:
            continue
        x = qb @ kb.transpose(1, 2) * scale
        size = qb.abs() @ kb.abs().transpose(1, 2) * scale
        th = torch.zeros_like(x)
        if cap:
            th = torch.tanh(x / cap)
            x = cap * th
        i, j = torch.arange(nq).view(-1, 1), torch.arange(nk).view(1, -1)
        away = (i + nk - nq - j).abs()
        if slopes is not None:
            bias = slopes.detach().cpu().double().view(-1, 1, 1) * away
            x = x - bias
            size = size + bias
        seen = torch.ones((nq, nk), dtype=torch.bool)
        if causal:
            seen = j <= i + nk - nq
            if prefix is not None:
                seen = seen | (j < int(prefix[b]))
        x = x.masked_fill(~seen, -math.inf)
        top = x.amax(dim=-1, keepdim=True)
        p = torch.exp(x - torch.where(top == -math.inf, torch.zeros_like(top), top))
        p = p / p.sum(dim=-1, keepdim=True).clamp(min=1e-300)
        o = p @ vb
        out[wq] = o.transpose(0, 1)
        # weights off by the scores' error: 2^-18 of the products' magnitude where it is large
        e = f + 2.0 ** -18 * (size + (cap or 0.0))
        off_o = ((u + e) * p) @ vb.abs() + e.amax(dim=-1, keepdim=True) * (p @ vb.abs())
        bo[wq] = (off_o + u * o.abs()).transpose(0, 1)
        if not train:
            continue
        gb = g64[wq].transpose(0, 1)
        dv = p.transpose(1, 2) @ gb
        dp = gb @ vb.transpose(1, 2)
        dpa = gb.abs() @ vb.abs().transpose(1, 2)
        delta = (gb * o).sum(-1, keepdim=True)
        slope = (1 - th * th) * scale
        ds = p * (dp - delta) * slope
        off_delta = (gb.abs() * (off_o + u * o.abs())).sum(-1, keepdim=True) + f * (gb * o).abs().sum(-1, keepdim=True)
        off_ds = (u + 2 * e) * ds.abs() + p * slope * (off_delta + f * dpa) + (p * (dp - delta).abs() * scale * 2.0 ** -18 * (1 + size) if cap else 0.0)
        dq, dk = ds @ kb, ds.transpose(1, 2) @ qb
        wide = e.amax(dim=-1, keepdim=True)
        oq = off_ds @ kb.abs() + f * (ds.abs() @ kb.abs()) + u * dq.abs()
        okk = off_ds.transpose(1, 2) @ qb.abs() + f * (ds.abs().transpose(1, 2) @ qb.abs())
        ov = ((u + e + wide) * p).transpose(1, 2) @ gb.abs()

        def shared(t):
            return t.unflatten(0, (G, R)).sum(1)

        gq[wq], bq[wq] = dq.transpose(0, 1), oq.transpose(0, 1)
        dk, dv = shared(dk), shared(dv)
        gk[wk], bk[wk] = dk.transpose(0, 1), (shared(okk) + u * dk.abs()).transpose(0, 1)
        gv[wk], bv[wk] = dv.transpose(0, 1), (shared(ov) + u * dv.abs()).transpose(0, 1)
    if train:
        return [out, gq, gk, gv], [bo, bq, bk, bv]
    return out, bo
